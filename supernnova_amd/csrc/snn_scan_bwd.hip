// snn_scan_bwd.hip -- gradients of the selective scan (include/snn_hip.h: snn_scan_backward).
//
// With g_t = dy_t silu(z_t) and the adjoint q_t = C_t g_t + a_{t+1} q_{t+1}, a_t = exp(s_t A):
//   dx = skip g + s (q . B)            ds = x (q . B) + sum_n w_n A_n,  w = a_t q_t h_{t-1};   ddelta = ds sigmoid(delta + bias)
//   dB_n = sum_d q_n s x               dC_n = sum_d g h_n               dA_n = sum_t w_n s       dz = dy y silu'(z)
//
// The tape holds the state every ScanTape<K>::STEPS steps.  A workgroup walks a chunk backwards segment by segment: it
// recomputes the segment's states and decays into registers (one exp per (step, channel, state), as the forward), then runs
// the adjoint over it; neither is ever divided by a decay.  Sums over states are two DPP adds a quad, dealt over it; sums over
// channels (dB, dC: 2K values a lane and step) are folded over the wave by v_permlane32_swap / v_permlane16_swap, each of which
// halves the number of live values while it adds, then DPP rotations, then LDS over the four waves, then -- layers wider than
// one workgroup's channels -- fp32 partial rows per channel block, added in order by scan_bc_sum_kernel.  Parameter gradients stay
// in fp32 registers: sums of at most 256 steps, then one addition for each such block over all chunks a workgroup takes, so that the
// rounding grows with the number of blocks and not of steps; scan_param_sum_kernel adds the workgroups' in fp64, in order.  No atomics.
//
// The vector unit bounds it: 108 instructions a lane's step of four states (27 to recompute, 56 for the adjoint, of which the
// channel sums take 22 issue slots; 25 per segment and chunk), at two waves a SIMD.  At their 256 registers it spills a little:
// gated bf16 of 16 states 12 vector registers into 52 bytes of scratch (8 states 16 into 68, fp32 up to 20 into 84), and 222 scalars
// (twelve views of 64-bit strides live through the time loop) into lanes of vector registers: 38 of a segment's instructions, 5 a
// step, bring them back, and some 190 a chunk.  Three or four waves a SIMD spill far more: 880 and 1254 us instead of 297.  4 x 2048 x 2048 bf16 of 16 states: adjoint pass 63, combination 6, this kernel 301, sums 8 + 17 us;
// 512 x 300 x 256 fp32: 323 us, sums 6 + 22 us.
#include <algorithm>
#include "snn_host.h"
#include "snn_scan.h"

#define HIP_CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { \
    snn_set_error("%s: %s", #x, hipGetErrorString(e_)); return SNN_ERR_HIP; } } while (0)

namespace {

__device__ __forceinline__ void swap32(float& a, float& b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap16(float& a, float& b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
// Sums over the wave's 64 / LN channels (lanes of equal lane % LN) of b[0..K), c[0..K).  Row r = lane / 16 receives, for
// i < K / 2, the sum of (r / 2 ? c : b)[i + (r % 2) K / 2], once for every channel of the row.
template <int K, int LN> __device__ __forceinline__ void channel_sums(float (&b)[K], float (&c)[K], float (&out)[K / 2])
{
#pragma unroll
    for (int i = 0; i < K; ++i) {
        swap32(b[i], c[i]);
        b[i] += c[i];
    }
#pragma unroll
    for (int i = 0; i < K / 2; ++i) {
        swap16(b[i], b[i + K / 2]);
        float v = b[i] + b[i + K / 2];
        if constexpr (LN <= 4) v += dpp<0x124>(v);        // row_ror:4
        if constexpr (LN <= 8) v += dpp<0x128>(v);        // row_ror:8
        out[i] = v;
    }
}

// floats of one slot's parameter gradients: dA (D, NP), dskip (D), dbias (D), and up to 16 bytes
__host__ __device__ __forceinline__ int64_t part_stride(int D, int NP) { return ((int64_t)D * (NP + 2) + 3) / 4 * 4; }

// What chunk c > 0 sends back from a zero adjoint, a_{t0} q_{t0}, into carry[b][c - 1], and the sum of its steps into csum[b][c].
template <typename T, int K, int LN, bool GATE> __global__ void __launch_bounds__(256) scan_adjoint_kernel(const ScanP<T> p)
{
    constexpr int SEG = SCAN_SEG, G = SEG / 4, NP = K * LN;
    __shared__ float sC[2][SEG * NP];
    const int tid = threadIdx.x, b = blockIdx.x, cb = blockIdx.y, c = blockIdx.z;
    const ScanCh ch = scan_channel<K, LN>(cb, p.cbg, p.dg, tid);
    const int j = ch.j, d = ch.d;
    const SeqRange r = seq_range(p.seq, b);
    const int t0 = c * p.tc, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
    if (c == 0 || t0 >= r.len) return;
    float w[K], A2[K];
    load_states<K>(p.A + (int64_t)d * p.N, ch.n, p.N, p.vec, A2);
    const float bias = p.dbias ? p.dbias[d] : 0.0f;
    float ssum = 0.0f;
    const int tl = t0 + (t1 - 1 - t0) / SEG * SEG;
    const int64_t first = r.row0 + tl + j;               // pointers to the last segment; they move back with it
    const T* dp = p.delta.p + first * p.delta.st + b * p.delta.sb + d;
    const T* zp = GATE ? p.z.p + first * p.z.st + b * p.z.sb + d : nullptr;
    const T* gp = p.dy.p + first * p.dy.st + b * p.dy.sb + d;
    LaneIn<T, G> di, zi, gi;
    RowStage<T, NP, SEG> Ci;
    Ci.init(p.C.p + (r.row0 + tl) * p.C.st + b * p.C.sb + ch.g * p.C_sg, p.C.st, p.N, tid);
    auto fetch = [&](int left) {
        di.load(dp, p.delta.st, j, left);
        if (GATE) zi.load(zp, p.z.st, j, left);
        gi.load(gp, p.dy.st, j, left);
        Ci.load(p.C.st, left);
        dp -= SEG * p.delta.st;
        if (GATE) zp -= SEG * p.z.st;
        gp -= SEG * p.dy.st;
        Ci.p -= SEG * p.C.st;
    };
    fetch(t1 - tl);
    decay_rates<K>(A2);
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = 0.0f;
    int buf = 0;
    for (int t = tl; t >= t0; t -= SEG, buf ^= 1) {
        Ci.store(sC[buf], tid);
        float s[G], g[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const float v = to_f32(di.v[i]) + bias;
            s[i] = p.softplus ? softplus_f32(v, nullptr) : v;
            g[i] = to_f32(gi.v[i]);
            if (GATE) {
                const float z = to_f32(zi.v[i]);
                g[i] *= z * sigmoid_f32(z);
            }
        }
        if (t + SEG > t1) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const bool live = t + 4 * i + j < t1;
                s[i] = live ? s[i] : 0.0f;
                g[i] = live ? g[i] : 0.0f;
            }
        }
        __syncthreads();
        if (t > t0) fetch(SEG);
        float Cv[2][K];                                  // of this step and the next
        lds_states<K>(&sC[buf][(SEG - 1) * NP], ch.n, Cv[1]);
#pragma unroll
        for (int i = G - 1; i >= 0; --i) {
            ssum += s[i];
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                const int m = 4 * i + q;
                if (m > 0) lds_states<K>(&sC[buf][(m - 1) * NP], ch.n, Cv[(m - 1) & 1]);
                pin_lds_reads();
                const float sq = qbc(s[i], q), gq = qbc(g[i], q);
#pragma unroll
                for (int k = 0; k < K; ++k) w[k] = __builtin_amdgcn_exp2f(sq * A2[k]) * fmaf(Cv[m & 1][k], gq, w[k]);
            }
        }
    }
    ssum = quad_sum(ssum);
    if (ch.ok) {
        store_states<K>(p.carry + (((int64_t)b * p.nc + c - 1) * p.D + d) * NP, ch.n, NP, true, w);
        if (ch.n == 0) p.csum[((int64_t)b * p.nc + c) * p.D + d] = ssum;
    }
}

template <typename T, int K, int LN, bool GATE> __global__ void __launch_bounds__(256, 2) scan_bwd_kernel(const ScanP<T> p)
{
    constexpr int SEG = ScanTape<K>::STEPS, G = SEG / 4, NP = K * LN, CH = 256 / LN;
    __shared__ float sB[2][SEG * NP], sC[2][SEG * NP], red[4][SEG][2 * NP];
    const int tid = threadIdx.x, nch = p.D / p.dg * p.cbg, cb = blockIdx.x % nch, slot = blockIdx.x / nch;
    const int wave = tid >> 6, lane = tid & 63;
    const ScanCh ch = scan_channel<K, LN>(cb, p.cbg, p.dg, tid);
    const int j = ch.j, d = ch.d;
    const int left_ch = p.dg - (cb - ch.g * p.cbg) * CH, d0 = ch.g * p.dg + p.dg - left_ch;
    float A2[K], dAs[K], dsks = 0.0f, dbss = 0.0f;      // sums over blocks of 256 steps; a block's own come first
    load_states<K>(p.A + (int64_t)d * p.N, ch.n, p.N, p.vec, A2);
    decay_rates<K>(A2);
#pragma unroll
    for (int k = 0; k < K; ++k) dAs[k] = 0.0f;
    const float bias = p.dbias ? p.dbias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
    const int64_t rows = p.seq.offsets ? p.seq.n_rows : (int64_t)p.seq.n_seq * p.seq.max_T;
    float* bcpart = p.bcpart ? p.bcpart + (int64_t)cb * rows * (2 * NP) : nullptr;
    const int items = p.seq.n_seq * p.nc;
    for (int item = slot; item < items; item += p.slots) {
        const int bi = item / p.nc, c = item - bi * p.nc, b = p.order ? p.order[bi] : bi;
        const SeqRange r = seq_range(p.seq, b);
        const int t0 = c * p.tc, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
        const int64_t rowb = p.seq.offsets ? r.row0 : (int64_t)b * p.seq.max_T;
        float w[K], dA[K], dsk = 0.0f, dbs = 0.0f;                // w: a_{t+1} q_{t+1}
#pragma unroll
        for (int k = 0; k < K; ++k) w[k] = dA[k] = 0.0f;
        if (p.nc > 1 && t0 < r.len) load_states<K>(p.carry + (((int64_t)b * p.nc + c) * p.D + d) * NP, ch.n, NP, true, w);
        else if (c == 0 && p.dhT) load_states<K>(p.dhT + ((int64_t)b * p.D + d) * p.N, ch.n, p.N, p.vec, w);
        if (t0 < t1) {
            const int tl = t0 + (t1 - 1 - t0) / SEG * SEG;
            const int64_t first = r.row0 + tl + j;       // pointers to the last segment; they move back with it
            const T* xp = p.x.p + first * p.x.st + b * p.x.sb + d;
            const T* dp = p.delta.p + first * p.delta.st + b * p.delta.sb + d;
            const T* zp = GATE ? p.z.p + first * p.z.st + b * p.z.sb + d : nullptr;
            const T* gp = p.dy.p + first * p.dy.st + b * p.dy.sb + d;
            T* dxp = p.dx.p + first * p.dx.st + b * p.dx.sb + d;
            T* ddp = p.ddelta.p + first * p.ddelta.st + b * p.ddelta.sb + d;
            T* dzp = GATE ? p.dz.p + first * p.dz.st + b * p.dz.sb + d : nullptr;
            const float* tape = p.tape + ((scan_tape_first(p.seq, r, b, SEG) + tl / SEG) * p.D + d) * NP + ch.n;
            LaneIn<T, G> xi, di, zi, gi;
            RowStage<T, NP, SEG> Bi, Ci;
            Bi.init(p.B.p + (r.row0 + tl) * p.B.st + b * p.B.sb + ch.g * p.B_sg, p.B.st, p.N, tid);
            Ci.init(p.C.p + (r.row0 + tl) * p.C.st + b * p.C.sb + ch.g * p.C_sg, p.C.st, p.N, tid);
            float hs[K];
            auto fetch = [&](int left) {
                xi.load(xp, p.x.st, j, left);
                di.load(dp, p.delta.st, j, left);
                if (GATE) zi.load(zp, p.z.st, j, left);
                gi.load(gp, p.dy.st, j, left);
                Bi.load(p.B.st, left);
                Ci.load(p.C.st, left);
                load_states<K>(tape, 0, NP, true, hs);
                xp -= SEG * p.x.st;
                dp -= SEG * p.delta.st;
                if (GATE) zp -= SEG * p.z.st;
                gp -= SEG * p.dy.st;
                Bi.p -= SEG * p.B.st;
                Ci.p -= SEG * p.C.st;
                tape -= (int64_t)p.D * NP;
            };
            fetch(t1 - tl);
            int buf = 0;
            for (int t = tl; t >= t0; t -= SEG, buf ^= 1) {
                Bi.store(sB[buf], tid);
                Ci.store(sC[buf], tid);
                float x[G], s[G], sig[G], z[G], dy[G], g[G], u[G], h[SEG + 1][K], a[SEG][K];
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    x[i] = to_f32(xi.v[i]);
                    const float v = to_f32(di.v[i]) + bias;
                    s[i] = v;
                    sig[i] = 1.0f;
                    if (p.softplus) s[i] = softplus_f32(v, &sig[i]);
                    dy[i] = to_f32(gi.v[i]);
                    z[i] = GATE ? to_f32(zi.v[i]) : 0.0f;
                }
                const int left = t1 - t;
                if (left < SEG || left_ch < CH) {        // steps behind the end leave the state, lanes without a channel add nothing
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        const bool live = 4 * i + j < left;
                        s[i] = live ? s[i] : 0.0f;
                        x[i] = live && ch.ok ? x[i] : 0.0f;
                        dy[i] = live && ch.ok ? dy[i] : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    u[i] = s[i] * x[i];
                    g[i] = GATE ? dy[i] * (z[i] * sigmoid_f32(z[i])) : dy[i];
                }
#pragma unroll
                for (int k = 0; k < K; ++k) h[0][k] = hs[k];
                __syncthreads();              // B, C staged; the last segment's partial sums have been read
                if (t > t0) fetch(SEG);
                // the segment's states and decays again
                float Bv[2][K], Cv[2][K];                // of this step and the next
                auto read = [&](int m, bool want_c) {
                    lds_states<K>(&sB[buf][m * NP], ch.n, Bv[m & 1]);
                    if (want_c) lds_states<K>(&sC[buf][m * NP], ch.n, Cv[m & 1]);
                };
                read(0, GATE);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    float yv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int m = 4 * i + q;
                        if (m + 1 < SEG) read(m + 1, GATE);
                        pin_lds_reads();
                        const float sq = qbc(s[i], q), uq = qbc(u[i], q);
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            a[m][k] = __builtin_amdgcn_exp2f(sq * A2[k]);
                            h[m + 1][k] = fmaf(a[m][k], h[m][k], uq * Bv[m & 1][k]);
                            if (GATE) yv[q] = fmaf(h[m + 1][k], Cv[m & 1][k], yv[q]);
                        }
                    }
                    if (GATE) {
                        const float y = fmaf(skip, x[i], step_sums<LN>(yv, j)), e = sigmoid_f32(z[i]);
                        if (ch.lead && 4 * i + j < left) dzp[4 * i * p.dz.st] = from_f32<T>(dy[i] * y * (e * fmaf(z[i], 1.0f - e, 1.0f)));
                    }
                }
                // the adjoint, backwards
                read(SEG - 1, true);
#pragma unroll
                for (int i = G - 1; i >= 0; --i) {
                    float s1[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = 3; q >= 0; --q) {
                        const int m = 4 * i + q;
                        const float sq = qbc(s[i], q), uq = qbc(u[i], q), gq = qbc(g[i], q);
                        if (m > 0) read(m - 1, true);
                        pin_lds_reads();
                        float pb[K], pc[K], sums[K / 2];
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            const float qk = fmaf(Cv[m & 1][k], gq, w[k]);
                            pc[k] = gq * h[m + 1][k];
                            pb[k] = qk * uq;
                            s1[q] = fmaf(qk, Bv[m & 1][k], s1[q]);
                            w[k] = a[m][k] * qk;
                            const float v = w[k] * h[m][k];
                            dA[k] = fmaf(v, sq, dA[k]);
                            s2[q] = fmaf(v, A2[k], s2[q]);
                        }
                        channel_sums<K, LN>(pb, pc, sums);
                        if ((lane & 15) < LN) {
                            float* o = &red[wave][m][(lane >> 5) * NP + ch.n + ((lane >> 4) & 1) * (K / 2)];
#pragma unroll
                            for (int k = 0; k < K / 2; ++k) o[k] = sums[k];
                        }
                    }
                    const float qB = step_sums<LN>(s1, j), wA = step_sums<LN>(s2, j) * SNN_LN2;
                    const float dd = fmaf(x[i], qB, wA) * sig[i];
                    if (ch.lead && 4 * i + j < left) {
                        dxp[4 * i * p.dx.st] = from_f32<T>(fmaf(skip, g[i], s[i] * qB));
                        ddp[4 * i * p.ddelta.st] = from_f32<T>(dd);
                        dbs += dd;
                        dsk = fmaf(g[i], x[i], dsk);
                    }
                }
                if (t % 256 == 0 || t == t0) {
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        dAs[k] += dA[k];
                        dA[k] = 0.0f;
                    }
                    dsks += dsk;
                    dbss += dbs;
                    dsk = dbs = 0.0f;
                }
                dxp -= SEG * p.dx.st;
                ddp -= SEG * p.ddelta.st;
                if (GATE) dzp -= SEG * p.dz.st;
                __syncthreads();
                for (int e = tid; e < SEG * 2 * NP; e += 256) {
                    const int m = e / (2 * NP), o = e % (2 * NP), half = o / NP, n = o % NP;
                    if (m < left) {
                        const float v = (red[0][m][o] + red[1][m][o]) + (red[2][m][o] + red[3][m][o]);
                        if (bcpart) bcpart[(rowb + t + m) * (2 * NP) + o] = v;
                        else if (n < p.N) {
                            const View<T>& q = half ? p.dC : p.dB;
                            q.p[(r.row0 + t + m) * q.st + b * q.sb + ch.g * p.N + n] = from_f32<T>(v);
                        }
                    }
                }
            }
            __syncthreads();                  // the next chunk stages into the buffers this one has read
        }
        if (c == 0 && p.dh0 && ch.ok) store_states<K>(p.dh0 + ((int64_t)b * p.D + d) * p.N, ch.n, p.N, p.vec, w);
        const FillRange f = fill_range(p.seq, r, b, t0, t0 + p.tc, c == p.nc - 1);
        const int n = left_ch < CH ? left_ch : CH;
        clear_channels(p.dx, r.row0 * p.dx.st + b * p.dx.sb, f, d0, n, tid);
        clear_channels(p.ddelta, r.row0 * p.ddelta.st + b * p.ddelta.sb, f, d0, n, tid);
        if (GATE) clear_channels(p.dz, r.row0 * p.dz.st + b * p.dz.sb, f, d0, n, tid);
        if (bcpart && p.seq.offsets) {
            for (int64_t e = f.a0 * (2 * NP) + tid; e < f.a1 * (2 * NP); e += 256) bcpart[rowb * (2 * NP) + e] = 0.0f;
            for (int64_t e = f.b0 * (2 * NP) + tid; e < f.b1 * (2 * NP); e += 256) bcpart[rowb * (2 * NP) + e] = 0.0f;
        } else if (!bcpart) {
            clear_channels(p.dB, r.row0 * p.dB.st + b * p.dB.sb + ch.g * p.N, f, 0, p.N, tid);
            clear_channels(p.dC, r.row0 * p.dC.st + b * p.dC.sb + ch.g * p.N, f, 0, p.N, tid);
        }
    }
    dsks = quad_sum(dsks);
    dbss = quad_sum(dbss);
    if (ch.ok) {
        float* q = p.part + (int64_t)slot * part_stride(p.D, NP);
        store_states<K>(q + (int64_t)d * NP, ch.n, NP, true, dAs);
        if (ch.n == 0) {
            q[(int64_t)p.D * NP + d] = dsks;
            q[(int64_t)p.D * (NP + 1) + d] = dbss;
        }
    }
}

// dA (D, N), dskip (D), dbias (D) from the slots' partial sums
__global__ void __launch_bounds__(1024) scan_param_sum_kernel(const float* __restrict__ part, int slots, int D, int N, int NP, float* dA, float* dskip,
                                                             float* dbias)
{
    int64_t col;
    double a;
    if (!column_sum(part, slots, part_stride(D, NP), (int64_t)D * (NP + 2), &col, &a)) return;
    if (col < (int64_t)D * NP) {
        const int d = (int)(col / NP), k = (int)(col - (int64_t)d * NP);
        if (k < N) dA[(int64_t)d * N + k] = (float)a;
    } else if (col < (int64_t)D * (NP + 1)) {
        if (dskip) dskip[col - (int64_t)D * NP] = (float)a;
    } else if (dbias) dbias[col - (int64_t)D * (NP + 1)] = (float)a;
}

// dB, dC rows from the channel blocks' partial rows, in block order, four states a thread.  In a padded batch the rows behind a
// sequence's end are recognised here and never written as partial rows; among ragged rows they have been cleared.
template <typename T> __global__ void __launch_bounds__(256) scan_bc_sum_kernel(const ScanP<T> p, int NP, int groups)
{
    const int64_t rows = p.seq.offsets ? p.seq.n_rows : (int64_t)p.seq.n_seq * p.seq.max_T;
    const int quads = NP / 2, per = groups * quads;                 // of a group's 2 NP partial sums
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * per) return;
    const int64_t row = id / per;
    const int e = (int)(id - row * per), g = e / quads, o = (e - g * quads) * 4, half = o >= NP, n = o - half * NP;
    int64_t t = row, b = 0;
    bool live = true;
    if (!p.seq.offsets) {
        b = row / p.seq.max_T;
        t = row - b * p.seq.max_T;
        live = t < seq_range(p.seq, (int)b).len;
    }
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (live) {
        const float* q = p.bcpart + ((int64_t)g * p.cbg * rows + row) * (2 * NP) + o;
        for (int i = 0; i < p.cbg; ++i, q += rows * (2 * NP)) {
            const float4 v = *(const float4*)q;
            a.x += v.x;
            a.y += v.y;
            a.z += v.z;
            a.w += v.w;
        }
    }
    const View<T>& w = half ? p.dC : p.dB;
    T* out = w.p + t * w.st + b * w.sb + g * p.N + n;
    const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < p.N) out[i] = from_f32<T>(v[i]);
}

struct Sizes { int64_t carry, csum, order, part, bc; int slots; };
// Slots: workgroups that share the chunks.  2048 of them all told keep four on every compute unit in turn and even out
// ragged lengths; more would only add partial sums to write and read.
Sizes sizes(const snn_scan_args* a, const ScanGrid& g)
{
    const int NP = scan_padded(a->states);
    const int64_t items = (int64_t)a->seq.n_seq * g.nc;
    Sizes z;
    z.slots = (int)std::min<int64_t>(items, std::max<int64_t>(1, 2048 / g.blocks_c));
    z.carry = g.nc > 1 ? items * a->channels * NP : 0;
    z.csum = g.nc > 1 ? (items * a->channels + 3) / 4 * 4 : 0;
    z.order = snn_scan_ordered(a, g) ? ((int64_t)a->seq.n_seq + 3) / 4 * 4 : 0;
    z.part = (int64_t)z.slots * part_stride(a->channels, NP);
    const int64_t rows = a->seq.offsets ? a->seq.n_rows : (int64_t)a->seq.n_seq * a->seq.max_T;
    z.bc = g.cbg > 1 ? (int64_t)g.blocks_c * rows * 2 * NP : 0;
    return z;
}

template <typename T, int K, int LN, bool GATE> int backward(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    ScanP<T> p = scan_params<T>(a, g);
    const Sizes z = sizes(a, g);
    p.carry = (float*)a->ws;
    p.csum = p.carry + z.carry;
    p.part = p.csum + z.csum + z.order;
    if (z.order) {
        snn_scan_launch_order(a->seq, (int*)(p.part - z.order), s);
        p.order = (const int*)(p.part - z.order);
    }
    p.bcpart = z.bc ? p.part + z.part : nullptr;
    p.slots = z.slots;
    if (g.nc > 1) {
        const dim3 grid((unsigned)a->seq.n_seq, (unsigned)g.blocks_c, (unsigned)g.nc);
        hipLaunchKernelGGL((scan_adjoint_kernel<T, K, LN, GATE>), grid, dim3(256), 0, s, p);
        snn_scan_launch_combine(a, g, a->dstate_out, p.carry, p.csum, true, s);
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, K, LN, GATE>), dim3((unsigned)(g.blocks_c * z.slots)), dim3(256), 0, s, p);
    const int64_t n = (int64_t)p.D * (K * LN + 2);
    hipLaunchKernelGGL(scan_param_sum_kernel, dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, s, (const float*)p.part, z.slots, p.D, p.N, K * LN,
                       a->dA, a->dskip, a->ddelta_bias);
    if (z.bc) {
        const int64_t rows = a->seq.offsets ? a->seq.n_rows : (int64_t)a->seq.n_seq * a->seq.max_T;
        const int64_t e = (rows * a->groups * (K * LN / 2) + 255) / 256;
        hipLaunchKernelGGL((scan_bc_sum_kernel<T>), dim3((unsigned)e), dim3(256), 0, s, p, K * LN, a->groups);
    }
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T, bool GATE> int by_states(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    if (a->states <= 8) return backward<T, 2, 4, GATE>(a, g, s);
    if (a->states <= 16) return backward<T, 4, 4, GATE>(a, g, s);
    if (a->states <= 32) return backward<T, 4, 8, GATE>(a, g, s);
    return backward<T, 4, 16, GATE>(a, g, s);
}

template <typename T> int run(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    return a->z.p ? by_states<T, true>(a, g, s) : by_states<T, false>(a, g, s);
}

}  // namespace

extern "C" int64_t snn_scan_workspace_bytes(const snn_scan_args* a, int32_t backward_pass)
{
    if (int rc = snn_scan_check(a, "snn_scan_workspace_bytes")) return rc;
    const ScanGrid g = snn_scan_grid(a);
    const Sizes z = sizes(a, g);
    return 4 * (z.carry + z.csum + z.order + (backward_pass ? z.part + z.bc : 0));
}

extern "C" int snn_scan_backward(const snn_scan_args* a, void* stream)
{
    if (int rc = snn_scan_check(a, "snn_scan_backward")) return rc;
    if (!a->x.p || !a->delta.p || !a->B.p || !a->C.p || !a->A || !a->dy.p || !a->tape || !a->dx.p || !a->ddelta.p || !a->dB.p || !a->dC.p ||
        !a->dA || !a->ws || (a->z.p && !a->dz.p) || ((uintptr_t)a->tape | (uintptr_t)a->ws) % 16) {
        snn_set_error("snn_scan_backward: null or misaligned pointer");
        return SNN_ERR_ARG;
    }
    const int64_t need = snn_scan_workspace_bytes(a, 1);
    if (a->ws_bytes < need || a->tape_floats < snn_scan_tape_floats(a)) {
        snn_set_error("snn_scan_backward: workspace of %lld bytes (%lld needed) or tape of %lld floats too small", (long long)a->ws_bytes,
                      (long long)need, (long long)a->tape_floats);
        return SNN_ERR_WORKSPACE;
    }
    const ScanGrid g = snn_scan_grid(a);
    const int64_t rows = a->seq.offsets ? a->seq.n_rows : (int64_t)a->seq.n_seq * a->seq.max_T;
    if ((int64_t)a->seq.n_seq * g.nc > 0x7fffffff || (rows * a->groups * (scan_padded(a->states) / 2) + 255) / 256 > SEQ_MAX_BLOCKS) {
        snn_set_error("snn_scan_backward: %lld rows of B and C are too many for one call", (long long)rows);
        return SNN_ERR_UNSUPPORTED;
    }
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == SNN_DT_F32 ? run<float>(a, g, s) : a->dtype == SNN_DT_BF16 ? run<bf16_t>(a, g, s) : run<f16_t>(a, g, s);
}
