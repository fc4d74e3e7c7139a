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
// halves the number of live values while it adds, then two DPP rotations, then LDS over the four waves, then -- layers wider than
// 64 channels -- fp32 partial rows per channel block, added in order by scan_bc_sum_kernel.  Parameter gradients stay in registers over
// all chunks a workgroup takes and are summed in fp64, in order, by scan_param_sum_kernel.  No atomics.
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
// Sums over the wave's 16 channels (lanes of equal lane % 4) of b[0..K), c[0..K).  Row r = lane / 16 receives, for
// i < K / 2, the sum of (r / 2 ? c : b)[i + (r % 2) K / 2], in all of its four quads.
template <int K> __device__ __forceinline__ void channel_sums(float (&b)[K], float (&c)[K], float (&out)[K / 2])
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
        v += dpp<0x124>(v);                      // row_ror:4
        out[i] = v + dpp<0x128>(v);              // row_ror:8
    }
}

// floats of one slot's parameter gradients: dA (D, 4K), dskip (D), dbias (D), and up to 16 bytes
__host__ __device__ __forceinline__ int64_t part_stride(int D, int NP) { return ((int64_t)D * (NP + 2) + 3) / 4 * 4; }

template <typename T, int G> struct BwdIn {
    T x[G], d[G], z[G], y[G];
    __device__ __forceinline__ void load(const ScanP<T>& p, int64_t xb, int64_t db, int64_t zb, int64_t gb, int t, int t1)
    {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if (t + 4 * i < t1) {
                x[i] = p.x.p[xb + (t + 4 * i) * p.x.st];
                d[i] = p.delta.p[db + (t + 4 * i) * p.delta.st];
                if (p.z.p) z[i] = p.z.p[zb + (t + 4 * i) * p.z.st];
                y[i] = p.dy.p[gb + (t + 4 * i) * p.dy.st];
            }
        }
    }
};

template <int Q> __device__ __forceinline__ float qb(float v) { return quad_bcast<Q>(v); }
__device__ __forceinline__ float qbc(float v, int q) { return q == 0 ? qb<0>(v) : q == 1 ? qb<1>(v) : q == 2 ? qb<2>(v) : qb<3>(v); }

// What chunk c > 0 sends back from a zero adjoint, a_{t0} q_{t0}, into carry[b][c - 1], and the sum of its steps into csum[b][c].
template <typename T, int K> __global__ void __launch_bounds__(256) scan_adjoint_kernel(const ScanP<T> p)
{
    constexpr int SEG = SCAN_SEG, G = SEG / 4;
    __shared__ float sC[2][SEG * 4 * K];
    const int tid = threadIdx.x, nch = p.D / p.dg * p.cbg, cb = blockIdx.x % nch;
    const int item = blockIdx.x / nch, b = item / p.nc, c = item - b * p.nc;
    const ScanCh ch = scan_channel(cb, p.cbg, p.dg, tid);
    const int j = ch.j, d = ch.d;
    const SeqRange r = seq_range(p.seq, b);
    const int t0 = c * p.tc, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
    if (c == 0 || t0 >= r.len) return;
    const int64_t xb = r.row0 * p.x.st + b * p.x.sb + d, db = r.row0 * p.delta.st + b * p.delta.sb + d;
    const int64_t zb = r.row0 * p.z.st + b * p.z.sb + d, gb = r.row0 * p.dy.st + b * p.dy.sb + d;
    const T* Cp = p.C.p + r.row0 * p.C.st + b * p.C.sb + ch.g * p.C_sg;
    float w[K], A2[K];
    load_states<K>(p.A + (int64_t)d * p.N, j, p.N, p.vec, A2);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        A2[k] *= SNN_LOG2E;
        w[k] = 0.0f;
    }
    const float bias = p.dbias ? p.dbias[d] : 0.0f;
    float ssum = 0.0f;
    BwdIn<T, G> in;
    BcStage<T, K, SEG> bc;
    const int tl = t0 + (t1 - 1 - t0) / SEG * SEG;
    in.load(p, xb, db, zb, gb, tl + j, t1);
    bc.template load<false>(Cp, p.C.st, Cp, p.C.st, tl, t1, p.N, tid);
    int buf = 0;
    for (int t = tl; t >= t0; t -= SEG, buf ^= 1) {
        bc.template store<false>(sC[buf], nullptr, tid);
        float s[G], g[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const bool live = t + 4 * i + j < t1;
            const float v = live ? to_f32(in.d[i]) + bias : 0.0f;
            const float sp = p.softplus ? softplus_f32(v, nullptr) : v;
            s[i] = live ? sp : 0.0f;
            g[i] = live ? to_f32(in.y[i]) : 0.0f;
            if (live && p.z.p) {
                const float z = to_f32(in.z[i]);
                g[i] *= z * sigmoid_f32(z);
            }
            ssum += s[i];
        }
        __syncthreads();
        if (t > t0) {
            in.load(p, xb, db, zb, gb, t - SEG + j, t1);
            bc.template load<false>(Cp, p.C.st, Cp, p.C.st, t - SEG, t1, p.N, tid);
        }
#pragma unroll
        for (int i = G - 1; i >= 0; --i) {
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                const float sq = qbc(s[i], q), gq = qbc(g[i], q);
                float Cv[K];
                lds_states<K>(&sC[buf][(4 * i + q) * 4 * K], j, Cv);
#pragma unroll
                for (int k = 0; k < K; ++k) w[k] = __builtin_amdgcn_exp2f(sq * A2[k]) * fmaf(Cv[k], gq, w[k]);
            }
        }
    }
    ssum = quad_sum(ssum);
    if (ch.ok) {
        store_states<K>(p.carry + (((int64_t)b * p.nc + c - 1) * p.D + d) * (4 * K), j, 4 * K, true, w);
        if (j == 0) p.csum[((int64_t)b * p.nc + c) * p.D + d] = ssum;
    }
}

template <typename T, int K> __global__ void __launch_bounds__(256, K == 16 ? 1 : 2) scan_bwd_kernel(const ScanP<T> p)
{
    constexpr int SEG = ScanTape<K>::STEPS, G = SEG / 4, NP = 4 * K;
    __shared__ float sB[2][SEG * NP], sC[2][SEG * NP], red[4][SEG][2 * NP];
    const int tid = threadIdx.x, nch = p.D / p.dg * p.cbg, cb = blockIdx.x % nch, slot = blockIdx.x / nch;
    const int wave = tid >> 6, lane = tid & 63;
    const ScanCh ch = scan_channel(cb, p.cbg, p.dg, tid);
    const int j = ch.j, d = ch.d;
    const float live_ch = ch.ok ? 1.0f : 0.0f;
    const int left = p.dg - (cb - ch.g * p.cbg) * SCAN_CH, d0 = ch.g * p.dg + p.dg - left;
    float A2[K], dA[K], dsk = 0.0f, dbs = 0.0f;
    load_states<K>(p.A + (int64_t)d * p.N, j, p.N, p.vec, A2);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        A2[k] *= SNN_LOG2E;
        dA[k] = 0.0f;
    }
    const float bias = p.dbias ? p.dbias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
    const int64_t rows = p.seq.offsets ? p.seq.n_rows : (int64_t)p.seq.n_seq * p.seq.max_T;
    float* bcpart = p.bcpart ? p.bcpart + (int64_t)cb * rows * (2 * NP) : nullptr;
    const int items = p.seq.n_seq * p.nc;
    for (int item = slot; item < items; item += p.slots) {
        const int b = item / p.nc, c = item - b * p.nc;
        const SeqRange r = seq_range(p.seq, b);
        const int t0 = c * p.tc, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
        const int64_t xb = r.row0 * p.x.st + b * p.x.sb + d, db = r.row0 * p.delta.st + b * p.delta.sb + d;
        const int64_t zb = r.row0 * p.z.st + b * p.z.sb + d, gb = r.row0 * p.dy.st + b * p.dy.sb + d;
        const int64_t dxb = r.row0 * p.dx.st + b * p.dx.sb, ddb = r.row0 * p.ddelta.st + b * p.ddelta.sb;
        const int64_t dzb = r.row0 * p.dz.st + b * p.dz.sb;
        const int64_t dBb = r.row0 * p.dB.st + b * p.dB.sb + ch.g * p.N, dCb = r.row0 * p.dC.st + b * p.dC.sb + ch.g * p.N;
        const int64_t rowb = p.seq.offsets ? r.row0 : (int64_t)b * p.seq.max_T;
        const T* Bp = p.B.p + r.row0 * p.B.st + b * p.B.sb + ch.g * p.B_sg;
        const T* Cp = p.C.p + r.row0 * p.C.st + b * p.C.sb + ch.g * p.C_sg;
        float w[K];                                               // a_{t+1} q_{t+1}
#pragma unroll
        for (int k = 0; k < K; ++k) w[k] = 0.0f;
        if (p.nc > 1 && t0 < r.len) load_states<K>(p.carry + (((int64_t)b * p.nc + c) * p.D + d) * NP, j, NP, true, w);
        else if (c == 0 && p.dhT) load_states<K>(p.dhT + ((int64_t)b * p.D + d) * p.N, j, p.N, p.vec, w);
        if (t0 < t1) {
            BwdIn<T, G> in;
            BcStage<T, K, SEG> bc;
            float hs[K];
            const int tl = t0 + (t1 - 1 - t0) / SEG * SEG;
            const float* tape = p.tape + ((scan_tape_first(p.seq, r, b, SEG) + tl / SEG) * p.D + d) * NP;
            in.load(p, xb, db, zb, gb, tl + j, t1);
            bc.template load<true>(Bp, p.B.st, Cp, p.C.st, tl, t1, p.N, tid);
            load_states<K>(tape, j, NP, true, hs);
            int buf = 0;
            for (int t = tl; t >= t0; t -= SEG, buf ^= 1) {
                bc.template store<true>(sB[buf], sC[buf], tid);
                float x[G], s[G], sig[G], z[G], dy[G], g[G], u[G], h[SEG + 1][K], a[SEG][K];
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const bool live = t + 4 * i + j < t1;
                    const float lc = live ? live_ch : 0.0f;       // lanes without a channel must add nothing to dB, dC
                    x[i] = live ? to_f32(in.x[i]) : 0.0f;
                    const float v = live ? to_f32(in.d[i]) + bias : 0.0f;
                    float sp = v;
                    sig[i] = 1.0f;
                    if (p.softplus) sp = softplus_f32(v, &sig[i]);
                    s[i] = live ? sp : 0.0f;
                    z[i] = live && p.z.p ? to_f32(in.z[i]) : 0.0f;
                    dy[i] = live && lc != 0.0f ? to_f32(in.y[i]) : 0.0f;
                    g[i] = p.z.p ? dy[i] * z[i] * sigmoid_f32(z[i]) : dy[i];
                    u[i] = lc != 0.0f ? s[i] * x[i] : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < K; ++k) h[0][k] = hs[k];
                __syncthreads();              // B, C staged; the last segment's partial sums have been read
                if (t > t0) {
                    in.load(p, xb, db, zb, gb, t - SEG + j, t1);
                    bc.template load<true>(Bp, p.B.st, Cp, p.C.st, t - SEG, t1, p.N, tid);
                    tape -= (int64_t)p.D * NP;
                    load_states<K>(tape, j, NP, true, hs);
                }
                // the segment's states and decays again
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    float yp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float sq = qbc(s[i], q), uq = qbc(u[i], q);
                        float Bv[K];
                        lds_states<K>(&sB[buf][(4 * i + q) * NP], j, Bv);
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            a[4 * i + q][k] = __builtin_amdgcn_exp2f(sq * A2[k]);
                            h[4 * i + q + 1][k] = fmaf(a[4 * i + q][k], h[4 * i + q][k], uq * Bv[k]);
                        }
                        if (p.z.p) {
                            float Cv[K];
                            lds_states<K>(&sC[buf][(4 * i + q) * NP], j, Cv);
#pragma unroll
                            for (int k = 0; k < K; ++k) yp[q] = fmaf(h[4 * i + q + 1][k], Cv[k], yp[q]);
                        }
                    }
                    if (p.z.p) {
                        const float y = fmaf(skip, x[i], quad_reduce_scatter(yp, j)), e = sigmoid_f32(z[i]);
                        const int tt = t + 4 * i + j;
                        if (ch.ok && tt < t1) p.dz.p[dzb + tt * p.dz.st + d] = from_f32<T>(dy[i] * y * (e * fmaf(z[i], 1.0f - e, 1.0f)));
                    }
                }
                // the adjoint, backwards
#pragma unroll
                for (int i = G - 1; i >= 0; --i) {
                    float s1[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = 3; q >= 0; --q) {
                        const int m = 4 * i + q;
                        const float sq = qbc(s[i], q), uq = qbc(u[i], q), gq = qbc(g[i], q);
                        float Bv[K], Cv[K], pb[K], pc[K], sums[K / 2];
                        lds_states<K>(&sB[buf][m * NP], j, Bv);
                        lds_states<K>(&sC[buf][m * NP], j, Cv);
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            const float qk = fmaf(Cv[k], gq, w[k]);
                            pc[k] = gq * h[m + 1][k];
                            pb[k] = qk * uq;
                            s1[q] = fmaf(qk, Bv[k], s1[q]);
                            w[k] = a[m][k] * qk;
                            const float v = w[k] * h[m][k];
                            dA[k] = fmaf(v, sq, dA[k]);
                            s2[q] = fmaf(v, A2[k], s2[q]);
                        }
                        channel_sums<K>(pb, pc, sums);
                        if ((lane & 12) == 0) {
                            float* o = &red[wave][m][(lane >> 5) * NP + j * K + ((lane >> 4) & 1) * (K / 2)];
#pragma unroll
                            for (int k = 0; k < K / 2; ++k) o[k] = sums[k];
                        }
                    }
                    const float qB = quad_reduce_scatter(s1, j), wA = quad_reduce_scatter(s2, j) * SNN_LN2;
                    const int tt = t + 4 * i + j;
                    const float dd = fmaf(x[i], qB, wA) * sig[i];
                    if (ch.ok && tt < t1) {
                        p.dx.p[dxb + tt * p.dx.st + d] = from_f32<T>(fmaf(skip, g[i], s[i] * qB));
                        p.ddelta.p[ddb + tt * p.ddelta.st + d] = from_f32<T>(dd);
                        dbs += dd;
                        dsk = fmaf(g[i], x[i], dsk);
                    }
                }
                __syncthreads();
                for (int e = tid; e < SEG * 2 * NP; e += 256) {
                    const int m = e / (2 * NP), o = e % (2 * NP), half = o / NP, n = o % NP, tt = t + m;
                    if (tt < t1) {
                        const float v = (red[0][m][o] + red[1][m][o]) + (red[2][m][o] + red[3][m][o]);
                        if (bcpart) bcpart[(rowb + tt) * (2 * NP) + o] = v;
                        else if (n < p.N) {
                            if (half) p.dC.p[dCb + tt * p.dC.st + n] = from_f32<T>(v);
                            else p.dB.p[dBb + tt * p.dB.st + n] = from_f32<T>(v);
                        }
                    }
                }
            }
            __syncthreads();                  // the next chunk stages into the buffers this one has read
        }
        if (c == 0 && p.dh0 && ch.ok) store_states<K>(p.dh0 + ((int64_t)b * p.D + d) * p.N, j, p.N, p.vec, w);
        const FillRange f = fill_range(p.seq, r, b, t0, t0 + p.tc, c == p.nc - 1);
        const int n = left < SCAN_CH ? left : SCAN_CH;
        clear_channels(p.dx, dxb, f, d0, n, tid);
        clear_channels(p.ddelta, ddb, f, d0, n, tid);
        if (p.dz.p) clear_channels(p.dz, dzb, f, d0, n, tid);
        if (bcpart) {
            for (int64_t e = f.a0 * (2 * NP) + tid; e < f.a1 * (2 * NP); e += 256) bcpart[rowb * (2 * NP) + e] = 0.0f;
            for (int64_t e = f.b0 * (2 * NP) + tid; e < f.b1 * (2 * NP); e += 256) bcpart[rowb * (2 * NP) + e] = 0.0f;
        } else {
            clear_channels(p.dB, dBb, f, 0, p.N, tid);
            clear_channels(p.dC, dCb, f, 0, p.N, tid);
        }
    }
    dsk = quad_sum(dsk);
    dbs = quad_sum(dbs);
    if (ch.ok) {
        float* q = p.part + (int64_t)slot * part_stride(p.D, NP);
        store_states<K>(q + (int64_t)d * NP, j, NP, true, dA);
        if (j == 0) {
            q[(int64_t)p.D * NP + d] = dsk;
            q[(int64_t)p.D * (NP + 1) + d] = dbs;
        }
    }
}

// dA (D, N), dskip (D), dbias (D) from the slots' partial sums: 32 columns x 8 rows of threads, fp64, fixed order
__global__ void __launch_bounds__(256) scan_param_sum_kernel(const float* __restrict__ part, int slots, int D, int N, int NP, float* dA, float* dskip,
                                                             float* dbias)
{
    __shared__ double s[8][32];
    const int64_t n = (int64_t)D * (NP + 2), stride = part_stride(D, NP), col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int row = threadIdx.x >> 5;
    double a = 0.0;
    if (col < n)
        for (int i = row; i < slots; i += 8) a += part[(int64_t)i * stride + col];
    s[row][threadIdx.x & 31] = a;
    __syncthreads();
    if (row == 0 && col < n) {
#pragma unroll
        for (int i = 1; i < 8; ++i) a += s[i][threadIdx.x];
        if (col < (int64_t)D * NP) {
            const int d = (int)(col / NP), k = (int)(col - (int64_t)d * NP);
            if (k < N) dA[(int64_t)d * N + k] = (float)a;
        } else if (col < (int64_t)D * (NP + 1)) {
            if (dskip) dskip[col - (int64_t)D * NP] = (float)a;
        } else if (dbias) dbias[col - (int64_t)D * (NP + 1)] = (float)a;
    }
}

// dB, dC rows from the channel blocks' partial rows (cleared rows included), in block order
template <typename T> __global__ void __launch_bounds__(256) scan_bc_sum_kernel(const ScanP<T> p, int NP, int groups)
{
    const int64_t rows = p.seq.offsets ? p.seq.n_rows : (int64_t)p.seq.n_seq * p.seq.max_T, per = (int64_t)groups * 2 * NP;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * per) return;
    const int64_t row = id / per;
    const int e = (int)(id - row * per), g = e / (2 * NP), o = e - g * 2 * NP, half = o / NP, n = o - half * NP;
    if (n >= p.N) return;
    const float* q = p.bcpart + ((int64_t)g * p.cbg * rows + row) * (2 * NP) + o;
    float a = 0.0f;
    for (int i = 0; i < p.cbg; ++i) a += q[(int64_t)i * rows * (2 * NP)];
    int64_t t = row, b = 0;
    if (!p.seq.offsets) {
        b = row / p.seq.max_T;
        t = row - b * p.seq.max_T;
    }
    if (half) p.dC.p[t * p.dC.st + b * p.dC.sb + g * p.N + n] = from_f32<T>(a);
    else p.dB.p[t * p.dB.st + b * p.dB.sb + g * p.N + n] = from_f32<T>(a);
}

struct Sizes { int64_t carry, csum, part, bc; int slots; };
// Slots: workgroups that share the chunks.  2048 of them all told keep four on every compute unit in turn and even out
// ragged lengths; more would only add partial sums to write and read.
Sizes sizes(const snn_scan_args* a, const ScanGrid& g)
{
    const int NP = 4 * scan_k(a->states);
    const int64_t items = (int64_t)a->seq.n_seq * g.nc;
    Sizes z;
    z.slots = (int)std::min<int64_t>(items, std::max<int64_t>(1, 2048 / g.blocks_c));
    z.carry = g.nc > 1 ? items * a->channels * NP : 0;
    z.csum = g.nc > 1 ? (items * a->channels + 3) / 4 * 4 : 0;
    z.part = (int64_t)z.slots * part_stride(a->channels, NP);
    const int64_t rows = a->seq.offsets ? a->seq.n_rows : (int64_t)a->seq.n_seq * a->seq.max_T;
    z.bc = g.cbg > 1 ? (int64_t)g.blocks_c * rows * 2 * NP : 0;
    return z;
}

template <typename T, int K> int backward(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    ScanP<T> p = scan_params<T>(a, g);
    const Sizes z = sizes(a, g);
    p.carry = (float*)a->ws;
    p.csum = p.carry + z.carry;
    p.part = p.csum + z.csum;
    p.bcpart = z.bc ? p.part + z.part : nullptr;
    p.slots = z.slots;
    const int64_t blocks = (int64_t)g.blocks_c * a->seq.n_seq * g.nc;
    if (g.nc > 1) {
        hipLaunchKernelGGL((scan_adjoint_kernel<T, K>), dim3((unsigned)blocks), dim3(256), 0, s, p);
        snn_scan_launch_combine(a, g, a->dstate_out, p.carry, p.csum, true, s);
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, K>), dim3((unsigned)(g.blocks_c * z.slots)), dim3(256), 0, s, p);
    const int64_t n = (int64_t)p.D * (4 * K + 2);
    hipLaunchKernelGGL(scan_param_sum_kernel, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, s, (const float*)p.part, z.slots, p.D, p.N, 4 * K,
                       a->dA, a->dskip, a->ddelta_bias);
    if (z.bc) {
        const int64_t rows = a->seq.offsets ? a->seq.n_rows : (int64_t)a->seq.n_seq * a->seq.max_T;
        const int64_t e = (rows * a->groups * 8 * K + 255) / 256;
        hipLaunchKernelGGL((scan_bc_sum_kernel<T>), dim3((unsigned)e), dim3(256), 0, s, p, 4 * K, a->groups);
    }
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T> int run(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    switch (scan_k(a->states)) {
    case 2: return backward<T, 2>(a, g, s);
    case 4: return backward<T, 4>(a, g, s);
    case 8: return backward<T, 8>(a, g, s);
    default: return backward<T, 16>(a, g, s);
    }
}

}  // namespace

extern "C" int64_t snn_scan_workspace_bytes(const snn_scan_args* a, int32_t backward_pass)
{
    if (int rc = snn_scan_check(a, "snn_scan_workspace_bytes")) return rc;
    const ScanGrid g = snn_scan_grid(a, backward_pass != 0);
    const Sizes z = sizes(a, g);
    return 4 * (z.carry + z.csum + (backward_pass ? z.part + z.bc : 0));
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
    const ScanGrid g = snn_scan_grid(a, true);
    const int64_t rows = a->seq.offsets ? a->seq.n_rows : (int64_t)a->seq.n_seq * a->seq.max_T;
    if ((int64_t)g.blocks_c * a->seq.n_seq * g.nc > 0x7fffffff || (rows * a->groups * 8 * scan_k(a->states) + 255) / 256 > 0x7fffffff) {
        snn_set_error("snn_scan_backward: grid too large");
        return SNN_ERR_UNSUPPORTED;
    }
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == SNN_DT_F32 ? run<float>(a, g, s) : a->dtype == SNN_DT_BF16 ? run<bf16_t>(a, g, s) : run<f16_t>(a, g, s);
}
