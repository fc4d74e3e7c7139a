// snn_scan.hip -- selective scan: forward (with the training tape) and the single step (include/snn_hip.h: snn_scan_*).
//
//   s_t = softplus(delta_t + bias),  h_t = exp(s_t A) h_{t-1} + s_t x_t B_t,  y_t = (C_t . h_t + skip x_t) silu(z_t)
//
// Per (step, channel, state): one product and one v_exp_f32 (half rate on gfx950) for the decay, one product, two
// fused multiply-adds: 6 issue slots, against 8 bytes (bf16, gated) per (step, channel) of up to 64 states.
// The vector unit bounds the scan, not the memory; so the state stays in registers, everything per step is done once per
// quad of lanes and not once per lane, and nothing is computed twice unless there is too little to do at once:
// where channels x sequences do not fill the chip, the time axis is cut into chunks that run side by side.  Then
// scan_fwd_kernel<STATE_ONLY> finds every chunk's last state from a zero start (and the sum of its steps: the decay over the
// whole chunk is exp(A sum s)), scan_combine_kernel runs over the chunks, and scan_fwd_kernel starts each chunk from its
// true state: 1.7 times the time of a single pass that filled the chip, over `nc` times the lanes.
// One prompt of 8191 x 4096 bf16, 16 states: 111 + 8 + 172 us, 22 and 33 vector instructions a lane's step of four states where the
// formula's (step, channel, state) terms take 16 and 20: the rest is per step (softplus, gate, sums over the states, conversions, loads
// and stores).  The vector unit is busy 0.96 and 0.89 of the time.  16384 sequences of up to 40 x 64 fp32: 120 us.
#include <algorithm>
#include "snn_host.h"
#include "snn_scan.h"

#define HIP_CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { \
    snn_set_error("%s: %s", #x, hipGetErrorString(e_)); return SNN_ERR_HIP; } } while (0)

namespace {

// STATE_ONLY: chunk c's last state from a zero start into carry[b][c + 1], the sum of its steps into csum[b][c].
template <typename T, int K, int LN, bool STATE_ONLY, bool GATE> __global__ void __launch_bounds__(256) scan_fwd_kernel(const ScanP<T> p)
{
    constexpr int SEG = SCAN_SEG, G = SEG / 4, TS = ScanTape<K>::STEPS, NP = K * LN, CH = 256 / LN;
    __shared__ float sB[2][SEG * NP], sC[2][STATE_ONLY ? 1 : SEG * NP];
    const int tid = threadIdx.x, c = blockIdx.z;
    const int b = p.order ? p.order[blockIdx.y] : blockIdx.x, cb = p.order ? blockIdx.x : blockIdx.y;
    const ScanCh ch = scan_channel<K, LN>(cb, p.cbg, p.dg, tid);
    const int j = ch.j, d = ch.d;
    const SeqRange r = seq_range(p.seq, b);
    const int t0 = c * p.tc, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
    if (STATE_ONLY && (t0 >= r.len || t0 + p.tc >= r.len)) return;      // nothing follows the chunk that ends the sequence
    float h[K], A2[K];
    load_states<K>(p.A + (int64_t)d * p.N, ch.n, p.N, p.vec, A2);
#pragma unroll
    for (int k = 0; k < K; ++k) h[k] = 0.0f;
    if (!STATE_ONLY) {
        if (c > 0) {
            if (t0 < r.len) load_states<K>(p.carry + (((int64_t)b * p.nc + c) * p.D + d) * NP, ch.n, NP, true, h);
        } else if (p.h0) load_states<K>(p.h0 + ((int64_t)b * p.D + d) * p.N, ch.n, p.N, p.vec, h);
    }
    float ssum = 0.0f;
    if (t0 < t1) {
        const float bias = p.dbias ? p.dbias[d] : 0.0f, skip = !STATE_ONLY && p.skip ? p.skip[d] : 0.0f;
        const int64_t first = r.row0 + t0 + j;
        const T* xp = p.x.p + first * p.x.st + b * p.x.sb + d;
        const T* dp = p.delta.p + first * p.delta.st + b * p.delta.sb + d;
        const T* zp = GATE ? p.z.p + first * p.z.st + b * p.z.sb + d : nullptr;
        T* yp = STATE_ONLY ? nullptr : p.y.p + first * p.y.st + b * p.y.sb + d;
        const bool keep = !STATE_ONLY && p.tape;
        float* tape = keep ? p.tape + ((scan_tape_first(p.seq, r, b, TS) + t0 / TS) * p.D + d) * NP + ch.n : nullptr;
        LaneIn<T, G> xi, di, zi;
        RowStage<T, NP, SEG> Bi, Ci;
        Bi.init(p.B.p + (r.row0 + t0) * p.B.st + b * p.B.sb + ch.g * p.B_sg, p.B.st, p.N, tid);
        if (!STATE_ONLY) Ci.init(p.C.p + (r.row0 + t0) * p.C.st + b * p.C.sb + ch.g * p.C_sg, p.C.st, p.N, tid);
        auto fetch = [&](int left) {                    // the next segment; `left` steps from its start to the chunk's end
            xi.load(xp, p.x.st, j, left);
            di.load(dp, p.delta.st, j, left);
            if (GATE) zi.load(zp, p.z.st, j, left);
            Bi.load(p.B.st, left);
            if (!STATE_ONLY) Ci.load(p.C.st, left);
            xp += SEG * p.x.st;
            dp += SEG * p.delta.st;
            if (GATE) zp += SEG * p.z.st;
            Bi.p += SEG * p.B.st;
            if (!STATE_ONLY) Ci.p += SEG * p.C.st;
        };
        fetch(t1 - t0);                                 // before anything waits for the loads above: one latency, not two
        decay_rates<K>(A2);
        int buf = 0;
        for (int t = t0; t < t1; t += SEG, buf ^= 1) {
            Bi.store(sB[buf], tid);
            if (!STATE_ONLY) Ci.store(sC[STATE_ONLY ? 0 : buf], tid);
            const int left = t1 - t;                     // steps from here to the chunk's end
            float u[G], s[G], xf[G], zf[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                if (4 * i >= left) break;
                xf[i] = to_f32(xi.v[i]);
                if (GATE) zf[i] = to_f32(zi.v[i]);
                const float v = to_f32(di.v[i]) + bias;
                s[i] = p.softplus ? softplus_f32(v, nullptr) : v;
                u[i] = s[i] * xf[i];
            }
            if (left < SEG) {                            // a step of zero leaves the state as it is
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    if (4 * i >= left) break;
                    const bool live = 4 * i + j < left;
                    s[i] = live ? s[i] : 0.0f;
                    u[i] = live ? u[i] : 0.0f;
                }
            }
            __syncthreads();      // one barrier a segment: the other buffer was last read before the barrier of the segment before
            if (left > SEG) fetch(left - SEG);
            float Bv[2][K], Cv[2][K];                    // of this step and the next
            auto read = [&](int m) {
                lds_states<K>(&sB[buf][m * NP], ch.n, Bv[m & 1]);
                if (!STATE_ONLY) lds_states<K>(&sC[STATE_ONLY ? 0 : buf][m * NP], ch.n, Cv[m & 1]);
            };
            read(0);
#pragma unroll
            for (int i = 0; i < G; ++i) {
                if (4 * i >= left) break;
                if (keep && (4 * i) % TS == 0) {
                    if (ch.ok) store_states<K>(tape, 0, NP, true, h);
                    tape += (int64_t)p.D * NP;
                }
                float yv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = 4 * i + q;
                    if (m + 1 < SEG) read(m + 1);
                    pin_lds_reads();
                    const float sq = qbc(s[i], q), uq = qbc(u[i], q);
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        h[k] = fmaf(__builtin_amdgcn_exp2f(sq * A2[k]), h[k], uq * Bv[m & 1][k]);
                        if (!STATE_ONLY) yv[q] = fmaf(h[k], Cv[m & 1][k], yv[q]);
                    }
                }
                if (STATE_ONLY) ssum += s[i];
                else {
                    float y = fmaf(skip, xf[i], step_sums<LN>(yv, j));
                    if (GATE) y *= zf[i] * sigmoid_f32(zf[i]);
                    if (ch.lead && 4 * i + j < left) yp[4 * i * p.y.st] = from_f32<T>(y);
                }
            }
            if (!STATE_ONLY) yp += SEG * p.y.st;
        }
    }
    if (STATE_ONLY) {
        ssum = quad_sum(ssum);
        if (ch.ok) {
            store_states<K>(p.carry + (((int64_t)b * p.nc + c + 1) * p.D + d) * NP, ch.n, NP, true, h);
            if (ch.n == 0) p.csum[((int64_t)b * p.nc + c) * p.D + d] = ssum;
        }
        return;
    }
    if (p.hT && ch.ok && (r.len > 0 ? t0 < r.len && r.len <= t0 + p.tc : c == 0))
        store_states<K>(p.hT + ((int64_t)b * p.D + d) * p.N, ch.n, p.N, p.vec, h);
    const int left = p.dg - (cb - ch.g * p.cbg) * CH;
    clear_channels(p.y, r.row0 * p.y.st + b * p.y.sb, fill_range(p.seq, r, b, t0, t0 + p.tc, c == p.nc - 1), ch.g * p.dg + p.dg - left,
                   left < CH ? left : CH, tid);
}

// order[r] = the sequence of rank r by length, longest first, equal ones by index: workgroups are dealt longest first, so that the
// last ones to run are short.  A wave counts the sequences in front of its own.
__global__ void __launch_bounds__(256) scan_order_kernel(const snn_seq seq, int* order)
{
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (b >= seq.n_seq) return;
    const int len = seq_range(seq, b).len;
    int rank = 0;
#pragma unroll 4
    for (int j = lane; j < seq.n_seq; j += 64) {
        const int l = seq_range(seq, j).len;
        rank += l > len || (l == len && j < b);
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) rank += __shfl_xor(rank, m);
    if (lane == 0) order[rank] = b;
}

// h 2^p + v.  2^p itself would overflow for p >= 128 (the decay over a chunk of growing states) where its product with a small h does
// not: the whole part of p goes to the exponent of h.  At 1000 and -1000 any h is inf or 0 already; a NaN stays.
struct Pow2 { float frac; int whole; };
__device__ __forceinline__ Pow2 pow2_parts(float p)
{
    const float q = p > 1000.0f ? 1000.0f : p, w = fmaxf(floorf(q), -1000.0f);
    return Pow2{__builtin_amdgcn_exp2f(q - w), (int)w};
}
__device__ __forceinline__ float decayed(float h, const Pow2& e, float v) { return fmaf(e.frac, ldexpf(h, e.whole), v); }

// carry[b][c] from the chunks' local results, over the chunks of a sequence.  Forward: slot c holds chunk c-1's local last
// state; state entering c = exp(A csum[c-1]) (state entering c-1) + slot c, from the initial state.  Reverse: slot c holds
// what chunk c+1 sends back from a zero start; entering c = slot c + exp(A csum[c+1]) (entering c+1), from `edge` (or 0) in
// the chunk that ends the sequence.
__global__ void __launch_bounds__(256) scan_combine_kernel(snn_seq seq, int D, int N, int NP, int tc, int nc, const float* A, const float* edge,
                                                           float* carry, const float* csum, int reverse)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)D * NP;
    if (id >= (int64_t)seq.n_seq * per) return;
    const int b = (int)(id / per), e = (int)(id - b * per), d = e / NP, n = e - d * NP;
    const int len = seq_range(seq, b).len, used = (len + tc - 1) / tc;
    float a2[1] = {n < N ? A[(int64_t)d * N + n] : 0.0f};
    decay_rates<1>(a2);
    float h = edge && n < N ? edge[((int64_t)b * D + d) * N + n] : 0.0f;
    float* q = carry + (int64_t)b * nc * per + e;
    const float* cs = csum + (int64_t)b * nc * D + d;
    // eight chunks' results and decays are fetched at a time: only the chain of multiply-adds is sequential
    const int n_steps = used - 1;
    if (reverse && used > 0) q[(int64_t)n_steps * per] = h;
    for (int i0 = 0; i0 < n_steps; i0 += 8) {
        float v[8];
        Pow2 e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = i0 + i < n_steps ? i0 + i : n_steps - 1, c = reverse ? n_steps - 1 - k : k + 1;
            v[i] = q[c * per];
            e[i] = pow2_parts(a2[0] * cs[(int64_t)(reverse ? c + 1 : c - 1) * D]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i < n_steps) {
                h = decayed(h, e[i], v[i]);
                q[(int64_t)(reverse ? n_steps - 1 - i0 - i : i0 + i + 1) * per] = h;
            }
        }
    }
}

// One step: 8 bytes of fp32 state per (channel, state) in and out, all else is a percent of that: the memory bounds it.
// The same lanes; a wave reads its neighbouring channels' states as one block, 16 bytes a lane.  256 sequences x 4096 channels x 16
// states: 31 us with the state in the last-level cache, 40 us a call at 151 MB; two or four sequences a thread: 41 and 42.
template <typename T, int K, int LN> __global__ void __launch_bounds__(256) scan_step_kernel(const ScanP<T> p)
{
    constexpr int CH = 256 / LN;
    const int cbs = (p.D + CH - 1) / CH, b = blockIdx.x / cbs, i = (blockIdx.x - b * cbs) * CH + threadIdx.x / LN;
    const bool ok = i < p.D;
    const int d = ok ? i : p.D - 1, g = d / p.dg, n = threadIdx.x % LN * K;
    float h[K], A2[K];
    T Bv[K], Cv[K];
    load_states<K>(p.h0 + ((int64_t)b * p.D + d) * p.N, n, p.N, p.vec, h);       // everything is fetched before anything is used
    const float x = to_f32(p.x.p[b * p.x.sb + d]), delta = to_f32(p.delta.p[b * p.delta.sb + d]);
    const float z = p.z.p ? to_f32(p.z.p[b * p.z.sb + d]) : 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int m = n + k < p.N ? n + k : p.N - 1;
        Bv[k] = p.B.p[b * p.B.sb + g * p.B_sg + m];
        Cv[k] = p.C.p[b * p.C.sb + g * p.C_sg + m];
    }
    load_states<K>(p.A + (int64_t)d * p.N, n, p.N, p.vec, A2);
    decay_rates<K>(A2);
    const float v = delta + (p.dbias ? p.dbias[d] : 0.0f), skip = p.skip ? p.skip[d] : 0.0f;
    const float s = p.softplus ? softplus_f32(v, nullptr) : v, u = s * x;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const bool in = n + k < p.N;
        h[k] = fmaf(__builtin_amdgcn_exp2f(s * A2[k]), h[k], in ? u * to_f32(Bv[k]) : 0.0f);
        y = in ? fmaf(h[k], to_f32(Cv[k]), y) : y;
    }
    y = quad_sum(y);
    if (LN >= 8) y += dpp<0x141>(y);
    if (LN >= 16) y += dpp<0x140>(y);
    if (!ok) return;
    store_states<K>(p.hT + ((int64_t)b * p.D + d) * p.N, n, p.N, p.vec, h);
    if (n == 0) {
        y = fmaf(skip, x, y);
        if (p.z.p) y *= z * sigmoid_f32(z);
        p.y.p[b * p.y.sb + d] = from_f32<T>(y);
    }
}

}  // namespace

// ---- host ---------------------------------------------------------------------------------------------------------
int snn_scan_check(const snn_scan_args* a, const char* fn)
{
    if (!a) { snn_set_error("%s: args is NULL", fn); return SNN_ERR_ARG; }
    if (a->seq.n_seq < 1 || a->seq.max_T < 1 || a->channels < 1 || a->groups < 1 || a->channels % a->groups || a->seq.n_rows < 0) {
        snn_set_error("%s: n_seq, max_T, channels and groups must be positive and groups divide channels", fn);
        return SNN_ERR_ARG;
    }
    if (a->dtype < 0 || a->dtype > 2 || a->states < 1 || a->states > 64) {
        snn_set_error("%s: dtype %d / %d states: supported are dtypes 0..2 (SNN_DT_*) and 1..64 states", fn, a->dtype, a->states);
        return SNN_ERR_UNSUPPORTED;
    }
    if (!snn_sizes_fit(a->seq, a->channels)) {
        snn_set_error("%s: at most 2^24 - 1 sequences, 2^30 steps and 2^19 channels", fn);
        return SNN_ERR_UNSUPPORTED;
    }
    if (a->seq.lengths && a->seq.offsets) { snn_set_error("%s: lengths and offsets exclude each other", fn); return SNN_ERR_ARG; }
    const int ch = 256 / scan_lanes(a->states);
    if ((int64_t)((a->channels / a->groups + ch - 1) / ch) * a->groups > 65535) {        // the grid's second dimension
        snn_set_error("%s: %d channels in %d groups are more than 65535 workgroups of %d", fn, a->channels, a->groups, ch);
        return SNN_ERR_UNSUPPORTED;
    }
    return SNN_OK;
}

// Chunks of the time axis.  One chunk (no arithmetic twice) once the workgroups of a single pass give every SIMD two waves
// (512 workgroups): whole calls of 1024 steps x 4096 channels bf16, split / not, 138 / 148 us at 256 workgroups, 185 / 194 at
// 384, 234 / 195 at 512.  Below that, as many chunks as bring the grid to 2048 workgroups, none shorter than 64 steps; 4096 for
// sequences of different lengths, whose empty chunks leave the chip half full otherwise.  scan_combine_kernel walks over the chunks
// one by one.  The count takes every sequence for one of max_T steps, so one long sequence among short ones is not split once they
// are 512 workgroups together, and then runs on its own ones alone: 8192 rows x 4096 bf16 261 us, with six sequences of 64 522, with
// seven (512 workgroups) 1302.  State pass + combination + scan in us, grids of 1024 / 2048 / 4096 / 8192 workgroups: one prompt of 8191 x 4096
// bf16 124 + 5 + 194 / 111 + 7 + 171 / 112 + 12 + 174 / 106 + 19 + 177; seven ragged prompts of up to 1501 x 1536 fp16
// 52 + 5 + 78 / 43 + 5 + 59 / 37 + 7 + 54 / 35 + 11 + 52.
ScanGrid snn_scan_grid(const snn_scan_args* a)
{
    ScanGrid g;
    const int dg = a->channels / a->groups;
    const int ch = 256 / scan_lanes(a->states);
    g.cbg = (dg + ch - 1) / ch;
    g.blocks_c = g.cbg * a->groups;
    const int64_t blocks = (int64_t)g.blocks_c * a->seq.n_seq;
    int64_t nc = 1;
    const int64_t target = a->seq.lengths || a->seq.offsets ? 4096 : 2048;
    if (blocks < 512) nc = std::min<int64_t>((target + blocks - 1) / blocks, (a->seq.max_T + 63) / 64);
    g.tc = (int)(((a->seq.max_T + nc - 1) / nc + SCAN_SEG - 1) / SCAN_SEG * SCAN_SEG);
    g.nc = (a->seq.max_T + g.tc - 1) / g.tc;
    return g;
}

// Longest first pays where the grid runs in a few rounds (512 workgroups and more, one chunk a sequence) over sequences of different
// lengths: training of 512 x 300 x 256 fp32 504 -> 410 us, the ranks' 2 x 5 us included.  Beyond 4096 sequences the rounds are many
// and even out, and the ranks, whose time goes with the square of the sequences, would cost more than they give.
bool snn_scan_ordered(const snn_scan_args* a, const ScanGrid& g)
{
    return (a->seq.lengths || a->seq.offsets) && (int64_t)g.blocks_c * a->seq.n_seq >= 512 && a->seq.n_seq > 1 && a->seq.n_seq <= 4096;
}
void snn_scan_launch_order(const snn_seq& seq, int* order, hipStream_t s)
{
    hipLaunchKernelGGL(scan_order_kernel, dim3((unsigned)((seq.n_seq + 3) / 4)), dim3(256), 0, s, seq, order);
}

template <typename T> ScanP<T> scan_params(const snn_scan_args* a, const ScanGrid& g)
{
    ScanP<T> p;
    p.seq = a->seq;
    p.x = snn_view_of<T>(a->x);
    p.delta = snn_view_of<T>(a->delta);
    p.z = snn_view_of<T>(a->z);
    p.B = snn_view_of<T>(a->B);
    p.C = snn_view_of<T>(a->C);
    p.y = snn_view_of<T>(a->y);
    p.B_sg = a->B_stride_g;
    p.C_sg = a->C_stride_g;
    p.A = a->A;
    p.skip = a->skip;
    p.dbias = a->delta_bias;
    p.h0 = a->state_in;
    p.hT = a->state_out;
    p.tape = a->tape;
    p.D = a->channels;
    p.N = a->states;
    p.dg = a->channels / a->groups;
    p.cbg = g.cbg;
    p.softplus = a->softplus;
    p.tc = g.tc;
    p.nc = g.nc;
    const int NP = scan_padded(a->states);
    p.carry = (float*)a->ws;
    p.csum = p.carry + (int64_t)a->seq.n_seq * g.nc * a->channels * NP;
    const uintptr_t al = (uintptr_t)a->A | (uintptr_t)a->state_in | (uintptr_t)a->state_out | (uintptr_t)a->dstate_out | (uintptr_t)a->dstate_in;
    p.vec = a->states == NP && al % 16 == 0;
    p.dy = snn_view_of<T>(a->dy);
    p.dx = snn_view_of<T>(a->dx);
    p.ddelta = snn_view_of<T>(a->ddelta);
    p.dz = snn_view_of<T>(a->dz);
    p.dB = snn_view_of<T>(a->dB);
    p.dC = snn_view_of<T>(a->dC);
    p.dhT = a->dstate_out;
    p.dh0 = a->dstate_in;
    p.part = p.bcpart = nullptr;
    p.slots = 0;
    p.order = nullptr;
    return p;
}
template ScanP<float> scan_params<float>(const snn_scan_args*, const ScanGrid&);
template ScanP<bf16_t> scan_params<bf16_t>(const snn_scan_args*, const ScanGrid&);
template ScanP<f16_t> scan_params<f16_t>(const snn_scan_args*, const ScanGrid&);

void snn_scan_launch_combine(const snn_scan_args* a, const ScanGrid& g, const float* edge, float* carry, const float* csum, bool reverse, hipStream_t s)
{
    const int NP = scan_padded(a->states);
    const int64_t n = (int64_t)a->seq.n_seq * a->channels * NP;
    hipLaunchKernelGGL(scan_combine_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a->seq, a->channels, a->states, NP, g.tc, g.nc,
                       a->A, edge, carry, csum, (int)reverse);
}

namespace {
template <typename T, int K, int LN> int forward(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    ScanP<T> p = scan_params<T>(a, g);
    dim3 grid((unsigned)a->seq.n_seq, (unsigned)g.blocks_c, (unsigned)g.nc);
    if (snn_scan_ordered(a, g)) {
        snn_scan_launch_order(a->seq, (int*)a->ws, s);
        p.order = (const int*)a->ws;
        std::swap(grid.x, grid.y);
    }
    if (g.nc > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<T, K, LN, true, false>), grid, dim3(256), 0, s, p);
        snn_scan_launch_combine(a, g, a->state_in, p.carry, p.csum, false, s);
    }
    if (a->z.p) hipLaunchKernelGGL((scan_fwd_kernel<T, K, LN, false, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((scan_fwd_kernel<T, K, LN, false, false>), grid, dim3(256), 0, s, p);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T, int K, int LN> int step(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    const ScanP<T> p = scan_params<T>(a, g);
    const int64_t blocks = (int64_t)((a->channels + 256 / LN - 1) / (256 / LN)) * a->seq.n_seq;
    if (blocks > SEQ_MAX_BLOCKS) { snn_set_error("snn_scan_step: %lld workgroups", (long long)blocks); return SNN_ERR_UNSUPPORTED; }
    hipLaunchKernelGGL((scan_step_kernel<T, K, LN>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T> int run(const snn_scan_args* a, const ScanGrid& g, bool one, hipStream_t s)
{
    if (a->states <= 8) return one ? step<T, 2, 4>(a, g, s) : forward<T, 2, 4>(a, g, s);
    if (a->states <= 16) return one ? step<T, 4, 4>(a, g, s) : forward<T, 4, 4>(a, g, s);
    if (a->states <= 32) return one ? step<T, 4, 8>(a, g, s) : forward<T, 4, 8>(a, g, s);
    return one ? step<T, 4, 16>(a, g, s) : forward<T, 4, 16>(a, g, s);
}
int dispatch(const snn_scan_args* a, bool one, hipStream_t s)
{
    const ScanGrid g = snn_scan_grid(a);
    return a->dtype == SNN_DT_F32 ? run<float>(a, g, one, s) : a->dtype == SNN_DT_BF16 ? run<bf16_t>(a, g, one, s) : run<f16_t>(a, g, one, s);
}
}  // namespace

extern "C" int64_t snn_scan_tape_floats(const snn_scan_args* a)
{
    if (int rc = snn_scan_check(a, "snn_scan_tape_floats")) return rc;
    return scan_tape_slots(a->seq, scan_tape_steps(a->states)) * a->channels * scan_padded(a->states);
}

extern "C" int snn_scan_forward(const snn_scan_args* a, void* stream)
{
    if (int rc = snn_scan_check(a, "snn_scan_forward")) return rc;
    if (!a->x.p || !a->delta.p || !a->B.p || !a->C.p || !a->y.p || !a->A || (a->state_out && a->state_out == a->state_in) ||
        ((uintptr_t)a->tape | (uintptr_t)a->ws) % 16) {
        snn_set_error("snn_scan_forward: null or misaligned pointer, or state_out is state_in");
        return SNN_ERR_ARG;
    }
    const int64_t need = snn_scan_workspace_bytes(a, 0);
    if (a->ws_bytes < need || (need && !a->ws) || (a->tape && a->tape_floats < snn_scan_tape_floats(a))) {
        snn_set_error("snn_scan_forward: workspace of %lld bytes (%lld needed) or tape of %lld floats too small", (long long)a->ws_bytes,
                      (long long)need, (long long)a->tape_floats);
        return SNN_ERR_WORKSPACE;
    }
    return dispatch(a, false, (hipStream_t)stream);
}

extern "C" int snn_scan_step(const snn_scan_args* a, void* stream)
{
    if (int rc = snn_scan_check(a, "snn_scan_step")) return rc;
    if (!a->x.p || !a->delta.p || !a->B.p || !a->C.p || !a->y.p || !a->A || !a->state_in || !a->state_out || a->seq.max_T != 1 ||
        a->seq.lengths || a->seq.offsets) {
        snn_set_error("snn_scan_step: null pointer, or max_T, lengths or offsets of more than one step");
        return SNN_ERR_ARG;
    }
    return dispatch(a, true, (hipStream_t)stream);
}
