// snn_scan.hip -- selective scan: forward (with the training tape) and the single step (include/snn_hip.h: snn_scan_*).
//
//   s_t = softplus(delta_t + bias),  h_t = exp(s_t A) h_{t-1} + s_t x_t B_t,  y_t = (C_t . h_t + skip x_t) silu(z_t)
//
// Per (step, channel, state): one product and one v_exp_f32 (a quarter-rate instruction) for the decay, one product, two
// fused multiply-adds: 8 issue slots for 7 operations, against 8 bytes (bf16, gated) per (step, channel) of up to 64 states.
// The vector unit bounds the scan, not the memory; so the state stays in registers, everything per step is done once per
// quad of lanes and not once per lane, and nothing is computed twice unless there is too little to do at once:
// where channels x sequences do not fill the chip, the time axis is cut into chunks that run side by side.  Then
// scan_state_kernel finds every chunk's last state from a zero start (and the sum of its steps: the decay over the
// whole chunk is exp(A sum s)), scan_combine_kernel runs over the chunks, and scan_fwd_kernel starts each chunk from its
// true state: 1.9 times the arithmetic over `nc` times the lanes.
#include <algorithm>
#include "snn_host.h"
#include "snn_scan.h"

#define HIP_CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { \
    snn_set_error("%s: %s", #x, hipGetErrorString(e_)); return SNN_ERR_HIP; } } while (0)

namespace {

// one segment's inputs of a lane: steps t + j, t + 4 + j, ... of four, prefetched a segment ahead
template <typename T, int G> struct SegIn {
    T x[G], d[G], z[G];
    __device__ __forceinline__ void load(const ScanP<T>& p, int64_t xb, int64_t db, int64_t zb, int t, int t1, bool state_only)
    {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if (t + 4 * i < t1) {
                x[i] = p.x.p[xb + (t + 4 * i) * p.x.st];
                d[i] = p.delta.p[db + (t + 4 * i) * p.delta.st];
                if (!state_only && p.z.p) z[i] = p.z.p[zb + (t + 4 * i) * p.z.st];
            }
        }
    }
};

// STATE_ONLY: chunk c's last state from a zero start into carry[b][c + 1], the sum of its steps into csum[b][c].
template <typename T, int K, bool STATE_ONLY> __global__ void __launch_bounds__(256) scan_fwd_kernel(const ScanP<T> p)
{
    constexpr int SEG = SCAN_SEG, G = SEG / 4, TS = ScanTape<K>::STEPS;
    __shared__ float sB[2][SEG * 4 * K], sC[2][STATE_ONLY ? 1 : SEG * 4 * K];
    const int tid = threadIdx.x, nch = p.D / p.dg * p.cbg, cb = blockIdx.x % nch;
    const int item = blockIdx.x / nch, b = item / p.nc, c = item - b * p.nc;
    const ScanCh ch = scan_channel(cb, p.cbg, p.dg, tid);
    const int j = ch.j, d = ch.d;
    const SeqRange r = seq_range(p.seq, b);
    const int t0 = c * p.tc, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
    const bool last = c == p.nc - 1;
    if (STATE_ONLY && (t0 >= r.len || t0 + p.tc >= r.len)) return;      // nothing follows the chunk that ends the sequence
    const int64_t xb = r.row0 * p.x.st + b * p.x.sb + d, db = r.row0 * p.delta.st + b * p.delta.sb + d;
    const int64_t zb = r.row0 * p.z.st + b * p.z.sb + d, yb = r.row0 * p.y.st + b * p.y.sb + d;
    const T* Bp = p.B.p + r.row0 * p.B.st + b * p.B.sb + ch.g * p.B_sg;
    const T* Cp = p.C.p + r.row0 * p.C.st + b * p.C.sb + ch.g * p.C_sg;
    float h[K], A2[K];
    load_states<K>(p.A + (int64_t)d * p.N, j, p.N, p.vec, A2);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        A2[k] *= SNN_LOG2E;
        h[k] = 0.0f;
    }
    if (!STATE_ONLY) {
        if (c > 0) {
            if (t0 < r.len) load_states<K>(p.carry + (((int64_t)b * p.nc + c) * p.D + d) * (4 * K), j, 4 * K, true, h);
        } else if (p.h0) load_states<K>(p.h0 + ((int64_t)b * p.D + d) * p.N, j, p.N, p.vec, h);
    }
    const float bias = p.dbias ? p.dbias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
    float* tape = nullptr;
    if (!STATE_ONLY && p.tape) tape = p.tape + ((scan_tape_first(p.seq, r, b, TS) + t0 / TS) * p.D + d) * (4 * K);
    float ssum = 0.0f;
    SegIn<T, G> in;
    BcStage<T, K, SEG> bc;
    if (t0 < t1) {
        in.load(p, xb, db, zb, t0 + j, t1, STATE_ONLY);
        bc.template load<!STATE_ONLY>(Bp, p.B.st, Cp, p.C.st, t0, t1, p.N, tid);
    }
    int buf = 0;
    for (int t = t0; t < t1; t += SEG, buf ^= 1) {
        bc.template store<!STATE_ONLY>(sB[buf], sC[STATE_ONLY ? 0 : buf], tid);
        float u[G], s[G], xf[G], zf[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const bool live = t + 4 * i + j < t1;
            xf[i] = live ? to_f32(in.x[i]) : 0.0f;
            zf[i] = live && !STATE_ONLY && p.z.p ? to_f32(in.z[i]) : 0.0f;
            const float v = live ? to_f32(in.d[i]) + bias : 0.0f;
            const float sp = p.softplus ? softplus_f32(v, nullptr) : v;
            s[i] = live ? sp : 0.0f;                            // a step of zero leaves the state as it is
            u[i] = s[i] * xf[i];
        }
        __syncthreads();      // one barrier a segment: the other buffer was last read before the barrier of the segment before
        if (t + SEG < t1) {
            in.load(p, xb, db, zb, t + SEG + j, t1, STATE_ONLY);
            bc.template load<!STATE_ONLY>(Bp, p.B.st, Cp, p.C.st, t + SEG, t1, p.N, tid);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if (!STATE_ONLY && tape && (4 * i) % TS == 0 && t + 4 * i < t1) {
                if (ch.ok) store_states<K>(tape, j, 4 * K, true, h);
                tape += (int64_t)p.D * (4 * K);
            }
            float yp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float sq = q == 0 ? quad_bcast<0>(s[i]) : q == 1 ? quad_bcast<1>(s[i]) : q == 2 ? quad_bcast<2>(s[i]) : quad_bcast<3>(s[i]);
                const float uq = q == 0 ? quad_bcast<0>(u[i]) : q == 1 ? quad_bcast<1>(u[i]) : q == 2 ? quad_bcast<2>(u[i]) : quad_bcast<3>(u[i]);
                float Bv[K], Cv[K];
                lds_states<K>(&sB[buf][(4 * i + q) * 4 * K], j, Bv);
                if (!STATE_ONLY) lds_states<K>(&sC[STATE_ONLY ? 0 : buf][(4 * i + q) * 4 * K], j, Cv);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    h[k] = fmaf(__builtin_amdgcn_exp2f(sq * A2[k]), h[k], uq * Bv[k]);
                    if (!STATE_ONLY) yp[q] = fmaf(h[k], Cv[k], yp[q]);
                }
            }
            if (STATE_ONLY) ssum += s[i];
            else {
                float y = fmaf(skip, xf[i], quad_reduce_scatter(yp, j));
                if (p.z.p) y *= zf[i] * sigmoid_f32(zf[i]);
                const int tt = t + 4 * i + j;
                if (ch.ok && tt < t1) p.y.p[yb + tt * p.y.st] = from_f32<T>(y);
            }
        }
    }
    if (STATE_ONLY) {
        ssum = quad_sum(ssum);
        if (ch.ok) {
            store_states<K>(p.carry + (((int64_t)b * p.nc + c + 1) * p.D + d) * (4 * K), j, 4 * K, true, h);
            if (j == 0) p.csum[((int64_t)b * p.nc + c) * p.D + d] = ssum;
        }
        return;
    }
    if (p.hT && ch.ok && (r.len > 0 ? t0 < r.len && r.len <= t0 + p.tc : c == 0))
        store_states<K>(p.hT + ((int64_t)b * p.D + d) * p.N, j, p.N, p.vec, h);
    const int left = p.dg - (cb - ch.g * p.cbg) * SCAN_CH;
    clear_channels(p.y, r.row0 * p.y.st + b * p.y.sb, fill_range(p.seq, r, b, t0, t0 + p.tc, last), ch.g * p.dg + p.dg - left,
                   left < SCAN_CH ? left : SCAN_CH, tid);
}

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
    const float a2 = n < N ? A[(int64_t)d * N + n] * SNN_LOG2E : 0.0f;
    float h = edge && n < N ? edge[((int64_t)b * D + d) * N + n] : 0.0f;
    float* q = carry + (int64_t)b * nc * per + e;
    const float* cs = csum + (int64_t)b * nc * D + d;
    if (!reverse) {
        for (int c = 1; c < used; ++c) {
            h = fmaf(__builtin_amdgcn_exp2f(a2 * cs[(int64_t)(c - 1) * D]), h, q[c * per]);
            q[c * per] = h;
        }
    } else {
        if (used > 0) q[(used - 1) * per] = h;
        for (int c = used - 2; c >= 0; --c) {
            h = fmaf(__builtin_amdgcn_exp2f(a2 * cs[(int64_t)(c + 1) * D]), h, q[c * per]);
            q[c * per] = h;
        }
    }
}

// One step: 8 bytes of fp32 state per (channel, state) in and out, all else is a percent of that: the memory bounds it.
// The same quads; a wave reads 16 neighbouring channels' states as one block of 16 bytes a lane.
template <typename T, int K> __global__ void __launch_bounds__(256) scan_step_kernel(const ScanP<T> p)
{
    const int64_t q = (int64_t)blockIdx.x * SCAN_CH + (threadIdx.x >> 2);
    const bool ok = q < (int64_t)p.seq.n_seq * p.D;
    const int64_t qq = ok ? q : (int64_t)p.seq.n_seq * p.D - 1;
    const int b = (int)(qq / p.D), d = (int)(qq - (int64_t)b * p.D), g = d / p.dg, j = threadIdx.x & 3;
    float h[K], A2[K], Bv[K], Cv[K];
    load_states<K>(p.h0 + qq * p.N, j, p.N, p.vec, h);
    load_states<K>(p.A + (int64_t)d * p.N, j, p.N, p.vec, A2);
    const T* Bp = p.B.p + b * p.B.sb + g * p.B_sg;
    const T* Cp = p.C.p + b * p.C.sb + g * p.C_sg;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const bool in = j * K + k < p.N;
        Bv[k] = in ? to_f32(Bp[j * K + k]) : 0.0f;
        Cv[k] = in ? to_f32(Cp[j * K + k]) : 0.0f;
    }
    const float x = to_f32(p.x.p[b * p.x.sb + d]), v = to_f32(p.delta.p[b * p.delta.sb + d]) + (p.dbias ? p.dbias[d] : 0.0f);
    const float s = p.softplus ? softplus_f32(v, nullptr) : v, u = s * x;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        h[k] = fmaf(__builtin_amdgcn_exp2f(s * (A2[k] * SNN_LOG2E)), h[k], u * Bv[k]);
        y = fmaf(h[k], Cv[k], y);
    }
    y = quad_sum(y);
    if (!ok) return;
    store_states<K>(p.hT + q * p.N, j, p.N, p.vec, h);
    if (j == 0) {
        if (p.skip) y = fmaf(p.skip[d], x, y);
        if (p.z.p) {
            const float z = to_f32(p.z.p[b * p.z.sb + d]);
            y *= z * sigmoid_f32(z);
        }
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
    if (a->seq.lengths && a->seq.offsets) { snn_set_error("%s: lengths and offsets exclude each other", fn); return SNN_ERR_ARG; }
    return SNN_OK;
}

// Chunks of the time axis.  One chunk (no arithmetic twice) once the workgroups of a single pass give every SIMD two waves
// (512 workgroups); below that, as many chunks as bring the grid to 1024 workgroups, none shorter than 64 steps.
ScanGrid snn_scan_grid(const snn_scan_args* a, bool backward)
{
    ScanGrid g;
    const int dg = a->channels / a->groups;
    g.cbg = (dg + SCAN_CH - 1) / SCAN_CH;
    g.blocks_c = g.cbg * a->groups;
    const int64_t blocks = (int64_t)g.blocks_c * a->seq.n_seq;
    int64_t nc = 1;
    if (blocks < 512) nc = std::min<int64_t>((1024 + blocks - 1) / blocks, (a->seq.max_T + 63) / 64);
    g.tc = (int)(((a->seq.max_T + nc - 1) / nc + SCAN_SEG - 1) / SCAN_SEG * SCAN_SEG);
    g.nc = (a->seq.max_T + g.tc - 1) / g.tc;
    return g;
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
    const int K = scan_k(a->states);
    p.carry = (float*)a->ws;
    p.csum = p.carry + (int64_t)a->seq.n_seq * g.nc * a->channels * 4 * K;
    const uintptr_t al = (uintptr_t)a->A | (uintptr_t)a->state_in | (uintptr_t)a->state_out | (uintptr_t)a->dstate_out | (uintptr_t)a->dstate_in;
    p.vec = a->states == 4 * K && al % 16 == 0;
    p.dy = snn_view_of<T>(a->dy);
    p.dx = snn_view_of<T>(a->dx);
    p.ddelta = snn_view_of<T>(a->ddelta);
    p.dz = snn_view_of<T>(a->dz);
    p.dB = snn_view_of<T>(a->dB);
    p.dC = snn_view_of<T>(a->dC);
    p.dhT = a->dstate_out;
    p.dh0 = a->dstate_in;
    p.part = p.bcpart = nullptr;
    p.slots = p.direct = 0;
    return p;
}
template ScanP<float> scan_params<float>(const snn_scan_args*, const ScanGrid&);
template ScanP<bf16_t> scan_params<bf16_t>(const snn_scan_args*, const ScanGrid&);
template ScanP<f16_t> scan_params<f16_t>(const snn_scan_args*, const ScanGrid&);

void snn_scan_launch_combine(const snn_scan_args* a, const ScanGrid& g, const float* edge, float* carry, const float* csum, bool reverse, hipStream_t s)
{
    const int NP = 4 * scan_k(a->states);
    const int64_t n = (int64_t)a->seq.n_seq * a->channels * NP;
    hipLaunchKernelGGL(scan_combine_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a->seq, a->channels, a->states, NP, g.tc, g.nc,
                       a->A, edge, carry, csum, (int)reverse);
}

namespace {
template <typename T, int K> int forward(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    const ScanP<T> p = scan_params<T>(a, g);
    const int64_t blocks = (int64_t)g.blocks_c * a->seq.n_seq * g.nc;
    if (blocks > 0x7fffffff) { snn_set_error("snn_scan_forward: %lld workgroups", (long long)blocks); return SNN_ERR_UNSUPPORTED; }
    if (g.nc > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<T, K, true>), dim3((unsigned)blocks), dim3(256), 0, s, p);
        snn_scan_launch_combine(a, g, a->state_in, p.carry, p.csum, false, s);
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, K, false>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T, int K> int step(const snn_scan_args* a, const ScanGrid& g, hipStream_t s)
{
    const ScanP<T> p = scan_params<T>(a, g);
    const int64_t blocks = ((int64_t)a->seq.n_seq * a->channels + SCAN_CH - 1) / SCAN_CH;
    if (blocks > 0x7fffffff) { snn_set_error("snn_scan_step: %lld workgroups", (long long)blocks); return SNN_ERR_UNSUPPORTED; }
    hipLaunchKernelGGL((scan_step_kernel<T, K>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T> int run(const snn_scan_args* a, const ScanGrid& g, bool one, hipStream_t s)
{
    switch (scan_k(a->states)) {
    case 2: return one ? step<T, 2>(a, g, s) : forward<T, 2>(a, g, s);
    case 4: return one ? step<T, 4>(a, g, s) : forward<T, 4>(a, g, s);
    case 8: return one ? step<T, 8>(a, g, s) : forward<T, 8>(a, g, s);
    default: return one ? step<T, 16>(a, g, s) : forward<T, 16>(a, g, s);
    }
}
int dispatch(const snn_scan_args* a, bool one, hipStream_t s)
{
    const ScanGrid g = snn_scan_grid(a, false);
    return a->dtype == SNN_DT_F32 ? run<float>(a, g, one, s) : a->dtype == SNN_DT_BF16 ? run<bf16_t>(a, g, one, s) : run<f16_t>(a, g, one, s);
}
}  // namespace

extern "C" int64_t snn_scan_tape_floats(const snn_scan_args* a)
{
    if (int rc = snn_scan_check(a, "snn_scan_tape_floats")) return rc;
    return scan_tape_slots(a->seq, scan_tape_steps(a->states)) * a->channels * 4 * scan_k(a->states);
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
