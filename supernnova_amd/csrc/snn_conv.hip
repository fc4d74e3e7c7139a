// snn_conv.hip -- depthwise causal convolution over the last 2..4 steps with silu: forward, backward, one step
// (include/snn_hip.h: snn_conv_*).
//
//   p_t = bias + sum_w weight[w] x_{t-W+1+w},   y_t = silu(p_t) = p_t s_t,  s_t = 1 / (1 + exp(-p_t))
//   dp_t = dy_t s_t (1 + p_t (1 - s_t));   dx_t = sum_w weight[w] dp_{t+W-1-w};   dweight[w] = sum dp_t x_{t-W+1+w}
//
// ~2W + 10 operations for two (backward: three) elements moved: the memory bounds it.  A thread owns V neighbouring channels
// (16 bytes of a row, 8 .. 16 in the backward) and walks a chunk of the time axis with the window in registers, so a row is
// read once but for the W - 1 rows in front of a chunk.  Threads are numbered (chunk of a sequence, channel vector), so
// narrow layers fill their waves too.  Measured: forward of 8192 x 4096 bf16 27.5 us = 4.9 TB/s (a large copy: 4.7); training of
// 2048 x 300 x 256 fp32, half of whose rows are padding, forward 197, backward 307, sums 10 us for 2.2 GB.
#include "snn_seq.h"
#include "snn_host.h"
#include <algorithm>
#include <type_traits>

#define HIP_CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { \
    snn_set_error("%s: %s", #x, hipGetErrorString(e_)); return SNN_ERR_HIP; } } while (0)

namespace {

template <typename T> struct ConvP {
    snn_seq seq;
    View<T> x, y, dy, dx;
    const float *weight, *bias;
    const T *s_in, *ds_out;
    T *s_out, *ds_in;
    float* part;
    int D, cv, tc, nc, slots, silu;     // channels, vectors per row, steps per chunk, chunks per sequence, backward: item slots
    int sh;                             // < 0: items are (sequence, chunk) of a grid of nc a sequence; else of seq_find_item, tc = 2^sh
    int64_t items;
};
template <typename T> __device__ __forceinline__ SeqItem chunk_of(const ConvP<T>& p, int64_t item)
{
    if (p.sh >= 0) return seq_find_item(p.seq, item, p.sh);
    const int b = (int)(item / p.nc);
    return SeqItem{b, item - (int64_t)b * p.nc};
}

template <typename T, int V> __device__ __forceinline__ void load_v(const T* p, float (&v)[V])
{
    const Pack<T, V> q = *(const Pack<T, V>*)p;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(q.v[i]);
}
template <typename T, int V> __device__ __forceinline__ void store_v(T* p, const float (&v)[V])
{
    Pack<T, V> q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = from_f32<T>(v[i]);
    *(Pack<T, V>*)p = q;
}
template <int V> __device__ __forceinline__ void zero_v(float (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
}
template <typename T, int V>
__device__ __forceinline__ void clear_rows(const View<T>& y, const FillRange& f, int64_t base)
{
    Pack<T, V> z;
#pragma unroll
    for (int i = 0; i < V; ++i) z.v[i] = (T)0.0f;
    for (int64_t t = f.a0; t < f.a1; ++t) *(Pack<T, V>*)(y.p + base + t * y.st) = z;
    for (int64_t t = f.b0; t < f.b1; ++t) *(Pack<T, V>*)(y.p + base + t * y.st) = z;
}
// step t (may lie before the first) of sequence b, channels d ..
template <typename T, int V, int W>
__device__ __forceinline__ void load_before(const ConvP<T>& p, int64_t xb, int b, int t, int d, float (&v)[V])
{
    if (t >= 0) load_v<T, V>(p.x.p + xb + t * p.x.st, v);
    else if (p.s_in) load_v<T, V>(p.s_in + ((int64_t)b * (W - 1) + (t + W - 1)) * p.D + d, v);
    else zero_v(v);
}
template <int V, int W> __device__ __forceinline__ void load_taps(const float* w, const float* bias, int d, float (&wt)[W][V], float (&bs)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) wt[k][i] = w[(int64_t)(d + i) * W + k];
        bs[i] = bias ? bias[d + i] : 0.0f;
    }
}

template <typename T, int V, int W> __global__ void __launch_bounds__(256) conv_fwd_kernel(const ConvP<T> p)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.items * p.cv) return;
    const int64_t item = id / p.cv;
    const SeqItem it = chunk_of(p, item);
    const int64_t c = it.c;
    if (c < 0) return;
    const int d = (int)(id - item * p.cv) * V, b = it.b;
    const SeqRange r = seq_range(p.seq, b);
    const int t0 = c * p.tc < r.len ? (int)(c * p.tc) : r.len, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
    const int64_t xb = r.row0 * p.x.st + b * p.x.sb + d, yb = r.row0 * p.y.st + b * p.y.sb + d;
    if (t0 < t1) {
        float wt[W][V], bs[V], win[W][V];
        load_taps<V, W>(p.weight, p.bias, d, wt, bs);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) load_before<T, V, W>(p, xb, b, t0 - (W - 1) + k, d, win[k]);
        constexpr int U = 4;                                   // rows in flight per thread
        Pack<T, V> raw[U];
        const T* xp = p.x.p + xb + t0 * p.x.st;
        T* yp = p.y.p + yb + t0 * p.y.st;
        for (int t = t0; t < t1; t += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = *(const Pack<T, V>*)(xp + (t + u < t1 ? u : 0) * p.x.st);
            xp += U * p.x.st;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u < t1) {
                    float out[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        win[W - 1][i] = to_f32(raw[u].v[i]);
                        float a = bs[i];
#pragma unroll
                        for (int k = 0; k < W; ++k) a = fmaf(wt[k][i], win[k][i], a);
                        out[i] = p.silu ? a * sigmoid_f32(a) : a;
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) win[k][i] = win[k + 1][i];
                    }
                    store_v<T, V>(yp + u * p.y.st, out);
                }
            }
            yp += U * p.y.st;
        }
    }
    if (p.s_out && (r.len > 0 ? t0 < r.len && r.len <= t0 + p.tc : c == 0)) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            float v[V];
            load_before<T, V, W>(p, xb, b, r.len - (W - 1) + k, d, v);
            store_v<T, V>(p.s_out + ((int64_t)b * (W - 1) + k) * p.D + d, v);
        }
    }
    clear_rows<T, V>(p.y, fill_of_chunk(p.seq, r, b, c, p.tc, p.sh < 0 && c == p.nc - 1), yb);
}

// A thread takes the chunks slot, slot + slots, .. so that the parameter gradients of many sequences add up in registers (fp32: their
// rounding grows with the chunks of a slot); part[slot][W + 1][D] is summed by conv_bwd_sum_kernel in fp64.
template <typename T, int V, int W> __global__ void __launch_bounds__(256) conv_bwd_kernel(const ConvP<T> p)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)p.slots * p.cv) return;
    const int slot = (int)(id / p.cv), d = (int)(id - (int64_t)slot * p.cv) * V;
    float wt[W][V], bs[V], dws[W][V], dbs[V];     // fp32 sums over a slot's chunks; a chunk's own come first: two short chains
    load_taps<V, W>(p.weight, p.bias, d, wt, bs);
    zero_v(dbs);
#pragma unroll
    for (int k = 0; k < W; ++k) zero_v(dws[k]);
    for (int64_t item = slot; item < p.items; item += p.slots) {
        const SeqItem it = chunk_of(p, item);
        const int b = it.b;
        const int64_t c = it.c;
        if (c < 0) continue;
        const SeqRange r = seq_range(p.seq, b);
        const int t0 = c * p.tc < r.len ? (int)(c * p.tc) : r.len, t1 = t0 + p.tc < r.len ? t0 + p.tc : r.len;
        const int64_t xb = r.row0 * p.x.st + b * p.x.sb + d, gb = r.row0 * p.dy.st + b * p.dy.sb + d;
        const int64_t ob = r.row0 * p.dx.st + b * p.dx.sb + d;
        if (t0 < t1 || c == 0) {                    // c == 0: the gradient of the initial state, also of an empty sequence
            float win[W][V], dpw[W][V], dw[W][V], db[V];             // dpw[k] = dp of k steps ago
            zero_v(db);
#pragma unroll
            for (int k = 0; k < W; ++k) zero_v(dw[k]);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) load_before<T, V, W>(p, xb, b, t0 - (W - 1) + k, d, win[k]);
#pragma unroll
            for (int k = 0; k < W; ++k) zero_v(dpw[k]);
            constexpr int U = 4;
            const int te = t1 + W - 1;              // dx of the chunk's last step needs the W - 1 steps behind it
            const T *xp = p.x.p + xb + t0 * p.x.st, *gp = p.dy.p + gb + t0 * p.dy.st;
            T* op = p.dx.p + ob + (t0 - (W - 1)) * p.dx.st;
            // steps tb .. tb + 3.  INNER: all of them are the chunk's, and so are the steps W - 1 before them, whose gradients
            // they complete: nothing to ask.
            auto group = [&](auto inner, int tb) {
                constexpr bool INNER = decltype(inner)::value;
                Pack<T, V> rx[U], rg[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (INNER || (tb + u < r.len && tb + u < te)) {
                        rx[u] = *(const Pack<T, V>*)(xp + u * p.x.st);
                        rg[u] = *(const Pack<T, V>*)(gp + u * p.dy.st);
                    }
                }
                xp += U * p.x.st;
                gp += U * p.dy.st;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int t = tb + u;
                    if (!INNER && t >= te) break;
                    const bool live = INNER || t < r.len, ours = INNER || t < t1;
                    float out[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float dp = 0.0f;
                        win[W - 1][i] = 0.0f;
                        if (live) {
                            win[W - 1][i] = to_f32(rx[u].v[i]);
                            float a = bs[i];
#pragma unroll
                            for (int k = 0; k < W; ++k) a = fmaf(wt[k][i], win[k][i], a);
                            dp = to_f32(rg[u].v[i]);
                            if (p.silu) {
                                const float s = sigmoid_f32(a);
                                dp *= s * fmaf(a, 1.0f - s, 1.0f);
                            }
                            if (ours) {
#pragma unroll
                                for (int k = 0; k < W; ++k) dw[k][i] = fmaf(dp, win[k][i], dw[k][i]);
                                db[i] += dp;
                            }
                        }
#pragma unroll
                        for (int k = W - 1; k > 0; --k) dpw[k][i] = dpw[k - 1][i];
                        dpw[0][i] = dp;
                        out[i] = wt[0][i] * dp;
#pragma unroll
                        for (int k = 1; k < W; ++k) out[i] = fmaf(wt[k][i], dpw[k][i], out[i]);
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) win[k][i] = win[k + 1][i];
                    }
                    const int tau = t - (W - 1);            // the step whose gradient is complete now
                    if (INNER) store_v<T, V>(op + u * p.dx.st, out);
                    else {
                        const int k = tau - r.len + W - 1;  // its place among the last W - 1 inputs
                        const bool mine = tau >= t0 || (c == 0 && tau < 0);
                        if (mine && p.ds_out && k >= 0 && k < W - 1) {
                            float e[V];
                            load_v<T, V>(p.ds_out + ((int64_t)b * (W - 1) + k) * p.D + d, e);
#pragma unroll
                            for (int i = 0; i < V; ++i) out[i] += e[i];
                        }
                        if (tau >= t0) store_v<T, V>(op + u * p.dx.st, out);
                        else if (mine && p.ds_in) store_v<T, V>(p.ds_in + ((int64_t)b * (W - 1) + (tau + W - 1)) * p.D + d, out);
                    }
                }
                op += U * p.dx.st;
            };
            int tb = t0;
            group(std::false_type{}, tb);           // the first W - 1 <= U steps complete the chunk's (or the state's) before
            for (tb += U; tb + U <= t1; tb += U) group(std::true_type{}, tb);
            for (; tb < te; tb += U) group(std::false_type{}, tb);
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int k = 0; k < W; ++k) dws[k][i] += dw[k][i];
                dbs[i] += db[i];
            }
        }
        clear_rows<T, V>(p.dx, fill_of_chunk(p.seq, r, b, c, p.tc, p.sh < 0 && c == p.nc - 1), ob);
    }
    float* q = p.part + (int64_t)slot * (W + 1) * p.D + d;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) q[k * p.D + i] = dws[k][i];
        q[W * p.D + i] = dbs[i];
    }
}

// dweight (D, W) and dbias (D) from the slots' partial sums
__global__ void __launch_bounds__(1024) conv_bwd_sum_kernel(const float* __restrict__ part, int slots, int W, int D, float* dweight, float* dbias)
{
    const int64_t n = (int64_t)(W + 1) * D;
    int64_t col;
    double a;
    if (!column_sum(part, slots, n, n, &col, &a)) return;
    const int k = (int)(col / D), d = (int)(col - (int64_t)k * D);
    if (k < W) dweight[(int64_t)d * W + k] = (float)a;
    else if (dbias) dbias[d] = (float)a;
}

template <typename T, int V, int W> __global__ void __launch_bounds__(256) conv_step_kernel(const ConvP<T> p)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.items * p.cv) return;
    const int b = (int)(id / p.cv), d = (int)(id - (int64_t)b * p.cv) * V;
    float wt[W][V], bs[V], win[W][V], out[V];
    const int64_t sb = (int64_t)b * (W - 1) * p.D + d;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load_v<T, V>(p.s_in + sb + (int64_t)k * p.D, win[k]);
    load_v<T, V>(p.x.p + b * p.x.sb + d, win[W - 1]);
    load_taps<V, W>(p.weight, p.bias, d, wt, bs);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float a = bs[i];
#pragma unroll
        for (int k = 0; k < W; ++k) a = fmaf(wt[k][i], win[k][i], a);
        out[i] = p.silu ? a * sigmoid_f32(a) : a;
    }
    store_v<T, V>(p.y.p + b * p.y.sb + d, out);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) store_v<T, V>(p.s_out + sb + (int64_t)k * p.D, win[k + 1]);
}

// ---- host ---------------------------------------------------------------------------------------------------------
enum { FWD = 0, BWD = 1, STEP = 2 };
const int ELEM[3] = {4, 2, 2};

int check_args(const snn_conv_args* a, int what, const char* fn)
{
    if (!a) { snn_set_error("%s: args is NULL", fn); return SNN_ERR_ARG; }
    if (a->seq.n_seq < 1 || a->seq.max_T < 1 || a->channels < 1 || a->seq.n_rows < 0) {
        snn_set_error("%s: n_seq, max_T and channels must be positive", fn);
        return SNN_ERR_ARG;
    }
    if (a->dtype < 0 || a->dtype > 2 || a->width < 2 || a->width > 4) {
        snn_set_error("%s: dtype %d / width %d: supported are dtypes 0..2 (SNN_DT_*) and 2..4 taps", fn, a->dtype, a->width);
        return SNN_ERR_UNSUPPORTED;
    }
    if (!snn_sizes_fit(a->seq, a->channels)) {
        snn_set_error("%s: at most 2^24 - 1 sequences, 2^30 steps and 2^19 channels", fn);
        return SNN_ERR_UNSUPPORTED;
    }
    if (a->seq.lengths && a->seq.offsets) { snn_set_error("%s: lengths and offsets exclude each other", fn); return SNN_ERR_ARG; }
    return SNN_OK;
}
// 16 bytes of a row per thread (backward: 4 channels) where every row starts at a multiple of that, one channel otherwise.
// 8192 x 4096 bf16: forward 27.5 us against 31.5 with one channel a thread, backward 48.5 against 59.
int vector_width(const snn_conv_args* a, int what)
{
    const int e = ELEM[a->dtype], v = what == BWD ? 4 : 16 / e;
    bool ok = a->channels % v == 0;
    auto view = [&](const snn_view& w) {
        ok = ok && ((uintptr_t)w.p % (v * e)) == 0 && w.stride_t % v == 0 && w.stride_n % v == 0;
    };
    auto ptr = [&](const void* q) { ok = ok && ((uintptr_t)q % (v * e)) == 0; };
    view(a->x);
    if (what != BWD) view(a->y);
    else { view(a->dy); view(a->dx); ptr(a->dstate_out); ptr(a->dstate_in); }
    ptr(a->state_in);
    if (what != BWD) ptr(a->state_out);
    return ok ? v : 1;
}
// Items of chunks of t steps.  A grid of max_T's chunks for every sequence, or, where more than half of that of ragged rows would be
// empty (one long sequence among short ones, or no bound known but the number of rows), the chunks that the rows can have, each of
// which then searches its sequence.  Grid / search, forward and backward: 4000 x up to 40 x 64 fp32 (grid 1.3 times the search's items)
// 11 / 18 and 39 / 50 us, 256 x up to 300 x 256 fp32 (1.8) 17.7 / 18.7 and 43 / 41, 7 x up to 1501 x 1536 fp16 (1.9) 15.8 / 12.2 and
// 36 / 27, 8192 + 7 x 64 x 4096 bf16 (7) 42 / 38 and 133 / 71.
int64_t grid_items(const snn_seq& s, int t) { return (int64_t)s.n_seq * ((s.max_T + t - 1) / t); }
int64_t row_items(const snn_seq& s, int t) { return s.n_rows / t + s.n_seq; }
bool by_rows(const snn_seq& s, int t) { return s.offsets && grid_items(s, t) > 2 * row_items(s, t); }
int64_t item_count(const snn_seq& s, int t) { return by_rows(s, t) ? row_items(s, t) : grid_items(s, t); }

// Steps per chunk: the longest of 64 (backward: 128) .. 16 that leaves 2^17 threads (two waves on every SIMD), so that long
// chunks (few repeated rows) go to large batches and short ones to single sequences.  Forward of 2048 x 300 x 256 fp32 with up
// to 64 / 128 / 512 steps: 193 / 208 / 206 us.
int chunk_steps(const snn_conv_args* a, int v, int what)
{
    const int64_t cv = (a->channels + v - 1) / v;
    int t = what == BWD ? 128 : 64;
    while (t > 16 && item_count(a->seq, t) * cv < (1 << 17)) t >>= 1;
    return t;
}
// Backward slots: about 2^17 threads (what its registers let the chip hold), never more than there are chunks.  2^18 take the
// same time and leave twice the partial sums: 18 instead of 10 us of adding up.
int bwd_slots(const snn_conv_args* a, int v)
{
    const int64_t cv = (a->channels + v - 1) / v, items = item_count(a->seq, chunk_steps(a, v, BWD));
    return (int)std::max<int64_t>(1, std::min<int64_t>(items, ((1 << 17) + cv - 1) / cv));
}

template <typename T, int V, int W> int launch(const snn_conv_args* a, int what, hipStream_t s)
{
    ConvP<T> p;
    p.seq = a->seq;
    p.x = snn_view_of<T>(a->x);
    p.y = snn_view_of<T>(a->y);
    p.dy = snn_view_of<T>(a->dy);
    p.dx = snn_view_of<T>(a->dx);
    p.weight = a->weight;
    p.bias = a->bias;
    p.s_in = (const T*)a->state_in;
    p.s_out = (T*)a->state_out;
    p.ds_out = (const T*)a->dstate_out;
    p.ds_in = (T*)a->dstate_in;
    p.part = (float*)a->ws;
    p.D = a->channels;
    p.cv = (a->channels + V - 1) / V;
    p.silu = a->silu;
    p.slots = 0;
    p.tc = what == STEP ? 1 : chunk_steps(a, V, what);
    p.sh = by_rows(a->seq, p.tc) ? __builtin_ctz(p.tc) : -1;
    p.nc = (a->seq.max_T + p.tc - 1) / p.tc;
    p.items = item_count(a->seq, p.tc);
    if (what == BWD) p.slots = bwd_slots(a, V);
    const int64_t blocks = ((what == BWD ? (int64_t)p.slots : p.items) * p.cv + 255) / 256;
    if (blocks > SEQ_MAX_BLOCKS) { snn_set_error("convolution: %lld workgroups", (long long)blocks); return SNN_ERR_UNSUPPORTED; }
    const dim3 g((unsigned)blocks), t(256);
    if constexpr (V != 4 || sizeof(T) == 4) {
        if (what == FWD) hipLaunchKernelGGL((conv_fwd_kernel<T, V, W>), g, t, 0, s, p);
        else if (what == STEP) hipLaunchKernelGGL((conv_step_kernel<T, V, W>), g, t, 0, s, p);
    }
    if constexpr (V <= 4) if (what == BWD) {
        hipLaunchKernelGGL((conv_bwd_kernel<T, V, W>), g, t, 0, s, p);
        hipLaunchKernelGGL(conv_bwd_sum_kernel, dim3((unsigned)(((int64_t)(W + 1) * p.D + 15) / 16)), dim3(1024), 0, s, (const float*)p.part, p.slots, W, p.D,
                           a->dweight, a->dbias);
    }
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
template <typename T, int V> int by_width(const snn_conv_args* a, int what, hipStream_t s)
{
    return a->width == 2 ? launch<T, V, 2>(a, what, s) : a->width == 3 ? launch<T, V, 3>(a, what, s) : launch<T, V, 4>(a, what, s);
}
int dispatch(const snn_conv_args* a, int what, hipStream_t s)
{
    const int v = vector_width(a, what);
    if (a->dtype == SNN_DT_F32) return v == 4 ? by_width<float, 4>(a, what, s) : by_width<float, 1>(a, what, s);
    if (a->dtype == SNN_DT_BF16)
        return v == 8 ? by_width<bf16_t, 8>(a, what, s) : v == 4 ? by_width<bf16_t, 4>(a, what, s) : by_width<bf16_t, 1>(a, what, s);
    return v == 8 ? by_width<f16_t, 8>(a, what, s) : v == 4 ? by_width<f16_t, 4>(a, what, s) : by_width<f16_t, 1>(a, what, s);
}

}  // namespace

extern "C" int snn_conv_forward(const snn_conv_args* a, void* stream)
{
    if (int rc = check_args(a, FWD, "snn_conv_forward")) return rc;
    if (!a->x.p || !a->y.p || !a->weight || (a->state_out && a->state_out == a->state_in)) {
        snn_set_error("snn_conv_forward: null pointer, or state_out is state_in");
        return SNN_ERR_ARG;
    }
    return dispatch(a, FWD, (hipStream_t)stream);
}

extern "C" int64_t snn_conv_workspace_bytes(const snn_conv_args* a)
{
    if (int rc = check_args(a, BWD, "snn_conv_workspace_bytes")) return rc;
    return (int64_t)bwd_slots(a, vector_width(a, BWD)) * (a->width + 1) * a->channels * 4;
}

extern "C" int snn_conv_backward(const snn_conv_args* a, void* stream)
{
    if (int rc = check_args(a, BWD, "snn_conv_backward")) return rc;
    if (!a->x.p || !a->dy.p || !a->dx.p || !a->weight || !a->dweight || !a->ws) {
        snn_set_error("snn_conv_backward: null pointer");
        return SNN_ERR_ARG;
    }
    if (a->ws_bytes < snn_conv_workspace_bytes(a)) {
        snn_set_error("snn_conv_backward: workspace of %lld bytes, %lld needed", (long long)a->ws_bytes, (long long)snn_conv_workspace_bytes(a));
        return SNN_ERR_WORKSPACE;
    }
    return dispatch(a, BWD, (hipStream_t)stream);
}

extern "C" int snn_conv_step(const snn_conv_args* a, void* stream)
{
    if (int rc = check_args(a, STEP, "snn_conv_step")) return rc;
    if (!a->x.p || !a->y.p || !a->weight || !a->state_in || !a->state_out || a->seq.max_T != 1 || a->seq.lengths || a->seq.offsets) {
        snn_set_error("snn_conv_step: null pointer, or max_T, lengths or offsets of more than one step");
        return SNN_ERR_ARG;
    }
    return dispatch(a, STEP, (hipStream_t)stream);
}
