// snn_seq.h -- what the sequence operators outside the LSTM stack share (snn_conv.hip, snn_scan.hip, snn_scan_bwd.hip):
// element types, the addressing of a batch of sequences, and cross-lane helpers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/snn_hip.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
// results are rounded once, to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// Sizes a call may have: t + chunk and (taps + 1) * channels stay below 2^31, and no grid has 2^32 threads.
constexpr int SEQ_MAX_STEPS = 1 << 30, SEQ_MAX_COUNT = (1 << 24) - 1, SEQ_MAX_CHANNELS = 1 << 19;
constexpr int64_t SEQ_MAX_BLOCKS = (1 << 24) - 1;
static inline bool snn_sizes_fit(const snn_seq& s, int channels)
{
    return s.n_seq <= SEQ_MAX_COUNT && s.max_T <= SEQ_MAX_STEPS && channels <= SEQ_MAX_CHANNELS;
}

// One view of the batch: element (sequence b, step t, channel d) is at p[t * st + b * sb + d].
template <typename T> struct View {
    T* p;
    int64_t st, sb;
};
template <typename T> static inline View<T> snn_view_of(const snn_view& v)
{
    return View<T>{(T*)v.p, v.stride_t, v.stride_n};
}

// First row and length of sequence b.  Whatever the device arrays hold, rows stay inside the tensors: a length is cut to
// [0, max_T], an offset to [0, n_rows], and a sequence whose end lies before its start is empty.
struct SeqRange { int64_t row0, end; int len; };
__device__ __forceinline__ SeqRange seq_range(const snn_seq& s, int b)
{
    SeqRange r;
    if (s.offsets) {
        int64_t o = s.offsets[b], e = s.offsets[b + 1];
        o = o < 0 ? 0 : (o > s.n_rows ? s.n_rows : o);
        e = e < o ? o : (e > s.n_rows ? s.n_rows : e);
        r.row0 = o;
        r.end = e;
        r.len = (int)(e - o < s.max_T ? e - o : s.max_T);
    } else {
        int l = s.lengths ? s.lengths[b] : s.max_T;
        r.row0 = 0;
        r.len = l < 0 ? 0 : (l > s.max_T ? s.max_T : l);
        r.end = s.max_T;
    }
    return r;
}
// Chunks of 2^sh steps as work items of a ragged batch: sequence b has the items from (offsets[b] >> sh) + b on, room for its every
// step, so that (n_rows >> sh) + n_seq hold all of them whatever bound on the lengths the caller knows; the last sequence has the
// rest, enough for the rows behind it.
struct SeqItem { int b; int64_t c; };                  // sequence, chunk
__device__ __forceinline__ int64_t seq_first_item(const snn_seq& s, int b, int sh)
{
    const int64_t o = s.offsets[b];
    return ((o < 0 ? 0 : (o > s.n_rows ? s.n_rows : o)) >> sh) + b;
}
// Which sequence an item of ragged rows belongs to: the last one whose first item is not behind it, by a search that asks seven
// places at once (a search by halves waits for log2 n_seq loads one after the other).  Offsets that decrease find some sequence, and
// maybe a chunk below 0, which the caller leaves out.
__device__ __forceinline__ SeqItem seq_find_item(const snn_seq& s, int64_t item, int sh)
{
    int lo = 0, hi = s.n_seq;                          // in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 7) >> 3;
        int n = 0;
#pragma unroll
        for (int k = 1; k < 8; ++k) {
            const int b = lo + k * step;
            n += b < hi && seq_first_item(s, b < hi ? b : lo, sh) <= item;
        }
        hi = lo + (n + 1) * step < hi ? lo + (n + 1) * step : hi;
        lo += n * step;
    }
    SeqItem r;
    r.b = lo;
    r.c = item - seq_first_item(s, lo, sh);
    return r;
}
// Rows (relative to row0) that belong to no step and that chunk [t0, t1) of sequence b has to clear, as two ranges:
// behind the sequence's end inside the padded batch, and -- ragged rows -- before the first and behind the last sequence.
struct FillRange { int64_t a0, a1, b0, b1; };
__device__ __forceinline__ FillRange fill_range(const snn_seq& s, const SeqRange& r, int b, int t0, int t1, bool last_chunk)
{
    FillRange f = {0, 0, 0, 0};
    if (s.offsets) {
        if (last_chunk) {                       // rows of the sequence past max_T, and behind the last sequence
            f.a0 = r.len;
            f.a1 = (b == s.n_seq - 1 ? s.n_rows : r.end) - r.row0;
        }
        if (b == 0 && t0 == 0) { f.b0 = -r.row0; f.b1 = 0; }
    } else {
        f.a0 = r.len > t0 ? r.len : t0;
        f.a1 = last_chunk ? s.max_T : t1;
    }
    return f;
}

// The same where every chunk c of tc steps clears its own steps' worth, and the sequence's last one (`last`, if any is) all behind.
__device__ __forceinline__ FillRange fill_of_chunk(const snn_seq& s, const SeqRange& r, int b, int64_t c, int tc, bool last)
{
    const int64_t t0 = c * tc, end = s.offsets ? (b == s.n_seq - 1 ? s.n_rows : r.end) - r.row0 : s.max_T;
    FillRange f = {r.len > t0 ? r.len : t0, last || end < t0 + tc ? end : t0 + tc, 0, 0};
    if (s.offsets && b == 0 && c == 0) f.b0 = -r.row0;
    return f;
}

// ---- cross-lane ---------------------------------------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ float dpp(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int S> __device__ __forceinline__ float quad_bcast(float v) { return dpp<S * 0x55>(v); }      // lane S of every quad
__device__ __forceinline__ float quad_xor1(float v) { return dpp<0xB1>(v); }
__device__ __forceinline__ float quad_xor2(float v) { return dpp<0x4E>(v); }
__device__ __forceinline__ float quad_sum(float v) { v += quad_xor1(v); return v + quad_xor2(v); }
// lane j of a quad receives the quad's sum of v[j]: 9 instructions for four sums
__device__ __forceinline__ float quad_reduce_scatter(const float v[4], int j)
{
    const bool o1 = j & 1, o2 = j & 2;
    const float r0 = (o1 ? v[1] : v[0]) + quad_xor1(o1 ? v[0] : v[1]);
    const float r1 = (o1 ? v[3] : v[2]) + quad_xor1(o1 ? v[2] : v[3]);
    return (o2 ? r1 : r0) + quad_xor2(o2 ? r0 : r1);
}

// ---- activations --------------------------------------------------------------------------------------------------
#define SNN_LOG2E 1.44269504088896341f
#define SNN_LN2 0.693147180559945309f
// silu and its slope take 2^(-v log2 e) as it comes: an error of |v| 6e-8 in the exponential, at most 2e-8 |v| in the sigmoid
__device__ __forceinline__ float sigmoid_f32(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -SNN_LOG2E)); }
// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) <= 1, and its derivative sigmoid(v).  Steps are small (v about -5), where
// log1p(e) ~ e, so e has to be relatively exact: the rounding error of |v| log2(e) is put back, and log1p(e) is
// log(u) + (e - (u - 1)), u = fl(1 + e): the second term is what the sum 1 + e dropped.
__device__ __forceinline__ float softplus_f32(float v, float* sigma)
{
    const float w = fminf(fabsf(v), 104.0f);                       // exp(-104) = 0
    const float hi = w * -SNN_LOG2E, lo = fmaf(w, -SNN_LOG2E, -hi);
    const float e0 = __builtin_amdgcn_exp2f(hi), e = fmaf(e0, lo * SNN_LN2, e0);
    const float u = 1.0f + e;
    const float l = fmaf(__builtin_amdgcn_logf(u), SNN_LN2, e - (u - 1.0f));     // v_log_f32: base 2
    if (sigma) *sigma = (v >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(u);
    return (v <= 0.0f ? 0.0f : v) + l;                             // not v > 0: a NaN stays
}

// ---- sums over workgroups -----------------------------------------------------------------------------------------
// Column `col` of part[slots][stride] in fp64 and in an order that depends on `slots` alone: a workgroup of 1024 threads sums 16
// columns, 64 rows at a time.  True for the 16 threads that receive a sum.
__device__ __forceinline__ bool column_sum(const float* __restrict__ part, int slots, int64_t stride, int64_t n, int64_t* col, double* sum)
{
    __shared__ double s[64][17];
    const int c = threadIdx.x & 15, row = threadIdx.x >> 4;
    *col = (int64_t)blockIdx.x * 16 + c;
    double a = 0.0;
    if (*col < n) {
        const float* q = part + (int64_t)row * stride + *col;
        int i = row;
        for (; i + 192 < slots; i += 256, q += 256 * stride) {          // four loads in flight
            const float v0 = q[0], v1 = q[64 * stride], v2 = q[128 * stride], v3 = q[192 * stride];
            a += ((double)v0 + v1) + ((double)v2 + v3);
        }
        for (; i < slots; i += 64, q += 64 * stride) a += *q;
    }
    s[row][c] = a;
    __syncthreads();
    if (row < 8) {
#pragma unroll
        for (int i = 1; i < 8; ++i) a += s[row + 8 * i][c];
        s[row][c] = a;
    }
    __syncthreads();
    if (row) return false;
#pragma unroll
    for (int i = 1; i < 8; ++i) a += s[i][c];
    *sum = a;
    return *col < n;
}
