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
// exp(v) to about an ulp: the product v * log2(e) is carried with its rounding error (|v| * 6e-8 of the result otherwise)
__device__ __forceinline__ float exp_f32(float v)
{
    const float hi = v * SNN_LOG2E;
    const float lo = fmaf(v, SNN_LOG2E, -hi) + v * 1.925963033500011e-08f;
    const float e = __builtin_amdgcn_exp2f(hi);
    return fabsf(hi) < 150.0f ? fmaf(e, lo * SNN_LN2, e) : e;          // infinite products have no rounding error to add
}
__device__ __forceinline__ float sigmoid_f32(float v) { return __builtin_amdgcn_rcpf(1.0f + exp_f32(-v)); }
// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) <= 1, and its derivative sigmoid(v).  log1p(e) = 2 atanh(s) with
// s = e / (2 + e) <= 1/3: seven terms of the odd series leave 1.4e-8 of the first, below fp32 rounding for every v.
__device__ __forceinline__ float softplus_f32(float v, float* sigma)
{
    const float e = exp_f32(-fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float p = fmaf(q, 1.0f / 13, 1.0f / 11);
    p = fmaf(q, p, 1.0f / 9);
    p = fmaf(q, p, 1.0f / 7);
    p = fmaf(q, p, 1.0f / 5);
    p = fmaf(q, p, 1.0f / 3);
    p = fmaf(q, p, 1.0f);
    if (sigma) *sigma = (v >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e);
    return (v > 0.0f ? v : (v == v ? 0.0f : v)) + 2.0f * s * p;
}
