// snn_clip.hip -- global gradient norm over many tensors, and clipping (include/snn_hip.h: snn_clip_grads).
//
//   norm = grad_scale (sum_i sum |g|^p)^(1/p),  coef = min(1, max_norm / (norm + 1e-6)),  g' = g coef
//
// Two passes over the gradients (every element's product needs the whole sum), 2-3 operations an element: the memory bounds
// both.  The tensors travel as kernel arguments, CLIP_TENSORS to a launch, so that nothing is copied to the device before a call
// and a captured call keeps its own table.  Work is cut into pieces of CLIP_PIECE elements; a workgroup finds its tensor in the
// table and leaves one fp64 partial sum per piece (squares of fp32 gradients overflow fp32 from 2e19 on).  Up to
// CLIP_DIRECT pieces -- this framework's own models -- every workgroup of the second pass adds the partial sums itself; above, a
// single workgroup does it in between: a call with limits of 0 / 1024 / 8192 at 30 pieces 27.6 / 24.4 / 25.0, at 250 27.5 / 24.3 /
// 24.6, at 1000 35.6 / 34.6 / 34.6, at 4000 143.5 / 143.5 / 146.3 us.
// 405 M bf16 elements in 168 tensors: first pass 104 + 57, sum 6, second pass 145 + 132 us: 2.4 GB at 5.5 TB/s (a large copy: 4.7;
// the end of the first pass is still in the last-level cache when the second begins there).
#include <hip/hip_runtime.h>
#include <math.h>
#include <algorithm>
#include <memory>
#include <new>
#include "snn_host.h"
#include "snn_seq.h"
#include "snn_update.h"

#define HIP_CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { \
    snn_set_error("%s: %s", #x, hipGetErrorString(e_)); return SNN_ERR_HIP; } } while (0)

namespace {

constexpr int CLIP_TENSORS = 96, CLIP_PIECE = 1 << 14, CLIP_DIRECT = 1024;

struct Table {                                  // 2.7 KB of the 4 KB of kernel arguments
    const void* src[CLIP_TENSORS];
    void* dst[CLIP_TENSORS];
    int64_t n[CLIP_TENSORS];
    int first[CLIP_TENSORS + 1];                // first piece of each tensor
    unsigned char dtype[CLIP_TENSORS];
    int count;
};
// 16 bytes at an address of any element alignment
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Loose { T v[16 / sizeof(T)]; };

__device__ __forceinline__ int find_tensor(const Table& t, int piece)
{
    int lo = 0, hi = t.count;                   // first[lo] <= piece < first[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (t.first[m] <= piece) lo = m;
        else hi = m;
    }
    return lo;
}
template <int P> __device__ __forceinline__ double join(double a, double v)
{
    if (P == 0) return v > a || v != v ? v : a;               // a NaN stays
    return a + v;
}
template <int P> __device__ __forceinline__ double magnitude(float v, double a)
{
    if (P == 2) return fma((double)v, (double)v, a);
    return join<P>(a, (double)fabsf(v));
}
template <int P, int THREADS = 256> __device__ __forceinline__ double block_join(double a)
{
    constexpr int WAVES = THREADS / 64;
    __shared__ double s[WAVES];
#pragma unroll
    for (int m = 32; m; m >>= 1) a = join<P>(a, __shfl_xor(a, m));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    a = s[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) a = join<P>(a, s[w]);
    return a;
}
template <typename T, int P> __device__ __forceinline__ double piece_sum(const T* g, int64_t n)
{
    constexpr int V = 16 / sizeof(T);
    double a[4] = {0.0, 0.0, 0.0, 0.0};
    const int64_t nv = n / V;
    int64_t i = threadIdx.x;
    for (; i + 3 * 256 < nv; i += 4 * 256) {                  // four loads in flight, four sums
        Loose<T> q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = *(const Loose<T>*)(g + (i + u * 256) * V);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < V; ++k) a[u] = magnitude<P>(to_f32(q[u].v[k]), a[u]);
    }
    for (; i < nv; i += 256) {
        const Loose<T> q = *(const Loose<T>*)(g + i * V);
#pragma unroll
        for (int k = 0; k < V; ++k) a[0] = magnitude<P>(to_f32(q.v[k]), a[0]);
    }
    for (int64_t e = nv * V + threadIdx.x; e < n; e += 256) a[0] = magnitude<P>(to_f32(g[e]), a[0]);
    return join<P>(join<P>(a[0], a[1]), join<P>(a[2], a[3]));
}
template <int P> __global__ void __launch_bounds__(256) clip_norm_kernel(const Table t, double* part)
{
    const int ti = find_tensor(t, blockIdx.x);
    const int64_t at = (int64_t)(blockIdx.x - t.first[ti]) * CLIP_PIECE, left = t.n[ti] - at, n = left < CLIP_PIECE ? left : CLIP_PIECE;
    const int dt = t.dtype[ti];
    double a;
    if (dt == SNN_DT_F32) a = piece_sum<float, P>((const float*)t.src[ti] + at, n);
    else if (dt == SNN_DT_BF16) a = piece_sum<bf16_t, P>((const bf16_t*)t.src[ti] + at, n);
    else a = piece_sum<f16_t, P>((const f16_t*)t.src[ti] + at, n);
    a = block_join<P>(a);
    if (threadIdx.x == 0) part[blockIdx.x] = a;
}
// norm and coefficient from the pieces' sums, by one workgroup, always in the same order
template <int P, int THREADS> __device__ __forceinline__ void finish(const double* part, int pieces, float max_norm, float grad_scale, float& norm, float& coef)
{
    double a = 0.0;
    int i = threadIdx.x;
    for (; i + 7 * THREADS < pieces; i += 8 * THREADS) {          // eight loads in flight
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = part[i + u * THREADS];
#pragma unroll
        for (int u = 0; u < 8; ++u) a = join<P>(a, v[u]);
    }
    for (; i < pieces; i += THREADS) a = join<P>(a, part[i]);
    a = block_join<P, THREADS>(a);
    norm = (float)((double)grad_scale * (P == 2 ? sqrt(a) : a));
    coef = max_norm / (norm + 1e-6f);
    coef = coef > 1.0f ? 1.0f : coef;                          // a NaN stays
}
template <int P> __global__ void __launch_bounds__(1024) clip_finish_kernel(const double* part, int pieces, float max_norm, float grad_scale, float* out)
{
    float norm, coef;
    finish<P, 1024>(part, pieces, max_norm, grad_scale, norm, coef);
    if (threadIdx.x == 0) {
        out[0] = norm;
        out[1] = coef;
    }
}
template <typename T> __device__ __forceinline__ void scale_piece(const T* g, T* o, int64_t n, float c)
{
    constexpr int V = 16 / sizeof(T);
    const int64_t nv = n / V;
    int64_t i = threadIdx.x;
    for (; i + 3 * 256 < nv; i += 4 * 256) {
        Loose<T> q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = *(const Loose<T>*)(g + (i + u * 256) * V);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int k = 0; k < V; ++k) q[u].v[k] = from_f32<T>(to_f32(q[u].v[k]) * c);
            *(Loose<T>*)(o + (i + u * 256) * V) = q[u];
        }
    }
    for (; i < nv; i += 256) {
        Loose<T> q = *(const Loose<T>*)(g + i * V);
#pragma unroll
        for (int k = 0; k < V; ++k) q.v[k] = from_f32<T>(to_f32(q.v[k]) * c);
        *(Loose<T>*)(o + i * V) = q;
    }
    for (int64_t e = nv * V + threadIdx.x; e < n; e += 256) o[e] = from_f32<T>(to_f32(g[e]) * c);
}
// DIRECT: the partial sums are added here, by every workgroup; workgroup 0 of the first launch writes `out`
template <int P, bool DIRECT>
__global__ void __launch_bounds__(256) clip_scale_kernel(const Table t, const double* part, int pieces, float max_norm, float grad_scale, float* out, int write_out)
{
    float norm, c;
    if (DIRECT) {
        finish<P, 256>(part, pieces, max_norm, grad_scale, norm, c);
        if (write_out && blockIdx.x == 0 && threadIdx.x == 0) {
            out[0] = norm;
            out[1] = c;
        }
    } else c = out[1];
    const int ti = find_tensor(t, blockIdx.x);
    if (c == 1.0f && t.src[ti] == t.dst[ti]) return;           // in place and not clipped: the product is the gradient
    const int64_t at = (int64_t)(blockIdx.x - t.first[ti]) * CLIP_PIECE, left = t.n[ti] - at, n = left < CLIP_PIECE ? left : CLIP_PIECE;
    const int dt = t.dtype[ti];
    if (dt == SNN_DT_F32) scale_piece<float>((const float*)t.src[ti] + at, (float*)t.dst[ti] + at, n, c);
    else if (dt == SNN_DT_BF16) scale_piece<bf16_t>((const bf16_t*)t.src[ti] + at, (bf16_t*)t.dst[ti] + at, n, c);
    else scale_piece<f16_t>((const f16_t*)t.src[ti] + at, (f16_t*)t.dst[ti] + at, n, c);
}

// The updates of snn_adam_step and snn_sgd_step (snn_update.h), gradients multiplied by grad_scale * *coef: the coefficient is
// read where clip_finish_kernel left it, so a clipped step reads the gradient twice and never writes it.
__global__ void __launch_bounds__(256) adam_clipped_kernel(int64_t n, float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                          float* __restrict__ v, float lr, float beta1, float beta2, float eps, float weight_decay,
                                                          float bc1, float bc2_sqrt, float grad_scale, const float* __restrict__ coef)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    adam_update(g[i] * grad_scale * *coef, p, m, v, i, lr, beta1, beta2, eps, weight_decay, bc1, bc2_sqrt);
}
__global__ void __launch_bounds__(256) sgd_clipped_kernel(int64_t n, float* __restrict__ p, const float* __restrict__ g, float* __restrict__ buf,
                                                         float lr, float momentum, float weight_decay, int first, float grad_scale,
                                                         const float* __restrict__ coef)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    sgd_update(g[i] * grad_scale * *coef, p, buf, i, lr, momentum, weight_decay, first);
}

int64_t pieces_of(int64_t n) { return (n + CLIP_PIECE - 1) / CLIP_PIECE; }

// tables of up to CLIP_TENSORS non-empty tensors, one launch of `f(table, pieces of the table, pieces before it)` each; `back`:
// from the last tensor to the first
template <typename F>
void each_table(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, bool back, F f)
{
    Table t;
    t.count = 0;
    int64_t before = 0;
    int here = 0;
    for (int k = 0; k < n_tensors; ++k) {
        const int i = back ? n_tensors - 1 - k : k;
        if (numel[i]) {
            t.src[t.count] = src[i];
            t.dst[t.count] = dst ? dst[i] : nullptr;
            t.n[t.count] = numel[i];
            t.dtype[t.count] = (unsigned char)dtype[i];
            t.first[t.count] = here;
            here += (int)pieces_of(numel[i]);
            t.first[++t.count] = here;
        }
        if (t.count && (t.count == CLIP_TENSORS || k == n_tensors - 1)) {
            f(t, here, before);
            before += here;
            here = t.count = 0;
        }
    }
}

template <int P>
void run(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, float max_norm, float grad_scale,
         float* out, double* part, int64_t pieces, hipStream_t s)
{
    const dim3 w(256);
    each_table(n_tensors, src, dst, numel, dtype, false, [&](const Table& t, int here, int64_t before) {
        hipLaunchKernelGGL((clip_norm_kernel<P>), dim3(here), w, 0, s, t, part + before);
    });
    const bool direct = dst && pieces && pieces <= CLIP_DIRECT;
    if (!direct) hipLaunchKernelGGL((clip_finish_kernel<P>), dim3(1), dim3(1024), 0, s, (const double*)part, (int)pieces, max_norm, grad_scale, out);
    if (dst)            // backwards: what the first pass read last is still in the last-level cache
        each_table(n_tensors, src, dst, numel, dtype, true, [&](const Table& t, int here, int64_t before) {
            if (direct)
                hipLaunchKernelGGL((clip_scale_kernel<P, true>), dim3(here), w, 0, s, t, (const double*)part, (int)pieces, max_norm, grad_scale, out, before == 0);
            else
                hipLaunchKernelGGL((clip_scale_kernel<P, false>), dim3(here), w, 0, s, t, (const double*)part, (int)pieces, max_norm, grad_scale, out, 0);
        });
}

// Results may not share memory with each other, nor with any gradient but their own (which they must then cover exactly): the
// workgroups of two tensors run at once.
struct Span { uintptr_t lo, hi; int i; };
int check_apart(int n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype)
{
    auto bytes = [&](int i) { return (uintptr_t)numel[i] * (dtype[i] == SNN_DT_F32 ? 4 : 2); };
    const std::unique_ptr<Span[]> to(new (std::nothrow) Span[n_tensors + 1]);
    if (!to) { snn_set_error("snn_clip_grads: out of host memory"); return SNN_ERR_ARG; }
    int n = 0;
    bool in_place = true;
    for (int i = 0; i < n_tensors; ++i) {
        if (!numel[i]) continue;
        to[n++] = Span{(uintptr_t)dst[i], (uintptr_t)dst[i] + bytes(i), i};
        in_place = in_place && dst[i] == src[i];
    }
    std::sort(to.get(), to.get() + n, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    for (int k = 1; k < n; ++k)
        if (to[k].lo < to[k - 1].hi) {
            snn_set_error("snn_clip_grads: a gradient or a place in out is listed twice, or two of them overlap (tensors %d, %d)", to[k - 1].i, to[k].i);
            return SNN_ERR_ARG;
        }
    for (int i = 0; i < n_tensors && !in_place; ++i) {
        if (!numel[i]) continue;
        const uintptr_t lo = (uintptr_t)src[i], hi = lo + bytes(i);
        // the first result that ends behind lo, and those that begin before hi
        const Span* s = std::upper_bound(to.get(), to.get() + n, lo, [](uintptr_t v, const Span& a) { return v < a.hi; });
        for (; s < to.get() + n && s->lo < hi; ++s)
            if (s->i != i || s->lo != lo) {
                snn_set_error("snn_clip_grads: out overlaps another gradient, or its own in part (tensors %d, %d)", s->i, i);
                return SNN_ERR_ARG;
            }
    }
    return SNN_OK;
}

}  // namespace

extern "C" int64_t snn_clip_scratch_doubles(int32_t n_tensors, const int64_t* numel)
{
    if (n_tensors < 0 || (n_tensors && !numel)) { snn_set_error("snn_clip_scratch_doubles: bad arguments"); return SNN_ERR_ARG; }
    int64_t p = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (numel[i] < 0) { snn_set_error("snn_clip_scratch_doubles: negative size"); return SNN_ERR_ARG; }
        p += pieces_of(numel[i]);
        if (p > 0x3fffffff) { snn_set_error("snn_clip_scratch_doubles: too many elements"); return SNN_ERR_UNSUPPORTED; }
    }
    return p;
}

extern "C" int snn_clip_grads(int32_t n_tensors, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype,
                              int32_t norm_type, float max_norm, float grad_scale, float* out, double* scratch, int64_t scratch_doubles, void* stream)
{
    const int64_t pieces = snn_clip_scratch_doubles(n_tensors, numel);
    if (pieces < 0) return (int)pieces;
    if (!out || (n_tensors && (!src || !dtype)) || (pieces && !scratch) || (norm_type != 0 && norm_type != 1 && norm_type != 2)) {
        snn_set_error("snn_clip_grads: null pointer, or norm_type %d (1, 2, 0 for the largest magnitude)", norm_type);
        return SNN_ERR_ARG;
    }
    if (scratch_doubles < pieces) {
        snn_set_error("snn_clip_grads: scratch of %lld doubles, %lld needed", (long long)scratch_doubles, (long long)pieces);
        return SNN_ERR_WORKSPACE;
    }
    for (int i = 0; i < n_tensors; ++i)
        if (numel[i] && (!src[i] || (dst && !dst[i]) || dtype[i] < 0 || dtype[i] > 2)) {
            snn_set_error("snn_clip_grads: tensor %d: null pointer or dtype %d", i, dtype[i]);
            return SNN_ERR_ARG;
        }
    if (dst)
        if (int rc = check_apart(n_tensors, src, dst, numel, dtype)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (norm_type == 2) run<2>(n_tensors, src, dst, numel, dtype, max_norm, grad_scale, out, scratch, pieces, s);
    else if (norm_type == 1) run<1>(n_tensors, src, dst, numel, dtype, max_norm, grad_scale, out, scratch, pieces, s);
    else run<0>(n_tensors, src, dst, numel, dtype, max_norm, grad_scale, out, scratch, pieces, s);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}

extern "C" int snn_adam_step_clipped(int64_t n, float* params, const float* grads, float* exp_avg, float* exp_avg_sq, int64_t step, float lr,
                                     float beta1, float beta2, float eps, float weight_decay, float grad_scale, const float* coef, void* stream)
{
    if (!params || !grads || !exp_avg || !exp_avg_sq || !coef || n < 1 || step < 1) {
        snn_set_error("snn_adam_step_clipped: null pointer, n < 1 or step < 1");
        return SNN_ERR_ARG;
    }
    const double bc1 = 1.0 - pow((double)beta1, (double)step), bc2 = 1.0 - pow((double)beta2, (double)step);
    hipLaunchKernelGGL(adam_clipped_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, n, params, grads, exp_avg,
                       exp_avg_sq, lr, beta1, beta2, eps, weight_decay, (float)bc1, (float)sqrt(bc2), grad_scale, coef);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}

extern "C" int snn_sgd_step_clipped(int64_t n, float* params, const float* grads, float* momentum_buf, int64_t step, float lr, float momentum,
                                    float weight_decay, float grad_scale, const float* coef, void* stream)
{
    if (!params || !grads || (momentum != 0.0f && !momentum_buf) || !coef || n < 1 || step < 1) {
        snn_set_error("snn_sgd_step_clipped: null pointer, n < 1 or step < 1");
        return SNN_ERR_ARG;
    }
    hipLaunchKernelGGL(sgd_clipped_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, n, params, grads, momentum_buf, lr,
                       momentum, weight_decay, step == 1 ? 1 : 0, grad_scale, coef);
    HIP_CHECK(hipGetLastError());
    return SNN_OK;
}
