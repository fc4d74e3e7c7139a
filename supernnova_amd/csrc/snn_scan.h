// snn_scan.h -- what the forward and the backward of the selective scan share (snn_scan.hip, snn_scan_bwd.hip).
#pragma once
#include "snn_seq.h"

// Mapping.  LN = 4, 8 or 16 neighbouring lanes own one channel: lane i of them holds the states i K .. i K + K-1 in registers,
// K = 4 (K = 2 for up to 8 states): 16, 32, 64 states.  States that do not exist have A = B = C = 0 and stay 0.  A wave covers
// 64 / LN channels, a workgroup of four waves 256 / LN, all of one group, so B_t and C_t are the workgroup's; they pass through
// LDS as fp32.  Per-step work that does not depend on the state (softplus, gate, loads, stores) is dealt over four lanes:
// lane j of every quad does it for step t + j of four, and the step's scalars reach the others by DPP, folded into the
// multiplication that takes them.
constexpr int SCAN_SEG = 16;                                              // steps per staged segment, forward
// Steps between the states kept on the tape = steps per segment of the backward, which holds h and a of a segment in
// registers: 64 of them.  16 steps of K = 4 would be 128, and spill 230 bytes a lane at two waves a SIMD (64: up to 84 bytes).
__host__ __device__ constexpr int scan_tape_steps(int states) { return states <= 8 ? 16 : 8; }
template <int K> struct ScanTape { static constexpr int STEPS = K == 2 ? 16 : 8; };
static inline int scan_lanes(int states) { return states <= 16 ? 4 : states <= 32 ? 8 : 16; }
static inline int scan_padded(int states) { return states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64; }
// tape slots: sequence b, segment s is slot first(b) + s with room for every sequence's last, partial segment
static inline int64_t scan_tape_slots(const snn_seq& s, int steps)
{
    return s.offsets ? s.n_rows / steps + s.n_seq + 1 : (int64_t)s.n_seq * ((s.max_T + steps - 1) / steps);
}
__device__ __forceinline__ int64_t scan_tape_first(const snn_seq& s, const SeqRange& r, int b, int steps)
{
    return s.offsets ? r.row0 / steps + b : (int64_t)b * ((s.max_T + steps - 1) / steps);
}

template <typename T> struct ScanP {
    snn_seq seq;
    View<T> x, delta, z, B, C, y;
    int64_t B_sg, C_sg;
    const float *A, *skip, *dbias, *h0;
    float *hT, *tape;
    float *carry, *csum;                // split over time: state (adjoint) entering chunk c, and the sum of steps of chunk c
    int D, N, dg, cbg, softplus;        // channels, states, channels per group, channel blocks per group
    int tc, nc;                         // steps per chunk, chunks
    const int* order;                   // sequences, longest first, or NULL
    int vec;                            // rows of N states start at multiples of 16 bytes and fill the lanes
    // backward
    View<T> dy, dx, ddelta, dz, dB, dC;
    const float* dhT;
    float *dh0, *part, *bcpart;         // per slot: dA (D, LN K), dskip, dbias (D); per channel block: dB, dC rows
    int slots;
};

// K states of a row of N fp32 states, from state n on
template <int K> __device__ __forceinline__ void load_states(const float* p, int n, int N, bool vec, float (&v)[K])
{
    if (vec) {
        if constexpr (K == 2) {
            const float2 q = *(const float2*)(p + n);
            v[0] = q.x;
            v[1] = q.y;
        } else {
            const float4 q = *(const float4*)(p + n);
            v[0] = q.x;
            v[1] = q.y;
            v[2] = q.z;
            v[3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] = n + i < N ? p[n + i] : 0.0f;
    }
}
template <int K> __device__ __forceinline__ void store_states(float* p, int n, int N, bool vec, const float (&v)[K])
{
    if (vec) {
        if constexpr (K == 2) *(float2*)(p + n) = make_float2(v[0], v[1]);
        else *(float4*)(p + n) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (n + i < N) p[n + i] = v[i];
    }
}

// A in powers of two.  Steps of zero -- those that fill up a sequence's last segment, too -- leave the state as it is, so the
// product must not be infinite: 0 x inf.  At the lowest finite value every other step still decays to 0.
template <int K> __device__ __forceinline__ void decay_rates(float (&A)[K])
{
#pragma unroll
    for (int k = 0; k < K; ++k) {
        A[k] *= SNN_LOG2E;
        A[k] = A[k] < -3.402823466e38f ? -3.402823466e38f : A[k];          // a NaN stays
    }
}

// Steps j, j + 4, .. of a segment of one tensor for lane j, G of them; p points at step j and moves with the segment.  A whole
// segment adds multiples of the stride, the same for every lane; the last one of a chunk reads the chunk's last step again
// instead of steps behind it, and the caller drops what it read there.
template <typename T, int G> struct LaneIn {
    T v[G];
    __device__ __forceinline__ void load(const T* p, int64_t st, int j, int left)       // left: steps to the chunk's end
    {
        if (left >= 4 * G) {
#pragma unroll
            for (int i = 0; i < G; ++i) v[i] = p[4 * i * st];
        } else {
#pragma unroll
            for (int i = 0; i < G; ++i) v[i] = p[((4 * i + j < left ? 4 * i + j : left - 1) - j) * st];
        }
    }
};

// The workgroup's rows of B or C, SEG steps at a time, into registers and from there into LDS as fp32: element e of thread tid
// is step e / NP, state e % NP; p moves with the segment.  Steps past the chunk's end and states past N are 0 and not read.
template <typename T, int NP, int SEG> struct RowStage {
    static constexpr int PER = (SEG * NP + 255) / 256, ROWS = 256 / NP;
    float v[PER];
    const T* p;
    int m;
    bool in;
    __device__ __forceinline__ void init(const T* base, int64_t st, int N, int tid)
    {
        const int n = tid % NP;
        m = tid / NP;
        in = n < N && (SEG * NP >= 256 || tid < SEG * NP);
        p = base + m * st + (n < N ? n : 0);
    }
    __device__ __forceinline__ void load(int64_t st, int left)       // left: steps to the chunk's end
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = in && m + i * ROWS < left ? to_f32(p[i * ROWS * st]) : 0.0f;
    }
    __device__ __forceinline__ void store(float* s, int tid)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (SEG * NP >= 256 || tid < SEG * NP) s[tid + i * 256] = v[i];
    }
};
template <int K> __device__ __forceinline__ void lds_states(const float* s, int n, float (&v)[K]) { load_states<K>(s, n, 0, true, v); }

// LDS reads stay on their side of this point; everything else may pass.  Left alone, the compiler puts a read right in front of
// its use and waits out its latency at every step.
__device__ __forceinline__ void pin_lds_reads() { __builtin_amdgcn_sched_barrier(0x611); }

// lane q of every quad, q a constant after unrolling
__device__ __forceinline__ float qbc(float v, int q)
{
    return q == 0 ? quad_bcast<0>(v) : q == 1 ? quad_bcast<1>(v) : q == 2 ? quad_bcast<2>(v) : quad_bcast<3>(v);
}
// v[q] of step q summed over the channel's lanes, to lane q of every quad.  Quads are joined by mirroring: the mirror image of
// lane j is lane 3 - j of another quad, so the quad is turned round first.
template <int LN> __device__ __forceinline__ float step_sums(const float (&v)[4], int j)
{
    float r = quad_reduce_scatter(v, j);
    if constexpr (LN >= 8) r += dpp<0x141>(dpp<0x1B>(r));        // row_half_mirror of quad_perm [3, 2, 1, 0]
    if constexpr (LN >= 16) r += dpp<0x140>(dpp<0x1B>(r));       // row_mirror
    return r;
}

// this lane's channel: group, channel, first state, lane of the quad; ok: the channel exists; lead: its first quad
struct ScanCh { int g, d, n, j; bool ok, lead; };
template <int K, int LN> __device__ __forceinline__ ScanCh scan_channel(int cb, int cbg, int dg, int tid)
{
    ScanCh c;
    c.g = cb / cbg;
    const int i = (cb - c.g * cbg) * (256 / LN) + tid / LN;
    c.ok = i < dg;
    c.d = c.g * dg + (c.ok ? i : dg - 1);          // lanes without a channel read the group's last one and write nothing
    c.n = tid % LN * K;
    c.j = tid & 3;
    c.lead = c.ok && tid % LN < 4;
    return c;
}
// rows of f cleared by the workgroup, channels d0 .. d0 + n (n <= 64): 16 rows at a time in words of four channels where those
// are aligned, else four rows at a time
template <typename T> __device__ __forceinline__ void clear_rows(T* p, int64_t st, int64_t rows, int n, int tid)
{
    if (((uintptr_t)p % (4 * sizeof(T)) | (st & 3) | (n & 3)) == 0) {
        Pack<T, 4> zero;
#pragma unroll
        for (int i = 0; i < 4; ++i) zero.v[i] = (T)0.0f;
        const int d = (tid & 15) * 4, t = tid >> 4;
        T* q = p + t * st + d;
        if (d < n)
            for (int64_t left = rows - t; left > 0; left -= 16, q += 16 * st) *(Pack<T, 4>*)q = zero;
    } else {
        const int d = tid & 63, t = tid >> 6;
        T* q = p + t * st + d;
        if (d < n)
            for (int64_t left = rows - t; left > 0; left -= 4, q += 4 * st) *q = (T)0.0f;
    }
}
template <typename T> __device__ __forceinline__ void clear_channels(const View<T>& y, int64_t base, const FillRange& f, int d0, int n, int tid)
{
    if (f.a1 > f.a0) clear_rows(y.p + base + f.a0 * y.st + d0, y.st, f.a1 - f.a0, n, tid);
    if (f.b1 > f.b0) clear_rows(y.p + base + f.b0 * y.st + d0, y.st, f.b1 - f.b0, n, tid);
}

// host: snn_scan.hip
int snn_scan_check(const snn_scan_args* a, const char* fn);
struct ScanGrid { int cbg, blocks_c, tc, nc; };
ScanGrid snn_scan_grid(const snn_scan_args* a);
bool snn_scan_ordered(const snn_scan_args* a, const ScanGrid& g);
void snn_scan_launch_order(const snn_seq& seq, int* order, hipStream_t s);
template <typename T> ScanP<T> scan_params(const snn_scan_args* a, const ScanGrid& g);
void snn_scan_launch_combine(const snn_scan_args* a, const ScanGrid& g, const float* edge, float* carry, const float* csum, bool reverse, hipStream_t s);
