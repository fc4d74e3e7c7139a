// snn_scan.h -- what the forward and the backward of the selective scan share (snn_scan.hip, snn_scan_bwd.hip).
#pragma once
#include "snn_seq.h"

// Mapping.  A quad of lanes owns one channel: lane j holds the states j*K .. j*K + K-1 in registers (K = 2, 4, 8, 16 for up
// to 8, 16, 32, 64 states; states that do not exist have A = B = C = 0 and stay 0).  A wave covers 16 channels, a workgroup
// of four waves SCAN_CH = 64, all of one group, so B_t and C_t are the workgroup's; they pass through LDS as fp32.
// Per-step work that does not depend on the state (softplus, gate, loads, stores) is dealt over the quad: lane j does
// it for step t + j of four, and the step's scalars reach the others by DPP.
constexpr int SCAN_CH = 64;
constexpr int SCAN_SEG = 16;                                              // steps per staged segment, forward
// Steps between the states kept on the tape = steps per segment of the backward, which holds h and a of a segment in
// registers.
__host__ __device__ constexpr int scan_tape_k(int k) { return k <= 2 ? 16 : k == 4 ? 8 : 4; }
template <int K> struct ScanTape { static constexpr int STEPS = scan_tape_k(K); };

static inline int scan_k(int states) { return states <= 8 ? 2 : states <= 16 ? 4 : states <= 32 ? 8 : 16; }
static inline int scan_tape_steps(int states) { return scan_tape_k(scan_k(states)); }
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
    int vec;                            // rows of N states start at multiples of 16 bytes and N == 4 K
    // backward
    View<T> dy, dx, ddelta, dz, dB, dC;
    const float* dhT;
    float *dh0, *part, *bcpart;         // per slot: dA (D, 4K), dskip, dbias (D); per channel block: dB, dC rows
    int slots, direct;
};

// lane j's K states of a row of N fp32 states
template <int K> __device__ __forceinline__ void load_states(const float* p, int j, int N, bool vec, float (&v)[K])
{
    if (vec) {
#pragma unroll
        for (int i = 0; i < K; i += (K < 4 ? 2 : 4)) {
            if constexpr (K < 4) {
                const float2 q = *(const float2*)(p + j * K + i);
                v[i] = q.x;
                v[i + 1] = q.y;
            } else {
                const float4 q = *(const float4*)(p + j * K + i);
                v[i] = q.x;
                v[i + 1] = q.y;
                v[i + 2] = q.z;
                v[i + 3] = q.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] = j * K + i < N ? p[j * K + i] : 0.0f;
    }
}
template <int K> __device__ __forceinline__ void store_states(float* p, int j, int N, bool vec, const float (&v)[K])
{
    if (vec) {
        if constexpr (K < 4) *(float2*)(p + j * K) = make_float2(v[0], v[1]);
        else {
#pragma unroll
            for (int i = 0; i < K; i += 4) *(float4*)(p + j * K + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (j * K + i < N) p[j * K + i] = v[i];
    }
}

// The workgroup's B (and C) rows of SEG steps from step t0 on, into registers and from there into LDS: element e of thread
// tid is step e / 4K, state e % 4K.  Steps at or past t1 and states past N are 0 and not read.
template <typename T, int K, int SEG> struct BcStage {
    static constexpr int PER = (SEG * 4 * K + 255) / 256;
    float b[PER], c[PER];
    template <bool WANT_C>
    __device__ __forceinline__ void load(const T* Bp, int64_t bst, const T* Cp, int64_t cst, int t0, int t1, int N, int tid)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + i * 256, t = t0 + e / (4 * K), n = e % (4 * K);
            const bool ok = e < SEG * 4 * K && t < t1 && n < N;
            b[i] = ok ? to_f32(Bp[t * bst + n]) : 0.0f;
            if (WANT_C) c[i] = ok ? to_f32(Cp[t * cst + n]) : 0.0f;
        }
    }
    template <bool WANT_C> __device__ __forceinline__ void store(float* Bs, float* Cs, int tid)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + i * 256;
            if (e < SEG * 4 * K) {
                Bs[e] = b[i];
                if (WANT_C) Cs[e] = c[i];
            }
        }
    }
};
template <int K> __device__ __forceinline__ void lds_states(const float* s, int j, float (&v)[K])
{
    if constexpr (K < 4) {
        const float2 q = *(const float2*)(s + j * K);
        v[0] = q.x;
        v[1] = q.y;
    } else {
#pragma unroll
        for (int i = 0; i < K; i += 4) {
            const float4 q = *(const float4*)(s + j * K + i);
            v[i] = q.x;
            v[i + 1] = q.y;
            v[i + 2] = q.z;
            v[i + 3] = q.w;
        }
    }
}

// this workgroup's channels: group, first channel, and the lane's channel (ok: it exists)
struct ScanCh { int g, d, j; bool ok; };
__device__ __forceinline__ ScanCh scan_channel(int cb, int cbg, int dg, int tid)
{
    ScanCh c;
    c.g = cb / cbg;
    const int i = (cb - c.g * cbg) * SCAN_CH + (tid >> 2);
    c.ok = i < dg;
    c.d = c.g * dg + (c.ok ? i : dg - 1);          // lanes without a channel read the group's last one and write nothing
    c.j = tid & 3;
    return c;
}
// rows of f cleared by the workgroup: 64 channels x 4 rows at a time
template <typename T> __device__ __forceinline__ void clear_channels(const View<T>& y, int64_t base, const FillRange& f, int d0, int n, int tid)
{
    const int d = tid & 63;
    if (d >= n) return;
    for (int64_t t = f.a0 + (tid >> 6); t < f.a1; t += 4) y.p[base + t * y.st + d0 + d] = (T)0.0f;
    for (int64_t t = f.b0 + (tid >> 6); t < f.b1; t += 4) y.p[base + t * y.st + d0 + d] = (T)0.0f;
}

// host: snn_scan.hip
int snn_scan_check(const snn_scan_args* a, const char* fn);
struct ScanGrid { int cbg, blocks_c, tc, nc; };
ScanGrid snn_scan_grid(const snn_scan_args* a, bool backward);
template <typename T> ScanP<T> scan_params(const snn_scan_args* a, const ScanGrid& g);
void snn_scan_launch_combine(const snn_scan_args* a, const ScanGrid& g, const float* edge, float* carry, const float* csum, bool reverse, hipStream_t s);
