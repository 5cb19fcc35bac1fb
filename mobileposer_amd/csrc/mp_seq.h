// Shared declarations of the sequence operators that take the caller's own tensors: the gated delta rule (mp_delta.hip), the linear
// layer with an adapter per sequence (mp_adapt.hip) and their entry points (mp_sequence.hip).
#pragma once
#include "mp_common.h"

namespace mpseq {

enum { kF32 = 0, kBF16 = 1 };           // MP_F32 / MP_BF16 of the boundary header

typedef uint16_t bf16raw;               // a bfloat16 as it lies in memory

// bf16 -> fp32 is exact; fp32 -> bf16 rounds to nearest even (NaN stays NaN): the one rounding of a bf16 output
static __device__ __forceinline__ float load_f(const float* p) { return *p; }
static __device__ __forceinline__ float load_f(const bf16raw* p) { return __uint_as_float((unsigned)*p << 16); }
static __device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
static __device__ __forceinline__ void store_f(bf16raw* p, float v) {
    const __bf16 b = (__bf16)v;
    *p = __builtin_bit_cast(uint16_t, b);
}

// ---------------------------------------------------------------- gated delta rule
// (strides in elements; q, k: [B][T][Hk][dk], v: [B][T][Hv][dv], g, beta: [B][T][Hv]; the last dimension is contiguous)
struct DeltaArgs {
    const void *q, *k, *v;
    const float *g, *beta;
    long sq[3], sk[3], sv[3], sg[3], sb[3];      // batch (or stream), time, head
    const int* lengths;                          // [B], clamped to 0..T on the device; nullptr: all T
    int B, T, Hk, Hv, dk, dv;
    float scale;
    void* o;                                     // [B][T][Hv][dv] contiguous, rows behind a sequence's end: zeros
    const float* s_in;                           // [B][Hv][dk][dv] or nullptr (zeros)
    float* s_out;                                // [B][Hv][dk][dv] or nullptr
    float* ws;
    int nchunk;
};
struct DeltaOnlineArgs {
    const void *q, *k, *v;
    const float *g, *beta;
    long sq[2], sk[2], sv[2], sg[2], sb[2];      // stream, head
    const int* slots;                            // [S] rows of `state`, or nullptr: stream s owns row s
    int S, n_slots, Hk, Hv, dk, dv;
    float scale;
    void* o;                                     // [S][Hv][dv]
    float* state;                                // [n_slots][Hv][dk][dv], updated in place
};
size_t delta_ws_floats(int B, int T, int Hv, int dk, int dv);
bool launch_delta(const DeltaArgs& a, int dtype, hipStream_t s);
int64_t delta_online_blocks(const DeltaOnlineArgs& a);        // workgroups of 256 threads
bool launch_delta_online(const DeltaOnlineArgs& a, int dtype, hipStream_t s);

// ---------------------------------------------------------------- linear layer with an adapter per sequence
struct AdaptArgs {
    const void* x;                               // [B][T][K], row strides below
    long sx[2];                                  // batch, time
    const void *w, *bias;                        // [M] rows of K, ldw apart; [M] or nullptr
    long ldw;
    const void *down, *up;                       // [n][r][K], [n][M][r]
    const float* scale;                          // [n] or nullptr (1)
    const int* ids;                              // [B]; negative: no adapter, >= n: the sequence's rows become NaN
    int B, T, K, M, n, r, relu;
    void* y;                                     // [B][T][M], row strides below
    long sy[2];                                  // batch, time
    float* ws;                                   // [B*T][r] fp32
    int vec;                                     // (set by the launcher) columns of y that can be stored at once: 2: 16 bytes, 1: four, 0: one
};
size_t adapt_ws_floats(int B, int T, int r);
bool adapt_fits(int B, int T, int M, int r);     // one call's launches can count these rows and columns
bool launch_adapt(const AdaptArgs& a, int dtype, hipStream_t s);

}  // namespace mpseq
