// Device helpers of the sequence operators: operands of the bf16 matrix instructions from bf16 or fp32 data.
//
// An fp32 value as three bf16 terms -- each the nearest to what the ones before it leave -- keeps all 24 bits, and a product of two
// such values is six products of terms: the three left out are below 2^-26 of it.  With fp32 accumulation that is the accuracy of
// an fp32 sum at 16 / 6 times the rate of the fp32 matrix instructions; beside a bf16 operand, which is its own only term, it is
// three products.  (An infinite value, or one above the largest bf16 by half a step, 3.396e38, gives NaN terms: inf - inf in the
// split.)
#pragma once
#include "mp_seq.h"

namespace mpseq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <class E> struct Arith;
template <> struct Arith<bf16raw> { static constexpr int P = 1; };               // planes of an input
template <> struct Arith<float> { static constexpr int P = 3; };

// eight consecutive elements as P planes of bf16 (rows need no alignment: a row of odd length starts anywhere)
template <class E> struct Oct;
template <> struct Oct<bf16raw> {
    u32x4 v;
    __device__ __forceinline__ void zero() { v = (u32x4){0, 0, 0, 0}; }
    __device__ __forceinline__ void arrived() const { asm volatile("" ::"v"(v)); }      // no load of it is in flight behind this
    __device__ __forceinline__ void load(const bf16raw* p) { __builtin_memcpy(&v, p, 16); }
    __device__ __forceinline__ void load_guarded(const bf16raw* p, int n) {
        bf16raw t[8];
        for (int i = 0; i < 8; ++i) t[i] = i < n ? p[i] : (bf16raw)0;
        __builtin_memcpy(&v, t, 16);
    }
    __device__ __forceinline__ void load_runs(const bf16raw* p, int) { load(p); }
    __device__ __forceinline__ void load_some_runs(const bf16raw* p, int, int n) { load_some(p, n); }
    __device__ __forceinline__ void load_clamped(const bf16raw* row, int d, int n) {
        bf16raw t[8];
        for (int i = 0; i < 8; ++i) t[i] = row[min(d + i, n - 1)];
        __builtin_memcpy(&v, t, 16);
    }
    __device__ __forceinline__ void shift(int s) {                // element i <- element i + s, zeros behind the last (s < 8)
        if (s & 4) { v[0] = v[2]; v[1] = v[3]; v[2] = v[3] = 0; }
        if (s & 2) { v[0] = v[1]; v[1] = v[2]; v[2] = v[3]; v[3] = 0; }
        if (s & 1) { v[0] = v[0] >> 16 | v[1] << 16; v[1] = v[1] >> 16 | v[2] << 16; v[2] = v[2] >> 16 | v[3] << 16; v[3] >>= 16; }
    }
    __device__ __forceinline__ void keep(int n) {                 // zeros from element n on
        for (int i = 0; i < 4; ++i) v[i] = 2 * i >= n ? 0 : 2 * i + 1 >= n ? v[i] & 0xffffu : v[i];
    }
    __device__ __forceinline__ void load_some(const bf16raw* p, int n) {
        if (n >= 8) load(p); else load_guarded(p, n);
    }
    __device__ __forceinline__ float dot(const Oct<float>& z, float s) const;
    __device__ __forceinline__ void planes(u32x4 (&o)[1]) const { o[0] = v; }
};
template <> struct Oct<float>;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// two floats -> their nearest bf16 (one word, a in the low half)
static __device__ __forceinline__ unsigned nearest_bf16(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
// the same, and what is left of them: x - bf16(x) is exact, and one v_dot2_f32_bf16 of the packed pair with (-1, 0) or (0, -1) does it
// without unpacking.  (The selectors come from registers: as a constant, 0xbf800000 is taken for the inline operand -1.0, whose
// halves are not what is meant.)
static __device__ __forceinline__ unsigned take_bf16(float& a, float& b) {
    unsigned first = 0x0000bf80u, second = 0xbf800000u;
    asm("" : "+s"(first));
    asm("" : "+s"(second));
    const bf16x2 w = __builtin_convertvector((f32x2){a, b}, bf16x2);
    a = __builtin_amdgcn_fdot2_f32_bf16(w, __builtin_bit_cast(bf16x2, first), a, false);
    b = __builtin_amdgcn_fdot2_f32_bf16(w, __builtin_bit_cast(bf16x2, second), b, false);
    return __builtin_bit_cast(unsigned, w);
}
template <> struct Oct<float> {
    float v[8];
    __device__ __forceinline__ void zero() { for (int i = 0; i < 8; ++i) v[i] = 0.f; }
    __device__ __forceinline__ void arrived() const { for (int i = 0; i < 8; ++i) asm volatile("" ::"v"(v[i])); }
    __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(v, p, 32); }
    __device__ __forceinline__ void load_guarded(const float* p, int n) {
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    }
    // two runs of four, `gap` apart; the first n of the row from p on are there
    __device__ __forceinline__ void load_runs(const float* p, int gap) {
        __builtin_memcpy(v, p, 16);
        __builtin_memcpy(v + 4, p + gap, 16);
    }
    __device__ __forceinline__ void load_some_runs(const float* p, int gap, int n) {
        for (int i = 0; i < 8; ++i) {
            const int at = (i & 3) + (i >> 2) * gap;
            v[i] = at < n ? p[at] : 0.f;
        }
    }
    __device__ __forceinline__ void load_clamped(const float* row, int d, int n) {
        for (int i = 0; i < 8; ++i) v[i] = row[min(d + i, n - 1)];
    }
    __device__ __forceinline__ void shift(int s) {
#pragma unroll
        for (int m = 4; m > 0; m >>= 1)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = s & m ? (i + m < 8 ? v[i + m < 8 ? i + m : 0] : 0.f) : v[i];
    }
    __device__ __forceinline__ void keep(int n) { for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : 0.f; }
    __device__ __forceinline__ void load_some(const float* p, int n) {
        if (n >= 8) load(p); else load_guarded(p, n);
    }
    __device__ __forceinline__ float dot(const Oct<float>& z, float s) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(z.v[i], v[i], s);
        return s;
    }
    __device__ __forceinline__ void planes(u32x4 (&o)[3]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = v[2 * i], b = v[2 * i + 1];
            o[0][i] = take_bf16(a, b);
            o[1][i] = take_bf16(a, b);
            o[2][i] = nearest_bf16(a, b);
        }
    }
};
__device__ __forceinline__ float Oct<bf16raw>::dot(const Oct<float>& z, float s) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(z.v[2 * i + 1], __uint_as_float(v[i] & 0xffff0000u), fmaf(z.v[2 * i], __uint_as_float(v[i] << 16), s));
    return s;
}
static __device__ __forceinline__ void store4(float* p, const float (&y)[4]) { *(float4*)p = {y[0], y[1], y[2], y[3]}; }
static __device__ __forceinline__ void store4(bf16raw* p, const float (&y)[4]) {
    *(uint2*)p = {nearest_bf16(y[0], y[1]), nearest_bf16(y[2], y[3])};
}
static __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// 4 x 16 blocks of 16-bit elements turned over on the way out of LDS: of 16 lanes each, lane 4 s + u reads elements 4 u .. 4 u + 3 of
// row s and receives element 16-lane index of rows 0..3
typedef short s16x4 __attribute__((ext_vector_type(4)));
static __device__ __forceinline__ uint2 read_turned(const char* lds_piece) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lds_piece));
}
// sum of the products of planes whose orders add up to less than the number of planes that matter, the small ones first
template <int PA, int PB>
static __device__ __forceinline__ f32x4 mfma_planes(const u32x4 (&a)[PA], const u32x4 (&b)[PB], f32x4 c) {
    constexpr int top = (PA > PB ? PA : PB) - 1;
#pragma unroll
    for (int s = top; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i)
            if (i < PA && s - i < PB) c = mfma32(a[i], b[s - i], c);
    return c;
}
// the same for N accumulators in turn, so that no product waits for the one before it
template <int N, int PA, int PB>
static __device__ __forceinline__ void mfma_planes_n(const u32x4 (&a)[N][PA], const u32x4 (&b)[PB], f32x4 (&c)[N]) {
    constexpr int top = (PA > PB ? PA : PB) - 1;
#pragma unroll
    for (int s = top; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i)
            if (i < PA && s - i < PB)
#pragma unroll
                for (int n = 0; n < N; ++n) c[n] = mfma32(a[n][i], b[s - i], c[n]);
}

}  // namespace mpseq
