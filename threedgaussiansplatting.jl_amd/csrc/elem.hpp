// elem.hpp — the element types of the decoder operators (float, bfloat16, half): vectors of
// eight, conversions, and the 32x32 matrix product of each type.
#pragma once

#include "common.hpp"

namespace tdgs {

typedef __bf16 bf16;
typedef _Float16 f16;

template <class T>
struct Elem {
    typedef T V8 __attribute__((ext_vector_type(8)));
    typedef T V8a __attribute__((ext_vector_type(8), aligned(16)));   // in memory: 16-byte aligned
    typedef T V4 __attribute__((ext_vector_type(4)));
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

inline bool known_dtype(int32_t dtype) { return dtype == TDGS_F32 || dtype == TDGS_BF16 || dtype == TDGS_F16; }
inline int64_t dtype_size(int32_t dtype) { return dtype == TDGS_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// f(T{}) for the element type of a dtype code (checked by the caller).
template <class F>
inline int with_dtype(int32_t dtype, F&& f) {
    switch (dtype) {
        case TDGS_F32: return f(float{});
        case TDGS_BF16: return f(bf16{});
        default: return f(f16{});
    }
}

// Eight elements at p, of which the first n exist (n <= 0: none); the others are zero. vec: p and
// every row it came from are 16-byte aligned.
template <class T>
__device__ __forceinline__ typename Elem<T>::V8 load8(const T* __restrict__ p, int n, bool vec) {
    typename Elem<T>::V8 r;
    if (vec && n >= 8) {
        r = *reinterpret_cast<const typename Elem<T>::V8a*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = i < n ? p[i] : (T)0.0f;
    }
    return r;
}

template <class T>
__device__ __forceinline__ typename Elem<T>::V8 zero8() {
    typename Elem<T>::V8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)0.0f;
    return r;
}

// acc += A B for one 32x32 block, 16 deep. A: lane l holds row l % 32, B: column l % 32; both the
// depth slots (l / 32) * 8 + i. acc: lane l holds column l % 32, register r row
// (r / 4) * 8 + (l / 32) * 4 + r % 4. Which depth a slot stands for is the caller's choice, as long as
// A and B agree: a block of results (its rows spread over the registers as above) can so be the next
// product's B without moving between lanes.
__device__ __forceinline__ f32x16 mma(Elem<bf16>::V8 a, Elem<bf16>::V8 b, f32x16 acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(Elem<f16>::V8 a, Elem<f16>::V8 b, f32x16 acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(Elem<float>::V8 a, Elem<float>::V8 b, f32x16 acc) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
    return acc;
}

// Both halves' values of x, in every lane (lane l gets those of lanes l % 32 and l % 32 + 32). The
// empty asm keeps the compiler from folding the two results of the swap into one.
__device__ __forceinline__ void both_halves(float x, float* lo, float* hi) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    uint32_t h = r[1];
    asm volatile("" : "+v"(h));
    *lo = __builtin_bit_cast(float, (uint32_t)r[0]);
    *hi = __builtin_bit_cast(float, h);
}
__device__ __forceinline__ float sum_halves(float x) {
    float lo, hi;
    both_halves(x, &lo, &hi);
    return lo + hi;
}
__device__ __forceinline__ float max_halves(float x) {
    float lo, hi;
    both_halves(x, &lo, &hi);
    return fmaxf(lo, hi);
}

// Division by a constant known on the host, for dividends below 2^31: with L = ceil(log2 d) and
// s = 31 + L, m = floor(2^s / d) + 1 < 2^32 + 1 exceeds 2^s / d by at most 1, so n m / 2^s exceeds
// n / d by less than 1 / d and has the same floor.
struct FastDiv {
    uint64_t m;
    uint32_t d, s;
    FastDiv() : m(0), d(1), s(0) {}
    explicit FastDiv(uint32_t div) : d(div) {
        uint32_t l = 0;
        while ((1ull << l) < div) ++l;
        s = 31 + l;
        m = (1ull << s) / div + 1;
    }
    __host__ __device__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> s); }
};

}  // namespace tdgs
