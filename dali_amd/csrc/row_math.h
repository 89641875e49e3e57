// What the kernels over rows of hidden states and logits share: 16-byte accesses at element alignment, folds over a wave and a workgroup,
// exponentials, and the argument checks of their C entries.
#ifndef DALI_HIP_ROW_MATH_H
#define DALI_HIP_ROW_MATH_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "runtime.h"

namespace dali_hip {

// 16 bytes of values that start at any element: global memory takes such an access as one instruction
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// one value of every thread -> the same fold of all in every thread, in an order that depends on nothing but the thread numbers.
// `scratch` holds one T per wave; it may be used again at once.
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
    return v;
}

template <int THREADS, typename T>
__device__ __forceinline__ T block_sum(T v, T* scratch) {
    v = wave_sum(v);
    if (THREADS == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = scratch[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) s += scratch[w];
    return s;
}

// ------------------------------------------------------------------------------------------------ arguments (host)
// The bytes that an operand covers, for refusing destinations that overlap what is still to be read
struct Span {
    const char* name;
    uintptr_t first = 0, lo = 0, hi = 0;  // of the first value, the lowest, and the end
    // rows of `width` values, `stride` values apart (either sign)
    Span(const char* n, const void* p, int64_t rows, int64_t width, int64_t stride, size_t size) : name(n) {
        if (!p || rows <= 0 || width <= 0) return;
        const int64_t last = (rows - 1) * stride;
        first = (uintptr_t)p;
        lo = (uintptr_t)p + (intptr_t)((last < 0 ? last : 0) * (int64_t)size);
        hi = (uintptr_t)p + (intptr_t)(((last > 0 ? last : 0) + width) * (int64_t)size);
    }
    Span(const char* n, const void* p, int64_t count, size_t size) : Span(n, p, 1, count, count, size) {}
    bool empty() const { return lo == hi; }
    bool meets(const Span& o) const { return !empty() && !o.empty() && lo < o.hi && o.lo < hi; }
    bool same(const Span& o) const { return first == o.first && lo == o.lo && hi == o.hi; }
};

// Destinations may not meet each other, nor an operand, except that the first `in_place` operands may be the first destination itself
inline int check_spans(const char* what, std::initializer_list<Span> outs, std::initializer_list<Span> ins, int in_place) {
    for (const Span* a = outs.begin(); a != outs.end(); ++a) {
        for (const Span* b = outs.begin(); b != a; ++b)
            if (a->meets(*b)) return fail("%s: %s and %s overlap", what, b->name, a->name);
        for (const Span* b = ins.begin(); b != ins.end(); ++b)
            if (a->meets(*b) && !(a == outs.begin() && b - ins.begin() < in_place && a->same(*b))) return fail("%s: %s overlaps %s", what, a->name, b->name);
    }
    return DALI_HIP_OK;
}

inline bool is_real(int dtype) { return dtype == DALI_HIP_FLOAT || dtype == DALI_HIP_DOUBLE; }

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DALI_HIP_OK : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace dali_hip

#endif
