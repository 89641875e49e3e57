// What the kernels over rows of hidden states and logits share: 16-byte accesses at element alignment, folds over a wave and a workgroup,
// exponentials, and the argument checks of their C entries.
#ifndef DALI_HIP_ROW_MATH_H
#define DALI_HIP_ROW_MATH_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "runtime.h"

namespace dali_hip {

// 16 bytes of values that start at any element: global memory takes such an access as one instruction
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// groups of 16 bytes in a row
template <typename T>
__host__ __device__ __forceinline__ int groups_of(int width) {
    return width / Vec<T>::N + (width % Vec<T>::N != 0);
}

// The group of values that begins at c, in two steps: the access, which reads the row's last whole group where c lies past its beginning, so that it needs no
// branch and many are under way at once; and the values, moved to their places, with `fill` past the row's end. Rows shorter than a group are read one by one;
// LONG: the row is known not to be, WHOLE: nor to end inside a group or before c.
template <bool LONG = false, bool WHOLE = false, typename T>
__device__ __forceinline__ typename Vec<T>::type ask_group(const T* x, int c, int width) {
    constexpr int N = Vec<T>::N;
    if constexpr (WHOLE) return *reinterpret_cast<const typename Vec<T>::type*>(x + c);
    if (LONG || width >= N) return *reinterpret_cast<const typename Vec<T>::type*>(x + min(c, width - N));
    typename Vec<T>::type g;
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = c + i < width ? x[c + i] : T(0);
    return g;
}
template <bool LONG = false, bool WHOLE = false, typename T>
__device__ __forceinline__ void take_group(const typename Vec<T>::type& g, int c, int width, T fill, T (&v)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = g[i];
    if constexpr (WHOLE) return;
    const int off = c - (width - N);
    if (off <= 0) return;
    if (LONG || width >= N) {
#pragma unroll
        for (int bit = 1; bit < N; bit *= 2)
            if (off & bit)
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = i + bit < N ? v[i + bit < N ? i + bit : 0] : fill;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < width ? v[i] : fill;
}
template <typename T>
__device__ __forceinline__ void load_group(const T* x, int c, int width, T fill, T (&v)[Vec<T>::N]) {
    take_group(ask_group(x, c, width), c, width, fill, v);
}

// (PAST: without taking room in the caches, for results that they would not hold until somebody reads them. A condition at run time does not do: the
// compiler merges the two stores into the ordinary one)
template <bool PAST = false, typename T>
__device__ __forceinline__ void store_group(T* out, int c, int width, const T (&v)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    if (c <= width - N) {
        typename Vec<T>::type g;
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = v[i];
        if constexpr (PAST) __builtin_nontemporal_store(g, reinterpret_cast<typename Vec<T>::type*>(out + c));
        else *reinterpret_cast<typename Vec<T>::type*>(out + c) = g;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < width) out[c + i] = v[i];
    }
}

// The value of the lane that is D away in the binary numbering of a wave, for folds that have already joined the lanes closer than D: `a` and `b` are
// the two halves' values, the same pair in both. Steps inside 16 lanes are data moves of the vector unit (within a quad, the mirror image of 8 and of 16 lanes),
// the others exchange half rows between two registers; none goes through LDS.
template <int D>
__device__ __forceinline__ void halves(unsigned v, unsigned& a, unsigned& b) {
    if constexpr (D <= 8) {
        constexpr int control = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;
        a = v;
        b = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, control, 0xf, 0xf, true);
    } else if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        a = r[0], b = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        a = r[0], b = r[1];
    }
}

template <int D, typename T>
__device__ __forceinline__ void halves_of(T v, T& a, T& b) {
    if constexpr (sizeof(T) == 4) {
        unsigned x, y;
        halves<D>(__builtin_bit_cast(unsigned, v), x, y);
        a = __builtin_bit_cast(T, x), b = __builtin_bit_cast(T, y);
    } else {
        const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
        unsigned x0, y0, x1, y1;
        halves<D>((unsigned)bits, x0, y0);
        halves<D>((unsigned)(bits >> 32), x1, y1);
        a = __builtin_bit_cast(T, (unsigned long long)x1 << 32 | x0);
        b = __builtin_bit_cast(T, (unsigned long long)y1 << 32 | y0);
    }
}

// the fold of LANES neighbouring lanes' values, the same in each of them; `op` is commutative, so the bits do not depend on the lane
template <int LANES, int D = 1, typename T, typename Op>
__device__ __forceinline__ T fold_lanes(T v, Op op) {
    if constexpr (D >= LANES) {
        return v;
    } else {
        T a, b;
        halves_of<D>(v, a, b);
        return fold_lanes<LANES, D * 2>(op(a, b), op);
    }
}

struct Sum {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const {
        return a + b;
    }
};
// (a NaN loses against a number)
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};

// the fold of one value of every thread, the same in each of them, in an order that depends on nothing but the thread numbers. `scratch` holds one T per wave;
// it may be used again at once.
template <int THREADS, typename T, typename Op>
__device__ __forceinline__ T fold_block(T v, T* scratch, Op op) {
    v = fold_lanes<64>(v, op);
    if constexpr (THREADS == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = scratch[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) s = op(s, scratch[w]);
    return s;
}

template <int THREADS, typename T>
__device__ __forceinline__ T block_sum(T v, T* scratch) {
    return fold_block<THREADS>(v, scratch, Sum());
}

// Whether a pass moves so much that the caches (256 MiB) would not hold its result until somebody reads it. Ordinary stores and those past the caches (us): gradient of log
// probabilities 8192x32000 408 and 392, layer norm 65536x1024 91.7 and 89.1, clipping 52 million values, whose second launch finds more of what the first read, 127 and 105.
// Smaller passes gain little (8192x1024 11.5 and 11.4, its gradient 24.2 and 22.6), and the next kernel would have to fetch their result.
inline bool past_caches(double bytes) { return bytes >= (double)(256L << 20); }

// f(true_type) or f(false_type)
template <typename F>
void either_way(bool condition, F f) {
    if (condition) f(std::true_type());
    else f(std::false_type());
}

// Results that another workgroup of the same launch reads: stored past the caches of this one's die, awaited, and announced with a ticket
template <typename T>
__device__ __forceinline__ void publish(T* p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T observe(const T* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether the calling workgroup is the last of `members` to arrive at the counter, which it then leaves at zero. All threads call it; `shared` is theirs. What
// any thread published before is acknowledged by memory before the ticket is drawn.
__device__ __forceinline__ bool last_to_arrive(unsigned* counter, unsigned members, unsigned* shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned ticket = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (ticket == members - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *shared = ticket;
    }
    __syncthreads();
    asm volatile("" ::: "memory");
    return *shared == members - 1;
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

inline bool off_elements(std::initializer_list<const void*> pointers, size_t size) {
    for (const void* p : pointers)
        if ((uintptr_t)p % size != 0) return true;
    return false;
}

inline bool is_real(int dtype) { return dtype == DALI_HIP_FLOAT || dtype == DALI_HIP_DOUBLE; }

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DALI_HIP_OK : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace dali_hip

#endif
