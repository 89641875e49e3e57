// The norm over all values of many arrays, and the arrays scaled so that it is at most a given one.
//
//   norm = sqrt(sum over all arrays of sum of squares),  scale = max_norm / norm where norm > max_norm, else 1
//
// Squares are summed in double (an fp32 value's square neither overflows nor vanishes there; squares of doubles go into three sums by the value's size, those of large and
// of small values scaled by a power of two: Squares). A workgroup sums the chunks that fall to it and leaves its partial sums; every workgroup of the second launch folds
// all of them in the same order before it scales, so the norm does not depend on scheduling and needs no launch of its own. (They lie where no other kernel writes until the
// second launch has been issued: Carried, runtime.h.) The second launch walks the chunks backwards: what the first read last is still in the cache. A norm that is not
// finite scales nothing: the arrays come back as they are and the norm says so, and arrays that are their own destinations are left alone whenever nothing is scaled.
// Bound by memory: 52 million fp32 values in 24 arrays 103 us, 38 for the norm (5.4 TB/s) and 64 to 68 for the scaling (6.3 TB/s read and written, half of the reading from
// the cache), in double 213 (5.9 TB/s read twice and written); 45 thousand in 12 arrays 11.8 us, where two launches and the host are all there is.
#include <algorithm>
#include <new>
#include <vector>

#include "row_math.h"

namespace dali_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 96;       // arrays per launch: their addresses travel with it (kernel arguments hold 4 KiB); up to kFew of them in a smaller form
constexpr int kFew = 16;
constexpr int kPartials = 2048;  // workgroups of the first launch, as far as one launch goes
constexpr int kMostArrays = 1 << 24;
constexpr int kLeast = 5;        // workgroups of a launch among many
constexpr long kOther = 1 << 20;  // partial sums before the others of their workgroups
static_assert((kMostArrays / kBatch + 1L) * kLeast <= kOther && 3 * kOther * sizeof(double) <= kCarriedBytes, "partial sums of as many launches");
constexpr int kUnroll = 4;       // groups of 16 bytes that a thread has in flight

// The sum of squares of fp32 values, or of doubles: those from 2^501 on times 2^-600, those below 2^-500 times 2^600, and the others, each in a sum of its own. 2^40 of
// them pass no sum's range, and none vanishes in it. (mid, large, small)
template <typename T>
struct Squares {
    static constexpr int SUMS = sizeof(T) == 4 ? 1 : 3;
    double sum[SUMS] = {};
    __device__ __forceinline__ void add(float v) { sum[0] += (double)v * (double)v; }
    __device__ __forceinline__ void add(double v) {
        const unsigned exponent = (unsigned)(__builtin_bit_cast(unsigned long long, v) >> 52) & 0x7ff;
        if (__builtin_expect(exponent - (1023 - 500) <= 1000, 1)) sum[0] += v * v;
        else if (exponent < 1023) sum[2] += (v * 0x1p600) * (v * 0x1p600);  // (zeros too)
        else sum[1] += (v * 0x1p-600) * (v * 0x1p-600);  // (infinities and NaN too)
    }
    __device__ __forceinline__ void join(const Squares& o) {
#pragma unroll
        for (int i = 0; i < SUMS; ++i) sum[i] += o.sum[i];
    }
    __device__ __forceinline__ double norm() const {
        if constexpr (SUMS == 1) {
            return sqrt(sum[0]);
        } else {
            if (ordinary()) return sqrt(sum[0]);
            const double s = sqrt(sum[2]) * 0x1p-600, m = sqrt(sum[0]) * 0x1p-600;
            if (sum[1] != 0) return sqrt(sum[1] + m * m) * 0x1p600;
            return sum[0] == 0 ? s : sqrt(sum[0] + s * s);
        }
    }
    __device__ __forceinline__ bool ordinary() const { return SUMS == 1 || (sum[SUMS > 1 ? 1 : 0] == 0 && sum[SUMS > 1 ? 2 : 0] == 0); }
    // over a workgroup, the same in each of its threads
    template <int THREADS>
    __device__ __forceinline__ void fold(double (&scratch)[THREADS / 64][SUMS]) {
#pragma unroll
        for (int i = 0; i < SUMS; ++i)
            if (i == 0 || __builtin_amdgcn_ballot_w64(sum[i] != 0) != 0) sum[i] = fold_lanes<64>(sum[i], Sum());  // (seldom)
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < SUMS; ++i) scratch[threadIdx.x >> 6][i] = sum[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SUMS; ++i) sum[i] = scratch[0][i];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w)
#pragma unroll
            for (int i = 0; i < SUMS; ++i) sum[i] += scratch[w][i];
    }
};

// What the arrays are multiplied by, in two factors: the first is 1 but where the product of both is below the normal numbers and would lose its digits. (In double: where the norm
// passes the largest float, the scale would lose them in one.) `none`: nothing is scaled.
struct Scale {
    double first = 1, second = 1;
    bool none;
    __device__ __forceinline__ Scale(double norm, double max_norm) : none(!(norm > max_norm && norm < (double)INFINITY)) {
        if (none) return;
        second = max_norm / norm;
        if (second < 0x1p-1000 && max_norm > 0) first = 0x1p-600, second = max_norm / (norm * 0x1p-600);  // (the norm is above 2^-74 then)
    }
    __device__ __forceinline__ float of(float v) const { return (float)((double)v * second); }  // (a second factor below 2^-1000 leaves nothing of a float)
    __device__ __forceinline__ double of(double v) const { return (v * first) * second; }
};

template <int MOST>
struct Batch {
    const void* in[MOST];
    void* out[MOST];
    long n[MOST];
    int first[MOST + 1];  // number of an array's first chunk in this launch
    int arrays, chunk;      // values to a chunk
    double *partial, *other;  // first launch: of its first workgroup (of doubles: their ordinary values; two sums more)
    int partials;           // second launch: all of them
    bool leave;             // second launch: nothing to scale, arrays in their own places stay as they are
    double max_norm;
    void* norm;             // written by the second launch, if this is its first batch (else NULL)
};

// the array that chunk b belongs to
template <int MOST>
__device__ __forceinline__ int array_of(const Batch<MOST>& a, int b) {
    int lo = 0, hi = a.arrays - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.first[mid] <= b) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// the groups of chunk b, four to a thread at a time: f(array, where in it, values, how many of them)
template <typename T, int MOST, typename F>
__device__ __forceinline__ void walk(const Batch<MOST>& a, int b, F f) {
    constexpr int N = Vec<T>::N, STEP = kThreads * N;
    const int i = array_of(a, b);
    if (a.leave && a.in[i] == a.out[i]) return;
    const long begin = (long)(b - a.first[i]) * a.chunk;
    const int count = (int)min((long)a.chunk, a.n[i] - begin);
    const T* x = (const T*)a.in[i] + begin;
    for (int c = threadIdx.x * N; c < count; c += kUnroll * STEP) {
        typename Vec<T>::type g[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) g[u] = ask_group(x, c + u * STEP, count);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            T v[N];
            take_group(g[u], c + u * STEP, count, T(0), v);
            f(i, begin, c + u * STEP, count, v);
        }
    }
}

template <typename T, int MOST>
__global__ __launch_bounds__(kThreads) void squares(Batch<MOST> a) {
    __shared__ double scratch[kThreads / 64][Squares<T>::SUMS];
    Squares<T> part[Vec<T>::N];
    for (int b = blockIdx.x; b < a.first[a.arrays]; b += gridDim.x)
        walk<T>(a, b, [&](int, long, int, int, const T(&v)[Vec<T>::N]) {
#pragma unroll
            for (int k = 0; k < Vec<T>::N; ++k) part[k].add(v[k]);
        });
#pragma unroll
    for (int k = 1; k < Vec<T>::N; ++k) part[0].join(part[k]);
    part[0].template fold<kThreads>(scratch);
    if (threadIdx.x == 0) {
        // (a sum below 0 says that the others are there to be read: a third of the bytes for the next launch, all of whose workgroups read them)
        a.partial[blockIdx.x] = part[0].ordinary() ? part[0].sum[0] : -part[0].sum[0];
        if constexpr (Squares<T>::SUMS > 1) {
            a.other[2 * (long)blockIdx.x] = part[0].sum[1];
            a.other[2 * (long)blockIdx.x + 1] = part[0].sum[2];
        }
    }
}

template <typename T, int MOST, bool PAST>
__global__ __launch_bounds__(kThreads) void rescale(Batch<MOST> a) {
    __shared__ double scratch[kThreads / 64][Squares<T>::SUMS];
    Squares<T> all;
    for (int i = threadIdx.x; i < a.partials; i += kThreads) {
        const double mid = a.partial[i];
        all.sum[0] += fabs(mid);
        if constexpr (Squares<T>::SUMS > 1)
            if (signbit(mid)) all.sum[1] += a.other[2 * (long)i], all.sum[2] += a.other[2 * (long)i + 1];
    }
    all.template fold<kThreads>(scratch);
    const double norm = all.norm();
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *(T*)a.norm = (T)norm;
    const Scale scale(norm, a.max_norm);
    a.leave = scale.none;
    for (int b = a.first[a.arrays] - 1 - (int)blockIdx.x; b >= 0; b -= gridDim.x)
        walk<T>(a, b, [&](int i, long begin, int c, int count, T(&v)[Vec<T>::N]) {
#pragma unroll
            for (int k = 0; k < Vec<T>::N; ++k) v[k] = scale.of(v[k]);
            if (c < count) store_group<PAST>((T*)a.out[i] + begin, c, count, v);
        });
}

// Few values in few arrays: one workgroup takes the norm and scales, in one launch (what it reads for the second time is in its cache). A wave takes units of 64
// groups, four at a time.
constexpr int kFewUnits = 32;  // (8192 fp32 values: 6 us; a compute unit alone moves some 20 GB/s, 45 thousand took 21 us, in two launches 11)
constexpr int kWaves = 16;
struct FewArrays {
    const void* in[kFew];
    void* out[kFew];
    int n[kFew];
    int first[kFew];  // number of an array's first unit; past the arrays: of none
    int units;
};

template <typename T, typename F>
__device__ __forceinline__ void walk_units(const FewArrays& a, F f) {
    constexpr int N = Vec<T>::N;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int unit = wave; unit < a.units; unit += kUnroll * kWaves) {
        typename Vec<T>::type g[kUnroll];
        int array[kUnroll], c[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int at = min(unit + u * kWaves, a.units - 1);  // (past the last unit: that one again, and not used)
            int i = 0;
#pragma unroll
            for (int k = 1; k < kFew; ++k) i += a.first[k] <= at ? 1 : 0;
            array[u] = i;
            c[u] = ((at - a.first[i]) * 64 + lane) * N;
            g[u] = ask_group((const T*)a.in[i], c[u], a.n[i]);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (unit + u * kWaves >= a.units) break;
            const int n = a.n[array[u]];
            T v[N];
            take_group(g[u], c[u], n, T(0), v);
            f(array[u], c[u], n, v);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves) void clip_few(FewArrays a, double max_norm, T* norm) {
    constexpr int N = Vec<T>::N;
    __shared__ double scratch[kWaves][Squares<T>::SUMS];
    Squares<T> all;
    walk_units<T>(a, [&](int, int, int, const T(&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) all.add(v[k]);
    });
    all.template fold<64 * kWaves>(scratch);
    const double length = all.norm();
    if (threadIdx.x == 0) *norm = (T)length;
    const Scale scale(length, max_norm);
    walk_units<T>(a, [&](int i, int c, int n, T(&v)[N]) {
        T* out = (T*)a.out[i];
        if (!out || (scale.none && a.in[i] == out)) return;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = scale.of(v[k]);
        store_group(out, c, n, v);
    });
}

// whether one workgroup takes the arrays, and their places in it
template <typename T>
bool taken_by_one(int count, const void* const* in, void* const* out, const int64_t* sizes, FewArrays* f) {
    constexpr int UNIT = 64 * Vec<T>::N;
    int arrays = 0;
    long units = 0;
    for (int i = 0; i < count; ++i) {
        if (sizes[i] == 0) continue;
        if (arrays == kFew || sizes[i] > (long)kFewUnits * UNIT) return false;
        f->in[arrays] = in[i];
        f->out[arrays] = out ? out[i] : nullptr;
        f->n[arrays] = (int)sizes[i];
        f->first[arrays++] = (int)units;
        units += (sizes[i] + UNIT - 1) / UNIT;
        if (units > kFewUnits) return false;
    }
    for (int k = arrays; k < kFew; ++k) f->first[k] = 0x7fffffff;
    f->units = (int)units;
    return true;
}

template <typename T, int MOST>
int clip_batches(int count, const void* const* in, void* const* out, const int64_t* sizes, double max_norm, T* norm) {
    const char* what = "dali_hip_clip_by_global_norm";
    const Carried carried;
    double *partial = (double*)carried.data(), *other = partial + kOther;
    long total = 0;
    for (int i = 0; i < count; ++i) total += sizes[i];
    constexpr int STEP = kThreads * Vec<T>::N * kUnroll;
    const int chunk = STEP;  // (of two, four, eight steps: 52 million values 103, 105, 113 us, this way 104; 4 million 12.6, 13.8, 18.5 and 13.1; 45 thousand 12.2, 12.6, 13.9 and 11.0)
    const int batches = (count + MOST - 1) / MOST, most = std::max(kPartials / std::max(batches, 1), kLeast);
    Batch<MOST> b;
    b.chunk = chunk;
    b.leave = false;
    b.max_norm = max_norm;
    // (what every launch gives is set in `launch`; a batch that is the only one stays as it is for the second round)
    bool filled = false;
    auto each = [&](auto&& launch) {
        for (int at = 0; at < count;) {
            if (filled && batches == 1) {
                at = count;
            } else {
                b.arrays = 0;
                b.first[0] = 0;
                for (; at < count && b.arrays < MOST; ++at) {
                    if (sizes[at] == 0) continue;
                    b.in[b.arrays] = in[at];
                    b.out[b.arrays] = out ? out[at] : nullptr;
                    b.n[b.arrays] = sizes[at];
                    b.first[b.arrays + 1] = b.first[b.arrays] + (int)((sizes[at] + chunk - 1) / chunk);
                    ++b.arrays;
                }
                filled = true;
            }
            if (!b.arrays) continue;
            launch(b.first[b.arrays]);
            if (launched(what)) return false;  // (and nothing is scaled by a norm that was not formed)
        }
        return true;
    };
    int partials = 0;
    const bool summed = each([&](int chunks) {
        const int blocks = std::min(chunks, most);
        b.partial = partial + partials;
        b.other = other + 2 * partials;
        hipLaunchKernelGGL((squares<T, MOST>), dim3(blocks), dim3(kThreads), 0, stream(), b);
        partials += blocks;
    });
    if (!summed) return DALI_HIP_ERROR;
    b.partial = partial;
    b.other = other;
    b.partials = partials;
    b.norm = norm;
    if (out && !each([&](int chunks) {
            either_way(past_caches(2.0 * sizeof(T) * total),
                       [&](auto p) { hipLaunchKernelGGL((rescale<T, MOST, decltype(p)::value>), dim3(std::min(chunks, 2048)), dim3(kThreads), 0, stream(), b); });
            b.norm = nullptr;
        }))
        return DALI_HIP_ERROR;
    if (b.norm) {  // the norm alone, or nothing to scale
        b.arrays = 0;
        b.first[0] = 0;
        hipLaunchKernelGGL((rescale<T, MOST, false>), dim3(1), dim3(kThreads), 0, stream(), b);
    }
    return launched(what);
}

template <typename T>
int clip(int count, const void* const* in, void* const* out, const int64_t* sizes, double max_norm, T* norm) {
    FewArrays few;
    if (taken_by_one<T>(count, in, out, sizes, &few)) {
        hipLaunchKernelGGL(clip_few<T>, dim3(1), dim3(64 * kWaves), 0, stream(), few, max_norm, norm);
        return launched("dali_hip_clip_by_global_norm");
    }
    if (count <= kFew) return clip_batches<T, kFew>(count, in, out, sizes, max_norm, norm);
    return clip_batches<T, kBatch>(count, in, out, sizes, max_norm, norm);
}

int checked(const char* what, int dtype, int count, const void* const* in, void* const* out, const int64_t* sizes, double max_norm, void* norm) {
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (count < 0 || !norm || (count > 0 && (!in || !sizes))) return fail("%s: NULL argument", what);
    if (out && !(max_norm >= 0)) return fail("%s: the largest norm must not be negative (got %g)", what, max_norm);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    for (int i = 0; i < count; ++i)
        if (sizes[i] < 0 || (sizes[i] > 0 && (!in[i] || (out && !out[i])))) return fail("%s: array %d has no memory or a negative size", what, i);
    // (partial sums: of kPartials workgroups, or of kLeast for every launch of kBatch arrays; chunks are numbered in 31 bits)
    if (count > kMostArrays) return fail("%s: %d arrays are more than there is room for", what, count);
    for (int i = 0; i < count; ++i)
        if (off_elements({in[i], out ? out[i] : nullptr, norm}, size)) return fail("%s: an address is off its type's size", what);
    const Span result("norm", norm, 1, size);
    for (int i = 0; i < count; ++i) {
        const Span a("an array", in[i], sizes[i], size);
        if (a.meets(result)) return fail("%s: the norm overlaps array %d", what, i);
        if (!out) continue;
        const Span o("a result", out[i], sizes[i], size);
        if (o.meets(result)) return fail("%s: the norm overlaps result %d", what, i);
    }
    if (out) {
        // A result may be its own array and must not meet anything else. Results in address order are apart from each other; those that an array
        // meets are then neighbours.
        struct Piece {
            uintptr_t lo, hi;
            int i;
        };
        std::vector<Piece> results;
        results.reserve(count);
        for (int i = 0; i < count; ++i)
            if (sizes[i] > 0) results.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + (uintptr_t)sizes[i] * size, i});
        std::sort(results.begin(), results.end(), [](const Piece& a, const Piece& b) { return a.lo < b.lo; });
        for (size_t j = 1; j < results.size(); ++j)
            if (results[j].lo < results[j - 1].hi) return fail("%s: results %d and %d overlap", what, results[j - 1].i, results[j].i);
        for (int i = 0; i < count; ++i) {
            const uintptr_t lo = (uintptr_t)in[i], hi = lo + (uintptr_t)sizes[i] * size;
            auto r = std::upper_bound(results.begin(), results.end(), lo, [](uintptr_t v, const Piece& p) { return v < p.hi; });
            for (; r != results.end() && r->lo < hi; ++r)
                if (r->i != i || r->lo != lo) return fail("%s: result %d overlaps array %d", what, r->i, i);
        }
    }
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT) return clip<float>(count, in, out, sizes, max_norm, (float*)norm);
    return clip<double>(count, in, out, sizes, max_norm, (double*)norm);
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_clip_by_global_norm(int dtype, int count, const void* const* in, void* const* out, const int64_t* sizes, double max_norm, void* norm) {
    const char* what = "dali_hip_clip_by_global_norm";
    try {
        return checked(what, dtype, count, in, out, sizes, max_norm, norm);
    } catch (const std::bad_alloc&) {  // (the list of results)
        return fail("%s: no host memory for %d arrays", what, count);
    }
}
