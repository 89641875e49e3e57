// The norm over all values of many arrays, and the arrays scaled so that it is at most a given one.
//
//   norm = sqrt(sum over all arrays of sum of squares),  scale = max_norm / norm where norm > max_norm, else 1
//
// Squares are summed in double (an fp32 value's square neither overflows nor vanishes there). A workgroup sums the chunks that fall to it and leaves one
// partial; every workgroup of the second launch folds all partials in the same order before it scales, so the norm does not depend on scheduling and needs no
// launch of its own. (The partials lie where no other kernel writes until the second launch has been issued: Carried, runtime.h.) The second launch walks the chunks backwards: what the first read last is still in the cache. A norm that is not finite
// scales nothing: the arrays come back as they are and the norm says so, and arrays that are their own destinations are left alone whenever nothing is scaled.
// Bound by memory: 52 million fp32 values in 24 arrays 103 us, 38 for the norm (5.4 TB/s) and 64 to 68 for the scaling (6.3 TB/s read and written, half of the reading from
// the cache); 45 thousand in 12 arrays 11 us, where two launches and the host are all there is.
#include <algorithm>
#include <vector>

#include "row_math.h"

namespace dali_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 96;       // arrays per launch: their addresses travel with it (kernel arguments hold 4 KiB); up to kFew of them in a smaller form
constexpr int kFew = 16;
constexpr int kPartials = 2048;  // workgroups of the first launch, as far as one launch goes
constexpr int kMostArrays = 1 << 24;
static_assert((kMostArrays / kBatch + 1L) * 16 * sizeof(double) <= kCarriedBytes, "partial sums of as many launches");
constexpr int kUnroll = 4;       // groups of 16 bytes that a thread has in flight

template <int MOST>
struct Batch {
    const void* in[MOST];
    void* out[MOST];
    long n[MOST];
    int first[MOST + 1];  // number of an array's first chunk in this launch
    int arrays, chunk;      // values to a chunk
    double* partial;        // first launch: of its first workgroup
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
    __shared__ double scratch[kThreads / 64];
    double part[Vec<T>::N] = {};
    for (int b = blockIdx.x; b < a.first[a.arrays]; b += gridDim.x)
        walk<T>(a, b, [&](int, long, int, int, const T(&v)[Vec<T>::N]) {
#pragma unroll
            for (int k = 0; k < Vec<T>::N; ++k) part[k] += (double)v[k] * (double)v[k];
        });
    double s = part[0];
#pragma unroll
    for (int k = 1; k < Vec<T>::N; ++k) s += part[k];
    s = block_sum<kThreads>(s, scratch);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

template <typename T, int MOST, bool PAST>
__global__ __launch_bounds__(kThreads) void rescale(Batch<MOST> a) {
    __shared__ double scratch[kThreads / 64];
    double s = 0;
    for (int i = threadIdx.x; i < a.partials; i += kThreads) s += a.partial[i];
    s = sqrt(block_sum<kThreads>(s, scratch));
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *(T*)a.norm = (T)s;
    // (in double: where the norm passes the largest float, the scale would lose its digits in one)
    const double scale = s > a.max_norm && s < (double)INFINITY ? a.max_norm / s : 1.0;
    a.leave = scale == 1.0;
    for (int b = a.first[a.arrays] - 1 - (int)blockIdx.x; b >= 0; b -= gridDim.x)
        walk<T>(a, b, [&](int i, long begin, int c, int count, T(&v)[Vec<T>::N]) {
#pragma unroll
            for (int k = 0; k < Vec<T>::N; ++k) v[k] = (T)((double)v[k] * scale);
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
    __shared__ double scratch[kWaves];
    double s = 0;
    walk_units<T>(a, [&](int, int, int, const T(&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) s += (double)v[k] * (double)v[k];
    });
    s = sqrt(block_sum<64 * kWaves>(s, scratch));
    if (threadIdx.x == 0) *norm = (T)s;
    const double scale = s > max_norm && s < (double)INFINITY ? max_norm / s : 1.0;
    walk_units<T>(a, [&](int i, int c, int n, T(&v)[N]) {
        T* out = (T*)a.out[i];
        if (!out || (scale == 1.0 && a.in[i] == out)) return;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (T)((double)v[k] * scale);
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
    const Carried carried;
    double* partial = (double*)carried.data();
    long total = 0;
    for (int i = 0; i < count; ++i) total += sizes[i];
    constexpr int STEP = kThreads * Vec<T>::N * kUnroll;
    const int chunk = STEP;  // (of two, four, eight steps: 52 million values 103, 105, 113 us, this way 104; 4 million 12.6, 13.8, 18.5 and 13.1; 45 thousand 12.2, 12.6, 13.9 and 11.0)
    const int batches = (count + MOST - 1) / MOST, most = std::max(kPartials / std::max(batches, 1), 16);
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
            if (b.arrays) launch(b.first[b.arrays]);
        }
    };
    int partials = 0;
    each([&](int chunks) {
        const int blocks = std::min(chunks, most);
        b.partial = partial + partials;
        hipLaunchKernelGGL((squares<T, MOST>), dim3(blocks), dim3(kThreads), 0, stream(), b);
        partials += blocks;
    });
    b.partial = partial;
    b.partials = partials;
    b.norm = norm;
    if (out)
        each([&](int chunks) {
            either_way(past_caches(2.0 * sizeof(T) * total),
                       [&](auto p) { hipLaunchKernelGGL((rescale<T, MOST, decltype(p)::value>), dim3(std::min(chunks, 2048)), dim3(kThreads), 0, stream(), b); });
            b.norm = nullptr;
        });
    if (b.norm) {  // the norm alone, or nothing to scale
        b.arrays = 0;
        b.first[0] = 0;
        hipLaunchKernelGGL((rescale<T, MOST, false>), dim3(1), dim3(kThreads), 0, stream(), b);
    }
    return launched("dali_hip_clip_by_global_norm");
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

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_clip_by_global_norm(int dtype, int count, const void* const* in, void* const* out, const int64_t* sizes, double max_norm, void* norm) {
    const char* what = "dali_hip_clip_by_global_norm";
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (count < 0 || !norm || (count > 0 && (!in || !sizes))) return fail("%s: NULL argument", what);
    if (out && !(max_norm >= 0)) return fail("%s: the largest norm must not be negative (got %g)", what, max_norm);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    for (int i = 0; i < count; ++i)
        if (sizes[i] < 0 || (sizes[i] > 0 && (!in[i] || (out && !out[i])))) return fail("%s: array %d has no memory or a negative size", what, i);
    // (partial sums: kPartials, or 16 for every launch of kBatch arrays; chunks are numbered in 31 bits)
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
