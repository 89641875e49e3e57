// The norm over all values of many arrays, and the arrays scaled so that it is at most a given one.
//
//   norm = sqrt(sum over all arrays of sum of squares),  scale = max_norm / norm where norm > max_norm, else 1
//
// Squares are summed in double (an fp32 value's square neither overflows nor vanishes there). Every workgroup sums one chunk and leaves one
// partial; one workgroup folds the partials in the order of the chunks, so the norm does not depend on scheduling. A norm that is not finite
// scales nothing: the arrays come back as they are and the norm says so.
#include <algorithm>
#include <vector>

#include "row_math.h"

namespace dali_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 96;  // arrays per launch: their addresses travel with it (kernel arguments hold 4 KiB)

struct Batch {
    const void* in[kBatch];
    void* out[kBatch];
    long n[kBatch];
    int first[kBatch + 1];  // number of an array's first chunk in this launch
    int arrays;
    long chunk;
    double* partial;  // of this launch's first chunk
    double* result;   // {scale}
};

// the array that chunk b belongs to
__device__ __forceinline__ int array_of(const Batch& a, int b) {
    int lo = 0, hi = a.arrays - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.first[mid] <= b) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void squares(Batch a) {
    __shared__ double scratch[kThreads / 64];
    const int i = array_of(a, blockIdx.x);
    const long begin = (blockIdx.x - a.first[i]) * a.chunk, end = min(begin + a.chunk, a.n[i]);
    const T* x = (const T*)a.in[i];
    double s = 0;
    for (long c = begin + threadIdx.x; c < end; c += kThreads) s += (double)x[c] * (double)x[c];
    s = block_sum<kThreads>(s, scratch);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void fold(const double* partial, int count, double max_norm, T* norm, double* scale) {
    __shared__ double scratch[kThreads / 64];
    double s = 0;
    for (int i = threadIdx.x; i < count; i += kThreads) s += partial[i];
    s = sqrt(block_sum<kThreads>(s, scratch));
    if (threadIdx.x == 0) {
        *norm = (T)s;
        *scale = s > max_norm && s < (double)INFINITY ? max_norm / s : 1.0;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void rescale(Batch a) {
    const int i = array_of(a, blockIdx.x);
    const long begin = (blockIdx.x - a.first[i]) * a.chunk, end = min(begin + a.chunk, a.n[i]);
    const T* x = (const T*)a.in[i];
    T* y = (T*)a.out[i];
    // (in double: where the norm passes the largest float, the scale would lose its digits in one)
    const double scale = *a.result;
    for (long c = begin + threadIdx.x; c < end; c += kThreads) y[c] = (T)((double)x[c] * scale);
}

template <typename T>
int clip(int count, const void* const* in, void* const* out, const int64_t* sizes, double max_norm, T* norm) {
    long total = 0;
    for (int i = 0; i < count; ++i) total += sizes[i];
    const long chunk = std::max(1024L, (total / 4096 + 1023) / 1024 * 1024);
    double* partial = (double*)(workspace() + kWorkspaceCounterBytes);
    double* scale = partial;
    ++partial;
    int done = 0;
    auto batches = [&](auto&& launch) {
        done = 0;
        for (int at = 0; at < count;) {
            Batch b;
            b.arrays = 0;
            b.first[0] = 0;
            for (; at < count && b.arrays < kBatch; ++at) {
                if (sizes[at] == 0) continue;
                b.in[b.arrays] = in[at];
                b.out[b.arrays] = out ? out[at] : nullptr;
                b.n[b.arrays] = sizes[at];
                b.first[b.arrays + 1] = b.first[b.arrays] + (int)((sizes[at] + chunk - 1) / chunk);
                ++b.arrays;
            }
            if (b.arrays == 0) continue;
            b.chunk = chunk;
            b.partial = partial + done;
            b.result = scale;
            launch(b, b.first[b.arrays]);
            done += b.first[b.arrays];
        }
    };
    batches([&](const Batch& b, int blocks) { hipLaunchKernelGGL(squares<T>, dim3(blocks), dim3(kThreads), 0, stream(), b); });
    hipLaunchKernelGGL(fold<T>, dim3(1), dim3(kThreads), 0, stream(), partial, done, max_norm, norm, scale);
    if (out) batches([&](const Batch& b, int blocks) { hipLaunchKernelGGL(rescale<T>, dim3(blocks), dim3(kThreads), 0, stream(), b); });
    return launched("dali_hip_clip_by_global_norm");
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
    // (one partial per chunk: at most 4096, and one more for each array)
    if (((size_t)count + 4096 + 2) * sizeof(double) > kWorkspacePartialBytes) return fail("%s: %d arrays are more than the workspace has room for", what, count);
    if (ensure_init()) return DALI_HIP_ERROR;
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
    if (dtype == DALI_HIP_FLOAT) return clip<float>(count, in, out, sizes, max_norm, (float*)norm);
    return clip<double>(count, in, out, sizes, max_norm, (double*)norm);
}
