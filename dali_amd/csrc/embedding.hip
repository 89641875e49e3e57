// Rows of an embedding table for tokens, scaled, and the gradient of the table. Beyond the reference (its gather has neither scale nor padding).
//
// y[i] = scale table[t_i], zeros where t_i lies outside the table. The gradient is written whole: dtable[r] = scale sum over i with t_i = r of dy[i], in the order
// of i, zeros for rows that no token names. The tokens are ordered first (stable, so a row's positions stay in their order), and a workgroup that owns
// neighbouring rows of the table finds where their runs begin by looking at 64 places of the ordered tokens at a time.
//
// Texts name a few tokens very often: positions that lie in a block of kChunk ordered tokens that are all the same are summed by a launch of their own before, so that a
// row's owner adds at most 2 (kChunk - 1) positions and the sums of whole blocks. What is summed in which order depends on the tokens alone, never on arrival.
#include <algorithm>
#include <cmath>

#include "row_math.h"

namespace dali_hip {
namespace {

// ------------------------------------------------------------------------------------------------ rows of tokens
// A team of LANES lanes copies a row: as many 16-byte groups at a time as it has lanes, four under way at once.
template <typename T, int LANES, bool PAST>
__global__ __launch_bounds__(256) void embedding_rows(const T* table, int64_t stride, int rows, int width, const int32_t* tokens, int64_t first, int64_t count, T scale, T* y) {
    constexpr int N = Vec<T>::N;
    const int64_t i = first + (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (i >= count) return;
    const int lane = threadIdx.x % LANES, token = tokens[i];
    T* out = y + i * width;
    if (token < 0 || token >= rows) {
        const T zeros[N] = {};
        for (int c = lane * N; c < width; c += LANES * N) store_group<PAST>(out, c, width, zeros);
        return;
    }
    const T* row = table + token * stride;
    for (int c = lane * N; c < width; c += 4 * LANES * N) {
        typename Vec<T>::type g[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j * LANES * N < width) g[j] = ask_group(row, c + j * LANES * N, width);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = c + j * LANES * N;
            if (at >= width) break;
            T v[N];
            take_group(g[j], at, width, T(0), v);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] *= scale;
            store_group<PAST>(out, at, width, v);
        }
    }
}

template <typename T>
int embedding(int64_t count, int rows, int width, const T* table, int64_t stride, const int32_t* tokens, double scale, T* y) {
    const int groups = groups_of<T>(width);
    const bool past = past_caches((double)count * width * sizeof(T));
    auto launch = [&](auto lanes, auto p) {
        constexpr int LANES = decltype(lanes)::value, PER = 256 / LANES;
        const int64_t most = (int64_t)1 << 23;  // workgroups of one launch, which has fewer than 2^32 threads
        for (int64_t first = 0; first < count; first += most * PER) {
            const int64_t blocks = std::min((count - first + PER - 1) / PER, most);
            embedding_rows<T, LANES, decltype(p)::value><<<dim3((unsigned)blocks), dim3(256), 0, stream()>>>(table, stride, rows, width, tokens, first, count, (T)scale, y);
            if (launched("dali_hip_embedding")) return DALI_HIP_ERROR;
        }
        return DALI_HIP_OK;
    };
    int status = DALI_HIP_OK;
    either_way(past, [&](auto p) {
        status = groups <= 8 ? launch(std::integral_constant<int, 8>(), p) : groups <= 32 ? launch(std::integral_constant<int, 32>(), p) : launch(std::integral_constant<int, 64>(), p);
    });
    return status;
}

// ------------------------------------------------------------------------------------------------ the gradient of the table
constexpr int kChunk = 64;

// The first of `n` ordered tokens that is not below `key`; all lanes of the wave take part. (Tokens outside the table come out behind the others, negative ones
// among them: read without a sign they are above any row's number.)
__device__ __forceinline__ int lower_bound(const int32_t* keys, int n, unsigned key) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;  // it lies in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;  // (at least one)
        const int at = lo + (lane + 1) * step - 1;
        const unsigned long long below = __ballot(at < hi && (unsigned)keys[min(at, n - 1)] < key);
        const int passed = __popcll(below);  // so many of the 64 places are below, the first ones
        hi = min(hi, lo + (passed + 1) * step - 1);
        lo = min(lo + passed * step, hi);
    }
    return lo;
}

// adds rows of dy to N sums of a lane, eight loads at a time; `place(p)` is the row at position p
template <bool LONG, typename T, typename Place>
__device__ __forceinline__ void add_rows(T (&sum)[Vec<T>::N], const T* from, int64_t stride, int c, int width, int begin, int end, Place place) {
    constexpr int N = Vec<T>::N;
    constexpr int DEEP = 8;
    int p = begin;
    for (; p + DEEP <= end; p += DEEP) {
        typename Vec<T>::type g[DEEP];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) g[j] = ask_group<LONG>(from + place(p + j) * stride, c, width);
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            T v[N];
            take_group<LONG>(g[j], c, width, T(0), v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += v[e];
        }
    }
    for (; p < end; ++p) {
        T v[N];
        load_group(from + place(p) * stride, c, width, T(0), v);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[e];
    }
}

// The sums of blocks of kChunk ordered tokens that are all the same: a wave takes 64 groups of columns of one.
template <typename T>
__global__ __launch_bounds__(256) void embedding_chunks(const T* dy, int64_t stride, int width, const int32_t* keys, const int32_t* positions, int rows, int first_chunk, T* partials) {
    constexpr int N = Vec<T>::N;
    const int chunk = first_chunk + blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t* k = keys + (int64_t)chunk * kChunk;
    const int first = k[0];
    if (first != k[kChunk - 1] || first < 0 || first >= rows) return;
    const int32_t* at = positions + (int64_t)chunk * kChunk;
    for (int c = (wave * 64 + lane) * N; c < width; c += 256 * N) {
        T sum[N] = {};
        add_rows<false>(sum, dy, stride, c, width, 0, kChunk, [&](int p) { return (int64_t)at[p]; });
        store_group(partials + (int64_t)chunk * width, c, width, sum);
    }
}

// A workgroup writes `per` neighbouring rows of the table (at most 16), its waves each a quarter of the columns.
template <typename T, bool PAST>
__global__ __launch_bounds__(256) void embedding_gradient(const T* dy, int64_t stride, int width, const int32_t* keys, const int32_t* positions, int count, int rows, int first_row,
                                                          int per, const T* partials, T scale, T* dtable) {
    constexpr int N = Vec<T>::N;
    __shared__ int begin[17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = first_row + blockIdx.x * per, here = min(per, rows - r0);
    for (int i = wave; i <= here; i += 4) {
        const int at = lower_bound(keys, count, (unsigned)(r0 + i));
        if (lane == 0) begin[i] = at;
    }
    __syncthreads();
    for (int r = 0; r < here; ++r) {
        const int from = begin[r], to = begin[r + 1];
        // whole blocks of this row's positions: [whole, whole_end) kChunk
        const int whole = (from + kChunk - 1) / kChunk, whole_end = to / kChunk;
        T* out = dtable + (int64_t)(r0 + r) * width;
        for (int c = (wave * 64 + lane) * N; c < width; c += 256 * N) {
            T sum[N] = {};
            const auto place = [&](int p) { return (int64_t)positions[p]; };
            if (whole < whole_end) {
                add_rows<false>(sum, dy, stride, c, width, from, whole * kChunk, place);
                add_rows<false>(sum, partials, (int64_t)width, c, width, whole, whole_end, [](int p) { return (int64_t)p; });
                add_rows<false>(sum, dy, stride, c, width, whole_end * kChunk, to, place);
            } else {
                add_rows<false>(sum, dy, stride, c, width, from, to, place);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] *= scale;
            store_group<PAST>(out, c, width, sum);
        }
    }
}

// what the gradient keeps beside its operands: ordered tokens, their positions, room for ordering them, and the sums of whole blocks
struct GradientSpace {
    size_t keys, positions, order, partials, bytes;
    GradientSpace(int64_t count, int width, size_t size) {
        const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
        keys = 0;
        positions = round((size_t)count * 4);
        order = 2 * positions;
        partials = order + round(argsort_scratch_bytes(count));
        bytes = partials + (size_t)(count / kChunk) * width * size;
    }
};

template <typename T>
int embedding_backward(int64_t count, int rows, int width, const T* dy, int64_t stride, const int32_t* tokens, double scale, T* dtable, char* space) {
    const char* what = "dali_hip_embedding_backward";
    const GradientSpace s(count, width, sizeof(T));
    int32_t *keys = (int32_t*)(space + s.keys), *positions = (int32_t*)(space + s.positions);
    T* partials = (T*)(space + s.partials);
    if (count && argsort_with(tokens, count, rows, keys, positions, space + s.order)) return DALI_HIP_ERROR;
    const int chunks = (int)(count / kChunk), most = 1 << 23;  // workgroups of one launch, which has fewer than 2^32 threads
    for (int first = 0; first < chunks; first += most) {
        embedding_chunks<T><<<dim3((unsigned)std::min(chunks - first, most)), dim3(256), 0, stream()>>>(dy, stride, width, keys, positions, rows, first, partials);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    const int per = std::max(1, std::min(16, rows / 2048));
    const bool past = past_caches((double)rows * width * sizeof(T));
    for (int64_t first = 0; first < rows; first += (int64_t)most * per) {
        const int64_t blocks = std::min((rows - first + per - 1) / per, (int64_t)most);
        either_way(past, [&](auto p) {
            embedding_gradient<T, decltype(p)::value>
                <<<dim3((unsigned)blocks), dim3(256), 0, stream()>>>(dy, stride, width, keys, positions, (int)count, rows, (int)first, per, partials, (T)scale, dtable);
        });
        if (launched(what)) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
}

int check_embedding(const char* what, int dtype, int64_t count, int rows, int width, double scale) {
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (count < 0 || count > 2147483647LL - 256) return fail("%s: %lld tokens", what, (long long)count);
    if (rows < 1) return fail("%s: a table of %d rows", what, rows);
    if (width < 1) return fail("%s: rows of %d values", what, width);
    if (!std::isfinite(scale)) return fail("%s: the scale must be finite (got %g)", what, scale);
    return DALI_HIP_OK;
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_embedding(int dtype, int64_t count, int rows, int width, const void* table, int64_t stride, const int32_t* tokens, double scale, void* y) {
    const char* what = "dali_hip_embedding";
    if (check_embedding(what, dtype, count, rows, width, scale)) return DALI_HIP_ERROR;
    if (count == 0) return DALI_HIP_OK;
    if (!table || !tokens || !y) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (off_elements({table, y}, size) || off_elements({tokens}, 4)) return fail("%s: an address is off its type's size", what);
    if (check_spans(what, {Span("y", y, count * width, size)}, {Span("table", table, rows, width, stride, size), Span("tokens", tokens, count, 4)}, 0)) return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    return dtype == DALI_HIP_FLOAT ? embedding(count, rows, width, (const float*)table, stride, tokens, scale, (float*)y)
                                   : embedding(count, rows, width, (const double*)table, stride, tokens, scale, (double*)y);
}

extern "C" int dali_hip_embedding_backward_workspace(int dtype, int64_t count, int rows, int width, size_t* bytes) {
    const char* what = "dali_hip_embedding_backward_workspace";
    if (check_embedding(what, dtype, count, rows, width, 1.0)) return DALI_HIP_ERROR;
    if (!bytes) return fail("%s: NULL argument", what);
    *bytes = GradientSpace(count, width, dtype == DALI_HIP_FLOAT ? 4 : 8).bytes;
    return DALI_HIP_OK;
}

extern "C" int dali_hip_embedding_backward(int dtype, int64_t count, int rows, int width, const void* dy, int64_t stride, const int32_t* tokens, double scale, void* dtable,
                                           void* workspace) {
    const char* what = "dali_hip_embedding_backward";
    if (check_embedding(what, dtype, count, rows, width, scale)) return DALI_HIP_ERROR;
    if (!dtable || (count && (!dy || !tokens || !workspace))) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (off_elements({dy, dtable}, size) || off_elements({tokens}, 4)) return fail("%s: an address is off its type's size", what);
    if (count && (uintptr_t)workspace % 256 != 0) return fail("%s: the workspace must lie on 256 bytes", what);
    const Span space("the workspace", count ? workspace : nullptr, (int64_t)GradientSpace(count, width, size).bytes, 1);
    if (check_spans(what, {Span("dtable", dtable, (int64_t)rows * width, size), space}, {Span("dy", dy, count, width, stride, size), Span("tokens", tokens, count, 4)}, 0))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    return dtype == DALI_HIP_FLOAT ? embedding_backward(count, rows, width, (const float*)dy, stride, tokens, scale, (float*)dtable, (char*)workspace)
                                   : embedding_backward(count, rows, width, (const double*)dy, stride, tokens, scale, (double*)dtable, (char*)workspace);
}
