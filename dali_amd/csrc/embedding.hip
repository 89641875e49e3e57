// Rows of an embedding table for tokens, scaled, and the gradient of the table. Beyond the reference (its gather has neither scale nor padding).
//
// y[i] = scale table[t_i], zeros where t_i lies outside the table. The gradient is written whole: dtable[r] = scale sum over i with t_i = r of dy[i], in the order of i, zeros
// for rows that no token names.
//
// The tokens are ordered first (stable, so a row's positions stay in their order). Texts name a few tokens very often and most words never, so the work is cut by places of the
// order, not by rows: a wave adds up the rows of dy at 16 to 128 neighbouring places, eight loads under way, and writes the runs that lie within them. A second launch
// joins the parts of longer runs and writes the rows that no token names. What is summed in which order depends on the tokens alone, never on arrival.
//
// Bound by memory. 65536 tokens of 1024 floats: rows 57 us (268 MB written past the caches, 4.7 TB/s); gradient 136: ordering the tokens 14 to 28 in six launches, 84 for reading dy
// (250 MB in the tokens' order, 3.0 TB/s), 31 for the second launch (131 MB written by both). 8 tokens: 3.9 us, the launch. fp64, 3001 tokens into 97 rows of 515: 36 us.
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
// the first of `n` ordered tokens that is not below `key`, sixteen lanes to a key. (Tokens outside the table come out behind the others, negative ones among
// them: read without a sign they are above any row's number.)
__device__ __forceinline__ int lower_bound(const int32_t* keys, int n, unsigned key) {
    const int lane = threadIdx.x & 15, shift = threadIdx.x & 48;
    int lo = 0, hi = n;  // it lies in [lo, hi]
    while (__any(lo < hi)) {
        const int step = (hi - lo + 15) / 16;
        const int at = lo + (lane + 1) * step - 1;
        const unsigned long long below = __ballot(step > 0 && at < hi && (unsigned)keys[min(max(at, 0), n - 1)] < key);
        const int passed = __popcll(below >> shift & 0xffffu);  // so many of the sixteen places are below, the first ones
        if (step > 0) {
            hi = min(hi, lo + (passed + 1) * step - 1);
            lo = min(lo + passed * step, hi);
        }
    }
    return lo;
}

// A wave takes 64 groups of columns of the rows at `chunk` neighbouring places of the order. A run of one token that lies within them is written to its row; what a run that
// goes on before or behind them comes to here is left in partials[chunk][0] (a run that the chunk begins with) or [1].
template <typename T>
__global__ __launch_bounds__(64) void embedding_chunks(const T* dy, int64_t stride, int width, const int32_t* keys, const int32_t* positions, int count, int rows, int chunk,
                                                       int first_chunk, T scale, T* dtable, T* partials) {
    constexpr int N = Vec<T>::N, DEEP = 8;
    const int lane = threadIdx.x, at = first_chunk + blockIdx.x, begin = at * chunk, end = min(begin + chunk, count);
    const int c = (blockIdx.y * 64 + lane) * N;
    T sum[N] = {};
    int run = begin;  // where the run at hand begins
    int token = __builtin_amdgcn_readfirstlane(keys[begin]);
    const bool goes_back = begin > 0 && keys[begin - 1] == token;
    // what the run at hand has come to, up to `to`; it goes on behind the chunk: `on`
    auto leave = [&](int to, bool on) {
        if ((unsigned)token < (unsigned)rows && c < width) {
            const bool part = on || (run == begin && goes_back);
            T* out = part ? partials + ((int64_t)at * 2 + (run == begin ? 0 : 1)) * width : dtable + (int64_t)token * width;
            T v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = part ? sum[e] : sum[e] * scale;
            store_group(out, c, width, v);
        }
        run = to;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0;
    };
    for (int p0 = begin; p0 < end; p0 += 64) {
        const int p = min(p0 + lane, end - 1), key = keys[p], place = positions[p], here = min(64, end - p0);
        // (the runs that begin here: the chunk's first is at hand already)
        const unsigned long long heads = __ballot(p0 + lane < end && p > begin && keys[max(p - 1, 0)] != key);
        for (int i = 0; i < here; i += DEEP) {
            typename Vec<T>::type g[DEEP];
#pragma unroll
            for (int j = 0; j < DEEP; ++j) {
                const int64_t row = __builtin_amdgcn_readlane(place, min(i + j, here - 1));
                if (c < width) g[j] = ask_group(dy + row * stride, c, width);
            }
#pragma unroll
            for (int j = 0; j < DEEP; ++j) {
                if (i + j >= here) break;
                if (heads >> (i + j) & 1) {
                    leave(p0 + i + j, false);
                    token = __builtin_amdgcn_readlane(key, i + j);
                }
                T v[N];
                take_group(g[j], c, width, T(0), v);
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] += v[e];
            }
        }
    }
    leave(end, end < count && keys[end] == token);
}

// What the chunks `first` to `last` of a row's run have come to, in their order, by a wave: columns from c0 on, the next ones `step` further. NARROW: the row has at most 32 groups; as many
// lanes read its groups as it takes, a power of two, and others parts further on, which are handed over in their order (a token of 1550 places in rows of 27: 23 us, so 16).
template <typename T, bool NARROW, bool PAST>
__device__ __forceinline__ void join_run(int width, int chunk, int from, int to, const T* partials, T scale, T* row, int c0, int step) {
    constexpr int N = Vec<T>::N, DEEP = 8;
    const int lane = threadIdx.x & 63, first = from / chunk, last = (to - 1) / chunk;
    const T* head = partials + ((int64_t)first * 2 + (from % chunk ? 1 : 0)) * width;
    int lanes = NARROW ? 1 : 64;
    if (NARROW)
        while (lanes * N < width) lanes *= 2;
    const int teams = 64 / lanes, team = lane / lanes;
    for (int c = c0 + lane % lanes * N; c < width || NARROW; c += step) {
        T sum[N];
        load_group(head, c, width, T(0), sum);
        for (int p = first + 1; p <= last; p += DEEP * teams) {
            typename Vec<T>::type g[DEEP];
#pragma unroll
            for (int j = 0; j < DEEP; ++j) g[j] = ask_group(partials + (int64_t)min(p + j * teams + team, last) * 2 * width, c, width);
#pragma unroll
            for (int j = 0; j < DEEP; ++j) {
                if (p + j * teams > last) break;
                T v[N];
                take_group(g[j], c, width, T(0), v);
                if constexpr (NARROW) {
                    for (int t = 0; t < teams && p + j * teams + t <= last; ++t)
#pragma unroll
                        for (int e = 0; e < N; ++e) sum[e] += __shfl(v[e], t * lanes + lane % lanes);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] += v[e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] *= scale;
        if (team == 0) store_group<PAST>(row, c, width, sum);
        if (NARROW) break;
    }
}

// A workgroup sees to `per` neighbouring rows of the table (at most 15): zeros where no token names one, and the parts of a run that lies in several chunks. A wave takes every fourth 64
// groups of columns, or, NARROW, every fourth row.
template <typename T, bool NARROW, bool PAST>
__global__ __launch_bounds__(256) void embedding_gradient(int width, const int32_t* keys, int count, int rows, int chunk, int first_row, int per, const T* partials, T scale,
                                                          T* dtable) {
    constexpr int N = Vec<T>::N;
    __shared__ int begin[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = first_row + blockIdx.x * per, here = min(per, rows - r0);
    {
        const int i = threadIdx.x / 16, at = lower_bound(keys, count, (unsigned)(r0 + min(i, here)));
        if (threadIdx.x % 16 == 0) begin[i] = at;
    }
    __syncthreads();
    for (int r = NARROW ? wave : 0; r < here; r += NARROW ? 4 : 1) {
        const int from = begin[r], to = begin[r + 1], c0 = NARROW ? 0 : wave * 64 * N;
        T* out = dtable + (int64_t)(r0 + r) * width;
        if (from < to) {
            if (from / chunk != (to - 1) / chunk) join_run<T, NARROW, PAST>(width, chunk, from, to, partials, scale, out, c0, 256 * N);  // (else written already)
            continue;
        }
        const T zeros[N] = {};
        for (int c = c0 + lane * N; c < width; c += (NARROW ? 64 : 256) * N) store_group<PAST>(out, c, width, zeros);
    }
}

// The same for tables most of whose rows no token names: up to 1024 rows or 32 KiB to a workgroup, whose zeros go over them as over one array, in groups on 16 bytes.
constexpr int kMostRowsEach = 1024, kBytesEach = 32768;

template <typename T, bool NARROW>
__global__ __launch_bounds__(256) void embedding_gradient_sparse(int width, unsigned width_m, int width_s, const int32_t* keys, int count, int rows, int chunk, int first_row, int per,
                                                                 const T* partials, T scale, T* dtable) {
    constexpr int N = Vec<T>::N;
    __shared__ int begin[kMostRowsEach + 1];
    __shared__ int ends[2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = first_row + blockIdx.x * per, here = min(per, rows - r0);
    if (wave == 0) {
        const int at = lower_bound(keys, count, (unsigned)(r0 + (lane < 16 ? 0 : here)));
        if (lane == 0 || lane == 16) ends[lane / 16] = at;
    }
    __syncthreads();
    const int low = ends[0], high = ends[1];
    T* out = dtable + (int64_t)r0 * width;
    const int n = here * width;                                                                        // (of many rows at most kBytesEach, else a row's width)
    const int head = (int)((16 - (uintptr_t)out % 16) % 16 / sizeof(T)), start = head ? head - N : 0;  // (the first group may begin before the rows)
    typedef T aligned_group __attribute__((ext_vector_type(N)));
    const auto zeros = [&](int64_t e) { *reinterpret_cast<aligned_group*>(out + e) = aligned_group{}; };
    if (low == high) {  // no token of these rows
        for (int64_t e = start + (int)threadIdx.x * N; e < n; e += 256 * N) {
            if (e >= 0 && e + N <= n) {
                zeros(e);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (e + i >= 0 && e + i < n) out[e + i] = T(0);
            }
        }
        return;
    }
    for (int i = threadIdx.x; i <= here; i += 256) {
        int lo = low, hi = high;
        while (lo < hi) {
            const int mid = lo + (hi - lo) / 2;
            if ((unsigned)keys[mid] < (unsigned)(r0 + i)) lo = mid + 1;
            else hi = mid;
        }
        begin[i] = lo;
    }
    __syncthreads();
    for (int64_t e = start + (int)threadIdx.x * N; e < n; e += 256 * N) {
        const int a = (int)max(e, (int64_t)0), b = (int)min(e + N, (int64_t)n) - 1;
        int r = (int)sgemm_row_map_div((unsigned)a, width_m, width_s);
        const bool one = r == (int)sgemm_row_map_div((unsigned)b, width_m, width_s);
        if (one && begin[r] != begin[r + 1]) continue;
        if (one && e >= 0 && e + N <= n) {
            zeros(e);
            continue;
        }
        int64_t end = (int64_t)(r + 1) * width;  // of row r
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t x = e + i;
            if (x < a || x > b) continue;
            while (x >= end) ++r, end += width;
            if (begin[r] == begin[r + 1]) out[x] = T(0);
        }
    }
    for (int base = 0, k = 0; base < here; base += 64) {
        const int mine = base + lane;
        unsigned long long rest = __ballot(mine < here && begin[min(mine, here - 1)] < begin[min(mine, here - 1) + 1] &&
                                           begin[min(mine, here - 1)] / chunk != (begin[min(mine, here - 1) + 1] - 1) / chunk);
        for (; rest; rest &= rest - 1, ++k) {
            const int r = base + __ffsll((long long)rest) - 1;
            if (!NARROW || (k & 3) == wave)
                join_run<T, NARROW, false>(width, chunk, begin[r], begin[r + 1], partials, scale, out + (int64_t)r * width, NARROW ? 0 : wave * 64 * N, 256 * N);
        }
    }
}

// Places of the order that a wave of the first launch takes: enough chunks to fill the chip, few enough parts of a frequent token
int chunk_of(int64_t count) {
    int chunk = 16;
    while (chunk < 128 && count / chunk > 1024) chunk *= 2;
    return chunk;
}

// what the gradient keeps beside its operands: ordered tokens, their positions, room for ordering them, and the parts of runs
struct GradientSpace {
    size_t keys, positions, order, partials, bytes;
    GradientSpace(int64_t count, int width, size_t size) {
        const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
        keys = 0;
        positions = round((size_t)count * 4);
        order = 2 * positions;
        partials = order + round(argsort_scratch_bytes(count));
        const int chunk = chunk_of(count);
        bytes = partials + 2 * (size_t)((count + chunk - 1) / chunk) * width * size;
    }
};

template <typename T>
int embedding_backward(int64_t count, int rows, int width, const T* dy, int64_t stride, const int32_t* tokens, double scale, T* dtable, char* space) {
    const char* what = "dali_hip_embedding_backward";
    const GradientSpace s(count, width, sizeof(T));
    int32_t *keys = (int32_t*)(space + s.keys), *positions = (int32_t*)(space + s.positions);
    T* partials = (T*)(space + s.partials);
    if (count && argsort_with(tokens, count, rows, keys, positions, space + s.order)) return DALI_HIP_ERROR;
    const int chunk = chunk_of(count), chunks = (int)((count + chunk - 1) / chunk), most = 1 << 23;  // workgroups along an axis of a launch, which has fewer than 2^32 threads
    const int across = (groups_of<T>(width) + 63) / 64;
    if (across > 65535) return fail("%s: rows of %d values are too wide", what, width);
    for (int first = 0; first < chunks; first += most) {
        embedding_chunks<T><<<dim3((unsigned)std::min(chunks - first, most), (unsigned)across), dim3(64), 0, stream()>>>(dy, stride, width, keys, positions, (int)count, rows, chunk,
                                                                                                                 first, (T)scale, dtable, partials);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    // A large table of which few rows are named is zeros for the most part: [44681,2199] for 34 tokens 134 us row by row, 90 (zeros alone 73), [119465,128] for one 59 and 20. Where the
    // named rows are more, the first launch has brought much of the table into the caches, and rows past them row by row are quicker ([43264,1344] fp64 for 5312 tokens 129 us, 150);
    // short rows gain as long as there are more of them than tokens ([79168,10] for 20084: 76, 47).
    const bool narrow = width <= 32 * Vec<T>::N, past = past_caches((double)rows * width * sizeof(T));
    const bool sparse = (rows >= 16384 || past) && (rows >= 16 * count || (narrow && rows > count));
    const int per = sparse ? std::max(1, std::min({(int)(kBytesEach / sizeof(T) / width), kMostRowsEach, rows / 1024})) : std::max(1, std::min(15, rows / 2048));
    int shift = 0;
    while (((int64_t)1 << shift) < width) ++shift;
    const unsigned times = (unsigned)((((uint64_t)1 << (31 + shift)) + width - 1) / width);  // (of an exact division by the width)
    for (int64_t first = 0; first < rows; first += (int64_t)most * per) {
        const dim3 grid((unsigned)std::min((rows - first + per - 1) / per, (int64_t)most));
        either_way(narrow, [&](auto n) {
            constexpr bool NARROW = decltype(n)::value;
            if (sparse)
                embedding_gradient_sparse<T, NARROW><<<grid, dim3(256), 0, stream()>>>(width, times, shift, keys, (int)count, rows, chunk, (int)first, per, partials, (T)scale, dtable);
            else
                either_way(past, [&](auto p) {
                    embedding_gradient<T, NARROW, decltype(p)::value><<<grid, dim3(256), 0, stream()>>>(width, keys, (int)count, rows, chunk, (int)first, per, partials, (T)scale, dtable);
                });
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
    if (!holds_scale(dtype, scale)) return fail("%s: the scale must be finite in its operands' type (got %g)", what, scale);
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
