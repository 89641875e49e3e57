// Softmax cross entropy of rows against a large vocabulary, from the hidden states and the projection, and its gradients: the logits are never kept. Beyond the reference
// (its softmax_cross_entropy takes logits).
//
// l = x w + bias; lse = m + ln S with the maximum m and S = sum e^(l - m); loss = (m - l_target) + ln S. The gradient of the logits is g = d (e^(l - lse) - [target]),
// from which dx = g w^T, dw = x^T g, dbias = sum over the rows of g.
//
// Many rows in fp32 go by products of matrices that are cut beforehand, with the softmax at their ends (further below). Else the vocabulary is taken in pieces, the rows in
// blocks, so that a piece of logits holds at most kPieceBytes and stays in the 256 MiB cache between the product that
// writes it and the kernel that reads it. Forward, every kSegment columns of a row leave a maximum and a sum of weights relative to it, and a last launch joins a
// row's (up to 1024 rows: the last workgroup of a row does). Backward, the piece is formed again and becomes g in its place; the products add it up in the order of pieces and
// blocks. Bound by the products: [8,1024].[1024,50257] 47.5 us, of which 41 read w; fp64 gradients of [301,515].[515,10007] 283, nearly all of it three products.
#include <algorithm>
#include <cmath>

#include "product_of_pieces.h"
#include "row_math.h"

namespace dali_hip {
namespace {

template <typename T>
struct Exponent;
template <>
struct Exponent<float> {
    static constexpr float lowest = -3.402823466e+38f;  // where a running maximum begins: finite, so that no difference to it is NaN
    static __device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }
    static __device__ __forceinline__ float ln(float s) { return logf(s); }
};
template <>
struct Exponent<double> {
    static constexpr double lowest = -1.7976931348623157e+308;
    static __device__ __forceinline__ double weight(double d) { return exp(d); }
    static __device__ __forceinline__ double ln(double s) { return log(s); }
};

constexpr int kGroupsEach = 4;  // of a lane, in a segment
template <typename T>
constexpr int kSegment = 64 * kGroupsEach * Vec<T>::N;  // 1024 floats, 512 doubles
constexpr int kChunkRows = 64;                          // that a workgroup of the gradient adds up for the bias, at most
constexpr size_t kPieceBytes = (size_t)128 << 20;
constexpr int kMostRows = 16384;
constexpr int kJoinRows = 1024;                         // up to which a row's segments are joined by the launch that forms them (with more that launch fills the chip)

// row-major C[m, n] = op(A) op(B) + beta C
int product(bool ta, bool tb, int m, int n, int k, const float* a, int lda, const float* b, int ldb, float beta, float* c, int ldc) {
    return dali_hip_sgemm(tb, ta, n, m, k, 1.0f, b, ldb, a, lda, beta, c, ldc);
}
int product(bool ta, bool tb, int m, int n, int k, const double* a, int lda, const double* b, int ldb, double beta, double* c, int ldc) {
    return dali_hip_dgemm(tb, ta, n, m, k, 1.0, b, ldb, a, lda, beta, c, ldc);
}
// The same where C may have few tiles and a long inner extent: the fp32 kernels cut that by themselves, the fp64 kernel into parts that lie in `parts` ([301, 10007] .
// [10007, 515] 600 us uncut)
size_t cut_bytes(float, int, int, int) { return 0; }
size_t cut_bytes(double, int m, int n, int k) { return dgemm_shares_bytes(m, n, k); }
int cut_product(bool ta, bool tb, int m, int n, int k, const float* a, int lda, const float* b, int ldb, float beta, float* c, int ldc, void*) {
    return product(ta, tb, m, n, k, a, lda, b, ldb, beta, c, ldc);
}
int cut_product(bool ta, bool tb, int m, int n, int k, const double* a, int lda, const double* b, int ldb, double beta, double* c, int ldc, void* parts) {
    return dgemm_shares(ta, tb, m, n, k, a, lda, b, ldb, beta, c, ldc, parts);
}

// How a call is cut, and what it keeps beside its operands
template <typename T>
struct Cut {
    int64_t rows;
    int inputs, vocab, block, piece, segments, chunk, chunks;
    size_t logits = 0, maxima, sums, chosen, inputs_kept, columns, parts, bytes;
    Cut(int64_t rows_, int inputs_, int vocab_, bool backward, bool bias) : rows(rows_), inputs(inputs_), vocab(vocab_) {
        const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
        block = (int)std::min<int64_t>(std::max<int64_t>(rows, 1), kMostRows);
        const int64_t fits = (int64_t)(kPieceBytes / sizeof(T)) / block / kSegment<T> * kSegment<T>;  // columns
        piece = (int)std::min<int64_t>(vocab, std::max<int64_t>(fits, kSegment<T>));
        segments = (int)(((int64_t)vocab + kSegment<T> - 1) / kSegment<T>);
        // (enough workgroups: fp64 301x10007 39 us with chunks of 64 rows, 10.7 with fewer)
        chunk = kChunkRows;
        while (chunk > 4 && (int64_t)((block + chunk - 1) / chunk) * ((piece + 256 * Vec<T>::N - 1) / (256 * Vec<T>::N)) < 1024) chunk /= 2;
        chunks = (block + chunk - 1) / chunk;
        maxima = round((size_t)block * piece * sizeof(T));
        sums = maxima + (backward ? 0 : round((size_t)block * segments * sizeof(T)));
        chosen = sums + (backward ? 0 : round((size_t)block * segments * sizeof(T)));
        inputs_kept = chosen + (backward ? 0 : round((size_t)block * sizeof(T)));
        columns = inputs_kept + (backward ? round((size_t)block * inputs * sizeof(T)) : 0);
        parts = columns + (backward && bias ? round((size_t)chunks * piece * sizeof(T)) : 0);
        bytes = parts;
        // (the last block and piece may be smaller, and cut more finely)
        const int b = (int)((std::max<int64_t>(rows, 1) - 1) % block) + 1, p = (vocab - 1) % piece + 1;
        for (const int m : {block, b})
            for (const int v : {piece, p}) {
                bytes = std::max(bytes, parts + cut_bytes(T(), m, v, inputs));
                if (backward) bytes = std::max({bytes, parts + cut_bytes(T(), m, inputs, v), parts + cut_bytes(T(), inputs, v, m), parts + cut_bytes(T(), v, inputs, m)});
            }
    }
};

// ------------------------------------------------------------------------------------------------ forward
// What the segments of a row come to, by `threads` neighbouring threads of which this is number `at`; all of them return it
template <typename T, int THREADS, typename Get>
__device__ __forceinline__ void entropy_row(int segments, int vocab, int target, int row, const Get& get, T* scratch, T* losses, T* lse) {
    typedef Exponent<T> E;
    T top = E::lowest, sum = 0;
    for (int i = threadIdx.x % THREADS; i < segments; i += THREADS) {
        T m, s, chosen;
        get(i, m, s, chosen);
        const T next = Max()(top, m);
        sum = sum * E::weight(top - next) + s * E::weight(m - next);
        top = next;
    }
    const T best = THREADS == 64 ? fold_lanes<64>(top, Max()) : fold_block<THREADS>(top, scratch, Max());
    sum *= E::weight(top - best);
    sum = THREADS == 64 ? fold_lanes<64>(sum, Sum()) : fold_block<THREADS>(sum, scratch, Sum());
    if (threadIdx.x % THREADS) return;
    T m, s, chosen;
    get(0, m, s, chosen);
    const T logarithm = E::ln(sum);
    lse[row] = best + logarithm;
    // (a row without weight leaves no probability for its target)
    losses[row] = target < 0 || target >= vocab ? T(0) : sum == T(0) ? T(INFINITY) : (best - chosen) + logarithm;
}

// A wave takes a segment of a row of the piece of logits that begins at column v0 of `width` columns, a workgroup up to four of one row. JOIN: the piece is all there is, and the last
// workgroup of a row to arrive joins its segments.
template <typename T, bool JOIN>
__global__ __launch_bounds__(256) void entropy_segments(const T* logits, int rows, int width, int v0, int segments, const T* bias, const int32_t* targets, int all, T* maxima,
                                                        T* sums, T* chosen, unsigned* counters, int counter_step, T* losses, T* lse) {
    constexpr int N = Vec<T>::N;
    typedef Exponent<T> E;
    const int here = (width + kSegment<T> - 1) / kSegment<T>, lane = threadIdx.x & 63, each = (here + 3) / 4;
    const int row = blockIdx.x / each, s = (blockIdx.x - row * each) * 4 + (threadIdx.x >> 6);
    if (!JOIN && s >= here) return;
    const T* x = logits + (int64_t)row * width;
    const int first = s * kSegment<T>;
    T v[kGroupsEach][N];
    typename Vec<T>::type g[kGroupsEach];
#pragma unroll
    for (int j = 0; j < kGroupsEach; ++j) {
        const int c = first + (j * 64 + lane) * N;
        if (c < width) g[j] = ask_group(x, c, width);
    }
    T top = E::lowest;
    const int target = targets[row] - v0;
#pragma unroll
    for (int j = 0; j < kGroupsEach; ++j) {
        const int c = first + (j * 64 + lane) * N;
        if (c < width) {
            take_group(g[j], c, width, T(-INFINITY), v[j]);
            if (bias) {
                T b[N];
                load_group(bias, c, width, T(0), b);
#pragma unroll
                for (int e = 0; e < N; ++e) v[j][e] += b[e];
            }
            if (target >= c && target < c + N && target < width) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (target == c + e) publish(chosen + row, v[j][e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[j][e] = T(-INFINITY);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) top = Max()(top, v[j][e]);
    }
    top = fold_lanes<64>(top, Max());
    T sum = 0;
#pragma unroll
    for (int j = 0; j < kGroupsEach; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) sum += E::weight(v[j][e] - top);
    sum = fold_lanes<64>(sum, Sum());
    if (lane == 0 && s < here) {
        const int64_t at = (int64_t)row * all + segments + s;
        publish(maxima + at, top);
        publish(sums + at, sum);
    }
    if constexpr (JOIN) {
        __shared__ unsigned ticket;
        __shared__ T scratch[4];
        if (each > 1) {
            if (!last_to_arrive(counters + row * counter_step, each, &ticket)) return;
        } else {  // nobody else to wait for
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        entropy_row<T, 256>(
            here, width, target, row,
            [&](int i, T& m, T& sum_of, T& c) { m = observe(maxima + (int64_t)row * all + i), sum_of = observe(sums + (int64_t)row * all + i), c = observe(chosen + row); }, scratch,
            losses, lse);
    }
}

// A wave joins the segments of a row.
template <typename T>
__global__ __launch_bounds__(256) void entropy_join(const T* maxima, const T* sums, const T* chosen, const int32_t* targets, int rows, int segments, int vocab, T* losses, T* lse) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    entropy_row<T, 64>(
        segments, vocab, targets[row], row,
        [&](int i, T& m, T& sum_of, T& c) { m = maxima[(int64_t)row * segments + i], sum_of = sums[(int64_t)row * segments + i], c = chosen[row]; }, (T*)nullptr, losses, lse);
}

template <typename T>
int cross_entropy(int64_t rows, int inputs, int vocab, const T* x, int64_t x_stride, const T* w, int64_t w_stride, bool w_by_columns, const T* bias, const int32_t* targets,
                  T* losses, T* lse, char* space) {
    const char* what = "dali_hip_projected_cross_entropy";
    const Cut<T> cut(rows, inputs, vocab, false, bias != nullptr);
    T *logits = (T*)(space + cut.logits), *maxima = (T*)(space + cut.maxima), *sums = (T*)(space + cut.sums), *chosen = (T*)(space + cut.chosen);
    const bool joins = cut.piece == vocab && cut.block <= kJoinRows;
    for (int64_t r = 0; r < rows; r += cut.block) {
        const int n = (int)std::min<int64_t>(cut.block, rows - r);
        for (int64_t v = 0; v < vocab; v += cut.piece) {
            const int width = (int)std::min<int64_t>(cut.piece, vocab - v), here = (width + kSegment<T> - 1) / kSegment<T>;
            if (cut_product(false, w_by_columns, n, width, inputs, x + r * x_stride, (int)x_stride, w_by_columns ? w + v * w_stride : w + v, (int)w_stride, T(0), logits, width, space + cut.parts))
                return DALI_HIP_ERROR;
            const dim3 grid((unsigned)(n * ((here + 3) / 4)));
            const T* b = bias ? bias + v : nullptr;
            const int segment = (int)(v / kSegment<T>);
            if (joins)
                entropy_segments<T, true><<<grid, dim3(256), 0, stream()>>>(logits, n, width, (int)v, segment, b, targets + r, cut.segments, maxima, sums, chosen,
                                                                           (unsigned*)workspace(), counter_step(n), losses + r, lse + r);
            else
                entropy_segments<T, false><<<grid, dim3(256), 0, stream()>>>(logits, n, width, (int)v, segment, b, targets + r, cut.segments, maxima, sums, chosen, nullptr, 0,
                                                                            nullptr, nullptr);
            if (launched(what)) return DALI_HIP_ERROR;
        }
        if (joins) continue;
        entropy_join<T><<<dim3((unsigned)((n + 3) / 4)), dim3(256), 0, stream()>>>(maxima, sums, chosen, targets + r, n, cut.segments, vocab, losses + r, lse + r);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
}

// ------------------------------------------------------------------------------------------------ backward
// x with zeros in the rows that have no target or no weight, whatever those hold: they have no part in dw
template <typename T>
__global__ __launch_bounds__(256) void entropy_inputs(const T* x, int64_t x_stride, int inputs, const int32_t* targets, const T* lse, int vocab, T* kept) {
    constexpr int N = Vec<T>::N;
    const int row = blockIdx.x, target = targets[row];
    const bool there = target >= 0 && target < vocab && lse[row] != T(-INFINITY);
    for (int c = threadIdx.x * N; c < inputs; c += 256 * N) {
        T v[N] = {};
        if (there) load_group(x + row * x_stride, c, inputs, T(0), v);
        store_group(kept + (int64_t)row * inputs, c, inputs, v);
    }
}

// A thread turns its group of columns of up to `chunk` rows of logits into their gradient and adds up what that comes to.
template <typename T>
__global__ __launch_bounds__(256) void entropy_gradient(T* logits, int rows, int width, int v0, int vocab, const T* bias, const int32_t* targets, const T* lse, const T* d_losses,
                                                        int chunk, T* columns) {
    constexpr int N = Vec<T>::N;
    typedef Exponent<T> E;
    const int c = (blockIdx.x * 256 + threadIdx.x) * N, r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
    if (c >= width) return;
    T b[N] = {}, sum[N] = {};
    if (bias) load_group(bias, c, width, T(0), b);
    // (rows of a piece that end inside a group: a thread's group holds its own columns only, so that no other thread writes what it reads)
    const bool whole = c + N <= width;
    for (int r = r0; r < r1; ++r) {
        T* x = logits + (int64_t)r * width;
        T v[N];
        if (whole) {
            const typename Vec<T>::type g = *reinterpret_cast<const typename Vec<T>::type*>(x + c);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = g[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = c + e < width ? x[c + e] : T(0);
        }
        const int target = targets[r];
        const T total = lse[r];
        const T d = target >= 0 && target < vocab ? d_losses[r] : T(0);
        // a row without a target has no gradient, nor one without weight
        const bool none = target < 0 || target >= vocab || total == T(-INFINITY);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const T p = E::weight(v[e] + b[e] - total) - (target == v0 + c + e ? T(1) : T(0));
            v[e] = none ? T(0) : d * p;
            sum[e] += v[e];
        }
        store_group(x, c, width, v);
    }
    if (columns) store_group(columns + (int64_t)blockIdx.y * width, c, width, sum);
}

// Sixteen waves add up the chunks of 64 columns, a lane a column, and are joined in their order.
template <typename T>
__global__ __launch_bounds__(1024) void entropy_bias(const T* columns, int chunks, int width, bool more, T* dbias) {
    __shared__ T parts[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    T sum = 0;
    if (c < width)
#pragma unroll 4
        for (int i = wave; i < chunks; i += 16) sum += columns[(int64_t)i * width + c];
    parts[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || c >= width) return;
    sum = more ? dbias[c] : T(0);
    for (int w = 0; w < 16; ++w) sum += parts[w][lane];
    dbias[c] = sum;
}

template <typename T>
__global__ __launch_bounds__(256) void entropy_zeros(T* out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = T(0);
}

template <typename T>
int cross_entropy_backward(int64_t rows, int inputs, int vocab, const T* d_losses, const T* x, int64_t x_stride, const T* w, int64_t w_stride, bool w_by_columns, const T* bias,
                           const int32_t* targets, const T* lse, T* dx, T* dw, bool dw_by_columns, T* dbias, char* space) {
    const char* what = "dali_hip_projected_cross_entropy_backward";
    const Cut<T> cut(rows, inputs, vocab, true, dbias != nullptr);
    T *g = (T*)(space + cut.logits), *kept = (T*)(space + cut.inputs_kept), *columns = dbias ? (T*)(space + cut.columns) : nullptr;
    void* parts = space + cut.parts;
    if (rows == 0) {  // (nothing is added up)
        entropy_zeros<T><<<dim3(1024), dim3(256), 0, stream()>>>(dw, (int64_t)inputs * vocab);
        if (!launched(what) && dbias) entropy_zeros<T><<<dim3(1024), dim3(256), 0, stream()>>>(dbias, (int64_t)vocab);
        return launched(what);
    }
    for (int64_t r = 0; r < rows; r += cut.block) {
        const int n = (int)std::min<int64_t>(cut.block, rows - r), chunks = (n + cut.chunk - 1) / cut.chunk;
        entropy_inputs<T><<<dim3((unsigned)n), dim3(256), 0, stream()>>>(x + r * x_stride, x_stride, inputs, targets + r, lse + r, vocab, kept);
        if (launched(what)) return DALI_HIP_ERROR;
        for (int64_t v = 0; v < vocab; v += cut.piece) {
            const int width = (int)std::min<int64_t>(cut.piece, vocab - v);
            const T* wp = w_by_columns ? w + v * w_stride : w + v;
            if (cut_product(false, w_by_columns, n, width, inputs, x + r * x_stride, (int)x_stride, wp, (int)w_stride, T(0), g, width, parts)) return DALI_HIP_ERROR;
            entropy_gradient<T><<<dim3((unsigned)((width + 256 * Vec<T>::N - 1) / (256 * Vec<T>::N)), (unsigned)chunks), dim3(256), 0, stream()>>>(
                g, n, width, (int)v, vocab, bias ? bias + v : nullptr, targets + r, lse + r, d_losses + r, cut.chunk, columns);
            if (launched(what)) return DALI_HIP_ERROR;
            if (cut_product(false, !w_by_columns, n, inputs, width, g, width, wp, (int)w_stride, T(v > 0), dx + r * inputs, inputs, parts)) return DALI_HIP_ERROR;
            const T more = T(r > 0);
            if (dw_by_columns ? cut_product(true, false, width, inputs, n, g, width, kept, inputs, more, dw + v * inputs, inputs, parts)
                              : cut_product(true, false, inputs, width, n, kept, inputs, g, width, more, dw + v, vocab, parts))
                return DALI_HIP_ERROR;
            if (dbias) {
                entropy_bias<T><<<dim3((unsigned)((width + 63) / 64)), dim3(1024), 0, stream()>>>(columns, chunks, width, r > 0, dbias + v);
                if (launched(what)) return DALI_HIP_ERROR;
            }
        }
    }
    return DALI_HIP_OK;
}

// ------------------------------------------------------------------------------------------------ many rows in fp32
// Products of images (product_of_pieces.h): x is cut once for all pieces of the vocabulary, a piece of w once for all products with it. The logits come out transposed, a
// row of them to a lane. Forward they are folded where they are and never leave the registers: every 64 columns leave a maximum and a sum. Backward they become g, which is
// written as an image at once for both products with it. Bound by the matrix pipe. [8192,1024].[1024,32000]: 2550 us forward (3580 through memory with products that cut
// their operands themselves), gradients 8170 (10840): logits 690, dx 670 and dw 670 for each of four pieces of the vocabulary.
constexpr size_t kWeightImageBytes = (size_t)256 << 20, kSlopeImageBytes = (size_t)512 << 20;

struct ImageCut {
    int block, piece, segments, chunks;
    size_t x, w, slopes, columns, parts, maxima, sums, chosen, bytes;
    ImageCut(int64_t rows, int inputs, int vocab, bool backward, bool bias) {
        using namespace pieces;
        const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
        block = (int)std::min<int64_t>(rows, kMostRows);
        size_t wide = std::min(kWeightImageBytes / ((size_t)blocks_of(inputs) * kBlock), (size_t)kMostInner / 16);
        if (backward) wide = std::min(wide, kSlopeImageBytes / ((size_t)blocks_of(block) * kBlock));
        // (pieces of like size, of whole rounds of tiles: 1024 columns are eight)
        const int64_t most = std::max<int64_t>(1024, (int64_t)wide * 16 / 1024 * 1024), count = (vocab + most - 1) / most;
        piece = (int)std::min<int64_t>(vocab, (vocab + count * 1024 - 1) / (count * 1024) * 1024);
        segments = (vocab + 63) / 64;
        chunks = (block + 63) / 64;
        x = 0;
        w = x + round(image_bytes(block, inputs));
        size_t at = w + round(image_bytes(inputs, piece));
        if (!backward) {
            maxima = at;
            sums = maxima + round((size_t)segments * block * sizeof(float));
            chosen = sums + round((size_t)segments * block * sizeof(float));
            bytes = chosen + round((size_t)block * sizeof(float));
            return;
        }
        slopes = at;
        columns = slopes + round(image_bytes(block, piece));
        parts = columns + (bias ? round((size_t)chunks * piece * sizeof(float)) : 0);
        bytes = parts;
        const int b = (int)((rows - 1) % block) + 1, p = (vocab - 1) % piece + 1;  // the last ones
        for (const int m : {block, b})
            for (const int v : {piece, p}) bytes = std::max({bytes, parts + shares_bytes(m, inputs, v), parts + shares_bytes(inputs, v, m), parts + shares_bytes(v, inputs, m)});
    }
};

// A wave's logits, transposed: f(row, of that row's 64 columns the first, the sums [32-column block][register])
template <typename F>
__device__ __forceinline__ void each_row(const pieces::floatx16 (&sum)[2][2], int n0, F f) {
#pragma unroll
    for (int j = 0; j < 2; ++j) f(j, n0 + 32 * j + (threadIdx.x & 31));
}
// bias of a lane's columns, zeros without and past the end
__device__ __forceinline__ void columns_bias(const float* bias, int c0, int width, float (&b)[2][16]) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int c = c0 + 32 * i + pieces::row_of(v, h);
            b[i][v] = bias && c < width ? bias[c] : 0.0f;
        }
}

__global__ __launch_bounds__(256, 3) void entropy_scores(pieces::Product g, int v0, const float* bias, const int32_t* targets, float* maxima, float* sums, float* chosen) {
    extern __shared__ __attribute__((aligned(16))) char pieces_lds[];
    pieces::product<true, false>(g, pieces_lds, [&](const pieces::floatx16 (&sum)[2][2], int c0, int n0, int) {
        typedef Exponent<float> E;
        if (c0 >= g.m) return;
        const int h = (threadIdx.x & 63) >> 5;
        float b[2][16];
        columns_bias(bias, c0, g.m, b);
        each_row(sum, n0, [&](int j, int row) {
            const int target = (row < g.n ? targets[row] : -1) - v0 - c0;
            float top = E::lowest, l[2][16];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int c = 32 * i + pieces::row_of(v, h);
                    l[i][v] = c0 + c < g.m ? sum[i][j][v] + b[i][v] : -INFINITY;
                    top = fmaxf(top, l[i][v]);
                    if (c == target && c0 + c < g.m) chosen[row] = l[i][v];
                }
            top = fold_lanes<64, 32>(top, Max());
            float all = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) all += E::weight(l[i][v] - top);
            all = fold_lanes<64, 32>(all, Sum());
            if (row < g.n && h == 0) {
                const int64_t at = (int64_t)((v0 + c0) / 64) * g.n + row;
                maxima[at] = top;
                sums[at] = all;
            }
        });
    });
}

// Sixteen waves join the segments of 64 rows, a lane a row.
__global__ __launch_bounds__(1024) void entropy_join_columns(const float* maxima, const float* sums, const float* chosen, const int32_t* targets, int rows, int segments, int vocab,
                                                             float* losses, float* lse) {
    typedef Exponent<float> E;
    __shared__ float tops[16][64], alls[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x * 64 + lane;
    float top = E::lowest, sum = 0;
    if (row < rows)
#pragma unroll 4
        for (int i = wave; i < segments; i += 16) {
            const float m = maxima[(int64_t)i * rows + row], s = sums[(int64_t)i * rows + row], next = fmaxf(top, m);
            sum = sum * E::weight(top - next) + s * E::weight(m - next);
            top = next;
        }
    tops[wave][lane] = top;
    alls[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || row >= rows) return;
    for (int w = 1; w < 16; ++w) top = fmaxf(top, tops[w][lane]);
    sum = 0;
    for (int w = 0; w < 16; ++w) sum += alls[w][lane] * E::weight(tops[w][lane] - top);
    const float logarithm = E::ln(sum);
    lse[row] = top + logarithm;
    const int target = targets[row];
    losses[row] = target < 0 || target >= vocab ? 0.0f : sum == 0.0f ? INFINITY : (top - chosen[row]) + logarithm;
}

__global__ __launch_bounds__(256, 3) void entropy_slopes(pieces::Product g, int v0, int vocab, const float* bias, const int32_t* targets, const float* lse, const float* d_losses,
                                                         char* slopes, int row_blocks, int col_blocks, float* columns) {
    extern __shared__ __attribute__((aligned(16))) char pieces_lds[];
    pieces::product<true, false>(g, pieces_lds, [&](const pieces::floatx16 (&sum)[2][2], int c0, int n0, int) {
        typedef Exponent<float> E;
        const int lane = threadIdx.x & 63, h = lane >> 5;
        float b[2][16], total[2][16];
        columns_bias(bias, c0, g.m, b);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) total[i][v] = 0;
        each_row(sum, n0, [&](int j, int row) {
            const bool there = row < g.n;
            const int target = there ? targets[row] : -1;
            const float level = there ? lse[row] : 0.0f;
            // a row without a target has no gradient, nor one without weight
            const bool none = target < 0 || target >= vocab || level == -INFINITY;
            const float d = none ? 0.0f : d_losses[row];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = c0 + 32 * i + 8 * q + 4 * h + e;
                        const float p = E::weight(sum[i][j][4 * q + e] + b[i][4 * q + e] - level) - (target == v0 + c ? 1.0f : 0.0f);
                        v[e] = none || c >= g.m ? 0.0f : d * p;
                        total[i][4 * q + e] += v[e];
                    }
                    const int block_row = row >> 4, block_col = (c0 + 32 * i + 8 * q) >> 4;
                    if (block_row >= row_blocks || block_col >= col_blocks) continue;
                    pieces::uintx2 hi, mid, low;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        unsigned x, y, z;
                        pieces::cut(v[2 * e], v[2 * e + 1], x, y, z);
                        hi[e] = x, mid[e] = y, low[e] = z;
                    }
                    char* to = slopes + ((int64_t)block_row * col_blocks + block_col) * pieces::kBlock + (row & 15) * 32 + pieces::half_at(row, q & 1) + 8 * h;
                    *reinterpret_cast<pieces::uintx2*>(to) = hi;
                    *reinterpret_cast<pieces::uintx2*>(to + pieces::kPlane) = mid;
                    *reinterpret_cast<pieces::uintx2*>(to + 2 * pieces::kPlane) = low;
                }
        });
        if (!columns || n0 >= g.n) return;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float s = fold_lanes<32>(total[i][v], Sum());
                const int c = c0 + 32 * i + pieces::row_of(v, h);
                if ((lane & 31) == 0 && c < g.m) columns[(int64_t)(n0 / 64) * g.m + c] = s;
            }
    });
}

int weight_image(const char* what, const float* w, int64_t w_stride, bool w_by_columns, int inputs, int width, char* image) {
    return w_by_columns ? pieces::image_of<true>(what, w, w_stride, inputs, width, {}, image) : pieces::image_of<false>(what, w, w_stride, inputs, width, {}, image);
}

int cross_entropy_by_images(int64_t rows, int inputs, int vocab, const float* x, int64_t x_stride, const float* w, int64_t w_stride, bool w_by_columns, const float* bias,
                            const int32_t* targets, float* losses, float* lse, char* space) {
    using namespace pieces;
    const char* what = "dali_hip_projected_cross_entropy";
    const ImageCut cut(rows, inputs, vocab, false, bias != nullptr);
    float *maxima = (float*)(space + cut.maxima), *sums = (float*)(space + cut.sums), *chosen = (float*)(space + cut.chosen);
    for (int64_t r = 0; r < rows; r += cut.block) {
        const int n = (int)std::min<int64_t>(cut.block, rows - r);
        const Image xs = {space + cut.x, blocks_of(n), blocks_of(inputs)};
        if (image_of<false>(what, x + r * x_stride, x_stride, n, inputs, {}, space + cut.x)) return DALI_HIP_ERROR;
        for (int64_t v = 0; v < vocab; v += cut.piece) {
            const int width = (int)std::min<int64_t>(cut.piece, vocab - v);
            const Image ws = {space + cut.w, blocks_of(inputs), blocks_of(width)};
            if (weight_image(what, w_by_columns ? w + v * w_stride : w + v, w_stride, w_by_columns, inputs, width, space + cut.w)) return DALI_HIP_ERROR;
            const Product g = product_for(ws, xs, width, n, xs.cols, 1);
            entropy_scores<<<dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(256), kLds, stream()>>>(g, (int)v, bias ? bias + v : nullptr, targets + r, maxima, sums, chosen);
            if (launched(what)) return DALI_HIP_ERROR;
        }
        entropy_join_columns<<<dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, stream()>>>(maxima, sums, chosen, targets + r, n, cut.segments, vocab, losses + r, lse + r);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
}

int cross_entropy_backward_by_images(int64_t rows, int inputs, int vocab, const float* d_losses, const float* x, int64_t x_stride, const float* w, int64_t w_stride,
                                     bool w_by_columns, const float* bias, const int32_t* targets, const float* lse, float* dx, float* dw, bool dw_by_columns, float* dbias,
                                     char* space) {
    using namespace pieces;
    const char* what = "dali_hip_projected_cross_entropy_backward";
    const ImageCut cut(rows, inputs, vocab, true, dbias != nullptr);
    float *parts = (float*)(space + cut.parts), *columns = dbias ? (float*)(space + cut.columns) : nullptr;
    for (int64_t r = 0; r < rows; r += cut.block) {
        const int n = (int)std::min<int64_t>(cut.block, rows - r), chunks = (n + 63) / 64;
        const Image xs = {space + cut.x, blocks_of(n), blocks_of(inputs)};
        if (image_of<false>(what, x + r * x_stride, x_stride, n, inputs, {targets + r, lse + r, vocab}, space + cut.x)) return DALI_HIP_ERROR;
        for (int64_t v = 0; v < vocab; v += cut.piece) {
            const int width = (int)std::min<int64_t>(cut.piece, vocab - v);
            const Image ws = {space + cut.w, blocks_of(inputs), blocks_of(width)}, gs = {space + cut.slopes, blocks_of(n), blocks_of(width)};
            if (weight_image(what, w_by_columns ? w + v * w_stride : w + v, w_stride, w_by_columns, inputs, width, space + cut.w)) return DALI_HIP_ERROR;
            const Product g = product_for(ws, xs, width, n, xs.cols, 1);
            entropy_slopes<<<dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(256), kLds, stream()>>>(g, (int)v, vocab, bias ? bias + v : nullptr, targets + r, lse + r, d_losses + r,
                                                                                                 space + cut.slopes, gs.rows, gs.cols, columns);
            if (launched(what)) return DALI_HIP_ERROR;
            if (kept_product<false, false>(what, gs, ws, n, inputs, {dx + r * inputs, inputs, 0, v > 0}, parts)) return DALI_HIP_ERROR;
            if (dw_by_columns ? kept_product<true, true>(what, gs, xs, width, inputs, {dw + v * inputs, inputs, 0, r > 0}, parts)
                              : kept_product<true, true>(what, xs, gs, inputs, width, {dw + v, vocab, 0, r > 0}, parts))
                return DALI_HIP_ERROR;
            if (dbias) {
                entropy_bias<float><<<dim3((unsigned)((width + 63) / 64)), dim3(1024), 0, stream()>>>(columns, chunks, width, r > 0, dbias + v);
                if (launched(what)) return DALI_HIP_ERROR;
            }
        }
    }
    return DALI_HIP_OK;
}

// Whether a call goes by images: where tiles fill the chip and the cutting of w, which takes as long for a few rows as for many, is a small part. us, by images and by fp32 products,
// inner extents of 32 to 1024. Taken: [512, 10000] forward 21 to 99 and 28 to 103, backward 85 to 225 and 98 to 296; [2048, 2048] 18 to 69 and 23 to 75, 86 to 184 and 81 to 234;
// [1024, 40000] 54 to 453 and 94 to 564, 247 to 1296 and 285 to 1655. Not taken: [256, 40000] 30 to 193 and 38 to 171, 152 to 467 and 130 to 499; [1024, 2048] 18 to 63 and 18
// to 44, 81 to 134 and 71 to 142; [128, 10000] 19 to 71 and 17 to 44, 67 to 132 and 80 to 146.
bool by_images(int dtype, int64_t rows, int inputs, int vocab) {
    const int64_t tiles = ((rows + pieces::kTile - 1) / pieces::kTile) * (((int64_t)vocab + pieces::kTile - 1) / pieces::kTile);
    return dtype == DALI_HIP_FLOAT && rows >= 512 && tiles >= 256 && inputs <= pieces::kMostInner;
}

int check_extents(const char* what, int dtype, int64_t rows, int inputs, int vocab) {
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (rows < 0 || rows > 2147483647LL) return fail("%s: %lld rows", what, (long long)rows);
    if (inputs < 1) return fail("%s: rows of %d values", what, inputs);
    if (vocab < 1 || vocab > 2147483647 - 4096) return fail("%s: a vocabulary of %d", what, vocab);
    return DALI_HIP_OK;
}

int check_strides(const char* what, int64_t rows, int inputs, int vocab, int64_t& x_stride, int64_t w_stride, bool w_by_columns) {
    if (rows <= 1) x_stride = inputs;
    if (x_stride < inputs || x_stride > 2147483647LL) return fail("%s: rows of x are %lld values apart and %d long", what, (long long)x_stride, inputs);
    if (w_stride < (w_by_columns ? inputs : vocab) || w_stride > 2147483647LL) return fail("%s: w's stride is %lld", what, (long long)w_stride);
    return DALI_HIP_OK;
}

size_t space_of(int dtype, int64_t rows, int inputs, int vocab, bool backward, bool bias) {
    if (by_images(dtype, rows, inputs, vocab)) return ImageCut(rows, inputs, vocab, backward, bias).bytes;
    return dtype == DALI_HIP_FLOAT ? Cut<float>(rows, inputs, vocab, backward, bias).bytes : Cut<double>(rows, inputs, vocab, backward, bias).bytes;
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_projected_cross_entropy_workspace(int dtype, int64_t rows, int inputs, int vocab, int backward, int with_bias, size_t* bytes) {
    const char* what = "dali_hip_projected_cross_entropy_workspace";
    if (check_extents(what, dtype, rows, inputs, vocab)) return DALI_HIP_ERROR;
    if (!bytes) return fail("%s: NULL argument", what);
    *bytes = rows ? space_of(dtype, rows, inputs, vocab, backward != 0, with_bias != 0) : 0;
    return DALI_HIP_OK;
}

extern "C" int dali_hip_projected_cross_entropy(int dtype, int64_t rows, int inputs, int vocab, const void* x, int64_t x_stride, const void* w, int64_t w_stride, int w_by_columns,
                                                const void* bias, const int32_t* targets, void* losses, void* lse, void* workspace) {
    const char* what = "dali_hip_projected_cross_entropy";
    if (check_extents(what, dtype, rows, inputs, vocab)) return DALI_HIP_ERROR;
    if (rows == 0) return DALI_HIP_OK;
    if (!x || !w || !targets || !losses || !lse || !workspace) return fail("%s: NULL argument", what);
    if (check_strides(what, rows, inputs, vocab, x_stride, w_stride, w_by_columns != 0)) return DALI_HIP_ERROR;
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (off_elements({x, w, bias, losses, lse}, size) || off_elements({targets}, 4)) return fail("%s: an address is off its type's size", what);
    if ((uintptr_t)workspace % 256 != 0) return fail("%s: the workspace must lie on 256 bytes", what);
    if (check_spans(what, {Span("losses", losses, rows, size), Span("lse", lse, rows, size),
                           Span("the workspace", workspace, (int64_t)space_of(dtype, rows, inputs, vocab, false, bias != nullptr), 1)},
                    {Span("x", x, rows, inputs, x_stride, size), Span("w", w, w_by_columns ? vocab : inputs, w_by_columns ? inputs : vocab, w_stride, size),
                     Span("bias", bias, vocab, size), Span("targets", targets, rows, 4)}, 0))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    if (by_images(dtype, rows, inputs, vocab))
        return cross_entropy_by_images(rows, inputs, vocab, (const float*)x, x_stride, (const float*)w, w_stride, w_by_columns != 0, (const float*)bias, targets, (float*)losses,
                                       (float*)lse, (char*)workspace);
    return dtype == DALI_HIP_FLOAT ? cross_entropy(rows, inputs, vocab, (const float*)x, x_stride, (const float*)w, w_stride, w_by_columns != 0, (const float*)bias, targets,
                                                   (float*)losses, (float*)lse, (char*)workspace)
                                   : cross_entropy(rows, inputs, vocab, (const double*)x, x_stride, (const double*)w, w_stride, w_by_columns != 0, (const double*)bias, targets,
                                                   (double*)losses, (double*)lse, (char*)workspace);
}

extern "C" int dali_hip_projected_cross_entropy_backward(int dtype, int64_t rows, int inputs, int vocab, const void* d_losses, const void* x, int64_t x_stride, const void* w,
                                                         int64_t w_stride, int w_by_columns, const void* bias, const int32_t* targets, const void* lse, void* dx, void* dw,
                                                         int dw_by_columns, void* dbias, void* workspace) {
    const char* what = "dali_hip_projected_cross_entropy_backward";
    if (check_extents(what, dtype, rows, inputs, vocab)) return DALI_HIP_ERROR;
    if (!w || !dw || (rows && (!d_losses || !x || !targets || !lse || !dx || !workspace))) return fail("%s: NULL argument", what);
    if (!bias != !dbias) return fail("%s: bias and dbias come together", what);
    if (check_strides(what, rows, inputs, vocab, x_stride, w_stride, w_by_columns != 0)) return DALI_HIP_ERROR;
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (off_elements({d_losses, x, w, bias, lse, dx, dw, dbias}, size) || off_elements({targets}, 4)) return fail("%s: an address is off its type's size", what);
    if (rows && (uintptr_t)workspace % 256 != 0) return fail("%s: the workspace must lie on 256 bytes", what);
    if (check_spans(what, {Span("dx", dx, rows * inputs, size), Span("dw", dw, (int64_t)inputs * vocab, size), Span("dbias", dbias, vocab, size),
                           Span("the workspace", rows ? workspace : nullptr, (int64_t)space_of(dtype, rows, inputs, vocab, true, bias != nullptr), 1)},
                    {Span("d_losses", d_losses, rows, size), Span("x", x, rows, inputs, x_stride, size),
                     Span("w", w, w_by_columns ? vocab : inputs, w_by_columns ? inputs : vocab, w_stride, size), Span("bias", bias, vocab, size), Span("targets", targets, rows, 4),
                     Span("lse", lse, rows, size)}, 0))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    if (by_images(dtype, rows, inputs, vocab))
        return cross_entropy_backward_by_images(rows, inputs, vocab, (const float*)d_losses, (const float*)x, x_stride, (const float*)w, w_stride, w_by_columns != 0,
                                                (const float*)bias, targets, (const float*)lse, (float*)dx, (float*)dw, dw_by_columns != 0, (float*)dbias, (char*)workspace);
    return dtype == DALI_HIP_FLOAT
               ? cross_entropy_backward(rows, inputs, vocab, (const float*)d_losses, (const float*)x, x_stride, (const float*)w, w_stride, w_by_columns != 0, (const float*)bias,
                                        targets, (const float*)lse, (float*)dx, (float*)dw, dw_by_columns != 0, (float*)dbias, (char*)workspace)
               : cross_entropy_backward(rows, inputs, vocab, (const double*)d_losses, (const double*)x, x_stride, (const double*)w, w_stride, w_by_columns != 0,
                                        (const double*)bias, targets, (const double*)lse, (double*)dx, (double*)dw, dw_by_columns != 0, (double*)dbias, (char*)workspace);
}
