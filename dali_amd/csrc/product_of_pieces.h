// Products of fp32 matrices that are cut beforehand, for operands that several products share: every value lies in memory as three bf16 pieces that add up to it, and the six
// products of pieces of weight 2^-16 and more are summed in fp32 on the bf16 matrix cores. (The cut and what is left out: sgemm_split.hip, which cuts its operands
// within the product, once for every tile that reads them; that takes as much of its time as the matrix instructions do.)
//
// A matrix lies as an image of blocks of 16 x 16 values, zeros past its ends: three planes of 16 rows of 32 bytes to a block, 1536 bytes; a row's two halves of 16 bytes change
// places where bit 2 of its number is set, so that the reads of eight rows' halves touch different banks. Loads bring such blocks into LDS as they are,
// and a wave reads operands of the matrix instruction from them either way: eight neighbours of a row at once where the inner extent runs along the rows, by the transposing read
// where it runs across them. So a matrix has one image for the products that sum over its rows and those that sum over its columns.
//
// A workgroup of four waves takes a tile of 128 x 128, a wave 64 x 64 of it as 2 x 2 sums of v_mfma_f32_32x32x16_bf16; slabs of 16 of the inner extent go through two stages of
// 24 KiB, written by the loads themselves; 48 KiB and at most 168 registers, so that three workgroups share a compute unit and two multiply while one waits (three stages and two
// workgroups: 2750 us against 2620 for [8192,1024].[1024,32000]). All six products go into one sum, four of the instruction's sums in turn. (sgemm_split.hip
// keeps the small ones apart, which costs registers and vector work and comes closer to double precision: gradients of [8192,1024].[1024,32000] 2.3e-7 away from it, here 1.0e-6, products in
// fp32 instructions 3.1e-6.)
//
// Bound by the matrix pipe: 0.81 of the cycles at the clock that the power limit leaves, 211 TFLOP/s in fp32 terms ([8192,1024].[1024,32000] 2550 us).
//
// A sum that is not finite (values from 2^111 and sums from 2^96 on, infinities, NaN): the tile is taken again with the fp32 instruction on the values, put together from their pieces.
#ifndef DALI_HIP_PRODUCT_OF_PIECES_H
#define DALI_HIP_PRODUCT_OF_PIECES_H

#include <algorithm>

#include "row_math.h"
#include "runtime.h"

namespace dali_hip {
namespace {
namespace pieces {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned int uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned int uintx2 __attribute__((ext_vector_type(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 1536, kPlane = 512;             // bytes
constexpr int kTile = 128, kOperand = 8 * kBlock;      // an operand's slab: eight blocks
constexpr int kStage = 2 * kOperand, kLds = 2 * kStage;
constexpr int kMostInner = 1 << 20;                    // of an image, so that eight blocks' distance fits 32 bits
static_assert(kLds <= 65536, "needs no reserving");

inline int blocks_of(int64_t n) { return (int)((n + 15) / 16); }
inline size_t image_bytes(int64_t rows, int64_t cols) { return (size_t)blocks_of(rows) * blocks_of(cols) * kBlock; }

// where in a row of a block its half `half` lies
__host__ __device__ __forceinline__ int half_at(int row, int half) { return (half ^ ((row >> 2) & 1)) * 16; }

struct Image {
    const char* data;
    int rows, cols;  // in blocks
};

// Two values' pieces, packed: of the value times 2^16, so that none is too small for its pieces. A value of 2^111 and more, an infinity or a NaN is NaN in the first piece, and its own
// bits in the other two.
constexpr float kUp = 0x1p16f, kDown = 0x1p-16f, kDownTwice = 0x1p-32f, kMost = 0x1p111f;
__device__ __forceinline__ void cut(float a, float b, unsigned& h, unsigned& m, unsigned& l) {
    const auto pack = [](float x, float y) { return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2{x, y}), bf16x2)); };
    const float as = a * kUp, bs = b * kUp;
    h = pack(as, bs);
    const float a1 = as - __uint_as_float(h << 16), b1 = bs - __uint_as_float(h & 0xffff0000u);
    m = pack(a1, b1);
    const float a2 = a1 - __uint_as_float(m << 16), b2 = b1 - __uint_as_float(m & 0xffff0000u);
    l = pack(a2, b2);
    const unsigned a_bits = __float_as_uint(a), b_bits = __float_as_uint(b);
    if (!(fabsf(a) < kMost)) h = (h & 0xffff0000u) | 0x7fc0u, m = (m & 0xffff0000u) | a_bits >> 16, l = (l & 0xffff0000u) | (a_bits & 0xffffu);
    if (!(fabsf(b) < kMost)) h = (h & 0xffffu) | 0x7fc00000u, m = (m & 0xffffu) | (b_bits & 0xffff0000u), l = (l & 0xffffu) | b_bits << 16;
}
__device__ __forceinline__ float together(const char* at) {
    const auto piece = [&](int p) { return (unsigned)*reinterpret_cast<const unsigned short*>(at + p * kPlane); };
    const float h = __uint_as_float(piece(0) << 16);
    return h == h ? (h + __uint_as_float(piece(1) << 16) + __uint_as_float(piece(2) << 16)) * kDown : __uint_as_float(piece(1) << 16 | piece(2));
}

// Which rows have a part in a gradient: those with a target and with weight (null: all of them)
struct Takes {
    const int32_t* targets;
    const float* lse;
    int vocab;
    __device__ __forceinline__ bool row(int r) const { return !targets || ((unsigned)targets[r] < (unsigned)vocab && lse[r] != -INFINITY); }
};

// The image of a matrix [rows, cols]: rows `ld` values apart (BY_COLUMNS: columns), a thread eight neighbours of a row. Rows that are not taken are zeros, whatever they hold.
template <bool BY_COLUMNS>
__global__ __launch_bounds__(256) void make_image(const float* x, int64_t ld, int rows, int cols, int row_blocks, int col_blocks, Takes takes, char* image) {
    const int t = threadIdx.x, r = BY_COLUMNS ? t & 15 : t >> 4, group = BY_COLUMNS ? t >> 4 : t & 15;
    const int across = (col_blocks + 7) / 8, rb = blockIdx.x / across, cb = (blockIdx.x - rb * across) * 8 + (group >> 1);
    if (rb >= row_blocks || cb >= col_blocks) return;
    const int row = rb * 16 + r, c = cb * 16 + (group & 1) * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (row < rows && takes.row(row)) {
        if (BY_COLUMNS) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) v[i] = x[(c + i) * ld + row];
        } else {
            float u[4], w[4];
            load_group(x + row * ld, c, cols, 0.0f, u);
            load_group(x + row * ld, c + 4, cols, 0.0f, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = c + i < cols ? u[i] : 0.0f, v[4 + i] = c + 4 + i < cols ? w[i] : 0.0f;
        }
    }
    uintx4 h, m, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned a, b, d;
        cut(v[2 * i], v[2 * i + 1], a, b, d);
        h[i] = a, m[i] = b, l[i] = d;
    }
    char* to = image + ((int64_t)rb * col_blocks + cb) * kBlock + r * 32 + half_at(r, group & 1);
    *reinterpret_cast<uintx4*>(to) = h;
    *reinterpret_cast<uintx4*>(to + kPlane) = m;
    *reinterpret_cast<uintx4*>(to + 2 * kPlane) = l;
}

template <bool BY_COLUMNS>
int image_of(const char* what, const float* x, int64_t ld, int rows, int cols, const Takes& takes, char* image) {
    const int row_blocks = blocks_of(rows), col_blocks = blocks_of(cols);
    const int64_t blocks = (int64_t)row_blocks * ((col_blocks + 7) / 8);
    make_image<BY_COLUMNS><<<dim3((unsigned)blocks), dim3(256), 0, stream()>>>(x, ld, rows, cols, row_blocks, col_blocks, takes, image);
    return launched(what);
}

// ------------------------------------------------------------------------------------------------ the product
struct Product {
    Image a, b;
    int m, n, k;  // k in blocks
    int tiles_m, tiles_n, shares;
};

__device__ __forceinline__ void to_lds(unsigned lds_address, unsigned offset, const char* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_address), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ const char* uniform(const char* p) {
    const unsigned long long b = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)b), hi = __builtin_amdgcn_readfirstlane((unsigned)(b >> 32));
    return (const char*)(((unsigned long long)hi << 32) | lo);
}
// what this wave has in LDS is there and every wave has come here; loads stay in flight
__device__ __forceinline__ void meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// An operand's side of the loads: two blocks to a wave and slab, three times 16 bytes to a lane. Along (the inner extent runs along the rows of the matrix): blocks of
// rows r0 / 16 + (0..7), a slab is a column of them; else columns, a slab is a row of them. Blocks past the matrix repeat its last one: what they sum up to is not kept.
template <bool ACROSS>
struct Side {
    const char* base;
    unsigned offset[3], to;
    int64_t step;
    __device__ __forceinline__ void start(const Image& image, int block0, int slab, unsigned to_) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        const int last = (ACROSS ? image.cols : image.rows) - 1;
        step = ACROSS ? (int64_t)image.cols * kBlock : kBlock;
        base = uniform(image.data + (ACROSS ? (int64_t)slab * image.cols + block0 : (int64_t)block0 * image.cols + slab) * kBlock);
        to = to_ + wave * 2 * kBlock;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int at = j * 1024 + lane * 16, which = at >= kBlock;
            const int block = min(2 * wave + which, last - block0);
            offset[j] = (unsigned)(block * (ACROSS ? 1 : image.cols)) * kBlock + (at - which * kBlock);
        }
    }
    __device__ __forceinline__ void ask(unsigned stage) {
#pragma unroll
        for (int j = 0; j < 3; ++j) to_lds(stage + to + j * 1024, offset[j], base);
        base += step;
    }
};

// Operand of 32 rows (columns) from row r of the tile on: lane l row l % 32, values 8 (l / 32) ... of the slab
template <bool ACROSS>
__device__ __forceinline__ void operand(const char* slab, int r, bf16x8 (&p)[3]) {
    const int lane = threadIdx.x & 63;
    const char* block = slab + (r / 16 + ((lane >> 4) & 1)) * kBlock;
    if (!ACROSS) {
#pragma unroll
        for (int q = 0; q < 3; ++q) p[q] = *reinterpret_cast<const bf16x8*>(block + q * kPlane + (lane & 15) * 32 + half_at(lane, lane >> 5));
    } else {
        // (of 16 lanes that take part in a transposing read, lane i brings 8 bytes of row i / 4, and gets column i of the four rows)
        const char* from = block + (8 * (lane >> 5) + ((lane & 15) >> 2)) * 32;
        const int first = (lane & 3) * 8, then = 4 * 32 + (first ^ 16);  // (four rows further the halves have changed places)
        typedef __attribute__((address_space(3))) shortx4 four;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((four*)(from + q * kPlane + first)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((four*)(from + q * kPlane + then));
            p[q] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
}
template <bool ACROSS>
__device__ __forceinline__ float value(const char* slab, int r, int k) {
    const int lane = threadIdx.x & 63;
    return together(slab + (r / 16 + ((lane >> 4) & 1)) * kBlock + (ACROSS ? k * 32 + half_at(k, (lane >> 3) & 1) + (lane & 7) * 2 : (lane & 15) * 32 + half_at(lane, k >> 3) + (k & 7) * 2));
}

// Row of a 32 x 32 sum that register v of a lane of half h holds; its column is lane % 32
__device__ __forceinline__ int row_of(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

// end(sums, first row, first column, share): what becomes of a wave's sums of 64 x 64
template <bool A_ACROSS, bool B_ACROSS, typename End>
__device__ __forceinline__ void product(const Product& g, char* lds, const End& end) {
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Every eighth workgroup runs on the same die: a die takes a run of neighbouring tiles, eight rows of tiles to a band, whose operands its cache holds.
    const int tiles = g.tiles_m * g.tiles_n, total = tiles * g.shares, per = total >> 3;
    int id = blockIdx.x;
    if (id < per * 8) id = (id & 7) * per + (id >> 3);
    const auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int share = same(id / tiles), tile = id - share * tiles;
    const int band = same(tile / (8 * g.tiles_n)), band_rows = min(8, g.tiles_m - 8 * band), in_band = tile - band * 8 * g.tiles_n;
    const int tn = same(in_band / band_rows), tm = 8 * band + in_band - tn * band_rows;
    const int begin = same((int)((int64_t)g.k * share / g.shares)), count = same((int)((int64_t)g.k * (share + 1) / g.shares)) - begin;
    const int wm = 64 * (wave >> 1), wn = 64 * (wave & 1);
    Side<A_ACROSS> a;
    Side<B_ACROSS> b;
    a.start(g.a, tm * 8, begin, lds0);
    b.start(g.b, tn * 8, begin, lds0 + kOperand);
    floatx16 sum[2][2];
    const auto clear = [&] {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) sum[i][j] = floatx16{};
    };
    clear();
    const auto ask = [&](int stage) {
        a.ask(stage * kStage);
        b.ask(stage * kStage);
    };
    ask(0);
    int stage = 0;
    for (int s = 0; s < count; ++s) {
        // this slab's loads of this wave are done, then everybody's; the next slab goes to the stage that all have left
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        meet();
        if (s + 1 < count) ask(stage ^ 1);
        const char* slab = lds + stage * kStage;
        bf16x8 left[2][3], right[2][3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            operand<A_ACROSS>(slab, wm + 32 * i, left[i]);
            operand<B_ACROSS>(slab + kOperand, wn + 32 * i, right[i]);
        }
        constexpr int of_left[6] = {0, 0, 1, 1, 0, 2}, of_right[6] = {0, 1, 0, 1, 2, 0};
#pragma unroll
        for (int p = 0; p < 6; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(left[i][of_left[p]], right[j][of_right[p]], sum[i][j], 0, 0, 0);
        stage ^= 1;
    }
    float probe = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) probe = fmaf(sum[i][j][v], 0.0f, probe);
    if (__syncthreads_or(probe != 0.0f)) {  // (0 * x is 0 for finite x and NaN else)
        const int lane = threadIdx.x & 63;
        clear();
        a.start(g.a, tm * 8, begin, lds0);
        b.start(g.b, tn * 8, begin, lds0 + kOperand);
        for (int s = 0; s < count; ++s) {
            ask(0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            meet();
            for (int k = 0; k < 16; k += 2) {
                float left[2], right[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    left[i] = value<A_ACROSS>(lds, wm + 32 * i, k + (lane >> 5));
                    right[i] = value<B_ACROSS>(lds + kOperand, wn + 32 * i, k + (lane >> 5));
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(left[i], right[j], sum[i][j], 0, 0, 0);
            }
            meet();
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) sum[i][j] *= kDownTwice;
    }
    end(sum, tm * kTile + wm, tn * kTile + wn, share);
}

// c[m, n] = product + (more ? c : 0), or a share of the product
struct Kept {
    float* c;
    int64_t ld, share_size;
    bool more;
};
template <bool A_ACROSS, bool B_ACROSS>
__global__ __launch_bounds__(256, 3) void product_kept(Product g, Kept to) {
    extern __shared__ __attribute__((aligned(16))) char pieces_lds[];
    product<A_ACROSS, B_ACROSS>(g, pieces_lds, [&](const floatx16 (&sum)[2][2], int m0, int n0, int share) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = n0 + 32 * j + (lane & 31), m = m0 + 32 * i;
                if (n >= g.n) continue;
                float* c = to.c + share * to.share_size + m * to.ld + n;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int r = row_of(v, lane >> 5);
                    if (m + r >= g.m) continue;
                    float* at = c + r * to.ld;
                    const float s = sum[i][j][v];
                    *at = to.more ? *at + s : s;
                }
            }
    });
}
// c = the shares in their order (+ c)
__global__ __launch_bounds__(256) void product_shares(const float* parts, int64_t share_size, int shares, int m, int n, Kept to) {
    const int64_t size = (int64_t)m * n;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
        float s = parts[i];
        for (int p = 1; p < shares; ++p) s += parts[p * share_size + i];
        const int64_t r = i / n;
        float* at = to.c + r * to.ld + (i - r * n);
        *at = to.more ? *at + s : s;
    }
}

constexpr int kSlots = 512;  // workgroups under way at once

// Shares of the inner extent, so that the workgroups come close to whole rounds; none has less than 32 slabs
inline int shares_for(int m, int n, int k) {
    const int64_t tiles = (int64_t)((m + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
    int best = 1;
    double least = 0;
    for (int s = 1; s <= 16 && (s == 1 || k / s >= 32); ++s) {
        // (in rounds of a whole inner extent; what a share costs beyond its slabs, and the folding of shares)
        const double time = (double)((tiles * s + kSlots - 1) / kSlots) / s * (1.0 + 8.0 * s / k) + (s > 1 ? 0.02 * s * (double)tiles / kSlots : 0.0);
        if (s == 1 || time < least) best = s, least = time;
    }
    return best;
}
inline size_t shares_bytes(int64_t m, int64_t n, int64_t k) {
    const int s = shares_for((int)m, (int)n, blocks_of(k));
    return s == 1 ? 0 : (size_t)s * m * n * sizeof(float);
}

inline Product product_for(const Image& a, const Image& b, int m, int n, int k, int shares) {
    return {a, b, m, n, k, (m + kTile - 1) / kTile, (n + kTile - 1) / kTile, shares};
}
// c [m, n] from two images whose inner extents agree; `parts` holds shares_bytes
template <bool A_ACROSS, bool B_ACROSS>
int kept_product(const char* what, const Image& a, const Image& b, int m, int n, Kept to, float* parts) {
    const int k = A_ACROSS ? a.rows : a.cols, shares = shares_for(m, n, k);
    const Product g = product_for(a, b, m, n, k, shares);
    const Kept part = {parts, n, (int64_t)m * n, false};
    product_kept<A_ACROSS, B_ACROSS><<<dim3((unsigned)(g.tiles_m * g.tiles_n * shares)), dim3(256), kLds, stream()>>>(g, shares > 1 ? part : to);
    if (launched(what)) return DALI_HIP_ERROR;
    if (shares > 1) {
        product_shares<<<dim3((unsigned)std::min<int64_t>(((int64_t)m * n + 255) / 256, 8192)), dim3(256), 0, stream()>>>(parts, part.share_size, shares, m, n, to);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
}

}  // namespace pieces
}  // namespace
}  // namespace dali_hip

#endif
