// Attention in fp32 on the bf16 matrix cores: every value is cut into three bf16 pieces that add up to it (as sgemm_split.hip does, after Henry, Tang and Heinecke, "Leveraging the
// bfloat16 Artificial Intelligence Datatype For Higher-Precision Computations", 2019), and the six products of pieces of weight 2^-16 and more are summed in fp32. What
// is left out comes to at most 2^-24 of a product, as much as rounding it once costs. A bf16 instruction does sixteen times the work of an fp32 one in the
// same time, so six of them take 3/8 of its time.
//
// Operands are multiplied by 2^16 as they are cut and sums by a power of two afterwards, so that no value is too small for its pieces. Values from 2^112 on, sums from 2^96 on,
// infinities and NaN leave something that is not finite behind: such a tile is taken again with the fp32 instructions on the values as they are, whatever that comes to.
//
// The arrangement is that of attention_tiles.h with instructions of 32x32x16: states by rows, a row of the problem (or a state, for the gradients of states) to a lane
// (lane % 32), whose scores leave the instruction in the order in which the next product takes them as its right operand. Left operands lie in LDS as three planes of rows,
// padded: along a row they are read 16 bytes at a time, across rows by the transposing read, four rows of a column to a lane.
//
// What bounds it: products fill 0.29 (forward) to 0.48 (gradient of states, heads of 128) of the cycles; cutting, exponentials and waits for LDS beside them, which two waves to a
// vector unit hide in part. us: 16x256x512 with 16 heads of 64 forward 53 (with fp32 instructions 84), its gradient 187 (280); 2x1999x4001, 8 heads on 2 of 128, gradient 1060 (2270).
// Registers decide how many waves that is: two to a unit, one with heads of 256, and some are spilled (84 and 73 of the forward pass with heads of 128 and 256).
#ifndef DALI_HIP_ATTENTION_SPLIT_H
#define DALI_HIP_ATTENTION_SPLIT_H

#include "attention_tiles.h"

namespace dali_hip {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned int uintx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));

constexpr float kUp = 0x1p16f, kDown = 0x1p-16f, kDownTwice = 0x1p-32f;

// two values' pieces, packed
__device__ __forceinline__ void cut_pair(float a, float b, unsigned& h, unsigned& m, unsigned& l) {
    const auto pack = [](float x, float y) { return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2{x, y}), bf16x2)); };
    h = pack(a, b);
    const float a1 = a - __uint_as_float(h << 16), b1 = b - __uint_as_float(h & 0xffff0000u);
    m = pack(a1, b1);
    const float a2 = a1 - __uint_as_float(m << 16), b2 = b1 - __uint_as_float(m & 0xffff0000u);
    l = pack(a2, b2);
}

// eight neighbours along the inner extent, in pieces
struct Pieces {
    bf16x8 p[3];
    __device__ __forceinline__ void cut(const float (&v)[8], float factor = 1.0f) {
        uintx4 h, m, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned x, y, z;
            cut_pair(v[2 * i] * factor, v[2 * i + 1] * factor, x, y, z);
            h[i] = x, m[i] = y, l[i] = z;
        }
        p[0] = __builtin_bit_cast(bf16x8, h), p[1] = __builtin_bit_cast(bf16x8, m), p[2] = __builtin_bit_cast(bf16x8, l);
    }
};

// the sum of products of pieces, the small ones first
__device__ __forceinline__ floatx16 multiply(const Pieces& a, const Pieces& b, floatx16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

// two of them in turn: neither waits for the result it has just asked for
__device__ __forceinline__ void multiply_both(const Pieces& a, const Pieces& b, floatx16& c, const Pieces& d, const Pieces& e, floatx16& f) {
    constexpr int left[6] = {2, 0, 1, 1, 0, 0}, right[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[left[i]], b.p[right[i]], c, 0, 0, 0);
        f = __builtin_amdgcn_mfma_f32_32x32x16_bf16(d.p[left[i]], e.p[right[i]], f, 0, 0, 0);
    }
}

// eight values of a row, zeros past its end
template <int D>
__device__ __forceinline__ void row_eight(const float* row, int c, int width, float (&v)[8]) {
    const auto a = row_group<D>(row, c, width), b = row_group<D>(row, c + 4, width);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}

// what a lane holds of 32 rows as a right operand: of row lane % 32, eight values of every sixteen
template <int D>
struct SplitFragment {
    Pieces step[D / 16];
    __device__ __forceinline__ void load(const float* row, int width, float factor) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            float v[8];
            row_eight<D>(row, 16 * s + 8 * (lane >> 5), width, v);
            step[s].cut(v, factor);
        }
    }
};

// R rows of D values in LDS as three planes, brought there by THREADS threads. Behind each row lie 32 bytes of padding: neither eight rows' sixteen bytes at one place nor four
// rows' 32 share banks.
template <int D, int R, int THREADS = 256>
struct SplitStaged {
    static constexpr int PITCH = 2 * D + 32, PLANE = R * PITCH, BYTES = 3 * PLANE, EIGHTS = D / 8, ALL = R * EIGHTS, EACH = (ALL + THREADS - 1) / THREADS;
    float v[EACH][8];
    __device__ __forceinline__ void fetch(const float* base, const Rows& rows, int first, int end, int width) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = threadIdx.x + i * THREADS, r = first + at / EIGHTS;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            if ((ALL % THREADS == 0 || at < ALL) && r < end) row_eight<D>(base + rows.at(r), at % EIGHTS * 8, width, v[i]);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = threadIdx.x + i * THREADS;
            if (ALL % THREADS && at >= ALL) break;
            char* to = lds + at / EIGHTS * PITCH + at % EIGHTS * 16;
            Pieces p;
            p.cut(v[i], kUp);
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x8*>(to + q * PLANE) = p.p[q];
        }
    }
    // left operand along the rows: row r + lane % 32, values 16 s + 8 (lane / 32) ...
    static __device__ __forceinline__ Pieces along(const char* lds, int r, int s) {
        const int lane = threadIdx.x & 63;
        const char* from = lds + (r + (lane & 31)) * PITCH + 32 * s + 16 * (lane >> 5);
        Pieces p;
#pragma unroll
        for (int q = 0; q < 3; ++q) p.p[q] = *reinterpret_cast<const bf16x8*>(from + q * PLANE);
        return p;
    }
    // Left operand across the rows: column c + lane % 32, of the 16 rows from r on those that a lane's scores are of: 4 (lane / 32) + (0..3) and 8 further. (Of 16 lanes that
    // take part in one transposing read, lane i brings 8 bytes of row i / 4, and gets column i of the four rows.)
    static __device__ __forceinline__ Pieces across(const char* lds, int r, int c) {
        const int lane = threadIdx.x & 63;
        const char* from = lds + (r + 4 * (lane >> 5) + ((lane & 15) >> 2)) * PITCH + 2 * (c + 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
        Pieces p;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            typedef __attribute__((address_space(3))) shortx4 lds_four;
            const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_four*)(from + q * PLANE));
            const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_four*)(from + q * PLANE + 8 * PITCH));
            p.p[q] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return p;
    }
};

// the weights of 16 states (or rows) as a right operand: the half `half` of what a lane holds of 32
__device__ __forceinline__ Pieces weights_of(const floatx16& s, int half) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s[8 * half + i];
    Pieces p;
    p.cut(v);
    return p;
}

// row of a tile's accumulator that a lane of half h holds in register v
__device__ __forceinline__ int split_row(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

// D columns of a transposed result
template <int D>
struct SplitColumns {
    floatx16 acc[D / 32];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < D / 32; ++b) acc[b] = floatx16{};
    }
    __device__ __forceinline__ void times(float f) {
#pragma unroll
        for (int b = 0; b < D / 32; ++b) acc[b] *= f;
    }
    __device__ __forceinline__ bool finite() const {
        float probe = 0.0f;  // (0 * x is 0 for finite x and NaN else)
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) probe = fmaf(acc[b][v], 0.0f, probe);
        return probe == 0.0f;
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float run[4] = {acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
                f(32 * b + 8 * q + 4 * h, run);
            }
    }
};

// ------------------------------------------------------------------------------------------------ forward
template <int D>
struct SplitForward {
    static constexpr int KT = ForwardShape<float, D>::KT;  // (the same: a tile that is taken again belongs to a part whose others are not)
    static constexpr int LDS = 2 * SplitStaged<D, KT>::BYTES > ForwardShape<float, D>::LDS ? 2 * SplitStaged<D, KT>::BYTES : ForwardShape<float, D>::LDS;
};

// A workgroup of four waves takes 128 rows of a problem over a part of the states, a wave 32 of them.
template <int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void attention_rows_split(Args a) {
    constexpr int KT = SplitForward<D>::KT;
    typedef SplitStaged<D, KT> Tile;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    char *ks = attention_lds, *vs = ks + Tile::BYTES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    const int problem = a.first + at, b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), slabs = (n + KT - 1) / KT;
    const int begin = (int)((int64_t)slabs * part / a.parts), end = (int)((int64_t)slabs * (part + 1) / a.parts);
    const float* q = (const float*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const float* k = (const float*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const float* v = (const float*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), k_rows(a.k), v_rows(a.v);
    const int row = tile * 128 + wave * 32 + (lane & 31);
    SplitFragment<D> qf;
    qf.load(q + q_rows.at(min(row, a.rows - 1)), a.width, (float)(a.scale * Matrix<float>::base * kUp));
    SplitColumns<D> y;
    y.clear();
    float top = Matrix<float>::lowest, sum = 0, lowest = 0;  // (of the scores as they are; of the lane's own states; of the scores times 2^32)
    Tile kt, vt;
    if (begin < end) {
        kt.fetch(k, k_rows, begin * KT, n, a.width);
        vt.fetch(v, v_rows, begin * KT, n, a.width);
    }
    for (int slab = begin; slab < end; ++slab) {
        __syncthreads();
        kt.store(ks);
        vt.store(vs);
        __syncthreads();
        if (slab + 1 < end) {
            kt.fetch(k, k_rows, (slab + 1) * KT, n, a.width);
            vt.fetch(v, v_rows, (slab + 1) * KT, n, a.width);
        }
        floatx16 s[KT / 32];
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) s[t] = floatx16{};
#pragma unroll
        for (int step = 0; step < D / 16; ++step)
#pragma unroll
            for (int t = 0; t < KT / 32; ++t) s[t] = multiply(Tile::along(ks, 32 * t, step), qf.step[step], s[t]);
        float best = -INFINITY;
        // (lowest: a sum that passed -2^128 on its way stays -inf and would weigh nothing; one that passed 2^128 makes its row NaN)
        if ((slab + 1) * KT > n) {
            asm volatile("");  // (a branch that the other slabs jump over, no selection that they all make)
#pragma unroll
            for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    lowest = fminf(lowest, s[t][e]);
                    if (slab * KT + 32 * t + split_row(e, h) >= n) s[t][e] = -INFINITY;
                    best = fmaxf(best, s[t][e]);
                }
        } else {
#pragma unroll
            for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) lowest = fminf(lowest, s[t][e]), best = fmaxf(best, s[t][e]);
        }
        best = fmaxf(top, fold_lanes<64, 32>(best, Max()) * kDownTwice);
        if (__any(best > top)) {
            const float again = Matrix<float>::weight(top - best);
            sum *= again;
            y.times(again);
            top = best;
        }
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[t][e] = Matrix<float>::weight(fmaf(s[t][e], kDownTwice, -top));
                sum += s[t][e];
            }
        }
#pragma unroll
        for (int t = 0; t < KT / 32; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const Pieces p = weights_of(s[t], half);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) y.acc[c] = multiply(Tile::across(vs, 32 * t + 16 * half, 32 * c), p, y.acc[c]);
            }
    }
    sum = fold_lanes<64, 32>(sum, Sum());
    // (a sum of 0: scores that are all -inf, or below what their pieces hold)
    const bool bad = begin < end && (!(sum > 0.0f && sum < INFINITY) || lowest == -INFINITY || !y.finite());
    if (__syncthreads_or(bad)) {
        constexpr int STEP = ForwardShape<float, D>::ROWS;
        for (int r = 0; r < 128 && tile * 128 + r < a.rows; r += STEP) {
            __syncthreads();
            rows_tile<float, D>(a, attention_lds, problem, part, tile * 128 + r);
        }
        return;
    }
    if (row >= a.rows) return;
    if (a.parts == 1) {
        const int64_t to = dense_row<float>(a, b, kvh, row);
        y.times(sum == 0.0f ? 0.0f : kDown / sum);
        float* out = (float*)a.y_out + to * a.width;
        y.each([&](int c, const auto& values) { store_run(out, c, a.width, values); });
        if (h == 0) ((float*)a.lse_out)[to] = sum == 0.0f ? -INFINITY : Matrix<float>::lse(top, sum);
    } else {
        const int64_t to = ((int64_t)part * a.batch * a.kv_heads + problem) * a.rows + row;
        float* out = (float*)a.parts_y + to * D;
        y.times(kDown);
        y.each([&](int c, const auto& values) { store_run(out, c, D, values); });
        if (h == 0) ((float*)a.parts_m)[to] = top, ((float*)a.parts_l)[to] = sum;
    }
}

// ------------------------------------------------------------------------------------------------ backward
// The gradients of the states: a workgroup takes 128 states, a wave 32 of them in its registers, and walks over the rows of a part, 32 at a time through LDS.
template <int D>
struct SplitStates {
    static constexpr int RT = 32;
    static constexpr int STAGE = 2 * SplitStaged<D, RT>::BYTES + 2 * RT * 4, MINE = 2 * STAGE, LDS = MINE > StatesShape<float, D>::LDS ? MINE : StatesShape<float, D>::LDS;
};

template <int D>
__global__ __launch_bounds__(256, D <= 64 ? 2 : 1) void attention_states_gradient_split(Args a) {
    constexpr int RT = SplitStates<D>::RT;
    typedef SplitStaged<D, RT> Tile;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    const int problem = a.first + at, b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), key = tile * 128 + wave * 32 + (lane & 31);
    const int begin = part_of(a, part, a.rows, RT), end = part_of(a, part + 1, a.rows, RT);
    const float* q = (const float*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const float* dy = (const float*)a.dy.p + b * a.dy.batch + (int64_t)kvh * a.group * a.dy.head;
    const float* k = (const float*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const float* v = (const float*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), dy_rows(a, a.dy);
    SplitColumns<D> dk, dv;
    dk.clear();
    dv.clear();
    float extreme = 0.0f;
    if (tile * 128 < n && begin < end) {
        SplitFragment<D> kf, vf;
        kf.load(k + min(key, n - 1) * a.k.row, a.width, (float)(a.scale * Matrix<float>::base * kUp));
        vf.load(v + min(key, n - 1) * a.v.row, a.width, kUp);
        Tile next;
        float level = 0, delta = 0;
        // what a thread holds of the rows' levels goes along with dy
        auto fetch_levels = [&](int r0) {
            if (threadIdx.x < RT) {
                const int r = r0 + threadIdx.x;
                level = INFINITY, delta = 0;
                if (r < end) {
                    const int64_t from = dense_row<float>(a, b, kvh, r);
                    level = level_of(((const float*)a.lse)[from]);
                    delta = ((const float*)a.delta)[from];
                }
            }
        };
        auto store_levels = [&](char* stage) {
            float* levels = reinterpret_cast<float*>(stage + 2 * Tile::BYTES);
            if (threadIdx.x < RT) levels[threadIdx.x] = level, levels[RT + threadIdx.x] = delta;
        };
        next.fetch(q, q_rows, begin, end, a.width);
        next.store(attention_lds);
        next.fetch(dy, dy_rows, begin, end, a.width);
        fetch_levels(begin);
        next.store(attention_lds + Tile::BYTES);
        store_levels(attention_lds);
        __syncthreads();
        int stage = 0;
        for (int r0 = begin; r0 < end; r0 += RT, stage ^= 1) {
            // (two stages: the next rows are cut and written while these are worked with)
            const char *qs = attention_lds + stage * SplitStates<D>::STAGE, *gs = qs + Tile::BYTES;
            const float *levels = reinterpret_cast<const float*>(gs + Tile::BYTES), *deltas = levels + RT;
            char* to = attention_lds + (stage ^ 1) * SplitStates<D>::STAGE;
            const bool more = r0 + RT < end;
            if (more) next.fetch(q, q_rows, r0 + RT, end, a.width);
            floatx16 s = floatx16{}, dp = floatx16{};
#pragma unroll
            for (int step = 0; step < D / 16; ++step) {
                multiply_both(Tile::along(qs, 0, step), kf.step[step], s, Tile::along(gs, 0, step), vf.step[step], dp);
                __builtin_amdgcn_sched_barrier(0);  // (operands of one step at a time: there are no registers for more)
            }
            if (more) {
                next.store(to);
                next.fetch(dy, dy_rows, r0 + RT, end, a.width);
                fetch_levels(r0 + RT);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float lev = levels[split_row(e, h)], del = deltas[split_row(e, h)];
                extreme = fmaxf(extreme, fabsf(s[e]));
                s[e] = lev == INFINITY ? 0.0f : Matrix<float>::weight(fmaf(s[e], kDownTwice, 16.0f - lev));  // (times 2^16, as the pieces want it)
                dp[e] = s[e] * fmaf(dp[e], kDownTwice, -del);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if constexpr (D == 32) {
                    multiply_both(Tile::across(gs, 16 * half, 0), weights_of(s, half), dv.acc[0], Tile::across(qs, 16 * half, 0), weights_of(dp, half), dk.acc[0]);
                } else {
                    const Pieces p = weights_of(s, half);
                    multiply_both(Tile::across(gs, 16 * half, 0), p, dv.acc[0], Tile::across(gs, 16 * half, 32), p, dv.acc[1]);
                    __builtin_amdgcn_sched_barrier(0);
                    const Pieces ds = weights_of(dp, half);
                    multiply_both(Tile::across(qs, 16 * half, 0), ds, dk.acc[0], Tile::across(qs, 16 * half, 32), ds, dk.acc[1]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (more) {
                next.store(to + Tile::BYTES);
                store_levels(to);
            }
            __syncthreads();
        }
    }
    if (__syncthreads_or(extreme == INFINITY || !dk.finite() || !dv.finite())) {
        constexpr int STEP = StatesShape<float, D>::STATES;
        for (int r = 0; r < 128; r += STEP) {
            __syncthreads();
            states_gradient_tile<float, D>(a, attention_lds, problem, part, tile * 128 + r);
        }
        return;
    }
    if (key >= a.keys) return;
    const int64_t to = part * a.part_size + (((int64_t)b * a.keys + key) * a.kv_heads + kvh) * a.width;
    // (behind the last state: what its stand-in came to is not the gradient, which is zero)
    dk.times(key < n ? kDownTwice : 0.0f);
    dk.times((float)a.scale);  // (a factor of its own: the product of the two may be too small for its digits)
    dv.times(key < n ? kDownTwice : 0.0f);
    dk.each([&](int c, const auto& values) { store_run((float*)a.dk + to, c, a.width, values); });
    dv.each([&](int c, const auto& values) { store_run((float*)a.dv + to, c, a.width, values); });
}

// The gradient of the rows: as the forward pass, with the weights known from lse.
template <int D>
struct SplitRows {
    static constexpr int KT = 32;
    static constexpr int STAGE = 2 * SplitStaged<D, KT>::BYTES, LDS = 2 * STAGE > RowsShape<float, D>::LDS ? 2 * STAGE : RowsShape<float, D>::LDS;
};

template <int D>
__global__ __launch_bounds__(256, 2) void attention_rows_gradient_split(Args a) {
    constexpr int KT = SplitRows<D>::KT;
    typedef SplitStaged<D, KT> Tile;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    const int problem = a.first + at, b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), row = tile * 128 + wave * 32 + (lane & 31), mine = min(row, a.rows - 1);
    const int begin = part_of(a, part, n, KT), end = part_of(a, part + 1, n, KT);
    const float* q = (const float*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const float* dy = (const float*)a.dy.p + b * a.dy.batch + (int64_t)kvh * a.group * a.dy.head;
    const float* k = (const float*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const float* v = (const float*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), dy_rows(a, a.dy), k_rows(a.k), v_rows(a.v);
    SplitFragment<D> qf, gf;
    qf.load(q + q_rows.at(mine), a.width, (float)(a.scale * Matrix<float>::base * kUp));
    gf.load(dy + dy_rows.at(mine), a.width, kUp);
    const int64_t own = dense_row<float>(a, b, kvh, mine);
    const float level = level_of(((const float*)a.lse)[own]), delta = ((const float*)a.delta)[own];
    SplitColumns<D> dq;
    dq.clear();
    float extreme = 0.0f;
    Tile next;
    if (begin < end) {
        next.fetch(k, k_rows, begin, end, a.width);
        next.store(attention_lds);
        next.fetch(v, v_rows, begin, end, a.width);
        next.store(attention_lds + Tile::BYTES);
    }
    __syncthreads();
    int stage = 0;
    for (int first = begin; first < end; first += KT, stage ^= 1) {
        const char *ks = attention_lds + stage * SplitRows<D>::STAGE, *vs = ks + Tile::BYTES;
        char* to = attention_lds + (stage ^ 1) * SplitRows<D>::STAGE;
        const bool more = first + KT < end;
        if (more) next.fetch(k, k_rows, first + KT, end, a.width);
        floatx16 s = floatx16{}, dp = floatx16{};
        Pieces left = Tile::along(ks, 0, 0), down = Tile::along(vs, 0, 0);
#pragma unroll
        for (int step = 0; step < D / 16; ++step) {
            Pieces left1 = left, down1 = down;
            if (step + 1 < D / 16) left1 = Tile::along(ks, 0, step + 1), down1 = Tile::along(vs, 0, step + 1);
            multiply_both(left, qf.step[step], s, down, gf.step[step], dp);
            __builtin_amdgcn_sched_barrier(0);
            left = left1, down = down1;
        }
        if (more) {
            next.store(to);
            next.fetch(v, v_rows, first + KT, end, a.width);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            extreme = fmaxf(extreme, fabsf(s[e]));
            const float p = Matrix<float>::weight(fmaf(s[e], kDownTwice, 16.0f - level));  // (times 2^16, as the pieces want it)
            dp[e] = p * fmaf(dp[e], kDownTwice, -delta);
        }
        if (first + KT > end) {
            asm volatile("");
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (first + split_row(e, h) >= end) dp[e] = 0.0f;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const Pieces ds = weights_of(dp, half);
            if constexpr (D == 32) {
                dq.acc[0] = multiply(Tile::across(ks, 16 * half, 0), ds, dq.acc[0]);
            } else {
#pragma unroll
                for (int c = 0; c < D / 32; c += 2)
                    multiply_both(Tile::across(ks, 16 * half, 32 * c), ds, dq.acc[c], Tile::across(ks, 16 * half, 32 * c + 32), ds, dq.acc[c + 1]);
            }
        }
        if (more) next.store(to + Tile::BYTES);
        __syncthreads();
    }
    if (__syncthreads_or(extreme == INFINITY || !dq.finite())) {
        constexpr int STEP = RowsShape<float, D>::ROWS;
        for (int r = 0; r < 128 && tile * 128 + r < a.rows; r += STEP) {
            __syncthreads();
            rows_gradient_tile<float, D>(a, attention_lds, problem, part, tile * 128 + r);
        }
        return;
    }
    if (row >= a.rows) return;
    float* out = (float*)a.dq + part * a.part_size + own * a.width;
    dq.times(kDownTwice);
    dq.times((float)a.scale);
    dq.each([&](int c, const auto& values) { store_run(out, c, a.width, values); });
}

// ------------------------------------------------------------------------------------------------ backward, wide heads
// Heads of more than 64: 32 columns of two operands and their sums would leave a wave's vector unit to itself, with nobody to work while it waits (heads of 128: 802 and 628 us for the
// states and the rows of 2x1999x4001, so 690 and 505). So a wave takes 16 with instructions of 16x16x32: half the registers, and two waves to a unit where heads have 128; each value
// read from LDS is used half as often.
// Lane l holds eight values of every 32 of its column l % 16, and of the results the rows 4 (l / 16) + (0..3).
__device__ __forceinline__ floatx4 narrow_mul(const Pieces& a, const Pieces& b, floatx4 c) {
    constexpr int left[6] = {2, 0, 1, 1, 0, 0}, right[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int i = 0; i < 6; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[left[i]], b.p[right[i]], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ void narrow_both(const Pieces& a, const Pieces& b, floatx4& c, const Pieces& d, const Pieces& e, floatx4& f) {
    constexpr int left[6] = {2, 0, 1, 1, 0, 0}, right[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[left[i]], b.p[right[i]], c, 0, 0, 0);
        f = __builtin_amdgcn_mfma_f32_16x16x32_bf16(d.p[left[i]], e.p[right[i]], f, 0, 0, 0);
    }
}

template <int D>
struct NarrowFragment {
    Pieces step[D / 32];
    __device__ __forceinline__ void load(const float* row, int width, float factor) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            float v[8];
            row_eight<D>(row, 32 * s + 8 * (lane >> 4), width, v);
            step[s].cut(v, factor);
        }
    }
};

// the tiles of SplitStaged as left operands: along row r + lane % 16, values 32 s + 8 (lane / 16) ...
template <typename Tile>
__device__ __forceinline__ Pieces narrow_along(const char* lds, int r, int s) {
    const int lane = threadIdx.x & 63;
    const char* from = lds + (r + (lane & 15)) * Tile::PITCH + 64 * s + 16 * (lane >> 4);
    Pieces p;
#pragma unroll
    for (int q = 0; q < 3; ++q) p.p[q] = *reinterpret_cast<const bf16x8*>(from + q * Tile::PLANE);
    return p;
}
// across all 32 rows: column c + lane % 16, rows 4 (lane / 16) + (0..3) and 16 further: those that a lane's scores of two tiles are of
template <typename Tile>
__device__ __forceinline__ Pieces narrow_across(const char* lds, int c) {
    const int lane = threadIdx.x & 63;
    const char* from = lds + (4 * (lane >> 4) + ((lane & 15) >> 2)) * Tile::PITCH + 2 * (c + 4 * (lane & 3));
    Pieces p;
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        typedef __attribute__((address_space(3))) shortx4 lds_four;
        const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_four*)(from + q * Tile::PLANE));
        const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_four*)(from + q * Tile::PLANE + 16 * Tile::PITCH));
        p.p[q] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return p;
}
__device__ __forceinline__ Pieces narrow_weights(const floatx4 (&s)[2]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s[i >> 2][i & 3];
    Pieces p;
    p.cut(v);
    return p;
}

template <int D>
struct NarrowColumns {
    floatx4 acc[D / 16];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < D / 16; ++b) acc[b] = floatx4{};
    }
    __device__ __forceinline__ bool finite() const {
        float probe = 0.0f;
#pragma unroll
        for (int b = 0; b < D / 16; ++b)
#pragma unroll
            for (int v = 0; v < 4; ++v) probe = fmaf(acc[b][v], 0.0f, probe);
        return probe == 0.0f;
    }
    // times both factors, one after the other (their product may be too small for its digits)
    __device__ __forceinline__ void put(float* row, int width, float first, float then) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int b = 0; b < D / 16; ++b) {
            const float run[4] = {acc[b][0] * first * then, acc[b][1] * first * then, acc[b][2] * first * then, acc[b][3] * first * then};
            store_run(row, 16 * b + 4 * g, width, run);
        }
    }
};

// Threads, and stages of 32 rows of two operands in LDS
template <int D>
struct Narrow {
    static constexpr int THREADS = D <= 128 ? 512 : 256, MINE = 16 * THREADS / 64, STAGES = D <= 128 ? 2 : 1;
    typedef SplitStaged<D, 32, THREADS> Tile;
    static constexpr int STAGE = 2 * Tile::BYTES + 64 * 4, OWN = STAGES * STAGE;
    static constexpr int STATES_LDS = OWN > StatesShape<float, D>::LDS ? OWN : StatesShape<float, D>::LDS, ROWS_LDS = OWN > RowsShape<float, D>::LDS ? OWN : RowsShape<float, D>::LDS;
    static_assert(StatesShape<float, D>::RK == 1 && RowsShape<float, D>::RQ == 1, "a tile that is taken again is of the same states and rows");
};

template <int D>
__global__ __launch_bounds__(Narrow<D>::THREADS, D <= 128 ? 2 : 1) void attention_states_gradient_narrow(Args a) {
    typedef Narrow<D> Z;
    typedef typename Z::Tile Tile;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    const int problem = a.first + at, b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), key = tile * Z::MINE + wave * 16 + (lane & 15);
    const int begin = part_of(a, part, a.rows, 32), end = part_of(a, part + 1, a.rows, 32);
    const float* q = (const float*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const float* dy = (const float*)a.dy.p + b * a.dy.batch + (int64_t)kvh * a.group * a.dy.head;
    const float* k = (const float*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const float* v = (const float*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), dy_rows(a, a.dy);
    NarrowColumns<D> dk, dv;
    dk.clear();
    dv.clear();
    float extreme = 0.0f;
    if (tile * Z::MINE < n && begin < end) {
        NarrowFragment<D> kf, vf;
        kf.load(k + min(key, n - 1) * a.k.row, a.width, (float)(a.scale * Matrix<float>::base * kUp));
        vf.load(v + min(key, n - 1) * a.v.row, a.width, kUp);
        Tile next;
        float level = 0, delta = 0;
        auto fetch_levels = [&](int r0) {
            if (threadIdx.x < 32) {
                const int r = r0 + threadIdx.x;
                level = INFINITY, delta = 0;
                if (r < end) {
                    const int64_t from = dense_row<float>(a, b, kvh, r);
                    level = level_of(((const float*)a.lse)[from]);
                    delta = ((const float*)a.delta)[from];
                }
            }
        };
        auto store_levels = [&](char* stage) {
            float* levels = reinterpret_cast<float*>(stage + 2 * Tile::BYTES);
            if (threadIdx.x < 32) levels[threadIdx.x] = level, levels[32 + threadIdx.x] = delta;
        };
        next.fetch(q, q_rows, begin, end, a.width);
        next.store(attention_lds);
        next.fetch(dy, dy_rows, begin, end, a.width);
        fetch_levels(begin);
        next.store(attention_lds + Tile::BYTES);
        store_levels(attention_lds);
        __syncthreads();
        int stage = 0;
        for (int r0 = begin; r0 < end; r0 += 32, stage ^= Z::STAGES - 1) {
            const char *qs = attention_lds + stage * Z::STAGE, *gs = qs + Tile::BYTES;
            const float *levels = reinterpret_cast<const float*>(gs + Tile::BYTES), *deltas = levels + 32;
            char* to = attention_lds + (stage ^ (Z::STAGES - 1)) * Z::STAGE;
            const bool more = r0 + 32 < end;
            if (more) next.fetch(q, q_rows, r0 + 32, end, a.width);
            floatx4 s[2] = {floatx4{}, floatx4{}}, dp[2] = {floatx4{}, floatx4{}};
            // (operands a step ahead of their products)
            Pieces left = narrow_along<Tile>(qs, 0, 0), down = narrow_along<Tile>(gs, 0, 0);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                Pieces left1 = left, down1 = down;
                if (i + 1 < D / 16) left1 = narrow_along<Tile>(qs, 16 * ((i + 1) & 1), (i + 1) / 2), down1 = narrow_along<Tile>(gs, 16 * ((i + 1) & 1), (i + 1) / 2);
                narrow_both(left, kf.step[i / 2], s[i & 1], down, vf.step[i / 2], dp[i & 1]);
                __builtin_amdgcn_sched_barrier(0);
                left = left1, down = down1;
            }
            if (Z::STAGES == 2 && more) {
                next.store(to);
                next.fetch(dy, dy_rows, r0 + 32, end, a.width);
                fetch_levels(r0 + 32);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const floatx4 lev = *reinterpret_cast<const floatx4*>(levels + 16 * t + 4 * g), del = *reinterpret_cast<const floatx4*>(deltas + 16 * t + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    extreme = fmaxf(extreme, fabsf(s[t][e]));
                    s[t][e] = lev[e] == INFINITY ? 0.0f : Matrix<float>::weight(fmaf(s[t][e], kDownTwice, 16.0f - lev[e]));  // (times 2^16, as the pieces want it)
                    dp[t][e] = s[t][e] * fmaf(dp[t][e], kDownTwice, -del[e]);
                }
            }
            left = narrow_across<Tile>(gs, 0), down = narrow_across<Tile>(gs, 16);
            Pieces weights = narrow_weights(s);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < 2 * D / 16; c += 2) {  // dv first, then dk
                Pieces left1 = left, down1 = down;
                const int then = c + 2;
                if (then < 2 * D / 16) {
                    const char* from = then < D / 16 ? gs : qs;
                    left1 = narrow_across<Tile>(from, 16 * (then % (D / 16))), down1 = narrow_across<Tile>(from, 16 * (then % (D / 16)) + 16);
                }
                if (c < D / 16) narrow_both(left, weights, dv.acc[c], down, weights, dv.acc[c + 1]);
                else narrow_both(left, weights, dk.acc[c - D / 16], down, weights, dk.acc[c - D / 16 + 1]);
                if (then == D / 16) weights = narrow_weights(dp);
                __builtin_amdgcn_sched_barrier(0);
                left = left1, down = down1;
            }
            if (Z::STAGES == 2) {
                if (more) {
                    next.store(to + Tile::BYTES);
                    store_levels(to);
                }
                __syncthreads();
            } else {
                __syncthreads();
                if (more) {
                    next.store(to);
                    next.fetch(dy, dy_rows, r0 + 32, end, a.width);
                    fetch_levels(r0 + 32);
                    next.store(to + Tile::BYTES);
                    store_levels(to);
                }
                __syncthreads();
            }
        }
    }
    if (__syncthreads_or(extreme == INFINITY || !dk.finite() || !dv.finite())) {
        states_gradient_tile<float, D, Z::THREADS>(a, attention_lds, problem, part, tile * Z::MINE);
        return;
    }
    if (key >= a.keys) return;
    const int64_t to = part * a.part_size + (((int64_t)b * a.keys + key) * a.kv_heads + kvh) * a.width;
    // (behind the last state: what its stand-in came to is not the gradient, which is zero)
    dk.put((float*)a.dk + to, a.width, key < n ? kDownTwice : 0.0f, (float)a.scale);
    dv.put((float*)a.dv + to, a.width, key < n ? kDownTwice : 0.0f, 1.0f);
}

template <int D>
__global__ __launch_bounds__(Narrow<D>::THREADS, D <= 128 ? 2 : 1) void attention_rows_gradient_narrow(Args a) {
    typedef Narrow<D> Z;
    typedef typename Z::Tile Tile;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    const int problem = a.first + at, b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), row = tile * Z::MINE + wave * 16 + (lane & 15), mine = min(row, a.rows - 1);
    const int begin = part_of(a, part, n, 32), end = part_of(a, part + 1, n, 32);
    const float* q = (const float*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const float* dy = (const float*)a.dy.p + b * a.dy.batch + (int64_t)kvh * a.group * a.dy.head;
    const float* k = (const float*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const float* v = (const float*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), dy_rows(a, a.dy), k_rows(a.k), v_rows(a.v);
    NarrowFragment<D> qf, gf;
    qf.load(q + q_rows.at(mine), a.width, (float)(a.scale * Matrix<float>::base * kUp));
    gf.load(dy + dy_rows.at(mine), a.width, kUp);
    const int64_t own = dense_row<float>(a, b, kvh, mine);
    const float level = level_of(((const float*)a.lse)[own]), delta = ((const float*)a.delta)[own];
    NarrowColumns<D> dq;
    dq.clear();
    float extreme = 0.0f;
    Tile next;
    if (begin < end) {
        next.fetch(k, k_rows, begin, end, a.width);
        next.store(attention_lds);
        next.fetch(v, v_rows, begin, end, a.width);
        next.store(attention_lds + Tile::BYTES);
    }
    __syncthreads();
    int stage = 0;
    for (int first = begin; first < end; first += 32, stage ^= Z::STAGES - 1) {
        const char *ks = attention_lds + stage * Z::STAGE, *vs = ks + Tile::BYTES;
        char* to = attention_lds + (stage ^ (Z::STAGES - 1)) * Z::STAGE;
        const bool more = first + 32 < end;
        if (more) next.fetch(k, k_rows, first + 32, end, a.width);
        floatx4 s[2] = {floatx4{}, floatx4{}}, dp[2] = {floatx4{}, floatx4{}};
        // (operands a step ahead of their products)
        Pieces left = narrow_along<Tile>(ks, 0, 0), down = narrow_along<Tile>(vs, 0, 0);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            Pieces left1 = left, down1 = down;
            if (i + 1 < D / 16) left1 = narrow_along<Tile>(ks, 16 * ((i + 1) & 1), (i + 1) / 2), down1 = narrow_along<Tile>(vs, 16 * ((i + 1) & 1), (i + 1) / 2);
            narrow_both(left, qf.step[i / 2], s[i & 1], down, gf.step[i / 2], dp[i & 1]);
            __builtin_amdgcn_sched_barrier(0);
            left = left1, down = down1;
        }
        if (Z::STAGES == 2 && more) {
            next.store(to);
            next.fetch(v, v_rows, first + 32, end, a.width);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                extreme = fmaxf(extreme, fabsf(s[t][e]));
                const float p = Matrix<float>::weight(fmaf(s[t][e], kDownTwice, 16.0f - level));  // (times 2^16, as the pieces want it)
                dp[t][e] = p * fmaf(dp[t][e], kDownTwice, -delta);
            }
        if (first + 32 > end) {
            asm volatile("");
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (first + 16 * t + 4 * g + e >= end) dp[t][e] = 0.0f;
        }
        const Pieces ds = narrow_weights(dp);
        left = narrow_across<Tile>(ks, 0), down = narrow_across<Tile>(ks, 16);
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
            Pieces left1 = left, down1 = down;
            if (c + 2 < D / 16) left1 = narrow_across<Tile>(ks, 16 * c + 32), down1 = narrow_across<Tile>(ks, 16 * c + 48);
            narrow_both(left, ds, dq.acc[c], down, ds, dq.acc[c + 1]);
            __builtin_amdgcn_sched_barrier(0);
            left = left1, down = down1;
        }
        if (Z::STAGES == 2) {
            if (more) next.store(to + Tile::BYTES);
            __syncthreads();
        } else {
            __syncthreads();
            if (more) {
                next.store(to);
                next.fetch(v, v_rows, first + 32, end, a.width);
                next.store(to + Tile::BYTES);
            }
            __syncthreads();
        }
    }
    if (__syncthreads_or(extreme == INFINITY || !dq.finite())) {
        rows_gradient_tile<float, D, Z::THREADS>(a, attention_lds, problem, part, tile * Z::MINE);
        return;
    }
    if (row >= a.rows) return;
    dq.put((float*)a.dq + part * a.part_size + own * a.width, a.width, kDownTwice, (float)a.scale);
}

}  // namespace
}  // namespace dali_hip

#endif
