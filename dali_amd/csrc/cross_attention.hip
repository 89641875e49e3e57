// Attention of a decoder's positions to an encoder's states, and its gradients. Beyond the reference.
//
// q [batch, queries, heads, width]; k, v [batch, keys, kv_heads, width]; head h looks at the states of kv head h / (heads / kv_heads); sequence b has counts[b] states,
// what lies behind them is not read. s = scale q.k, lse = ln sum e^s, p = e^(s - lse), y = sum p v. With delta = dy.y: ds = p (dy.v - delta), dq = scale sum ds k,
// dk = scale sum ds q, dv = sum p dy. The scores are never kept: they are formed tile by tile beside a running maximum and sum, and again on the way back.
//
// The positions of all heads that share a kv head are the rows of one problem, whose states are read once for all of them: row r is position r / group of head r % group.
//
// Everything is formed transposed, states by rows: a 16x16 tile of s comes out of the matrix instruction with one row of the problem to a lane (lane % 16) and four
// states to its registers, which is what the next product takes as its right operand if its inner extent is walked in the order (register, lane / 16). So
// the weights never leave their registers, a lane's running maximum, sum and rescaling are of one row, and maxima over the states are folded over two
// exchanges of half rows. The left operands are tiles of states in LDS, read 16 bytes at a time both along a state (for s) and across states (for y).
#include <algorithm>
#include <cmath>

#include "attention_split.h"
#include "attention_tiles.h"

namespace dali_hip {
namespace {

// ------------------------------------------------------------------------------------------------ many rows
template <typename T, int D, bool LATE>
__global__ __launch_bounds__(256, D * sizeof(T) <= 1024 ? 2 : 1) void attention_rows(Args a) {
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    rows_tile<T, D, LATE>(a, attention_lds, a.first + at, part, tile * ForwardShape<T, D>::ROWS);
}

template <typename T, int D, bool LATE>
__global__ __launch_bounds__(256, D * sizeof(T) <= 512 ? 2 : 1) void attention_states_gradient(Args a) {
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    states_gradient_tile<T, D, 256, LATE>(a, attention_lds, a.first + at, part, tile * StatesShape<T, D>::STATES);
}

template <typename T, int D, bool LATE>
__global__ __launch_bounds__(256, D * sizeof(T) <= 512 ? 2 : 1) void attention_rows_gradient(Args a) {
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int id = on_die(blockIdx.x, gridDim.x), at = id / (a.tiles * a.parts), rest = id - at * a.tiles * a.parts, part = rest / a.tiles, tile = rest - part * a.tiles;
    rows_gradient_tile<T, D, 256, LATE>(a, attention_lds, a.first + at, part, tile * RowsShape<T, D>::ROWS);
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 RQ rows: nobody shares a state with another wave, so each of the four takes states of its own, straight from memory into the operands (16 at a time,
// 64-byte pieces of a state), and they are joined in LDS. 32x1x2048 with 16 heads on 4 of 64, 101 MB: 28.4 us, of which reading at the rate of a copy takes 20 and the start of a launch and
// the meeting of its parts 8.
template <typename T, int D, int RQ>
__global__ __launch_bounds__(256, D * sizeof(T) <= 512 ? 2 : 1) void attention_few(Args a) {
    typedef Matrix<T> M;
    constexpr int N = Vec<T>::N, C = D / (4 * N);
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    T* tops = reinterpret_cast<T*>(attention_lds);  // [4][16 RQ]
    T* sums = tops + 64 * RQ;
    T* ys = sums + 64 * RQ;  // [16 RQ][D + N]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int id = on_die(blockIdx.x, gridDim.x);
    const int at = id / a.parts, part = id - at * a.parts, problem = a.first + at;
    const int b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    // (a sequence with fewer states has fewer parts, not shorter ones)
    const int n = count_of(a, b), slabs = (n + 15) / 16, mine = part * 4 + wave, most = ((a.keys + 15) / 16 + a.parts - 1) / a.parts;
    const int parts = max(1, (slabs + most - 1) / max(most, 1));
    if (part >= parts) return;
    const int begin = (int)((int64_t)slabs * mine / (4 * parts)), end = (int)((int64_t)slabs * (mine + 1) / (4 * parts));
    const T* q = (const T*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const T* k = (const T*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const T* v = (const T*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q);
    Fragment<T, D> qf[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) qf[i].load(q + q_rows.at(min(16 * i + (lane & 15), a.rows - 1)), a.width, (T)(a.scale * M::base));
    Columns<T, D> y[RQ];
    Running<T> run[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) y[i].clear();
    // 16 states as left operands, along them and across them (the last state stands in for those behind it, whose scores are -inf and whose values become zeros)
    struct Slab {
        typename Vec<T>::type left[C];
        typename Columns<T, D>::values across[4][Columns<T, D>::BLOCKS];
    };
    auto fetch = [&](Slab& to, int slab) {
        const T* k_row = k + min(slab * 16 + (lane & 15), n - 1) * a.k.row;
#pragma unroll
        for (int c = 0; c < C; ++c) to.left[c] = row_group<D>(k_row, (4 * c + g) * N, a.width);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T* v_row = v + min(slab * 16 + M::row_of(e, g), n - 1) * a.v.row;
#pragma unroll
            for (int blk = 0; blk < Columns<T, D>::BLOCKS; ++blk) {
                constexpr int NV = Columns<T, D>::NV;
                const int c = (16 * blk + (lane & 15)) * NV;
                typedef T loose __attribute__((ext_vector_type(NV), aligned(sizeof(T))));
                if (c + NV <= a.width) {
                    to.across[e][blk] = *reinterpret_cast<const loose*>(v_row + c);
                } else {
#pragma unroll
                    for (int i = 0; i < NV; ++i) to.across[e][blk][i] = c + i < a.width ? v_row[c + i] : T(0);
                }
            }
        }
    };
    auto take = [&](Slab& from, int slab) {
        typename M::acc s[RQ][1];
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            s[i][0] = typename M::acc{};
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < N; ++e) s[i][0] = M::mul(from.left[c][e], qf[i].g[c][e], s[i][0]);
        }
        if (slab * 16 + 16 > n) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (slab * 16 + M::row_of(e, g) >= n) {
#pragma unroll
                    for (int i = 0; i < RQ; ++i) s[i][0][e] = T(-INFINITY);
#pragma unroll
                    for (int blk = 0; blk < Columns<T, D>::BLOCKS; ++blk) from.across[e][blk] = typename Columns<T, D>::values{};
                }
        }
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            T again;
            if (run[i].template take<1>(s[i], again)) y[i].times(again);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int blk = 0; blk < Columns<T, D>::BLOCKS; ++blk)
#pragma unroll
                for (int c = 0; c < Columns<T, D>::NV; ++c)
#pragma unroll
                    for (int i = 0; i < RQ; ++i) y[i].acc[blk][c] = M::mul(from.across[e][blk][c], s[i][0][e], y[i].acc[blk][c]);
    };
    if constexpr (D * sizeof(T) <= 512) {  // the next slab is under way while one is worked on
        Slab even, odd;
        if (begin < end) fetch(even, begin);
        for (int slab = begin; slab < end; slab += 2) {
            if (slab + 1 < end) fetch(odd, slab + 1);
            take(even, slab);
            if (slab + 1 >= end) break;
            if (slab + 2 < end) fetch(even, slab + 2);
            take(odd, slab + 1);
        }
    } else {
        for (int slab = begin; slab < end; ++slab) {
            Slab one;
            fetch(one, slab);
            take(one, slab);
        }
    }
    // the four waves' parts: maxima and sums first, then the rows, one wave after the other
    T sum[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) {
        sum[i] = fold_row(run[i].sum, Sum());
        if (g == 0) {
            tops[wave * 16 * RQ + 16 * i + lane] = run[i].top;
            sums[wave * 16 * RQ + 16 * i + lane] = sum[i];
        }
    }
    __syncthreads();
    T best[RQ], all[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) {
        best[i] = M::lowest, all[i] = 0;
        for (int w = 0; w < 4; ++w) best[i] = Max()(best[i], tops[w * 16 * RQ + 16 * i + (lane & 15)]);
        for (int w = 0; w < 4; ++w) all[i] += sums[w * 16 * RQ + 16 * i + (lane & 15)] * M::weight(tops[w * 16 * RQ + 16 * i + (lane & 15)] - best[i]);
        y[i].times(M::weight(run[i].top - best[i]));
    }
    for (int w = 0; w < 4; ++w) {
        if (wave == w)
#pragma unroll
            for (int i = 0; i < RQ; ++i) {
                T* row = ys + (16 * i + (lane & 15)) * (D + N);
                y[i].each([&](int c, const auto& values) {
#pragma unroll
                    for (int e = 0; e < Columns<T, D>::NV; ++e) row[c + e] = w == 0 ? values[e] : row[c + e] + values[e];
                });
            }
        __syncthreads();
    }
    // (every wave holds the maximum and the sum of a lane's row)
    const int64_t pitch = (int64_t)a.batch * a.kv_heads * a.rows, own = (int64_t)problem * a.rows;  // of a part; this problem's rows in it
    if (wave == 0 && g == 0) {
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            const int r = 16 * i + lane;
            sums[r] = all[i];  // from here on the row's own
            if (r >= a.rows) continue;
            if (parts == 1) {
                ((T*)a.lse_out)[dense_row<T>(a, b, kvh, r)] = all[i] == T(0) ? T(-INFINITY) : M::lse(best[i], all[i]);
            } else {
                publish((T*)a.parts_m + part * pitch + own + r, best[i]);
                publish((T*)a.parts_l + part * pitch + own + r, all[i]);
            }
        }
    }
    __syncthreads();
    const int groups = a.rows * (D / N);
    if (parts == 1) {
        for (int at = threadIdx.x; at < groups; at += 256) {
            const int r = at / (D / N), c = at % (D / N) * N;
            if (c >= a.width) continue;
            T values[N];
#pragma unroll
            for (int e = 0; e < N; ++e) values[e] = sums[r] == T(0) ? T(0) : ys[r * (D + N) + c + e] / sums[r];
            store_group((T*)a.y_out + dense_row<T>(a, b, kvh, r) * a.width, c, a.width, values);
        }
        return;
    }
    // The parts of a problem meet in the workspace; the last workgroup to arrive joins them, in their order.
    for (int at = threadIdx.x; at < groups; at += 256) {
        const int r = at / (D / N), c = at % (D / N) * N;
#pragma unroll
        for (int e = 0; e < N; ++e) publish((T*)a.parts_y + (part * pitch + own + r) * D + c + e, ys[r * (D + N) + c + e]);
    }
    __shared__ unsigned ticket;
    if (!last_to_arrive(a.counters + at * a.counter_step, parts, &ticket)) return;
    const T *pm = (const T*)a.parts_m + own, *pl = (const T*)a.parts_l + own, *py = (const T*)a.parts_y + own * D;
    for (int at = threadIdx.x; at < groups; at += 256) {
        const int r = at / (D / N), c = at % (D / N) * N;
        T top = M::lowest, sum = 0, values[N] = {};
#pragma unroll 4
        for (int p = 0; p < parts; ++p) top = Max()(top, observe(pm + p * pitch + r));
#pragma unroll 4
        for (int p = 0; p < parts; ++p) {
            const T f = M::weight(observe(pm + p * pitch + r) - top);
            sum += observe(pl + p * pitch + r) * f;
#pragma unroll
            for (int e = 0; e < N; ++e) values[e] += observe(py + (p * pitch + r) * D + c + e) * f;
        }
        const int64_t to = dense_row<T>(a, b, kvh, r);
        if (c == 0) ((T*)a.lse_out)[to] = sum == T(0) ? T(-INFINITY) : M::lse(top, sum);
        if (c >= a.width) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) values[e] = sum == T(0) ? T(0) : values[e] / sum;
        store_group((T*)a.y_out + to * a.width, c, a.width, values);
    }
}

// A wave joins the parts of a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_join(Args a) {
    typedef Matrix<T> M;
    const int64_t problems = (int64_t)a.batch * a.kv_heads, unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= problems * a.rows) return;
    const int lane = threadIdx.x & 63, problem = (int)(unit / a.rows), r = (int)(unit - (int64_t)problem * a.rows);
    const T *m = (const T*)a.parts_m + unit, *l = (const T*)a.parts_l + unit, *y = (const T*)a.parts_y + unit * D;
    const int64_t pitch = problems * a.rows;
    T top = M::lowest, sum = 0;
    for (int p = 0; p < a.parts; ++p) top = Max()(top, m[p * pitch]);
    constexpr int EACH = (D + 63) / 64;
    T out[EACH] = {};
    for (int p = 0; p < a.parts; ++p) {
        const T f = M::weight(m[p * pitch] - top);
        sum += l[p * pitch] * f;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (i * 64 + lane < D) out[i] += y[p * pitch * D + i * 64 + lane] * f;
    }
    const int64_t to = dense_row<T>(a, problem / a.kv_heads, problem % a.kv_heads, r);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (i * 64 + lane < a.width) ((T*)a.y_out)[to * a.width + i * 64 + lane] = sum == T(0) ? T(0) : out[i] / sum;
    if (lane == 0) ((T*)a.lse_out)[to] = sum == T(0) ? T(-INFINITY) : M::lse(top, sum);
}

// delta = dy.y of every row: 16 lanes to a row. Bound by memory (16x256 rows of 16 heads of 64: 34 MB, 8 to 9.7 us).
template <typename T>
__global__ __launch_bounds__(256) void attention_delta(Args a, int64_t first) {
    constexpr int N = Vec<T>::N;
    const int64_t row = first + (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const bool there = row < (int64_t)a.batch * a.queries * a.heads;
    T sum = 0;
    if (there) {
        const int64_t bt = row / a.heads;
        const int h = (int)(row - bt * a.heads), b = (int)(bt / a.queries), t = (int)(bt - (int64_t)b * a.queries);
        const T *dy = (const T*)a.dy.p + b * a.dy.batch + t * a.dy.row + h * a.dy.head, *y = (const T*)a.y + row * a.width;
        for (int c = threadIdx.x % 16 * N; c < a.width; c += 16 * N) {
            T u[N], v[N];
            load_group(dy, c, a.width, T(0), u);
            load_group(y, c, a.width, T(0), v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += u[e] * v[e];
        }
    }
    sum = fold_lanes<16>(sum, Sum());
    if (there && threadIdx.x % 16 == 0) ((T*)a.delta)[row] = sum;
}

// A gradient from what parts of the rows or states came to, in their order. Bound by memory (two parts of 16 MB: 5.6 us).
template <typename T>
__global__ __launch_bounds__(256) void attention_gradient_join(const T* parts, int64_t part_size, int count, int64_t size, T* out) {
    constexpr int N = Vec<T>::N;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N; i < size; i += (int64_t)gridDim.x * 256 * N) {
        const int here = (int)min((int64_t)N, size - i);
        T sum[N] = {};
        for (int p = 0; p < count; ++p) {
            T v[N];
            load_group(parts + p * part_size + i, 0, here, T(0), v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += v[e];
        }
        store_group(out + i, 0, here, sum);
    }
}

// ------------------------------------------------------------------------------------------------ launches (host)
constexpr int kUnits = 256;  // compute units that work is cut for

// Parts that the states (or rows) are cut into, so that every compute unit has about `per_unit` workgroups, none with less than `least` slabs. As many to a unit as it holds at once
// does best: gradients with heads of up to 64 two (4x1000x2000, heads of 64: 801 us with one, 686 with two, 738 with three), of more than 64 one (4x512x1024, heads of 256:
// 501, 536, 565); single positions with heads of up to 64 floats three (32x1x2048: 30.3 us with two, 28.2 with three), wider ones two (8x1x4096, 32 heads
// on 8 of 128: 59, 81), and at most 32 for a problem, since one workgroup joins them (1x1x8000, 16 heads of 64: 22 us, 26 with 48).
// within: no more workgroups than those, since one to a unit that is left for a second round takes as long as the first
int parts_for(int64_t workgroups, int slabs, int per_unit, int least, bool within = false) {
    if (workgroups >= kUnits * per_unit) return 1;
    const int64_t wanted = ((int64_t)kUnits * per_unit + (within ? 0 : workgroups - 1)) / workgroups;
    return (int)std::max<int64_t>(1, std::min<int64_t>({wanted, slabs / least, 64}));
}

int padded(int width) { return width <= 32 ? 32 : width <= 64 ? 64 : width <= 128 ? 128 : 256; }

// how the forward pass is cut
struct ForwardPlan {
    bool few;
    int rq, tiles, parts;
    template <typename T, int D>
    void set(const Args& a) {
        typedef ForwardShape<T, D> S;
        const int64_t problems = (int64_t)a.batch * a.kv_heads;
        few = a.rows <= (D * sizeof(T) <= 512 ? 32 : 16);  // (wider rows: 32 would not fit a wave's registers)
        rq = a.rows <= 16 ? 1 : 2;
        const int rows = std::is_same_v<T, float> ? 128 : S::ROWS;
        tiles = few ? 1 : (a.rows + rows - 1) / rows;
        parts = few ? std::min(32, parts_for(problems, (a.keys + 63) / 64, D * sizeof(T) <= 256 ? 3 : 2, 2)) : parts_for(problems * tiles, (a.keys + S::KT - 1) / S::KT, Halves<T, D>::H == 1 ? 2 : 4, 4);
    }
};

// how the gradients are cut: tiles of the states over parts of the rows, tiles of the rows over parts of the states
struct BackwardPlan {
    int state_tiles, state_parts, row_tiles, row_parts;
    int64_t state_size, row_size;  // values of a gradient
    template <typename T, int D>
    void set(const Args& a) {
        const int64_t problems = (int64_t)a.batch * a.kv_heads;
        // (float: rows and states of a tile by the kernels of attention_split.h)
        constexpr bool exact = !std::is_same_v<T, float>;
        constexpr int states = exact ? StatesShape<T, D>::STATES : D <= 128 ? 128 : 64, rows = exact ? RowsShape<T, D>::ROWS : states;
        state_tiles = (a.keys + states - 1) / states, row_tiles = (a.rows + rows - 1) / rows;
        // (Heads of more than 64 doubles: a slab is 3.4 to 6.8 us of work, so two make a part: gradients of 1x448x969, one head of 128, 299 us with eight, 98 with two. More than 128: four
        // workgroups to a unit, one after the other, even out lengths: gradients of 3x878x3987, 4 heads of 256, 4780 us with one, 4190 with four)
        constexpr int slab = exact ? StatesShape<T, D>::RT : 32, least = exact && D > 64 ? 2 : 8, per_unit = Halves<T, D>::H > 1 ? 4 : D <= 64 ? 2 : 1;
        constexpr bool within = exact && D > 64 && per_unit == 1;
        static_assert(!exact || slab == RowsShape<T, D>::KT, "the same slabs of rows and states");
        state_parts = a.keys && a.rows ? parts_for(problems * state_tiles, (a.rows + slab - 1) / slab, per_unit, least, within) : 1;
        row_parts = a.keys && a.rows ? parts_for(problems * row_tiles, (a.keys + slab - 1) / slab, per_unit, least, within) : 1;
        const auto round = [](int64_t n) { return (n + 63) / 64 * 64; };
        state_size = round((int64_t)a.batch * a.keys * a.kv_heads * a.width), row_size = round((int64_t)a.batch * a.queries * a.heads * a.width);
    }
    // of what the parts came to, in values
    int64_t space() const { return std::max(state_parts > 1 ? 2 * state_parts * state_size : 0, row_parts > 1 ? row_parts * row_size : 0); }
};

template <typename F>
auto by_width(int dtype, int width, F f) {
    const int d = padded(width);
    if (dtype == DALI_HIP_FLOAT) {
        if (d == 32) return f(float(), std::integral_constant<int, 32>());
        if (d == 64) return f(float(), std::integral_constant<int, 64>());
        if (d == 128) return f(float(), std::integral_constant<int, 128>());
        return f(float(), std::integral_constant<int, 256>());
    }
    if (d == 32) return f(double(), std::integral_constant<int, 32>());
    if (d == 64) return f(double(), std::integral_constant<int, 64>());
    if (d == 128) return f(double(), std::integral_constant<int, 128>());
    return f(double(), std::integral_constant<int, 256>());
}

size_t round256(size_t b) { return (b + 255) / 256 * 256; }

// bytes of the workspace, and where its parts lie
size_t lay_out(int dtype, Args& a, bool backward, char* space) {
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8, rows = (size_t)a.batch * a.queries * a.heads;
    if (backward)
        return by_width(dtype, a.width, [&](auto t, auto d) -> size_t {
            BackwardPlan plan;
            plan.set<decltype(t), decltype(d)::value>(a);
            a.delta = space, a.parts_y = space + round256(rows * size);
            return round256(rows * size) + (size_t)plan.space() * size;
        });
    return by_width(dtype, a.width, [&](auto t, auto d) -> size_t {
        ForwardPlan plan;
        plan.set<decltype(t), decltype(d)::value>(a);
        a.parts = plan.parts, a.tiles = plan.tiles;
        if (plan.parts == 1) return 0;
        const size_t y = round256(rows * plan.parts * padded(a.width) * size), one = round256(rows * plan.parts * size);
        a.parts_y = space, a.parts_m = space + y, a.parts_l = space + y + one;
        return y + 2 * one;
    });
}

// `each` workgroups for each of the problems, in launches of fewer than 2^32 threads
template <typename K>
int launch(const char* what, K kernel, int64_t problems, int64_t each, int lds, Args a, int threads = 256) {
    if (lds > 65536) {
        const hipError_t e = reserve_dynamic_lds((const void*)kernel, lds);
        if (e != hipSuccess) return fail("%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
    }
    const int64_t most = std::max<int64_t>(1, (1 << 22) / each);
    for (int64_t first = 0; first < problems; first += most) {
        a.first = (int)first;
        kernel<<<dim3((unsigned)(std::min(problems - first, most) * each)), dim3(threads), lds, stream()>>>(a);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
}

// f(false_type), or f(true_type) where attention_tiles.h has a form of its own for heads that do not fill D
template <typename T, int D, typename F>
int by_fill(int width, F f) {
    if constexpr (Halves<T, D>::H > 1)
        if (width != D) return f(std::true_type());
    return f(std::false_type());
}

template <typename T, int D>
int forward(const char* what, Args a) {
    ForwardPlan plan;
    plan.set<T, D>(a);
    a.parts = plan.parts, a.tiles = plan.tiles;
    const int64_t problems = (int64_t)a.batch * a.kv_heads;
    if (plan.few && plan.parts > 1) {  // (so few problems that one launch takes them all)
        a.counters = (unsigned*)workspace();
        a.counter_step = counter_step(problems);
    }
    const int few_lds = 16 * plan.rq * (D + Vec<T>::N + 8) * (int)sizeof(T);
    if (plan.few) {
        if constexpr (D * sizeof(T) <= 512)
            if (plan.rq == 2) return launch(what, attention_few<T, D, 2>, problems, plan.parts, few_lds, a);
        return launch(what, attention_few<T, D, 1>, problems, plan.parts, few_lds, a);
    }
    int status;
    if constexpr (std::is_same_v<T, float>)
        status = launch(what, attention_rows_split<D>, problems, plan.tiles * plan.parts, SplitForward<D>::LDS, a);
    else
        status = by_fill<T, D>(a.width, [&](auto late) {
            return launch(what, attention_rows<T, D, decltype(late)::value>, problems, plan.tiles * plan.parts, ForwardShape<T, D>::LDS, a);
        });
    if (status || plan.parts == 1) return status;
    return launch(what, attention_join<T, D>, 1, (problems * a.rows + 3) / 4, 0, a);
}

template <typename T>
int join(const char* what, const T* parts, int64_t part_size, int count, int64_t size, void* out) {
    const int64_t groups = (size + Vec<T>::N - 1) / Vec<T>::N;
    attention_gradient_join<T><<<dim3((unsigned)std::min<int64_t>((groups + 255) / 256, 8 * kUnits)), dim3(256), 0, stream()>>>(parts, part_size, count, size, (T*)out);
    return launched(what);
}

template <typename T, int D>
int backward(const char* what, Args a) {
    const int64_t problems = (int64_t)a.batch * a.kv_heads, rows = (int64_t)a.batch * a.queries * a.heads;
    const int64_t most = (int64_t)1 << 26;
    for (int64_t first = 0; first < rows; first += most) {
        attention_delta<T><<<dim3((unsigned)((std::min(rows - first, most) + 15) / 16)), dim3(256), 0, stream()>>>(a, first);
        if (launched(what)) return DALI_HIP_ERROR;
    }
    BackwardPlan plan;
    plan.set<T, D>(a);
    constexpr bool split = std::is_same_v<T, float>;
    T* parts = (T*)a.parts_y;
    if (a.keys > 0) {
        Args b = a;
        b.tiles = plan.state_tiles, b.parts = plan.state_parts;
        if (b.parts > 1) b.part_size = plan.state_size, b.dk = parts, b.dv = parts + b.parts * plan.state_size;
        const int64_t each = (int64_t)b.tiles * b.parts;
        if constexpr (split && D > 64) {
            if (launch(what, attention_states_gradient_narrow<D>, problems, each, Narrow<D>::STATES_LDS, b, Narrow<D>::THREADS)) return DALI_HIP_ERROR;
        } else if constexpr (split) {
            if (launch(what, attention_states_gradient_split<D>, problems, each, SplitStates<D>::LDS, b)) return DALI_HIP_ERROR;
        } else {
            if (by_fill<T, D>(a.width, [&](auto late) { return launch(what, attention_states_gradient<T, D, decltype(late)::value>, problems, each, StatesShape<T, D>::LDS, b); }))
                return DALI_HIP_ERROR;
        }
        if (b.parts > 1) {
            const int64_t size = (int64_t)a.batch * a.keys * a.kv_heads * a.width;
            if (join(what, (const T*)b.dk, b.part_size, b.parts, size, a.dk) || join(what, (const T*)b.dv, b.part_size, b.parts, size, a.dv)) return DALI_HIP_ERROR;
        }
    }
    if (rows == 0) return DALI_HIP_OK;
    Args b = a;
    b.tiles = plan.row_tiles, b.parts = plan.row_parts;
    if (b.parts > 1) b.part_size = plan.row_size, b.dq = parts;
    const int64_t each = (int64_t)b.tiles * b.parts;
    int status;
    if constexpr (split && D > 64) status = launch(what, attention_rows_gradient_narrow<D>, problems, each, Narrow<D>::ROWS_LDS, b, Narrow<D>::THREADS);
    else if constexpr (split) status = launch(what, attention_rows_gradient_split<D>, problems, each, SplitRows<D>::LDS, b);
    else status = by_fill<T, D>(a.width, [&](auto late) { return launch(what, attention_rows_gradient<T, D, decltype(late)::value>, problems, each, RowsShape<T, D>::LDS, b); });
    return status || b.parts == 1 ? status : join(what, (const T*)parts, b.part_size, b.parts, rows * a.width, a.dq);
}

// ------------------------------------------------------------------------------------------------ arguments (host)
int check_extents(const char* what, int dtype, int batch, int queries, int keys, int heads, int kv_heads, int width, double scale, Args& a) {
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (batch < 0 || queries < 0 || keys < 0) return fail("%s: %d sequences of %d positions and %d states", what, batch, queries, keys);
    if (heads < 1 || kv_heads < 1 || heads % kv_heads) return fail("%s: %d heads cannot share %d", what, heads, kv_heads);
    if (width < 1 || width > DALI_HIP_MAX_HEAD_WIDTH) return fail("%s: heads are from 1 to %d wide (got %d)", what, DALI_HIP_MAX_HEAD_WIDTH, width);
    if (!holds_scale(dtype, scale) || (dtype == DALI_HIP_FLOAT && !holds_scale(dtype, scale * Matrix<float>::base)))
        return fail("%s: the scale must be finite in its operands' type, in float times log2 e too (got %g)", what, scale);
    const int group = heads / kv_heads;
    if ((int64_t)queries * group > 1 << 28 || keys > 1 << 28 || (int64_t)batch * kv_heads > 2147483647LL)
        return fail("%s: %d sequences of %d positions and %d states with %d heads are too many", what, batch, queries, keys, heads);
    a = {};
    a.batch = batch, a.queries = queries, a.keys = keys, a.heads = heads, a.kv_heads = kv_heads, a.width = width, a.group = group, a.rows = queries * group, a.scale = scale;
    while ((1 << a.group_s) < group) ++a.group_s;
    a.group_m = (unsigned)((((uint64_t)1 << (31 + a.group_s)) + group - 1) / group);
    return DALI_HIP_OK;
}

Operand operand(const void* p, const int64_t* strides) { return {p, strides[0], strides[1], strides[2]}; }

// what an operand of [batch, rows, heads, width] values covers
Span span_of(const char* name, const Operand& o, int batch, int rows, int heads, int width, size_t size) {
    Span s(name, nullptr, 0, size);
    if (!o.p || batch < 1 || rows < 1) return s;
    int64_t lo = 0, hi = width;
    for (const int64_t reach : {(batch - 1) * o.batch, (rows - 1) * o.row, (heads - 1) * o.head}) (reach < 0 ? lo : hi) += reach;
    s.first = (uintptr_t)o.p;
    s.lo = (uintptr_t)o.p + (intptr_t)(lo * (int64_t)size);
    s.hi = (uintptr_t)o.p + (intptr_t)(hi * (int64_t)size);
    return s;
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_cross_attention_workspace(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int width, int backward, size_t* bytes) {
    const char* what = "dali_hip_cross_attention_workspace";
    Args a;
    if (check_extents(what, dtype, batch, queries, keys, heads, kv_heads, width, 1.0, a)) return DALI_HIP_ERROR;
    if (!bytes) return fail("%s: NULL argument", what);
    *bytes = batch && queries ? lay_out(dtype, a, backward != 0, nullptr) : 0;
    return DALI_HIP_OK;
}

extern "C" int dali_hip_cross_attention(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int width, const void* q, const int64_t* q_strides, const void* k,
                                        const int64_t* k_strides, const void* v, const int64_t* v_strides, const int32_t* counts, double scale, void* y, void* lse,
                                        void* workspace) {
    const char* what = "dali_hip_cross_attention";
    Args a;
    if (check_extents(what, dtype, batch, queries, keys, heads, kv_heads, width, scale, a)) return DALI_HIP_ERROR;
    if (batch == 0 || queries == 0) return DALI_HIP_OK;
    if (!q || !q_strides || !y || !lse || (keys && (!k || !k_strides || !v || !v_strides))) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    a.q = operand(q, q_strides);
    if (keys) a.k = operand(k, k_strides), a.v = operand(v, v_strides);
    a.counts = counts, a.y_out = y, a.lse_out = lse;
    const size_t bytes = lay_out(dtype, a, false, (char*)workspace);
    if (bytes && !workspace) return fail("%s: NULL argument", what);
    if (off_elements({q, k, v, y, lse}, size) || off_elements({counts}, 4)) return fail("%s: an address is off its type's size", what);
    if (bytes && (uintptr_t)workspace % 256 != 0) return fail("%s: the workspace must lie on 256 bytes", what);
    const int64_t rows = (int64_t)batch * queries * heads;
    if (check_spans(what, {Span("y", y, rows * width, size), Span("lse", lse, rows, size), Span("the workspace", bytes ? workspace : nullptr, (int64_t)bytes, 1)},
                    {span_of("q", a.q, batch, queries, heads, width, size), span_of("k", a.k, batch, keys, kv_heads, width, size),
                     span_of("v", a.v, batch, keys, kv_heads, width, size), Span("key_counts", counts, batch, 4)}, 0))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    return by_width(dtype, width, [&](auto t, auto d) { return forward<decltype(t), decltype(d)::value>(what, a); });
}

extern "C" int dali_hip_cross_attention_backward(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int width, const void* dy, const int64_t* dy_strides,
                                                 const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                                 const void* y, const void* lse, const int32_t* counts, double scale, void* dq, void* dk, void* dv, void* workspace) {
    const char* what = "dali_hip_cross_attention_backward";
    Args a;
    if (check_extents(what, dtype, batch, queries, keys, heads, kv_heads, width, scale, a)) return DALI_HIP_ERROR;
    if (batch == 0 || (queries == 0 && keys == 0)) return DALI_HIP_OK;
    if ((queries && (!dy || !dy_strides || !q || !q_strides || !y || !lse || !dq || !workspace)) || (keys && (!k || !k_strides || !v || !v_strides || !dk || !dv)))
        return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (queries) a.q = operand(q, q_strides), a.dy = operand(dy, dy_strides);
    if (keys) a.k = operand(k, k_strides), a.v = operand(v, v_strides);
    a.counts = counts, a.y = y, a.lse = lse, a.dq = dq, a.dk = dk, a.dv = dv;
    const size_t bytes = queries ? lay_out(dtype, a, true, (char*)workspace) : 0;
    if (off_elements({dy, q, k, v, y, lse, dq, dk, dv}, size) || off_elements({counts}, 4)) return fail("%s: an address is off its type's size", what);
    if (bytes && (uintptr_t)workspace % 256 != 0) return fail("%s: the workspace must lie on 256 bytes", what);
    const int64_t rows = (int64_t)batch * queries * heads, states = (int64_t)batch * keys * kv_heads;
    if (check_spans(what, {Span("dq", dq, rows * width, size), Span("dk", dk, states * width, size), Span("dv", dv, states * width, size),
                           Span("the workspace", bytes ? workspace : nullptr, (int64_t)bytes, 1)},
                    {span_of("dy", a.dy, batch, queries, heads, width, size), span_of("q", a.q, batch, queries, heads, width, size),
                     span_of("k", a.k, batch, keys, kv_heads, width, size), span_of("v", a.v, batch, keys, kv_heads, width, size), Span("y", y, rows * width, size),
                     Span("lse", lse, rows, size), Span("key_counts", counts, batch, 4)}, 0))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    return by_width(dtype, width, [&](auto t, auto d) { return backward<decltype(t), decltype(d)::value>(what, a); });
}
