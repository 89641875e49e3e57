// What the kernels of attention share: the operands of a call, tiles of them in registers and LDS, the running softmax, and what a workgroup does for a tile of rows or of
// states in the type's own arithmetic (cross_attention.hip; attention_split.h, where its own does not serve).
#ifndef DALI_HIP_ATTENTION_TILES_H
#define DALI_HIP_ATTENTION_TILES_H

#include "row_math.h"
#include "runtime.h"

namespace dali_hip {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef double doublex4 __attribute__((ext_vector_type(4)));

// The 16x16x4 matrix instruction: lane l holds a[l % 16][l / 16] and b[l / 16][l % 16], and of the result column l % 16, rows row_of(0..3, l / 16).
// Exponents are those of 2 in fp32 (the instruction's base) and of e in fp64.
template <typename T>
struct Matrix;
template <>
struct Matrix<float> {
    typedef floatx4 acc;
    static constexpr float lowest = -3.402823466e+38f;
    static constexpr double base = 1.4426950408889634074;  // exponents are counted in powers of 2
    static __device__ __forceinline__ int row_of(int v, int g) { return 4 * g + v; }
    static __device__ __forceinline__ acc mul(float a, float b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(d); }
    static __device__ __forceinline__ float lse(float top, float sum) { return (top + log2f(sum)) * 0.693147180559945309f; }
};
template <>
struct Matrix<double> {
    typedef doublex4 acc;
    static constexpr double lowest = -1.7976931348623157e+308;
    static constexpr double base = 1.0;
    static __device__ __forceinline__ int row_of(int v, int g) { return 4 * v + g; }
    static __device__ __forceinline__ acc mul(double a, double b, acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ double weight(double d) { return exp(d); }
    static __device__ __forceinline__ double lse(double top, double sum) { return top + log(sum); }
};

struct Operand {
    const void* p;
    int64_t batch, row, head;  // strides in values
};

struct Args {
    int batch, queries, keys, heads, kv_heads, width, group, rows;  // group: heads that share a kv head; rows: queries * group
    Operand q, k, v, dy;
    const int32_t* counts;
    const void *y, *lse;  // dense
    double scale;
    void *y_out, *lse_out, *dq, *dk, *dv;  // dense
    void* delta;                            // [batch, queries, heads]
    // results of parts of the states (or rows): [part][problem][row][D], and maxima and sums [part][problem][row]
    void *parts_y, *parts_m, *parts_l;
    int64_t part_size;  // of the gradients: values from one part's to the next one's, which lie as the gradients do
    int parts, tiles;
    unsigned* counters;  // of arrivals, counter_step words apart
    int counter_step;
    int first;  // problem of a launch's first workgroup
    // r / group for rows r: an exact division by a product (sgemm_row_map_div)
    unsigned group_m;
    int group_s;
    __device__ __forceinline__ int position_of(int r) const { return group == 1 ? r : (int)sgemm_row_map_div((unsigned)r, group_m, group_s); }
};

// Rows that neighbouring heads share: row r lies at position r / group of head r % group
struct Rows {
    int64_t row, head;
    int group;
    unsigned group_m;
    int group_s;
    __device__ __forceinline__ Rows(const Args& a, const Operand& o) : row(o.row), head(o.head), group(a.group), group_m(a.group_m), group_s(a.group_s) {}
    __device__ __forceinline__ explicit Rows(const Operand& o) : row(o.row), head(0), group(1), group_m(0), group_s(0) {}
    __device__ __forceinline__ int64_t at(int r) const {
        if (group == 1) return r * row;
        const int t = (int)sgemm_row_map_div((unsigned)r, group_m, group_s);
        return t * row + (r - t * group) * head;
    }
};

__device__ __forceinline__ int count_of(const Args& a, int b) { return a.counts ? max(0, min(a.counts[b], a.keys)) : a.keys; }

// neighbouring workgroups, which share operands, run on the same die (every eighth one does)
__device__ __forceinline__ int on_die(int id, int total) {
    const int per = total >> 3;
    return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

// A group of values of a row, zeros past the row's end
template <int D, typename T>
__device__ __forceinline__ typename Vec<T>::type row_group(const T* row, int c, int width) {
    if (width == D) return *reinterpret_cast<const typename Vec<T>::type*>(row + c);
    T v[Vec<T>::N];
    typename Vec<T>::type g = {};
    if (c < width) {
        load_group(row, c, width, T(0), v);
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i) g[i] = v[i];
    }
    return g;
}
// LATE, below: heads of more than 128 doubles that are not 256 wide. All that a thread brings is asked for before any is put in its place. (Put there at once, each group is waited for:
// gradients of 23x420x102 with 2 heads of 187 535 us, and 302. Narrower heads are quicker without, their registers are full; for whole rows there is nothing to put in its place, and a kernel
// that does either at run time spills.)

// What a lane holds of 16 rows as a right operand: row lane % 16, groups lane / 16 of every four, from value c0 of W on
template <typename T, int D, int W = D, bool LATE = false>
struct Fragment {
    static constexpr int N = Vec<T>::N, C = D / (4 * N);
    typename Vec<T>::type g[C];
    __device__ __forceinline__ void load(const T* row, int width, T factor, int c0 = 0) {
        const int lane = threadIdx.x & 63;
        if constexpr (!LATE) {
#pragma unroll
            for (int c = 0; c < C; ++c) g[c] = row_group<W>(row, c0 + (4 * c + (lane >> 4)) * N, width) * factor;
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) g[c] = ask_group<true>(row, c0 + (4 * c + (lane >> 4)) * N, width);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                T v[N];
                take_group<true>(g[c], c0 + (4 * c + (lane >> 4)) * N, width, T(0), v);
#pragma unroll
                for (int e = 0; e < N; ++e) g[c][e] = v[e] * factor;
            }
        }
    }
};

// Heads of more than 128 doubles: two waves share 16 rows (or states), each with half of the width, since operands and sums of all of it do not fit a wave's registers (up to 696 of them
// were spilled, and the gradients of the states took two launches). Each forms half of a score's sum, and they meet in LDS; results are the half's own. The halves are whole blocks of 32,
// as even as that allows. Gradients of 3x878x3987, 4 heads of 256: 9990 us, so 3790; forward 4x500x1000, 8 heads on 4 of 256: 977, 502. Bound by the matrix pipe for half of the
// time (one wave to a vector unit: nobody works while it waits).
template <typename T, int D>
struct Halves {
    static constexpr int H = D * sizeof(T) > 1024 ? 2 : 1, W = D / H;  // waves that share rows, and the most that one has of the width
    static constexpr int GROUPS = 4 / H;                              // of waves in a workgroup of four
    int wave, group, c0, mine;                                        // the wave; its group; what it has of the width: from c0 on, `mine`
    __device__ __forceinline__ explicit Halves(int width) : wave(threadIdx.x >> 6) {
        group = wave / H;
        mine = H == 1 ? D : (width + 63) / 64 * 32;
        c0 = wave % H * mine;
    }
    // whether the wave's share ends before its value c
    __device__ __forceinline__ bool ends(int c) const { return H > 1 && c >= mine; }
    static constexpr int bytes(int tiles) { return H == 1 ? 0 : 2 * 4 * tiles * 256 * (int)sizeof(T); }
    // the sums of both halves, by way of `space` ([2][4 waves][tiles][4][64], whose halves are written in turn: with one barrier a time nobody writes what another still reads)
    template <int TILES>
    __device__ __forceinline__ void meet(T* space, int& turn, typename Matrix<T>::acc* (&s)[TILES]) const {
        if constexpr (H > 1) {
            const int lane = threadIdx.x & 63;
            T* all = space + turn * 4 * TILES * 256 + lane;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) all[((wave * TILES + t) * 4 + v) * 64] = (*s[t])[v];
            __syncthreads();
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) (*s[t])[v] += all[(((wave ^ 1) * TILES + t) * 4 + v) * 64];
            turn ^= 1;
        }
    }
};

// A tile of R rows of D values in LDS, a group of padding behind each row: sixteen rows' groups at one place lie in different banks
template <typename T, int D, int R, int THREADS = 256, bool LATE = false>
struct Staged {
    static constexpr int N = Vec<T>::N, PITCH = D + N, GROUPS = D / N, EACH = R * GROUPS / THREADS;
    static constexpr int BYTES = R * PITCH * sizeof(T);
    static_assert(R * GROUPS % THREADS == 0, "whole groups to every thread");
    typename Vec<T>::type g[EACH];
    int there;  // rows of the tile
    // rows [first, first + R) of those below `end` (first is), zeros elsewhere
    __device__ __forceinline__ void fetch(const T* base, const Rows& rows, int first, int end, int width) {
        there = end - first;
        if constexpr (!LATE) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = threadIdx.x + i * THREADS, r = first + at / GROUPS;
                g[i] = r < end ? row_group<D>(base + rows.at(r), at % GROUPS * N, width) : typename Vec<T>::type{};
            }
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = threadIdx.x + i * THREADS;
                g[i] = ask_group<true>(base + rows.at(min(first + at / GROUPS, end - 1)), at % GROUPS * N, width);
            }
        }
    }
    __device__ __forceinline__ void store(T* lds, int width) const {
        typedef T aligned_group __attribute__((ext_vector_type(16 / sizeof(T))));
        if constexpr (!LATE) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = threadIdx.x + i * THREADS;
                *reinterpret_cast<aligned_group*>(lds + at / GROUPS * PITCH + at % GROUPS * N) = g[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = threadIdx.x + i * THREADS, c = at % GROUPS * N;
                T v[N];
                take_group<true>(g[i], c, width, T(0), v);
                aligned_group to;
#pragma unroll
                for (int e = 0; e < N; ++e) to[e] = at / GROUPS < there ? v[e] : T(0);
                *reinterpret_cast<aligned_group*>(lds + at / GROUPS * PITCH + c) = to;
            }
        }
    }
    // the left operand along the rows: row r + lane % 16, group 4 c + lane / 16
    static __device__ __forceinline__ typename Vec<T>::type along(const T* lds, int r, int c) {
        typedef T aligned_group __attribute__((ext_vector_type(16 / sizeof(T))));
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const aligned_group*>(lds + (r + (lane & 15)) * PITCH + (4 * c + (lane >> 4)) * N);
    }
};

// How the D columns of a transposed result lie in accumulators: block b, tile t of it (NV tiles to a block), row i of the tile: column (16 b + i) NV + t, so
// that a lane reads the left operand of NV tiles, and writes NV neighbours of the result, at once.
template <typename T, int D>
struct Columns {
    static constexpr int NV = D % (16 * Vec<T>::N) == 0 ? Vec<T>::N : Vec<T>::N / 2, BLOCKS = D / (16 * NV);
    static_assert(D % (16 * NV) == 0, "whole blocks");
    typedef T values __attribute__((ext_vector_type(NV)));
    typename Matrix<T>::acc acc[BLOCKS][NV];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int t = 0; t < NV; ++t) acc[b][t] = typename Matrix<T>::acc{};
    }
    __device__ __forceinline__ void times(T f) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int t = 0; t < NV; ++t) acc[b][t] *= f;
    }
    // the left operand across rows: row `r`, the lane's values of block b
    static __device__ __forceinline__ values across(const T* row, int b) { return *reinterpret_cast<const values*>(row + (16 * b + (threadIdx.x & 15)) * NV); }
    // f(column, NV values) for every run of neighbours that the lane holds
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                T run[NV];
#pragma unroll
                for (int t = 0; t < NV; ++t) run[t] = acc[b][t][v];
                f((16 * b + Matrix<T>::row_of(v, g)) * NV, run);
            }
    }
};

template <int NV, typename T>
__device__ __forceinline__ void store_run(T* row, int c, int width, const T (&run)[NV]) {
    typedef T values __attribute__((ext_vector_type(NV), aligned(sizeof(T))));
    if (c + NV <= width) {
        values g;
#pragma unroll
        for (int i = 0; i < NV; ++i) g[i] = run[i];
        *reinterpret_cast<values*>(row + c) = g;
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (c + i < width) row[c + i] = run[i];
    }
}

// folds over the four lanes that hold a row
template <typename T, typename Op>
__device__ __forceinline__ T fold_row(T v, Op op) {
    return fold_lanes<64, 16>(v, op);
}

// The running softmax of the row of a lane
template <typename T>
struct Running {
    T top = Matrix<T>::lowest, sum = 0;  // (the sum of the lane's own states)
    // takes the scores of a tile, which become weights; true where the sums so far have to be multiplied by `again`
    template <int TILES>
    __device__ __forceinline__ bool take(typename Matrix<T>::acc (&s)[TILES], T& again) {
        T best = top;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) best = Max()(best, s[t][v]);
        best = fold_row(best, Max());
        const bool rises = __any(best > top);
        again = Matrix<T>::weight(top - best);
        T here = 0;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                s[t][v] = Matrix<T>::weight(s[t][v] - best);
                here += s[t][v];
            }
        sum = sum * again + here;
        top = best;
        return rises;
    }
};

template <typename T>
__device__ __forceinline__ int64_t dense_row(const Args& a, int b, int kvh, int r) {
    const int t = a.position_of(r);
    return ((int64_t)b * a.queries + t) * a.heads + (int64_t)kvh * a.group + (r - t * a.group);
}

// ------------------------------------------------------------------------------------------------ forward
// A workgroup of four waves takes 64 RQ rows of a problem, a wave (or two) 16 RQ of them, over a part of the states, KT at a time through LDS.
template <typename T, int D>
struct ForwardShape {
    static constexpr int KT = D * sizeof(T) <= 256 ? 64 : D * sizeof(T) <= 1024 ? 32 : 16, RQ = D * sizeof(T) <= 512 ? 2 : 1, ROWS = 16 * RQ * Halves<T, D>::GROUPS;
    static constexpr int TILES = 2 * Staged<T, D, KT>::BYTES, LDS = TILES + Halves<T, D>::bytes(KT / 16);
};

// (LATE: see above; else heads of more than 128 doubles are 256 wide)
template <typename T, int D, bool LATE = false>
__device__ __forceinline__ void rows_tile(const Args& a, char* lds, int problem, int part, int first_row) {
    typedef Matrix<T> M;
    typedef ForwardShape<T, D> S;
    typedef Halves<T, D> Z;
    constexpr int KT = S::KT, RQ = S::RQ, N = Vec<T>::N, W = Z::W, C = W / (4 * N);
    static_assert(Z::H == 1 || (RQ == 1 && KT == 16), "one tile of scores meets at a time");
    T *ks = reinterpret_cast<T*>(lds), *vs = ks + KT * Staged<T, D, KT>::PITCH;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int width = Z::H > 1 && !LATE ? D : a.width;
    const Z z(width);
    int turn = 0;
    const int b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), slabs = (n + KT - 1) / KT;
    const int begin = (int)((int64_t)slabs * part / a.parts), end = (int)((int64_t)slabs * (part + 1) / a.parts);
    const T* q = (const T*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const T* k = (const T*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const T* v = (const T*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), k_rows(a.k), v_rows(a.v);
    const int r0 = first_row + z.group * 16 * RQ;
    Fragment<T, W, D, LATE> qf[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) qf[i].load(q + q_rows.at(min(r0 + 16 * i + (lane & 15), a.rows - 1)), width, (T)(a.scale * M::base), z.c0);
    Columns<T, W> y[RQ];
    Running<T> run[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) y[i].clear();
    Staged<T, D, KT, 256, LATE> kt, vt;
    if (begin < end) {
        kt.fetch(k, k_rows, begin * KT, n, width);
        vt.fetch(v, v_rows, begin * KT, n, width);
    }
    for (int slab = begin; slab < end; ++slab) {
        __syncthreads();
        kt.store(ks, width);
        vt.store(vs, width);
        __syncthreads();
        if (slab + 1 < end) {
            kt.fetch(k, k_rows, (slab + 1) * KT, n, width);
            vt.fetch(v, v_rows, (slab + 1) * KT, n, width);
        }
        typename M::acc s[RQ][KT / 16];
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
#pragma unroll
            for (int i = 0; i < RQ; ++i) s[i][t] = typename M::acc{};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (z.ends(c * 4 * N)) break;
                const typename Vec<T>::type left = Staged<T, D, KT>::along(ks + z.c0, 16 * t, c);
#pragma unroll
                for (int e = 0; e < N; ++e)
#pragma unroll
                    for (int i = 0; i < RQ; ++i) s[i][t] = M::mul(left[e], qf[i].g[c][e], s[i][t]);
            }
        }
        if constexpr (Z::H > 1) {
            typename M::acc* halves[1] = {&s[0][0]};
            z.meet(reinterpret_cast<T*>(lds + S::TILES), turn, halves);
        }
        if ((slab + 1) * KT > n) {
#pragma unroll
            for (int t = 0; t < KT / 16; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (slab * KT + 16 * t + M::row_of(e, g) >= n)
#pragma unroll
                        for (int i = 0; i < RQ; ++i) s[i][t][e] = T(-INFINITY);
        }
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            T again;
            if (run[i].template take<KT / 16>(s[i], again)) y[i].times(again);
        }
#pragma unroll
        for (int t = 0; t < KT / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const T* row = vs + (16 * t + M::row_of(e, g)) * Staged<T, D, KT>::PITCH + z.c0;
#pragma unroll
                for (int blk = 0; blk < Columns<T, W>::BLOCKS; ++blk) {
                    if (z.ends(blk * 16 * Columns<T, W>::NV)) break;
                    const auto left = Columns<T, W>::across(row, blk);
#pragma unroll
                    for (int c = 0; c < Columns<T, W>::NV; ++c)
#pragma unroll
                        for (int i = 0; i < RQ; ++i) y[i].acc[blk][c] = M::mul(left[c], s[i][t][e], y[i].acc[blk][c]);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < RQ; ++i) {
        const int r = r0 + 16 * i + (lane & 15);
        const T sum = fold_row(run[i].sum, Sum());
        if (r >= a.rows) continue;
        if (a.parts == 1) {
            const int64_t to = dense_row<T>(a, b, kvh, r);
            y[i].times(sum == T(0) ? T(0) : T(1) / sum);
            T* out = (T*)a.y_out + to * width;
            y[i].each([&](int c, const auto& values) {
                if (c < z.mine) store_run(out, z.c0 + c, width, values);
            });
            if (g == 0 && z.c0 == 0) ((T*)a.lse_out)[to] = sum == T(0) ? T(-INFINITY) : M::lse(run[i].top, sum);
        } else {
            const int64_t to = ((int64_t)part * a.batch * a.kv_heads + problem) * a.rows + r;
            T* out = (T*)a.parts_y + to * D;
            y[i].each([&](int c, const auto& values) {
                if (c < z.mine) store_run(out, z.c0 + c, D, values);
            });
            if (g == 0 && z.c0 == 0) ((T*)a.parts_m)[to] = run[i].top, ((T*)a.parts_l)[to] = sum;
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward
// where part `part` of `n` rows or states begins: on whole slabs
__device__ __forceinline__ int part_of(const Args& a, int part, int n, int slab) { return min(n, (int)((int64_t)((n + slab - 1) / slab) * part / a.parts) * slab); }

// what weights of a row are relative to: a row without weight has none anywhere
template <typename T>
__device__ __forceinline__ T level_of(T lse) {
    return lse == T(-INFINITY) ? T(INFINITY) : lse * (T)Matrix<T>::base;
}

// The gradients of the states: a workgroup takes 64 RK states (of four waves), a wave (or two) 16 RK of them in its registers, and walks over the rows of a part of them, RT at a time
// through LDS.
template <typename T, int D>
struct StatesShape {
    typedef Halves<T, D> Z;
    static constexpr int RT = Z::H == 1 ? 32 : 16, RK = sizeof(T) == 8 && D <= 32 ? 2 : 1, STATES = 16 * RK * Z::GROUPS;  // (float: where pieces do not serve)
    static constexpr int TILES = 2 * Staged<T, D, RT>::BYTES + 2 * RT * (int)sizeof(T), LDS = TILES + Z::bytes(2);
};

template <typename T, int D, int THREADS = 256, bool LATE = false>
__device__ __forceinline__ void states_gradient_tile(const Args& a, char* lds, int problem, int part, int first_state) {
    typedef Matrix<T> M;
    typedef StatesShape<T, D> S;
    typedef Halves<T, D> Z;
    constexpr int RT = S::RT, RK = S::RK, N = Vec<T>::N, W = Z::W, C = W / (4 * N), PITCH = Staged<T, D, RT, THREADS>::PITCH;
    static_assert(Z::H == 1 || (RK == 1 && THREADS == 256), "two tiles of scores meet at a time");
    T *qs = reinterpret_cast<T*>(lds), *gs = qs + RT * PITCH, *levels = gs + RT * PITCH, *deltas = levels + RT;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int width = Z::H > 1 && !LATE ? D : a.width;
    const Z z(a.width);  // (asked at every step whether its share ends, also where that is known: without the branches the compiler reads further ahead and spills 64 registers)
    int turn = 0;
    const int b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), k0 = first_state + z.group * 16 * RK;
    const int begin = part_of(a, part, a.rows, RT), end = part_of(a, part + 1, a.rows, RT);
    const T* q = (const T*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const T* dy = (const T*)a.dy.p + b * a.dy.batch + (int64_t)kvh * a.group * a.dy.head;
    const T* k = (const T*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const T* v = (const T*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), dy_rows(a, a.dy);
    Columns<T, W> dk[RK], dv[RK];
#pragma unroll
    for (int i = 0; i < RK; ++i) dk[i].clear(), dv[i].clear();
    if (first_state < n) {
        Fragment<T, W, D, LATE> kf[RK], vf[RK];
#pragma unroll
        for (int i = 0; i < RK; ++i) {
            const int key = min(k0 + 16 * i + (lane & 15), n - 1);
            kf[i].load(k + key * a.k.row, width, (T)(a.scale * M::base), z.c0);
            vf[i].load(v + key * a.v.row, width, T(1), z.c0);
        }
        Staged<T, D, RT, THREADS, LATE> qt, gt;
        T level = 0, delta = 0;
        auto fetch = [&](int r0) {
            qt.fetch(q, q_rows, r0, end, width);
            gt.fetch(dy, dy_rows, r0, end, width);
            if (threadIdx.x < RT) {
                const int r = r0 + threadIdx.x;
                level = T(INFINITY), delta = 0;
                if (r < end) {
                    const int64_t at = dense_row<T>(a, b, kvh, r);
                    level = level_of(((const T*)a.lse)[at]);
                    delta = ((const T*)a.delta)[at];
                }
            }
        };
        if (begin < end) fetch(begin);
        for (int r0 = begin; r0 < end; r0 += RT) {
            __syncthreads();
            qt.store(qs, width);
            gt.store(gs, width);
            if (threadIdx.x < RT) levels[threadIdx.x] = level, deltas[threadIdx.x] = delta;
            __syncthreads();
            if (r0 + RT < end) fetch(r0 + RT);
#pragma unroll
            for (int t = 0; t < RT / 16; ++t) {
                typename M::acc s[RK], dp[RK];
#pragma unroll
                for (int i = 0; i < RK; ++i) s[i] = dp[i] = typename M::acc{};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (z.ends(c * 4 * N)) break;
                    const typename Vec<T>::type left = Staged<T, D, RT, THREADS>::along(qs + z.c0, 16 * t, c), down = Staged<T, D, RT, THREADS>::along(gs + z.c0, 16 * t, c);
#pragma unroll
                    for (int e = 0; e < N; ++e)
#pragma unroll
                        for (int i = 0; i < RK; ++i) s[i] = M::mul(left[e], kf[i].g[c][e], s[i]);
#pragma unroll
                    for (int e = 0; e < N; ++e)
#pragma unroll
                        for (int i = 0; i < RK; ++i) dp[i] = M::mul(down[e], vf[i].g[c][e], dp[i]);
                }
                if constexpr (Z::H > 1) {
                    typename M::acc* halves[2] = {&s[0], &dp[0]};
                    z.meet(reinterpret_cast<T*>(lds + S::TILES), turn, halves);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 16 * t + M::row_of(e, g);
                    const T lev = levels[r], del = deltas[r];
#pragma unroll
                    for (int i = 0; i < RK; ++i) {
                        s[i][e] = lev == T(INFINITY) ? T(0) : M::weight(s[i][e] - lev);
                        dp[i][e] = s[i][e] * (dp[i][e] - del);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 16 * t + M::row_of(e, g);
#pragma unroll
                    for (int blk = 0; blk < Columns<T, W>::BLOCKS; ++blk) {
                        if (z.ends(blk * 16 * Columns<T, W>::NV)) break;
                        const auto of_values = Columns<T, W>::across(gs + r * PITCH + z.c0, blk), of_keys = Columns<T, W>::across(qs + r * PITCH + z.c0, blk);
#pragma unroll
                        for (int c = 0; c < Columns<T, W>::NV; ++c)
#pragma unroll
                            for (int i = 0; i < RK; ++i) dv[i].acc[blk][c] = M::mul(of_values[c], s[i][e], dv[i].acc[blk][c]);
#pragma unroll
                        for (int c = 0; c < Columns<T, W>::NV; ++c)
#pragma unroll
                            for (int i = 0; i < RK; ++i) dk[i].acc[blk][c] = M::mul(of_keys[c], dp[i][e], dk[i].acc[blk][c]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RK; ++i) {
        const int key = k0 + 16 * i + (lane & 15);
        if (key >= a.keys) continue;
        const int64_t to = part * a.part_size + (((int64_t)b * a.keys + key) * a.kv_heads + kvh) * width;
        // (behind the last state: what its stand-in came to is not the gradient, which is zero)
        const bool there = key < n;
        auto put = [&](T* out, const Columns<T, W>& sums, T factor) {
            sums.each([&](int c, const auto& values) {
                T run[Columns<T, W>::NV];
#pragma unroll
                for (int e = 0; e < Columns<T, W>::NV; ++e) run[e] = there ? values[e] * factor : T(0);
                if (c < z.mine) store_run(out + to, z.c0 + c, width, run);
            });
        };
        put((T*)a.dk, dk[i], (T)a.scale);
        put((T*)a.dv, dv[i], T(1));
    }
}

// The gradient of the rows: as the forward pass, with the weights known from lse.
template <typename T, int D>
struct RowsShape {
    typedef Halves<T, D> Z;
    static constexpr int KT = Z::H == 1 ? 32 : 16, RQ = sizeof(T) == 8 && D <= 32 ? 2 : 1, ROWS = 16 * RQ * Z::GROUPS;
    static constexpr int TILES = 2 * Staged<T, D, KT>::BYTES, LDS = TILES + Z::bytes(2);
};

template <typename T, int D, int THREADS = 256, bool LATE = false>
__device__ __forceinline__ void rows_gradient_tile(const Args& a, char* lds, int problem, int part, int first_row) {
    typedef Matrix<T> M;
    typedef RowsShape<T, D> S;
    typedef Halves<T, D> Z;
    constexpr int KT = S::KT, RQ = S::RQ, N = Vec<T>::N, W = Z::W, C = W / (4 * N), PITCH = Staged<T, D, KT, THREADS>::PITCH;
    static_assert(Z::H == 1 || (RQ == 1 && THREADS == 256), "two tiles of scores meet at a time");
    T *ks = reinterpret_cast<T*>(lds), *vs = ks + KT * PITCH;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int width = Z::H > 1 && !LATE ? D : a.width;
    const Z z(width);
    int turn = 0;
    const int b = problem / a.kv_heads, kvh = problem - b * a.kv_heads;
    const int n = count_of(a, b), begin = part_of(a, part, n, KT), end = part_of(a, part + 1, n, KT);
    const T* q = (const T*)a.q.p + b * a.q.batch + (int64_t)kvh * a.group * a.q.head;
    const T* dy = (const T*)a.dy.p + b * a.dy.batch + (int64_t)kvh * a.group * a.dy.head;
    const T* k = (const T*)a.k.p + b * a.k.batch + kvh * a.k.head;
    const T* v = (const T*)a.v.p + b * a.v.batch + kvh * a.v.head;
    const Rows q_rows(a, a.q), dy_rows(a, a.dy), k_rows(a.k), v_rows(a.v);
    const int r0 = first_row + z.group * 16 * RQ;
    Fragment<T, W, D, LATE> qf[RQ], gf[RQ];
    Columns<T, W> dq[RQ];
    T level[RQ], delta[RQ];
#pragma unroll
    for (int i = 0; i < RQ; ++i) {
        const int r = min(r0 + 16 * i + (lane & 15), a.rows - 1);
        qf[i].load(q + q_rows.at(r), width, (T)(a.scale * M::base), z.c0);
        gf[i].load(dy + dy_rows.at(r), width, T(1), z.c0);
        const int64_t at = dense_row<T>(a, b, kvh, r);
        level[i] = level_of(((const T*)a.lse)[at]);
        delta[i] = ((const T*)a.delta)[at];
        dq[i].clear();
    }
    Staged<T, D, KT, THREADS, LATE> kt, vt;
    if (begin < end) {
        kt.fetch(k, k_rows, begin, end, width);
        vt.fetch(v, v_rows, begin, end, width);
    }
    for (int first = begin; first < end; first += KT) {
        __syncthreads();
        kt.store(ks, width);
        vt.store(vs, width);
        __syncthreads();
        if (first + KT < end) {
            kt.fetch(k, k_rows, first + KT, end, width);
            vt.fetch(v, v_rows, first + KT, end, width);
        }
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            typename M::acc s[RQ], dp[RQ];
#pragma unroll
            for (int i = 0; i < RQ; ++i) s[i] = dp[i] = typename M::acc{};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (z.ends(c * 4 * N)) break;
                const typename Vec<T>::type left = Staged<T, D, KT, THREADS>::along(ks + z.c0, 16 * t, c), down = Staged<T, D, KT, THREADS>::along(vs + z.c0, 16 * t, c);
#pragma unroll
                for (int e = 0; e < N; ++e)
#pragma unroll
                    for (int i = 0; i < RQ; ++i) {
                        s[i] = M::mul(left[e], qf[i].g[c][e], s[i]);
                        dp[i] = M::mul(down[e], gf[i].g[c][e], dp[i]);
                    }
            }
            if constexpr (Z::H > 1) {
                typename M::acc* halves[2] = {&s[0], &dp[0]};
                z.meet(reinterpret_cast<T*>(lds + S::TILES), turn, halves);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool there = first + 16 * t + M::row_of(e, g) < end;
#pragma unroll
                for (int i = 0; i < RQ; ++i) dp[i][e] = there ? M::weight(s[i][e] - level[i]) * (dp[i][e] - delta[i]) : T(0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const T* row = ks + (16 * t + M::row_of(e, g)) * PITCH + z.c0;
#pragma unroll
                for (int blk = 0; blk < Columns<T, W>::BLOCKS; ++blk) {
                    if (z.ends(blk * 16 * Columns<T, W>::NV)) break;
                    const auto left = Columns<T, W>::across(row, blk);
#pragma unroll
                    for (int c = 0; c < Columns<T, W>::NV; ++c)
#pragma unroll
                        for (int i = 0; i < RQ; ++i) dq[i].acc[blk][c] = M::mul(left[c], dp[i][e], dq[i].acc[blk][c]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RQ; ++i) {
        const int r = r0 + 16 * i + (lane & 15);
        if (r >= a.rows) continue;
        T* out = (T*)a.dq + part * a.part_size + dense_row<T>(a, b, kvh, r) * width;
        dq[i].times((T)a.scale);
        dq[i].each([&](int c, const auto& values) {
            if (c < z.mine) store_run(out, z.c0 + c, width, values);
        });
    }
}

}  // namespace
}  // namespace dali_hip

#endif
