// Layer normalisation along the last axis and its gradient.
//
//   mean = sum(x) / n,  rstd = 1 / sqrt(sum((x - mean)^2) / n + epsilon),  y = (x - mean) rstd gamma + beta
//   u = (x - mean) rstd,  a = dy gamma,  dx = rstd (a - mean(a) - u mean(a u)),  dgamma = sum over rows of dy u,  dbeta = that of dy
//
// Sums are held in the operands' own type (32 bits or more). The variance is the mean of squared distances from the mean, with the mean's own
// rounding error taken out again (x - mean sums to delta n where the mean is off by delta): rows far from zero keep their digits. Rows for which
// this is not enough, because delta is most of the distances or because sums pass the type's range, are taken again (norm_apart).
#include <algorithm>
#include <type_traits>

#include "row_math.h"

namespace dali_hip {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct NormArgs {
    const T *x, *gamma, *beta;
    T *y, *mean, *rstd;
    long rows, stride;
    int width;
    T epsilon;
};

// Sums over the team of TEAM threads that holds a row: lanes of a wave, or whole waves of a workgroup, all of which meet once per call. `scratch` has two halves
// that take turns, so that a wave may write the next sums while another still reads these.
template <typename T, int TEAM, int TEAMS = 1>
struct TeamScratch {
    T v[TEAM > 64 ? 2 : 1][TEAM > 64 ? TEAMS * TEAM / 64 : 1][2];
};
// (AT_ONCE: waves whose sums are read side by side, in as many registers)
template <int TEAM, int AT_ONCE = 16, typename T, int TEAMS>
__device__ __forceinline__ void team_sum(T& p, T& q, TeamScratch<T, TEAM, TEAMS>& scratch, int& turn) {
    p = fold_lanes<(TEAM < 64 ? TEAM : 64)>(p, Sum());
    q = fold_lanes<(TEAM < 64 ? TEAM : 64)>(q, Sum());
    if constexpr (TEAM > 64) {
        auto& s = scratch.v[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6][0] = p, s[threadIdx.x >> 6][1] = q;
        __syncthreads();
        const int from = TEAMS == 1 ? 0 : threadIdx.x / TEAM * (TEAM / 64);
        p = s[from][0], q = s[from][1];
#pragma unroll AT_ONCE
        for (int w = 1; w < TEAM / 64; ++w) p += s[from + w][0], q += s[from + w][1];
    }
}

template <typename T>
__device__ __forceinline__ T root_of(T variance, T epsilon) {
    // (below zero by rounding alone; a NaN stays)
    return T(1) / sqrt((variance < T(0) ? T(0) : variance) + epsilon);
}

// Whether a row's variance can be taken as the mean square `spread` of its distances from the mean less the square of their own mean `off`: that keeps its digits (three
// quarters of the spread are left, or what is lost is nothing beside epsilon), and nothing has passed the type's range.
template <typename T>
__device__ __forceinline__ bool settled(T off, T spread, T epsilon) {
    return (off * off <= T(0.25) * spread + T(1.0 / 4096) * epsilon) & (spread < T(INFINITY));
}

// A row that is not is marked by an rstd below 0 and taken again once its team is through with all others: its y is not written until then, so it is still there where
// y takes its place, and the kernels' registers stay those of ordinary rows (as further passes over a row in registers 72 became 76 to 100, and
// 65536x200 took 24.0 us instead of 21.4).
template <typename T>
__device__ __forceinline__ T mark(T spread) {
    return spread < T(INFINITY) ? T(-1) : T(-2);
}

// The row is read times a power of two where something passed the range (so 2^31 of the largest squares do not), and the distances are made good by their mean
// before the squares are taken: they are small multiples of the values' last place where that matters, so both differences are exact, and a row
// of one value has distances of 0. Four readings a value at a time, the later ones in the caches: 8192x1024 of nothing but such rows 27 us, of others 11.7.
template <typename T>
struct Scaled;
template <>
struct Scaled<float> {
    static constexpr float down = 0x1p-81f, up = 0x1p81f;
};
template <>
struct Scaled<double> {
    static constexpr double down = 0x1p-540, up = 0x1p540;
};
template <int TEAM, typename T, typename Scratch>
__device__ __forceinline__ void norm_apart(const NormArgs<T>& a, long r, int l, T down, Scratch& scratch, int& turn) {
    const T* x = a.x + r * a.stride;
    const T count = a.width;
    T s = 0, off = 0, rest = 0, square = 0, none = 0;
#pragma unroll 1
    for (long c = l; c < a.width; c += TEAM) s += x[c] * down;
    team_sum<TEAM, 1>(s, none, scratch, turn);
    const T near = s / count;
#pragma unroll 1
    for (long c = l; c < a.width; c += TEAM) off += x[c] * down - near;
    team_sum<TEAM, 1>(off, none, scratch, turn);
    off /= count;
#pragma unroll 1
    for (long c = l; c < a.width; c += TEAM) {
        const T d = (x[c] * down - near) - off;
        rest += d;
        square += d * d;
    }
    team_sum<TEAM, 1>(rest, square, scratch, turn);
    rest /= count;
    T variance = square / count - rest * rest;
    variance = variance < T(0) ? T(0) : variance;
    // (scaled down, epsilon may vanish: beside any variance that is not 0 it is nothing)
    const T unit = variance == T(0) ? root_of(variance, a.epsilon) : root_of(variance, a.epsilon * down * down);
    T* y = a.y + r * a.width;
#pragma unroll 1
    for (long c = l; c < a.width; c += TEAM) {
        const T u = (((x[c] * down - near) - off) - rest) * unit;
        y[c] = u * (a.gamma ? a.gamma[c] : T(1)) + (a.beta ? a.beta[c] : T(0));
    }
    if (l == 0) {
        const T mean = (near + off) + rest;
        a.mean[r] = down < T(1) ? mean * Scaled<T>::up : mean;
        a.rstd[r] = variance == T(0) ? unit : unit * down;
    }
}
template <int TEAM, int TEAMS, typename T, typename Scratch>
__device__ __forceinline__ void norm_marked(const NormArgs<T>& a, Scratch& scratch, int& turn) {
    int l = threadIdx.x % TEAM;
    asm volatile("" : "+v"(l)::"memory");  // (no address is kept in registers for this)
#pragma unroll 1
    for (long first = (long)blockIdx.x * TEAMS; first < a.rows; first += (long)gridDim.x * TEAMS) {
        const long r = first + threadIdx.x / TEAM;
        if (r >= a.rows) continue;
        T marked = l == 0 ? a.rstd[r] : T(0), none = 0;  // (of the thread that wrote it)
        team_sum<TEAM, 1>(marked, none, scratch, turn);
        if (marked < T(0)) norm_apart<TEAM>(a, r, l, marked == mark(T(0)) ? T(1) : Scaled<T>::down, scratch, turn);
    }
}

// A team of TEAM threads per row, which lives in their registers, E groups of 16 bytes to a thread: read once, written once, which bounds it. WHOLE: the teams' groups are
// the row exactly. The weights stay in registers from row to row where they fit. 8192x1024 11.6 us (5.8 TB/s), 65536x1024 89 us (6.0), 32768x4096 183 us (5.9); 8x1024 4.2 us
// among others, 2.9 of them on the device.
// (the bound on waves: of 3001x2047 in double 18.4 us, without it 19.5; of 32768x2999 in float 150, without it 141)
template <typename T, int TEAM, int E, bool WHOLE, bool PAST>
__global__ __launch_bounds__(TEAM > kThreads ? TEAM : kThreads, TEAM == 256 && E == 4 && sizeof(T) == 8 ? 5 : 1) void norm_team(NormArgs<T> a) {
    constexpr int N = Vec<T>::N, BLOCK = TEAM > kThreads ? TEAM : kThreads, TEAMS = BLOCK / TEAM;
    constexpr bool HOLD = E * N <= 16, LONG = TEAM > 8;  // (8 threads are given the shortest rows)
    __shared__ TeamScratch<T, TEAM> scratch;
    int turn = 0;
    const int l = threadIdx.x % TEAM;
    const T count = a.width;
    T gamma[HOLD ? E : 1][N], beta[HOLD ? E : 1][N];
    auto weights = [&](int e, T (&g)[N], T (&b)[N]) {
        const int c = (l + e * TEAM) * N;
        if (a.gamma) {
            load_group(a.gamma, c, a.width, T(0), g);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = T(1);
        }
        if (a.beta) {
            load_group(a.beta, c, a.width, T(0), b);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) b[i] = T(0);
        }
    };
    if constexpr (HOLD) {
#pragma unroll
        for (int e = 0; e < E; ++e) weights(e, gamma[e], beta[e]);
    }
    bool apart = false;
    for (long first = (long)blockIdx.x * TEAMS; first < a.rows; first += (long)gridDim.x * TEAMS) {
        const long row = first + threadIdx.x / TEAM, r = row < a.rows ? row : a.rows - 1;  // (a team without a row goes along with the last)
        const T* x = a.x + r * a.stride;
        typename Vec<T>::type group[E];
        T v[E][N];
        T s = 0, none = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) group[e] = ask_group<LONG, WHOLE>(x, (l + e * TEAM) * N, a.width);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            take_group<LONG, WHOLE>(group[e], (l + e * TEAM) * N, a.width, T(0), v[e]);
#pragma unroll
            for (int i = 0; i < N; ++i) s += v[e][i];
        }
        team_sum<TEAM>(s, none, scratch, turn);
        const T near = s / count;
        T off = 0, square = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[e][i] -= near;
                const T d = WHOLE || (l + e * TEAM) * N + i < a.width ? v[e][i] : T(0);
                off += d;
                square += d * d;
            }
        team_sum<TEAM>(off, square, scratch, turn);
        off /= count;
        const T spread = square / count;
        const bool plain = settled(off, spread, a.epsilon);
        apart |= !plain;
        const T rstd = root_of(spread - off * off, a.epsilon);
        if (row < a.rows) {
            if (l == 0) {
                a.mean[r] = near + off;
                a.rstd[r] = plain ? rstd : mark(spread);
            }
            if (!plain) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                T g[N], b[N];
                if constexpr (!HOLD) weights(e, g, b);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const T gi = HOLD ? gamma[HOLD ? e : 0][i] : g[i], bi = HOLD ? beta[HOLD ? e : 0][i] : b[i];
                    v[e][i] = (v[e][i] - off) * rstd * gi + bi;
                }
                store_group<PAST>(a.y + r * a.width, (l + e * TEAM) * N, a.width, v[e]);
            }
        }
    }
    if (__builtin_amdgcn_ballot_w64(apart) != 0) norm_marked<TEAM, TEAMS>(a, scratch, turn);
}

// Rows that no workgroup's registers hold, or not without spilling: a workgroup walks each three times, the later ones in the caches
template <typename T, bool PAST>
__global__ __launch_bounds__(1024) void norm_rows(NormArgs<T> a) {
    constexpr int N = Vec<T>::N, BLOCK = 1024;
    __shared__ TeamScratch<T, BLOCK> scratch;
    int turn = 0;
    const int groups = groups_of<T>(a.width);
    const T count = a.width;
    bool apart = false;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = a.x + r * a.stride;
        T* y = a.y + r * a.width;
        T s = 0, none = 0, v[N], g[N], b[N];
        for (int j = threadIdx.x; j < groups; j += BLOCK) {
            load_group(x, j * N, a.width, T(0), v);
#pragma unroll
            for (int i = 0; i < N; ++i) s += v[i];
        }
        team_sum<BLOCK>(s, none, scratch, turn);
        const T near = s / count;
        T off = 0, square = 0;
        for (int j = threadIdx.x; j < groups; j += BLOCK) {
            load_group(x, j * N, a.width, near, v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const T d = v[i] - near;
                off += d;
                square += d * d;
            }
        }
        team_sum<BLOCK>(off, square, scratch, turn);
        off /= count;
        const T spread = square / count;
        if (!settled(off, spread, a.epsilon)) {
            apart = true;
            if (threadIdx.x == 0) a.rstd[r] = mark(spread);
            continue;
        }
        const T rstd = root_of(spread - off * off, a.epsilon);
        for (int j = threadIdx.x; j < groups; j += BLOCK) {
            load_group(x, j * N, a.width, T(0), v);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = T(1), b[i] = T(0);
            if (a.gamma) load_group(a.gamma, j * N, a.width, T(0), g);
            if (a.beta) load_group(a.beta, j * N, a.width, T(0), b);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = ((v[i] - near) - off) * rstd * g[i] + b[i];
            store_group<PAST>(y, j * N, a.width, v);
        }
        if (threadIdx.x == 0) {
            a.mean[r] = near + off;
            a.rstd[r] = rstd;
        }
    }
    if (__builtin_amdgcn_ballot_w64(apart) != 0) norm_marked<BLOCK, 1>(a, scratch, turn);
}

template <typename T>
struct NormBackwardArgs {
    const T *dy, *x, *mean, *rstd, *gamma;
    T *dx, *dgamma, *dbeta;
    T* partial;  // [parts][2][width]
    long rows, dy_stride, x_stride;
    int width, parts;
};

// u = (x - mean) rstd of a row, from halves: x - mean may pass the type's range where x and mean do not. (Nothing is lost by it: what halving rounds off is
// below the smallest normal number, and an rstd that is finite stands for a deviation far above.)
template <typename T>
struct Normalised {
    T mean, twice;
    __device__ __forceinline__ Normalised(T row_mean, T rstd) : mean(row_mean * T(0.5)), twice(rstd * T(2)) {}
    __device__ __forceinline__ T operator()(T x) const { return (x * T(0.5) - mean) * twice; }
};

// the value of the lane D further on in its half (D = 8: of 16 lanes) or in the other half, without a condition on closer lanes
template <int D, typename T>
__device__ __forceinline__ T plus_across(T v) {
    if constexpr (D >= 16) {
        T a, b;
        halves_of<D>(v, a, b);
        return a + b;
    } else {
        static_assert(D == 8, "lanes 8, 16 or 32 apart");
        const auto rotated = [](unsigned w) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xf, 0xf, true); };
        if constexpr (sizeof(T) == 4) {
            return v + __builtin_bit_cast(T, rotated(__builtin_bit_cast(unsigned, v)));
        } else {
            const unsigned long long w = __builtin_bit_cast(unsigned long long, v);
            return v + __builtin_bit_cast(T, (unsigned long long)rotated((unsigned)(w >> 32)) << 32 | rotated((unsigned)w));
        }
    }
}

// The gradient with the rows in registers as above; a thread also keeps the sums of its columns over all rows that its team takes. At the end the teams of a
// workgroup are joined, lanes first and then waves through LDS, in halves, and the workgroup leaves one row of partial sums for each weight. So x and dy are read once for all
// three gradients. Bound by memory: 32768x4096 280 us (5.7 TB/s), 65536x1024 148 us (5.4); 8192x1024 22.3 us, of which 18 to 20 are this launch (a wave has four rows) and 2
// to 4 the fold; 3001x2047 in double 36 us. The next row is asked for before this one is worked on (8192x1024 24.2 without, 65536x1024 154).
template <typename T, int TEAM, int TEAMS, int E, bool WHOLE, bool WEIGHTS, bool PAST>
__global__ __launch_bounds__(TEAM * TEAMS) void norm_backward_team(NormBackwardArgs<T> a) {
    constexpr int N = Vec<T>::N, BLOCK = TEAM * TEAMS;
    constexpr bool LONG = TEAM > 8;  // (8 threads are given the shortest rows)
    // (waves that hold the same columns; LDS for half of them)
    constexpr int SPAN = TEAM > 64 ? TEAM : 64, SAME = BLOCK / SPAN;
    __shared__ TeamScratch<T, TEAM, TEAMS> scratch;
    __shared__ T joined[WEIGHTS && SAME > 1 ? SAME / 2 : 1][WEIGHTS && SAME > 1 ? 2 * E * N : 1][WEIGHTS && SAME > 1 ? SPAN : 1];
    int turn = 0;
    const int l = threadIdx.x % TEAM;
    const T count = a.width;
    T gamma[E][N], dgamma[E][N], dbeta[E][N];
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int i = 0; i < N; ++i) gamma[e][i] = T(1), dgamma[e][i] = dbeta[e][i] = T(0);
        if (a.gamma) load_group(a.gamma, (l + e * TEAM) * N, a.width, T(0), gamma[e]);
    }
    // The next row is under way while one is worked on, where the registers hold both
    constexpr bool AHEAD = TEAM <= 512 || E <= 2;
    typename Vec<T>::type asked_x[E], asked_dy[E];
    T mean, rstd;
    const long stride = (long)gridDim.x * TEAMS;
    auto ask = [&](long row) {
        const long r = row < a.rows ? row : a.rows - 1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            asked_x[e] = ask_group<LONG, WHOLE>(a.x + r * a.x_stride, (l + e * TEAM) * N, a.width);
            asked_dy[e] = ask_group<LONG, WHOLE>(a.dy + r * a.dy_stride, (l + e * TEAM) * N, a.width);
        }
        mean = a.mean[r], rstd = a.rstd[r];
    };
    if constexpr (AHEAD) ask((long)blockIdx.x * TEAMS + threadIdx.x / TEAM);
    for (long first = (long)blockIdx.x * TEAMS; first < a.rows; first += stride) {
        const long row = first + threadIdx.x / TEAM, r = row < a.rows ? row : a.rows - 1;
        const bool live = row < a.rows;  // (a team without a row goes along with the last, and adds nothing)
        if constexpr (!AHEAD) ask(row);
        const Normalised<T> normalised(mean, rstd);
        const T row_rstd = rstd;
        T u[E][N], d[E][N];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            take_group<LONG, WHOLE>(asked_x[e], (l + e * TEAM) * N, a.width, T(0), u[e]);
            take_group<LONG, WHOLE>(asked_dy[e], (l + e * TEAM) * N, a.width, T(0), d[e]);
        }
        if constexpr (AHEAD)
            if (first + stride < a.rows) ask(row + stride);
        T level = 0, along = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = WHOLE || (l + e * TEAM) * N + i < a.width;
                u[e][i] = in ? normalised(u[e][i]) : T(0);
                if constexpr (WEIGHTS) {
                    dgamma[e][i] += live ? d[e][i] * u[e][i] : T(0);
                    dbeta[e][i] += live ? d[e][i] : T(0);
                }
                d[e][i] *= gamma[e][i];
                level += d[e][i];
                along += d[e][i] * u[e][i];
            }
        team_sum<TEAM>(level, along, scratch, turn);
        level /= count;
        along /= count;
        if (live) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
#pragma unroll
                for (int i = 0; i < N; ++i) d[e][i] = row_rstd * ((d[e][i] - level) - u[e][i] * along);
                store_group<PAST>(a.dx + r * a.width, (l + e * TEAM) * N, a.width, d[e]);
            }
        }
    }
    if constexpr (WEIGHTS) {
        auto every = [&](auto&& f) {
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < N; ++i) f(dgamma[e][i], 2 * (e * N + i)), f(dbeta[e][i], 2 * (e * N + i) + 1);
        };
        if constexpr (TEAM < 64) {
            every([&](T& v, int) {
                if constexpr (TEAM <= 8) v = plus_across<8>(v);
                if constexpr (TEAM <= 16) v = plus_across<16>(v);
                v = plus_across<32>(v);
            });
        }
        const int at = threadIdx.x % SPAN, group = threadIdx.x / SPAN;
#pragma unroll
        for (int half = SAME / 2; half >= 1; half /= 2) {
            __syncthreads();
            if (group >= half && group < 2 * half) every([&](T& v, int k) { joined[group - half][k][at] = v; });
            __syncthreads();
            if (group < half) every([&](T& v, int k) { v += joined[group][k][at]; });
        }
        if (threadIdx.x < TEAM) {
            T* g = a.parts == 1 ? a.dgamma : a.partial + (long)blockIdx.x * 2 * a.width;
            T* b = a.parts == 1 ? a.dbeta : g + a.width;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                store_group(g, (l + e * TEAM) * N, a.width, dgamma[e]);
                store_group(b, (l + e * TEAM) * N, a.width, dbeta[e]);
            }
        }
    }
}

// Longer rows: dx by a workgroup that walks each row twice ...
template <typename T, bool PAST>
__global__ __launch_bounds__(1024) void norm_backward_rows(NormBackwardArgs<T> a) {
    constexpr int N = Vec<T>::N, BLOCK = 1024;
    __shared__ TeamScratch<T, BLOCK> scratch;
    int turn = 0;
    const int groups = groups_of<T>(a.width);
    const T count = a.width;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = a.x + r * a.x_stride, *dy = a.dy + r * a.dy_stride;
        T* dx = a.dx + r * a.width;
        const T mean = a.mean[r], rstd = a.rstd[r];
        const Normalised<T> normalised(mean, rstd);
        T level = 0, along = 0, u[N], d[N], g[N];
        auto load = [&](int j) {
            load_group(x, j * N, a.width, mean, u);
            load_group(dy, j * N, a.width, T(0), d);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = T(1);
            if (a.gamma) load_group(a.gamma, j * N, a.width, T(0), g);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                u[i] = normalised(u[i]);
                d[i] *= g[i];
            }
        };
        for (int j = threadIdx.x; j < groups; j += BLOCK) {
            load(j);
#pragma unroll
            for (int i = 0; i < N; ++i) level += d[i], along += d[i] * u[i];
        }
        team_sum<BLOCK>(level, along, scratch, turn);
        level /= count;
        along /= count;
        for (int j = threadIdx.x; j < groups; j += BLOCK) {
            load(j);
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = rstd * ((d[i] - level) - u[i] * along);
            store_group<PAST>(dx, j * N, a.width, d);
        }
    }
}

// ... and the weights by columns, over one part of the rows
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_weights(NormBackwardArgs<T> a) {
    const long c = (long)blockIdx.x * kThreads + threadIdx.x;  // (may pass 31 bits in the last workgroup)
    if (c >= a.width) return;
    T g = 0, b = 0;
#pragma unroll 4
    for (long r = blockIdx.y; r < a.rows; r += a.parts) {
        const T d = a.dy[r * a.dy_stride + c];
        g += d * Normalised<T>(a.mean[r], a.rstd[r])(a.x[r * a.x_stride + c]);
        b += d;
    }
    if (a.parts == 1) {
        a.dgamma[c] = g;
        a.dbeta[c] = b;
        return;
    }
    T* p = a.partial + (long)blockIdx.y * 2 * a.width + c;
    p[0] = g;
    p[a.width] = b;
}

// The parts in order: 16 threads of a column take every 16th part each, and are joined in a tree. Partial rows of dgamma and dbeta lie one behind the other, so
// both are columns of one matrix [parts, 2 width].
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_fold(NormBackwardArgs<T> a) {
    __shared__ T joined[16][17];
    const int i = threadIdx.x & 15, p = threadIdx.x >> 4;
    const long c = (long)blockIdx.x * 16 + i, columns = 2L * a.width;
    T s = 0;
    if (c < columns) {
        const T* from = a.partial + c;
#pragma unroll 16
        for (int k = p; k < a.parts; k += 16) s += from[k * columns];
    }
    joined[p][i] = s;
#pragma unroll
    for (int half = 8; half >= 1; half /= 2) {
        __syncthreads();
        if (p < half) joined[p][i] += joined[p + half][i];
    }
    __syncthreads();
    if (p == 0 && c < columns) (c < a.width ? a.dgamma[c] : a.dbeta[c - a.width]) = joined[0][i];
}

// Threads to a row and groups to a thread that hold a row of `groups` groups; false: none up to MOST. The forward pass, which holds a row and no sums, takes fewer threads
// with more groups (256 threads with 2, 512 with 1: 32768x1500 73 and 87 us; 256 with 4, 512 with 2: 32768x3000 143 and 149; 512 with 4, 1024 with 2: 16384x8192 182 and 188).
template <int MOST, typename F>
bool team_for(int groups, F launch) {
    auto with = [&](auto team, auto e) {
        launch(team, e);
        return true;
    };
    using std::integral_constant;
    if (groups <= 8) return with(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (groups <= 16) return with(integral_constant<int, 16>(), integral_constant<int, 1>());
    if (groups <= 32) return with(integral_constant<int, 32>(), integral_constant<int, 1>());
    if (groups <= 64) return with(integral_constant<int, 64>(), integral_constant<int, 1>());
    if (groups <= 128) return with(integral_constant<int, 64>(), integral_constant<int, 2>());
    if (groups <= 192) return with(integral_constant<int, 64>(), integral_constant<int, 3>());
    if (groups <= 256) return with(integral_constant<int, 64>(), integral_constant<int, 4>());
    if constexpr (MOST > 4096) {
        if (groups <= 512) return with(integral_constant<int, 256>(), integral_constant<int, 2>());
        if (groups <= 1024) return with(integral_constant<int, 256>(), integral_constant<int, 4>());
        if (groups <= 2048) return with(integral_constant<int, 512>(), integral_constant<int, 4>());
    }
    if (groups <= 512) return with(integral_constant<int, 512>(), integral_constant<int, 1>());
    if (groups <= 1024) return with(integral_constant<int, 512>(), integral_constant<int, 2>());
    if (groups <= 2048) return with(integral_constant<int, 1024>(), integral_constant<int, 2>());
    if (groups <= 4096) return with(integral_constant<int, 1024>(), integral_constant<int, 4>());
    if constexpr (MOST > 4096)
        if (groups <= 8192) return with(integral_constant<int, 1024>(), integral_constant<int, 8>());
    return false;
}

template <typename T>
int forward(NormArgs<T> a) {
    const bool past = past_caches(2.0 * sizeof(T) * a.rows * a.width);
    const int groups = groups_of<T>(a.width);
    // Rows of more than 4096 groups that are not whole do not fit the registers without spilling some. Held and walked three times (us): 4096x20000 180 and 155, 4096x31000 226
    // and 261, 8x20000 10.3 and 7.3; in double 4096x9001 227 and 158, 4096x15000 272 and 254, and whole 4096x16384 198 and 291.
    const bool walked = groups > 4096 && a.width != 8192 * Vec<T>::N && (groups <= 6144 || sizeof(T) == 8);
    const bool held = !walked && team_for<8192>(groups, [&](auto team, auto e) {
        constexpr int TEAM = decltype(team)::value, E = decltype(e)::value, BLOCK = TEAM > kThreads ? TEAM : kThreads, TEAMS = BLOCK / TEAM;
        const dim3 grid((unsigned)std::min((a.rows + TEAMS - 1) / TEAMS, 8192L * kThreads / BLOCK));
        either_way(past, [&](auto p) {
            either_way(a.width == TEAM * E * Vec<T>::N, [&](auto whole) {
                if constexpr (E < 8 || sizeof(T) == 4 || decltype(whole)::value)
                    hipLaunchKernelGGL((norm_team<T, TEAM, E, decltype(whole)::value, decltype(p)::value>), grid, dim3(BLOCK), 0, stream(), a);
            });
        });
    });
    if (!held)
        either_way(past, [&](auto p) { hipLaunchKernelGGL((norm_rows<T, decltype(p)::value>), dim3((unsigned)std::min(a.rows, 65536L)), dim3(1024), 0, stream(), a); });
    return launched("dali_hip_layer_norm");
}

template <typename T>
int backward(NormBackwardArgs<T> a) {
    const char* what = "dali_hip_layer_norm_backward";
    const bool past = past_caches(3.0 * sizeof(T) * a.rows * a.width);
    const long fit = (long)(kCarriedBytes / (2 * sizeof(T) * (size_t)a.width));  // rows of partial sums that there is room for
    const Carried carried;  // (to the launch that folds them)
    a.partial = (T*)carried.data();
    a.parts = 1;
    if (a.rows == 0) {
        if (a.dgamma) hipLaunchKernelGGL(norm_weights<T>, dim3((unsigned)(((long)a.width + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream(), a);
        return launched(what);
    }
    const bool held = team_for<4096>(groups_of<T>(a.width), [&](auto team, auto e) {
        constexpr int TEAM = decltype(team)::value, E = decltype(e)::value;
        // as many workgroups as the registers let run at once, each with all the rows that fall to it
        auto run = [&](auto teams) {
            constexpr int TEAMS = decltype(teams)::value, per_unit = TEAM > 64 || E == 4 ? 1 : TEAM == 64 && E == 1 ? 4 : 2;
            a.parts = (int)std::max(1L, std::min({(a.rows + TEAMS - 1) / TEAMS, 256L * per_unit, fit}));
            const dim3 grid((unsigned)a.parts);
            either_way(past, [&](auto p) {
                either_way(a.width == TEAM * E * Vec<T>::N, [&](auto whole) {
                    either_way(a.dgamma != nullptr, [&](auto weights) {
                        hipLaunchKernelGGL((norm_backward_team<T, TEAM, TEAMS, E, decltype(whole)::value, decltype(weights)::value, decltype(p)::value>), grid, dim3(TEAM * TEAMS), 0,
                                           stream(), a);
                    });
                });
            });
        };
        // Two teams of 512 threads share a workgroup and its partial sums; where rows are many and a team holds two groups to a thread, one team to a compute unit
        // streams faster (32768x4096: 280 us, two teams 305; 4000x4096: 46 and 43)
        if constexpr (TEAM == 512) {
            if (E == 2 && a.rows >= 8192) run(std::integral_constant<int, 1>());
            else run(std::integral_constant<int, 2>());
        } else {
            run(std::integral_constant<int, (TEAM > 512 ? 1 : 512 / TEAM)>());
        }
    });
    if (!held && a.dgamma) {
        // (the weights first: dx may take the place of x or dy)
        a.parts = (int)std::max(1L, std::min({64L, a.rows, fit}));
        hipLaunchKernelGGL(norm_weights<T>, dim3((unsigned)(((long)a.width + kThreads - 1) / kThreads), a.parts), dim3(kThreads), 0, stream(), a);
    }
    if (launched(what)) return DALI_HIP_ERROR;
    if (a.dgamma && a.parts > 1) hipLaunchKernelGGL(norm_fold<T>, dim3((unsigned)((2L * a.width + 15) / 16)), dim3(kThreads), 0, stream(), a);
    if (launched(what)) return DALI_HIP_ERROR;
    if (!held)
        either_way(past, [&](auto p) { hipLaunchKernelGGL((norm_backward_rows<T, decltype(p)::value>), dim3((unsigned)std::min(a.rows, 65536L)), dim3(1024), 0, stream(), a); });
    return launched(what);
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_layer_norm(int dtype, int64_t rows, int width, const void* x, int64_t x_stride, const void* gamma, const void* beta, double epsilon, void* y,
                                   void* mean, void* rstd) {
    const char* what = "dali_hip_layer_norm";
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (rows < 0 || width < 1) return fail("%s: %lld rows of %d values", what, (long long)rows, width);
    if (!(epsilon >= 0) || epsilon > 1e30) return fail("%s: epsilon must be from 0 to 1e30 (got %g)", what, epsilon);
    if (rows == 0) return DALI_HIP_OK;
    if (!x || !y || !mean || !rstd) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (check_spans(what, {Span("y", y, rows * width, size), Span("mean", mean, rows, size), Span("rstd", rstd, rows, size)},
                    {Span("x", x, rows, width, x_stride, size), Span("gamma", gamma, width, size), Span("beta", beta, width, size)}, 1))
        return DALI_HIP_ERROR;
    if (off_elements({x, gamma, beta, y, mean, rstd}, size)) return fail("%s: an address is off its type's size", what);
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT)
        return forward<float>({(const float*)x, (const float*)gamma, (const float*)beta, (float*)y, (float*)mean, (float*)rstd, (long)rows, (long)x_stride, width, (float)epsilon});
    return forward<double>({(const double*)x, (const double*)gamma, (const double*)beta, (double*)y, (double*)mean, (double*)rstd, (long)rows, (long)x_stride, width, epsilon});
}

extern "C" int dali_hip_layer_norm_backward(int dtype, int64_t rows, int width, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* mean,
                                            const void* rstd, const void* gamma, void* dx, void* dgamma, void* dbeta) {
    const char* what = "dali_hip_layer_norm_backward";
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (rows < 0 || width < 1) return fail("%s: %lld rows of %d values", what, (long long)rows, width);
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return fail("%s: NULL argument", what);
    if (!dgamma != !dbeta) return fail("%s: dgamma and dbeta come together", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (check_spans(what, {Span("dx", dx, rows * width, size), Span("dgamma", dgamma, width, size), Span("dbeta", dbeta, width, size)},
                    {Span("dy", dy, rows, width, dy_stride, size), Span("x", x, rows, width, x_stride, size), Span("mean", mean, rows, size), Span("rstd", rstd, rows, size),
                     Span("gamma", gamma, width, size)},
                    2))
        return DALI_HIP_ERROR;
    if (off_elements({dy, x, mean, rstd, gamma, dx, dgamma, dbeta}, size)) return fail("%s: an address is off its type's size", what);
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT)
        return backward<float>({(const float*)dy, (const float*)x, (const float*)mean, (const float*)rstd, (const float*)gamma, (float*)dx, (float*)dgamma, (float*)dbeta, nullptr,
                                (long)rows, (long)dy_stride, (long)x_stride, width, 1});
    return backward<double>({(const double*)dy, (const double*)x, (const double*)mean, (const double*)rstd, (const double*)gamma, (double*)dx, (double*)dgamma, (double*)dbeta,
                             nullptr, (long)rows, (long)dy_stride, (long)x_stride, width, 1});
}
