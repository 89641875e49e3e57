// Log probabilities of given tokens under softmax(logits), row by row, with the entropy of the row and its best alternatives; and the gradient.
//
//   m = max x,  S = sum e^(x - m),  T = sum e^(x - m) (x - m)
//   lse = m + ln S,  log p(t) = x_t - lse,  entropy = -sum p ln p = ln S - T / S
//   d x = d log p(t) (delta_t - p) - d entropy p (ln p + entropy)
//
// A value of -inf (or far below m) has weight 0 and adds nothing to the entropy. A row of -inf alone has lse = -inf, entropy 0 and no gradient.
// A NaN or +inf makes its row's results NaN. A token outside [0, vocab) stands for none: its log probability is 0 and has no gradient.
#include <algorithm>
#include <type_traits>

#include "row_math.h"

namespace dali_hip {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct Real;
template <>
struct Real<float> {
    static constexpr float lowest = -3.402823466e+38f;  // where a running maximum begins: finite, so that no difference to it is NaN
    static constexpr float under = -1e30f;              // an exponent whose weight is 0: what an infinite one is replaced by where it meets a weight
    static __device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }
    static __device__ __forceinline__ float ln(float s) { return logf(s); }
};
template <>
struct Real<double> {
    static constexpr double lowest = -1.7976931348623157e+308;
    static constexpr double under = -1e300;
    static __device__ __forceinline__ double weight(double d) { return exp(d); }
    static __device__ __forceinline__ double ln(double s) { return log(s); }
};

template <typename T>
struct LogProbArgs {
    const T* logits;
    const int* tokens;
    T *log_probs, *entropy, *lse, *top;
    int* top_tokens;
    long rows, stride;
    int vocab, k;
    // rows in segments: `per` groups of Vec<T>::N logits to a segment
    int segments, per;
    T* sums;         // [rows][segments][3]
    T* best;         // [rows][segments][k]
    int* positions;  // the same
    unsigned* counters;
    int counter_step;
};

// of two entries the better: the larger value, the lower position among equals
template <typename T>
__device__ __forceinline__ bool better(T v, int i, T w, int j) {
    return v > w || (v == w && i < j);
}

// a NaN counts as -inf among the alternatives
template <typename T>
__device__ __forceinline__ T ranked(T v) {
    return Max()(v, T(-INFINITY));
}

// the best entry that LANES neighbouring lanes hold
template <int LANES, int D = 1, typename T>
__device__ __forceinline__ void best_of_lanes(T& v, int& i) {
    if constexpr (D < LANES) {
        T va, vb;
        int ia, ib;
        halves_of<D>(v, va, vb);
        halves_of<D>(i, ia, ib);
        const bool first = better(va, ia, vb, ib);
        v = first ? va : vb;
        i = first ? ia : ib;
        best_of_lanes<LANES, D * 2>(v, i);
    }
}

template <typename T>
__host__ __device__ __forceinline__ int groups_of(int vocab) {
    return vocab / Vec<T>::N + (vocab % Vec<T>::N != 0);
}

// group c / N of the row, with -inf in the place of what lies past its end
template <typename T>
__device__ __forceinline__ void load_group(const T* x, int c, int vocab, T (&v)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    if (c <= vocab - N) {
        const typename Vec<T>::type g = *reinterpret_cast<const typename Vec<T>::type*>(x + c);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = g[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = c + i < vocab ? x[c + i] : T(-INFINITY);
    }
}

// what a row's sums come to
template <typename T>
struct RowResult {
    T m, ln, lse;
    bool nothing;
};
template <typename T>
__device__ __forceinline__ RowResult<T> result_of(T m, T s) {
    const T ln = Real<T>::ln(s);
    return {m, ln, m + ln, s == T(0)};
}
template <typename T>
__device__ __forceinline__ void write_row(const LogProbArgs<T>& a, long r, const RowResult<T>& q, T s, T t, int token, T own) {
    a.lse[r] = q.nothing ? T(-INFINITY) : q.lse;
    a.entropy[r] = q.nothing ? T(0) : q.ln - t / s;
    a.log_probs[r] = token < 0 || token >= a.vocab ? T(0) : q.nothing ? T(-INFINITY) : (own - q.m) - q.ln;
}

// Rows that LANES lanes hold in registers, E groups each: every statistic is exact after one reading, and an alternative is one fold over what is left.
template <typename T, int LANES, int E>
__global__ __launch_bounds__(kThreads) void log_prob_short(LogProbArgs<T> a) {
    constexpr int N = Vec<T>::N;
    const int l = threadIdx.x % LANES;
    const long row = (long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    const long r = row < a.rows ? row : a.rows - 1;  // (lanes without a row go along with the last)
    const T* x = a.logits + r * a.stride;
    T v[E][N];
#pragma unroll
    for (int e = 0; e < E; ++e) load_group(x, (l + e * LANES) * N, a.vocab, v[e]);
    const int token = a.tokens[r];
    const T own = token >= 0 && token < a.vocab ? x[token] : T(0);
    T m = Real<T>::lowest;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < N; ++i) m = Max()(m, v[e][i]);
    m = fold_lanes<LANES>(m, Max());
    T s = 0, t = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const T d = v[e][i] - m, w = Real<T>::weight(d);
            s += w;
            t += w * Max()(d, Real<T>::under);
        }
    s = fold_lanes<LANES>(s, Sum());
    t = fold_lanes<LANES>(t, Sum());
    const RowResult<T> q = result_of(m, s);
    if (l == 0 && row < a.rows) write_row(a, r, q, s, t, token, own);
    // one alternative after the other; an entry that has been named is no longer free
    unsigned unnamed = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < N; ++i) unnamed |= ((l + e * LANES) * N + i < a.vocab ? 1u : 0u) << (e * N + i);
    for (int n = 0; n < a.k; ++n) {
        T bv = -INFINITY;
        int at = 0x7fffffff, slot = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const T w = ranked(v[e][i]);
                const bool take = (unnamed >> (e * N + i) & 1) && (w > bv || at == 0x7fffffff);
                bv = take ? w : bv;
                at = take ? (l + e * LANES) * N + i : at;
                slot = take ? e * N + i : slot;
            }
        const int mine = at;
        best_of_lanes<LANES>(bv, at);
        if (mine == at) unnamed &= ~(1u << slot);
        if (l == 0 && row < a.rows) {
            a.top[r * a.k + n] = q.nothing ? T(-INFINITY) : bv == T(-INFINITY) ? x[at] - q.lse : bv - q.lse;
            a.top_tokens[r * a.k + n] = at;
        }
    }
}

constexpr int kList = 512;   // entries that may be ranked at once
constexpr int kQuads = kThreads / 4;

// The k best of `n` entries in LDS, in order: an entry's place is the number of better ones
template <typename T, typename Put>
__device__ __forceinline__ void rank_list(const T* value, const int* position, int n, int k, Put put) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const T v = value[i];
        const int p = position[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += better(value[j], position[j], v, p) ? 1 : 0;
        if (place < k) put(place, v, p);
    }
}

// One workgroup per row, or per segment of a row: a thread walks its groups once with a running maximum, the sum of weights below it and the sum of weights
// times exponents, which are rescaled when the maximum rises (once per four groups). For the alternatives it also keeps its best group. Of the k units (quads of threads,
// or threads where more than 16 alternatives are asked for) with the best groups, the k-th best group's value and position bound the k best entries from below, and
// entries above that bound lie in those units alone: they are read again, what passes the bound is collected and ranked.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void log_prob_long(LogProbArgs<T> a) {
    constexpr int N = Vec<T>::N, U = 4;
    __shared__ T scratch[4], list[kList], key[TOP ? kThreads : 1], bound;
    __shared__ int places[kList], group[TOP ? kThreads : 1], unit[TOP ? DALI_HIP_MAX_ALTERNATIVES : 1], bound_group, count;
    __shared__ unsigned arrived;
    const int tid = threadIdx.x, lane = tid & 63;
    const long r = blockIdx.x / (unsigned)a.segments;
    const int segment = (int)(blockIdx.x - (unsigned)r * (unsigned)a.segments);
    const T* x = a.logits + r * a.stride;
    const int groups = groups_of<T>(a.vocab), begin = segment * a.per, end = min(groups, begin + a.per), whole = min(end, a.vocab / N);
    const int token = a.tokens[r];
    const T own = token >= 0 && token < a.vocab ? x[token] : T(0);
    T m = Real<T>::lowest, s = 0, t = 0, top = -INFINITY;
    int top_group = begin + tid < end ? begin + tid : 0x7fffffff;
    auto raise = [&](T to) {
        const T by = Max()(m - to, Real<T>::under), w = Real<T>::weight(by);
        t = w * (t + by * s);
        s *= w;
        m = to;
    };
    auto add = [&](T v) {
        const T d = v - m, w = Real<T>::weight(d);
        s += w;
        t += w * Max()(d, Real<T>::under);
    };
    int j = begin + tid;
    for (; j + (U - 1) * kThreads < whole; j += U * kThreads) {
        typename Vec<T>::type v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const typename Vec<T>::type*>(x + (long)(j + u * kThreads) * N);
        T high = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            T g = v[u][0];
#pragma unroll
            for (int i = 1; i < N; ++i) g = Max()(g, v[u][i]);
            high = Max()(high, g);
            if (TOP && g > top) top = g, top_group = j + u * kThreads;
        }
        raise(high);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) add(v[u][i]);
    }
    for (; j < end; j += kThreads) {
        T v[N];
        load_group(x, j * N, a.vocab, v);
        T g = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) g = Max()(g, v[i]);
        if (TOP && g > top) top = g, top_group = j;
        raise(Max()(m, g));
#pragma unroll
        for (int i = 0; i < N; ++i) add(v[i]);
    }
    // the workgroup's sums
    const T mine = m;
    m = fold_block<kThreads>(m, scratch, Max());
    {
        const T by = Max()(mine - m, Real<T>::under), w = Real<T>::weight(by);
        t = block_sum<kThreads>(w * (t + by * s), scratch);
        s = block_sum<kThreads>(w * s, scratch);
    }
    int found = 0;
    if constexpr (TOP) {
        const bool quads = a.k <= 16;
        if (quads) {
            best_of_lanes<4>(top, top_group);
            if ((tid & 3) == 0) key[tid >> 2] = top, group[tid >> 2] = top_group;
        } else {
            key[tid] = top, group[tid] = top_group;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        if (quads) {
            if (tid < 64) {
                T kv = key[lane];
                int kg = group[lane];
                for (int n = 0; n < a.k; ++n) {
                    T bv = kv;
                    int bg = kg;
                    best_of_lanes<64>(bv, bg);
                    if (kg == bg) {  // (a group belongs to one unit)
                        unit[n] = lane;
                        if (n == a.k - 1) bound = bv, bound_group = bg;
                        kv = -INFINITY, kg = 0x7fffffff;
                    }
                }
            }
        } else {
            int place = 0;
            for (int i = 0; i < kThreads; ++i) place += better(key[i], group[i], top, top_group) ? 1 : 0;
            if (place < a.k) unit[place] = tid;
            if (place == a.k - 1) bound = top, bound_group = top_group;
        }
        __syncthreads();
        // the units' entries again
        const T low = bound;
        const int low_group = bound_group, wide = quads ? 4 : 1, walks = (end - begin + kThreads - 1) / kThreads * wide;
        for (int i = tid; i < a.k * walks; i += kThreads) {
            const int n = i / walks, step = i - n * walks;
            const int g = begin + unit[n] * wide + (quads ? (step & 3) + (step >> 2) * kThreads : step * kThreads);
            if (g >= end) continue;
            T v[N];
            load_group(x, g * N, a.vocab, v);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const T w = ranked(v[e]);
                if (g * N + e < a.vocab && (w > low || (w == low && g <= low_group))) {
                    const int slot = atomicAdd(&count, 1);
                    if (slot < kList) list[slot] = w, places[slot] = g * N + e;
                }
            }
        }
        __syncthreads();
        found = count;
        if (found > kList) {
            // (so many of the best side by side in few units: one after the other over the whole segment)
            T last = INFINITY;
            int last_at = -1;
            for (int n = 0; n < a.k; ++n) {
                T bv = -INFINITY;
                int at = 0x7fffffff;
                for (long c = (long)begin * N + tid; c < min((long)a.vocab, (long)end * N); c += kThreads) {
                    const T w = ranked(x[c]);
                    if (better(last, last_at, w, (int)c) && better(w, (int)c, bv, at)) bv = w, at = (int)c;
                }
                best_of_lanes<64>(bv, at);
                __syncthreads();
                if (lane == 0) key[tid >> 6] = bv, group[tid >> 6] = at;
                __syncthreads();
                for (int w = 0; w < kThreads / 64; ++w)
                    if (better(key[w], group[w], bv, at)) bv = key[w], at = group[w];
                if (tid == 0) list[n] = bv, places[n] = at;
                last = bv;
                last_at = at;
            }
            found = a.k;
            __syncthreads();
        }
    }
    if (a.segments > 1) {
        const long cell = r * a.segments + segment;
        if (tid == 0) {
            publish(a.sums + cell * 3, m);
            publish(a.sums + cell * 3 + 1, s);
            publish(a.sums + cell * 3 + 2, t);
        }
        if constexpr (TOP)
            rank_list(list, places, found, a.k, [&](int place, T v, int p) {
                publish(a.best + cell * a.k + place, v);
                publish(a.positions + cell * a.k + place, p);
            });
        if (!last_to_arrive(a.counters + r * a.counter_step, (unsigned)a.segments, &arrived)) return;
        // the row's sums and candidates, from all segments
        const T* sums = a.sums + r * a.segments * 3;
        const bool have = lane < a.segments;
        m = have ? observe(sums + lane * 3) : Real<T>::lowest;
        s = have ? observe(sums + lane * 3 + 1) : T(0);
        t = have ? observe(sums + lane * 3 + 2) : T(0);
        if constexpr (TOP) {
            found = a.segments * a.k;
            for (int i = tid; i < found; i += kThreads) list[i] = observe(a.best + r * found + i), places[i] = observe(a.positions + r * found + i);
        }
        const T part = m;
        m = fold_lanes<64>(m, Max());
        const T by = Max()(part - m, Real<T>::under), w = Real<T>::weight(by);
        t = fold_lanes<64>(w * (t + by * s), Sum());
        s = fold_lanes<64>(w * s, Sum());
        __syncthreads();
    }
    const RowResult<T> q = result_of(m, s);
    if (tid == 0) write_row(a, r, q, s, t, token, own);
    if constexpr (TOP)
        rank_list(list, places, found, a.k, [&](int place, T v, int p) {
            a.top[r * a.k + place] = q.nothing ? T(-INFINITY) : v == T(-INFINITY) ? x[p] - q.lse : v - q.lse;
            a.top_tokens[r * a.k + place] = p;
        });
}

template <typename T>
struct LogProbBackwardArgs {
    const T *d_log_probs, *d_entropy, *logits, *lse, *entropy;
    const int* tokens;
    T* d_logits;
    long rows, stride;
    int vocab, pieces;
};

// what is the same for a whole row of the gradient
template <typename T>
struct RowGradient {
    T lse, g, h, entropy;
    int token;
    __device__ __forceinline__ RowGradient(const LogProbBackwardArgs<T>& a, long r) {
        token = a.tokens[r];
        const T l = a.lse[r];
        const bool nothing = l == T(-INFINITY);
        lse = nothing ? T(0) : l;  // (then all weights are 0)
        g = token < 0 || token >= a.vocab || nothing ? T(0) : a.d_log_probs[r];
        h = a.d_entropy ? a.d_entropy[r] : T(0);
        entropy = a.d_entropy ? a.entropy[r] : T(0);
    }
    __device__ __forceinline__ T of(T x, int c) const {
        const T d = x - lse;
        return (c == token ? g : T(0)) - Real<T>::weight(d) * (g + h * (Max()(d, Real<T>::under) + entropy));
    }
};

template <typename T>
__device__ __forceinline__ void store_group(T* out, int c, int vocab, const T (&v)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    if (c <= vocab - N) {
        typename Vec<T>::type g;
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = v[i];
        *reinterpret_cast<typename Vec<T>::type*>(out + c) = g;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < vocab) out[c + i] = v[i];
    }
}

// LANES lanes to a row
template <typename T, int LANES, int E>
__global__ __launch_bounds__(kThreads) void log_prob_backward_short(LogProbBackwardArgs<T> a) {
    constexpr int N = Vec<T>::N;
    const int l = threadIdx.x % LANES;
    const long r = (long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (r >= a.rows) return;
    const T* x = a.logits + r * a.stride;
    T v[E][N];
#pragma unroll
    for (int e = 0; e < E; ++e) load_group(x, (l + e * LANES) * N, a.vocab, v[e]);
    const RowGradient<T> q(a, r);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = (l + e * LANES) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) v[e][i] = q.of(v[e][i], c + i);
        store_group(a.d_logits + r * a.vocab, c, a.vocab, v[e]);
    }
}

// a workgroup to a piece of a row, four groups to a thread
template <typename T>
__global__ __launch_bounds__(kThreads) void log_prob_backward_long(LogProbBackwardArgs<T> a) {
    constexpr int N = Vec<T>::N, U = 4;
    const long r = blockIdx.x / (unsigned)a.pieces;
    const int piece = (int)(blockIdx.x - (unsigned)r * (unsigned)a.pieces);
    const T* x = a.logits + r * a.stride;
    const RowGradient<T> q(a, r);
    const int first = (piece * U * kThreads + (int)threadIdx.x) * N;  // (the last group of the longest row ends at 2^31 - 1)
    T v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) load_group(x, min((long)first + u * kThreads * N, (long)a.vocab), a.vocab, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long c = (long)first + u * kThreads * N;
        if (c >= a.vocab) break;
#pragma unroll
        for (int i = 0; i < N; ++i) v[u][i] = q.of(v[u][i], (int)c + i);
        store_group(a.d_logits + r * a.vocab, (int)c, a.vocab, v[u]);
    }
}

// lanes and groups per lane that hold a row of `groups` groups; false: none
template <typename F>
bool short_rows(int groups, F launch) {
    if (groups <= 8) launch(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    else if (groups <= 16) launch(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    else if (groups <= 32) launch(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    else if (groups <= 64) launch(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    else if (groups <= 128) launch(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    else if (groups <= 256) launch(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    else return false;
    return true;
}

template <typename T>
int forward(LogProbArgs<T> all) {
    const int groups = groups_of<T>(all.vocab);
    const bool is_short = groups <= 256;
    // a launch numbers its workgroups in 31 bits
    for (long done = 0; done < all.rows;) {
        LogProbArgs<T> a = all;
        a.rows = std::min(all.rows - done, 1L << 24);
        a.logits += done * a.stride;
        a.tokens += done;
        a.log_probs += done, a.entropy += done, a.lse += done;
        if (a.k) a.top += done * a.k, a.top_tokens += done * a.k;
        done += a.rows;
        a.segments = 1;
        a.per = groups;
        if (is_short) {
            short_rows(groups, [&](auto lanes, auto e) {
                constexpr int per = kThreads / decltype(lanes)::value;
                hipLaunchKernelGGL((log_prob_short<T, decltype(lanes)::value, decltype(e)::value>), dim3((unsigned)((a.rows + per - 1) / per)), dim3(kThreads), 0, stream(), a);
            });
            continue;
        }
        // Few rows are cut into segments of at least 512 groups, two for a thread, until there are 512 workgroups or so; their candidates are ranked in one list
        const long cut = std::min({512L / a.rows, (long)groups / 512, (long)kList / std::max(a.k, 1), 64L});
        if (cut > 1) {
            a.segments = (int)cut;
            a.per = (groups + a.segments - 1) / a.segments;
            a.segments = (groups + a.per - 1) / a.per;
            a.counters = (unsigned*)workspace();
            a.counter_step = counter_step(a.rows);
            a.sums = (T*)(workspace() + kWorkspaceCounterBytes);
            a.best = a.sums + a.rows * a.segments * 3;
            a.positions = (int*)(a.best + a.rows * a.segments * a.k);
        }
        const dim3 grid((unsigned)(a.rows * a.segments));
        if (a.k) hipLaunchKernelGGL((log_prob_long<T, true>), grid, dim3(kThreads), 0, stream(), a);
        else hipLaunchKernelGGL((log_prob_long<T, false>), grid, dim3(kThreads), 0, stream(), a);
    }
    return launched("dali_hip_token_log_probs");
}

template <typename T>
int backward(LogProbBackwardArgs<T> all) {
    const int groups = groups_of<T>(all.vocab);
    const long pieces = ((long)groups + 4 * kThreads - 1) / (4 * kThreads);
    for (long done = 0; done < all.rows;) {
        LogProbBackwardArgs<T> a = all;
        a.rows = std::min(all.rows - done, std::max(1L, (1L << 24) / pieces));
        a.logits += done * a.stride;
        a.d_logits += done * a.vocab;
        a.tokens += done;
        a.d_log_probs += done, a.lse += done;
        if (a.d_entropy) a.d_entropy += done, a.entropy += done;
        done += a.rows;
        a.pieces = (int)pieces;
        if (short_rows(groups, [&](auto lanes, auto e) {
                constexpr int per = kThreads / decltype(lanes)::value;
                hipLaunchKernelGGL((log_prob_backward_short<T, decltype(lanes)::value, decltype(e)::value>), dim3((unsigned)((a.rows + per - 1) / per)), dim3(kThreads), 0, stream(), a);
            }))
            continue;
        hipLaunchKernelGGL(log_prob_backward_long<T>, dim3((unsigned)(a.rows * pieces)), dim3(kThreads), 0, stream(), a);
    }
    return launched("dali_hip_token_log_probs_backward");
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_token_log_probs(int dtype, int64_t rows, int vocab, const void* logits, int64_t stride, const int32_t* tokens, int k, void* log_probs, void* entropy,
                                        void* lse, void* top_log_probs, int32_t* top_tokens) {
    const char* what = "dali_hip_token_log_probs";
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (rows < 0 || vocab < 1) return fail("%s: %lld rows of %d logits", what, (long long)rows, vocab);
    if (k < 0 || k > DALI_HIP_MAX_ALTERNATIVES || k > vocab)
        return fail("%s: %d alternatives of %d logits (at most %d are served)", what, k, vocab, DALI_HIP_MAX_ALTERNATIVES);
    if (rows == 0) return DALI_HIP_OK;
    if (!logits || !tokens || !log_probs || !entropy || !lse || (k && (!top_log_probs || !top_tokens))) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (check_spans(what,
                    {Span("log_probs", log_probs, rows, size), Span("entropy", entropy, rows, size), Span("lse", lse, rows, size),
                     Span("top_log_probs", top_log_probs, rows * k, size), Span("top_tokens", top_tokens, rows * k, 4)},
                    {Span("logits", logits, rows, vocab, stride, size), Span("tokens", tokens, rows, 4)}, 0))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT)
        return forward<float>({(const float*)logits, tokens, (float*)log_probs, (float*)entropy, (float*)lse, (float*)top_log_probs, top_tokens, (long)rows, (long)stride, vocab, k});
    return forward<double>(
        {(const double*)logits, tokens, (double*)log_probs, (double*)entropy, (double*)lse, (double*)top_log_probs, top_tokens, (long)rows, (long)stride, vocab, k});
}

extern "C" int dali_hip_token_log_probs_backward(int dtype, int64_t rows, int vocab, const void* d_log_probs, const void* d_entropy, const void* logits, int64_t stride,
                                                 const int32_t* tokens, const void* lse, const void* entropy, void* d_logits) {
    const char* what = "dali_hip_token_log_probs_backward";
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (rows < 0 || vocab < 1) return fail("%s: %lld rows of %d logits", what, (long long)rows, vocab);
    if (rows == 0) return DALI_HIP_OK;
    if (!d_log_probs || !logits || !tokens || !lse || !d_logits || (d_entropy && !entropy)) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (check_spans(what, {Span("d_logits", d_logits, rows * vocab, size)},
                    {Span("logits", logits, rows, vocab, stride, size), Span("d_log_probs", d_log_probs, rows, size), Span("d_entropy", d_entropy, rows, size),
                     Span("tokens", tokens, rows, 4), Span("lse", lse, rows, size), Span("entropy", entropy, rows, size)},
                    1))
        return DALI_HIP_ERROR;
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT)
        return backward<float>({(const float*)d_log_probs, (const float*)d_entropy, (const float*)logits, (const float*)lse, (const float*)entropy, tokens, (float*)d_logits,
                                (long)rows, (long)stride, vocab, 1});
    return backward<double>({(const double*)d_log_probs, (const double*)d_entropy, (const double*)logits, (const double*)lse, (const double*)entropy, tokens, (double*)d_logits,
                             (long)rows, (long)stride, vocab, 1});
}
