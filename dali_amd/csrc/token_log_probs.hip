// Log probabilities of given tokens under softmax(logits), row by row, with the entropy of the row and its best alternatives; and the gradient.
//
//   m = max x,  S = sum e^(x - m),  T = sum e^(x - m) (x - m)
//   lse = m + ln S,  log p(t) = x_t - lse,  entropy = -sum p ln p = ln S - T / S
//   d x = d log p(t) (delta_t - p) - d entropy p (ln p + entropy)
//
// Log probabilities are written as (x - m) - ln S, which keeps the digits of rows far from 0; p of the gradient is e^(x - lse) with lse as it was rounded.
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
    static constexpr float under = -200.0f;             // an exponent whose weight is 0: what a lower one is replaced by where it meets a weight or a gradient
    static __device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }
    static __device__ __forceinline__ float ln(float s) { return logf(s); }
};
template <>
struct Real<double> {
    static constexpr double lowest = -1.7976931348623157e+308;
    static constexpr double under = -1000.0;
    static __device__ __forceinline__ double weight(double d) { return exp(d); }
    static __device__ __forceinline__ double ln(double s) { return log(s); }
};

// a NaN counts as -inf among the alternatives
template <typename T>
__device__ __forceinline__ T ranked(T v) {
    return Max()(v, T(-INFINITY));
}

// An entry of a row (or the best of a group of entries, by the group's number): of two the better has the larger value, or among equals the lower position. A NaN
// counts as -inf. Of fp32 it is one whole number that grows with the value and falls with the position; there a zero is a zero of either sign.
template <typename T>
struct Entry;
template <>
struct Entry<float> {
    unsigned long long key;
    static __device__ __forceinline__ Entry of(float v, int position) {
        const unsigned b = __builtin_bit_cast(unsigned, fmaxf(v, -INFINITY) + 0.0f);
        return {(unsigned long long)(b ^ ((unsigned)((int)b >> 31) | 0x80000000u)) << 32 | (0xffffffffu - (unsigned)position)};
    }
    static __device__ __forceinline__ Entry none() { return {0}; }  // worse than any
    static __device__ __forceinline__ Entry either(bool first, const Entry& a, const Entry& b) { return {first ? a.key : b.key}; }
    __device__ __forceinline__ float value() const {
        const unsigned b = (unsigned)(key >> 32);
        return __builtin_bit_cast(float, b ^ ((unsigned)((int)~b >> 31) | 0x80000000u));
    }
    __device__ __forceinline__ int position() const { return (int)(0xffffffffu - (unsigned)key); }
    __device__ __forceinline__ bool better(const Entry& o) const { return key > o.key; }
    template <int D>
    __device__ __forceinline__ void halves(Entry& a, Entry& b) const {
        halves_of<D>(key, a.key, b.key);
    }
    __device__ __forceinline__ Entry lane(int l) const {
        return {(unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(key >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)key, l)};
    }
    __device__ __forceinline__ void publish(Entry* p) const { dali_hip::publish(&p->key, key); }
    static __device__ __forceinline__ Entry observe(const Entry* p) { return {dali_hip::observe(&p->key)}; }
};
template <>
struct Entry<double> {
    double v;
    long at;
    static __device__ __forceinline__ Entry of(double v, int position) { return {fmax(v, -(double)INFINITY), position}; }
    static __device__ __forceinline__ Entry none() { return {-INFINITY, 1L << 40}; }
    static __device__ __forceinline__ Entry either(bool first, const Entry& a, const Entry& b) { return {first ? a.v : b.v, first ? a.at : b.at}; }
    __device__ __forceinline__ double value() const { return v; }
    __device__ __forceinline__ int position() const { return (int)at; }
    __device__ __forceinline__ bool better(const Entry& o) const { return v > o.v || (v == o.v && at < o.at); }
    template <int D>
    __device__ __forceinline__ void halves(Entry& a, Entry& b) const {
        halves_of<D>(v, a.v, b.v);
        halves_of<D>(at, a.at, b.at);
    }
    static __device__ __forceinline__ long word(long w, int l) {
        return (long)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(w >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)w, l));
    }
    __device__ __forceinline__ Entry lane(int l) const { return {__builtin_bit_cast(double, word(__builtin_bit_cast(long, v), l)), word(at, l)}; }
    __device__ __forceinline__ void publish(Entry* p) const {
        dali_hip::publish(&p->v, v);
        dali_hip::publish(&p->at, at);
    }
    static __device__ __forceinline__ Entry observe(const Entry* p) { return {dali_hip::observe(&p->v), dali_hip::observe(&p->at)}; }
};

// the best entry that LANES neighbouring lanes hold
template <int LANES, int D = 1, typename T>
__device__ __forceinline__ Entry<T> best_of_lanes(const Entry<T>& e) {
    if constexpr (D >= LANES) {
        return e;
    } else {
        Entry<T> a, b;
        e.template halves<D>(a, b);
        return best_of_lanes<LANES, D * 2>(Entry<T>::either(a.better(b), a, b));
    }
}

// how many of a wave's entries are better than the lane's own: its place among them
template <typename T>
__device__ __forceinline__ int place_in_wave(const Entry<T>& e) {
    int place = 0;
#pragma unroll 16
    for (int l = 0; l < 64; ++l) place += e.lane(l).better(e) ? 1 : 0;
    return place;
}

// The k-th best of a wave's entries, in every lane: a few by taking the best away one after the other, more by counting places
constexpr int kOneByOne = 10;  // (65536x1000 with 4, 8, 12, 16 alternatives: 62, 76, 92, 110 us one by one, 85, 89, 91, 93 by places)
template <typename T>
__device__ __forceinline__ Entry<T> kth_of_wave(Entry<T> e, int k) {
    if (k > kOneByOne) return e.lane(__builtin_ctzll(__ballot(place_in_wave(e) == k - 1)));
    for (int n = 1; n < k; ++n) {
        const Entry<T> best = best_of_lanes<64>(e);
        e = Entry<T>::either(best.better(e), e, Entry<T>::none());
    }
    return best_of_lanes<64>(e);
}

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
    Entry<T>* best;  // [rows][segments][k], in order
    unsigned* counters;
    int counter_step;
};

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

template <typename T>
__device__ __forceinline__ void write_alternative(const LogProbArgs<T>& a, long r, const T* x, const RowResult<T>& q, int place, const Entry<T>& e) {
    const T v = e.value();
    const int p = e.position();
    // (as the given token's is written: lse would round away digits of rows far from 0. A NaN was ranked as -inf)
    a.top[r * a.k + place] = q.nothing ? T(-INFINITY) : ((v == T(-INFINITY) ? x[p] : v) - q.m) - q.ln;
    a.top_tokens[r * a.k + place] = p;
}

// Entries of one wave that are ranked at once
constexpr int kWaveList = 128;

// The k best of the entries that a wave holds in registers, E groups to a lane, E > 1: the k-th best of the lanes' best groups (`top`, and the group's number) bounds
// them, what passes it is collected and ranked. False where the list does not hold them.
template <typename T, int E, typename Put>
__device__ __forceinline__ bool best_by_bound(const T (&v)[E][Vec<T>::N], T top, int top_group, int l, int vocab, int k, Entry<T>* list, int* count, Put put) {
    constexpr int N = Vec<T>::N;
    const Entry<T> mine = l * N < vocab ? Entry<T>::of(top, top_group) : Entry<T>::none();
    const Entry<T> bound = kth_of_wave(mine, k);
    const T low = bound.value();
    if (l == 0) *count = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int e = 0; e < E; ++e) {
        T g = ranked(v[e][0]);
#pragma unroll
        for (int i = 1; i < N; ++i) g = Max()(g, v[e][i]);
        if (g < low) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (l + e * 64) * N + i;
            // (the bound's position is a group's: any of its entries may be the one)
            if (c < vocab && !bound.better(Entry<T>::of(v[e][i], l + e * 64))) {
                const int slot = atomicAdd(count, 1);
                if (slot < kWaveList) list[slot] = Entry<T>::of(v[e][i], c);
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int n = __builtin_amdgcn_readfirstlane(*(volatile int*)count);
    if (n > kWaveList) return false;
    for (int i = l; i < n; i += 64) {
        const Entry<T> e = list[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) place += list[j].better(e) ? 1 : 0;
        if (place < k) put(place, e);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return true;
}

// One alternative after the other of the entries that LANES lanes hold: an entry that has been named is no longer free
template <typename T, int LANES, int E, typename Put>
__device__ __forceinline__ void best_one_by_one(const T (&v)[E][Vec<T>::N], int l, int vocab, int k, Put put) {
    constexpr int N = Vec<T>::N;
    unsigned long long unnamed = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < N; ++i) unnamed |= ((l + e * LANES) * N + i < vocab ? 1ull : 0ull) << (e * N + i);
    for (int n = 0; n < k; ++n) {
        Entry<T> best = Entry<T>::none();
        int slot = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const Entry<T> w = Entry<T>::of(v[e][i], (l + e * LANES) * N + i);
                const bool take = (unnamed >> (e * N + i) & 1) && w.better(best);
                best = Entry<T>::either(take, w, best);
                slot = take ? e * N + i : slot;
            }
        const int mine = best.position();
        best = best_of_lanes<LANES>(best);
        if (mine == best.position()) unnamed &= ~(1ull << slot);
        if (l == 0) put(n, best);
    }
}

// The same for fp32 rows of one group to a lane, where the lanes lie in the order of the positions: each orders its four once, and the next alternative is the
// head of the first lane whose head is the largest of all heads. They go into `list` in order.
template <int LANES>
__device__ __forceinline__ void best_by_heads(const float (&v)[1][4], int l, int vocab, int k, Entry<float>* list) {
    unsigned key[4];
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        key[i] = l * 4 + i < vocab ? (unsigned)(Entry<float>::of(v[0][i], 0).key >> 32) : 0u;  // (0 is worse than any entry's)
        at[i] = l * 4 + i;
    }
    auto order = [&](int i, int j) {
        const bool swap = key[j] > key[i] || (key[j] == key[i] && at[j] < at[i]);
        const unsigned hi = swap ? key[j] : key[i], lo = swap ? key[i] : key[j];
        const int p = swap ? at[j] : at[i], q = swap ? at[i] : at[j];
        key[i] = hi, key[j] = lo, at[i] = p, at[j] = q;
    };
    order(0, 1), order(2, 3), order(0, 2), order(1, 3), order(1, 2);
    const int lane = threadIdx.x & 63, base = lane & ~(LANES - 1);
    const unsigned long long team = (LANES == 64 ? ~0ull : ((1ull << (LANES % 64)) - 1)) << base;
    for (int n = 0; n < k; ++n) {
        const unsigned high = fold_lanes<LANES>(key[0], [](unsigned a, unsigned b) { return a > b ? a : b; });
        if (__builtin_ctzll(__ballot(key[0] == high) & team) == lane) {
            list[n].key = (unsigned long long)key[0] << 32 | (0xffffffffu - (unsigned)at[0]);
            key[0] = key[1], key[1] = key[2], key[2] = key[3], key[3] = 0;
            at[0] = at[1], at[1] = at[2], at[2] = at[3];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Rows that LANES lanes hold in registers, E groups each: every statistic is exact after one reading, and no workgroup meets. Bound by memory without alternatives
// (65536x1500 66 us, 5.9 TB/s; 51200x97 7.6 us, where the launch is half of it), by arithmetic with them (51200x97 with 5 14.5 us, 65536x1000 64 us, 4.1 TB/s: a
// comparison of all lanes costs a row as much as its exponentials).
template <typename T, int LANES, int E, bool TOP>
__global__ __launch_bounds__(kThreads) void log_prob_short(LogProbArgs<T> a) {
    constexpr int N = Vec<T>::N;
    // lists: of a wave that bounds its best, or of a row whose lanes' heads are compared
    constexpr bool HEADS = TOP && E == 1 && sizeof(T) == 4, LIST = TOP && (E > 1 || HEADS);
    constexpr int LISTS = HEADS ? kThreads / LANES : kThreads / 64, LENGTH = HEADS ? (LANES * N < DALI_HIP_MAX_ALTERNATIVES ? LANES * N : DALI_HIP_MAX_ALTERNATIVES) : kWaveList;
    __shared__ Entry<T> lists[LIST ? LISTS : 1][LIST ? LENGTH : 1];
    __shared__ int counts[LIST ? kThreads / 64 : 1];
    const int l = threadIdx.x % LANES;
    const long row = (long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    const bool live = row < a.rows;
    const long r = live ? row : a.rows - 1;  // (lanes without a row go along with the last)
    const T* x = a.logits + r * a.stride;
    typename Vec<T>::type g[E];
    T v[E][N];
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = ask_group<(LANES > 8)>(x, (l + e * LANES) * N, a.vocab);
#pragma unroll
    for (int e = 0; e < E; ++e) take_group<(LANES > 8)>(g[e], (l + e * LANES) * N, a.vocab, T(-INFINITY), v[e]);
    const int token = a.tokens[r];
    const T own = token >= 0 && token < a.vocab ? x[token] : T(0);
    T m = Real<T>::lowest, top = -INFINITY;
    int top_group = l;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        T h = v[e][0];
#pragma unroll
        for (int i = 1; i < N; ++i) h = Max()(h, v[e][i]);
        m = Max()(m, h);
        if (TOP && E > 1 && h > top) top = h, top_group = l + e * LANES;
    }
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
    if (l == 0 && live) write_row(a, r, q, s, t, token, own);
    if constexpr (TOP) {
        auto put = [&](int place, const Entry<T>& e) {
            if (live) write_alternative(a, r, x, q, place, e);
        };
        if constexpr (E == 1 && sizeof(T) == 4) {
            Entry<T>* list = lists[threadIdx.x / LANES];
            best_by_heads<LANES>(v, l, a.vocab, a.k, list);
            for (int n = l; n < a.k; n += LANES) put(n, list[n]);
        } else if constexpr (E == 1) {
            best_one_by_one<T, LANES, E>(v, l, a.vocab, a.k, put);
        } else {
            const int wave = threadIdx.x >> 6;
            if (!best_by_bound<T, E>(v, top, top_group, l, a.vocab, a.k, lists[wave], &counts[wave], put)) best_one_by_one<T, LANES, E>(v, l, a.vocab, a.k, put);
        }
    }
}

constexpr int kList = 512;    // entries that are ranked at once
constexpr int kMerge = 64;    // segments of a row, one to a lane of the wave that joins them
constexpr int kParts = 4;     // of a thread's walk, each with a best group
constexpr int kByHeads = 8;   // up to so many alternatives, the segments' lists are joined one after the other
constexpr int kByQuads = 32;  // up to so many alternatives, the best of 64 quads of threads bound them; beyond, those of the threads themselves, which bound them closer but
                              // take longer to compare (quads and threads, 8192x32000: 236 and 232 us with 24, 283 and 268 with 48; 1x50257: 10.6 and 13.0, 12.6 and 14.1)

// The running sums of a row or a part of it: the maximum, the weights relative to it and their product with the exponents
template <typename T>
struct Sums {
    T m = Real<T>::lowest, s = 0, t = 0;
    __device__ __forceinline__ void raise(T to) {
        const T by = Max()(m - to, Real<T>::under), w = Real<T>::weight(by);
        t = w * (t + by * s);
        s *= w;
        m = to;
    }
    __device__ __forceinline__ void add(T v) {
        const T d = v - m, w = Real<T>::weight(d);
        s += w;
        t += w * Max()(d, Real<T>::under);
    }
    __device__ __forceinline__ void over_wave() {
        raise(fold_lanes<64>(m, Max()));
        s = fold_lanes<64>(s, Sum());
        t = fold_lanes<64>(t, Sum());
    }
    __device__ __forceinline__ void join(Sums o) {
        const T high = Max()(m, o.m);
        raise(high);
        o.raise(high);
        s += o.s;
        t += o.t;
    }
};

// What the workgroups of the long forms share
template <typename T, bool TOP>
struct Shared {
    T sums[kThreads / 64][3];
    unsigned arrived;
    int count, units;
    Entry<T> list[TOP ? kList : 1], key[TOP ? kThreads : 1], bound;
    unsigned short unit[TOP ? kParts * kThreads : 1];
};

template <typename T, bool TOP>
__device__ __forceinline__ void over_block(Sums<T>& q, Shared<T, TOP>& sh) {
    q.over_wave();
    if ((threadIdx.x & 63) == 0) {
        T* p = sh.sums[threadIdx.x >> 6];
        p[0] = q.m, p[1] = q.s, p[2] = q.t;
    }
    __syncthreads();
    q.m = sh.sums[0][0], q.s = sh.sums[0][1], q.t = sh.sums[0][2];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) {
        Sums<T> o;
        o.m = sh.sums[w][0], o.s = sh.sums[w][1], o.t = sh.sums[w][2];
        q.join(o);
    }
}

// The k-th best of the best groups that the quads of threads hold (or the threads): k groups have an entry that good, so the k best entries of all are no worse
template <typename T>
__device__ __forceinline__ Entry<T> find_bound(const Entry<T>& mine, int k, Shared<T, true>& sh) {
    const int tid = threadIdx.x;
    if (tid == 0) sh.count = sh.units = 0;
    if (k <= kByQuads) {
        const Entry<T> quad = best_of_lanes<4>(mine);
        if ((tid & 3) == 0) sh.key[tid >> 2] = quad;
        __syncthreads();
        if (tid < 64) {
            const Entry<T> kth = kth_of_wave(sh.key[tid], k);
            if (tid == 0) sh.bound = kth;
        }
    } else {
        sh.key[tid] = mine;
        __syncthreads();
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < kThreads; ++i) place += sh.key[i].better(mine) ? 1 : 0;
        if (place == k - 1) sh.bound = mine;
    }
    __syncthreads();
    return sh.bound;
}

// the entries of group g that pass the bound join the list
template <typename T>
__device__ __forceinline__ void collect(const T (&v)[Vec<T>::N], int g, int vocab, const Entry<T>& bound, Shared<T, true>& sh) {
    const T low = bound.value();
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) {
        if (ranked(v[e]) < low) continue;
        // (the bound's position is a group's: any of its entries may be the one)
        const Entry<T> w = Entry<T>::of(v[e], g);
        if (g * Vec<T>::N + e < vocab && !bound.better(w)) {
            const int slot = atomicAdd(&sh.count, 1);
            if (slot < kList) sh.list[slot] = Entry<T>::of(v[e], g * Vec<T>::N + e);
        }
    }
}

// The k best of `n` entries of the list, in order: an entry's place is the number of better ones
template <typename T, typename Put>
__device__ __forceinline__ void rank_list(const Shared<T, true>& sh, int n, int k, Put put) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const Entry<T> e = sh.list[i];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) place += sh.list[j].better(e) ? 1 : 0;
        if (place < k) put(place, e);
    }
}

// So many of the best side by side in few units that the list does not hold them: one after the other over all groups, into the list
template <typename T>
__device__ __forceinline__ void one_by_one(const LogProbArgs<T>& a, const T* x, int begin, int end, Shared<T, true>& sh) {
    Entry<T> last = Entry<T>::none();
    for (int n = 0; n < a.k; ++n) {
        Entry<T> best = Entry<T>::none();
        for (long c = (long)begin * Vec<T>::N + threadIdx.x; c < min((long)a.vocab, (long)end * Vec<T>::N); c += kThreads) {
            const Entry<T> w = Entry<T>::of(x[c], (int)c);
            if ((n == 0 || last.better(w)) && w.better(best)) best = w;
        }
        best = best_of_lanes<64>(best);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.key[threadIdx.x >> 6] = best;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; ++w)
            if (sh.key[w].better(best)) best = sh.key[w];
        if (threadIdx.x == 0) sh.list[n] = best;
        last = best;
    }
    __syncthreads();
}

// The end of a row: straight to the results, or by way of the workspace where the row has several segments, whose last workgroup joins them. `found` entries
// of the list hold the k best of the segment.
template <typename T, bool TOP>
__device__ __forceinline__ void finish(const LogProbArgs<T>& a, long r, int segment, const T* x, Sums<T> q, int found, int token, T own, Shared<T, TOP>& sh) {
    const int tid = threadIdx.x;
    if (a.segments == 1) {
        const RowResult<T> done = result_of(q.m, q.s);
        if (tid == 0) write_row(a, r, done, q.s, q.t, token, own);
        if constexpr (TOP) rank_list(sh, found, a.k, [&](int place, const Entry<T>& e) { write_alternative(a, r, x, done, place, e); });
        return;
    }
    const long cell = r * a.segments + segment;
    if (tid == 0) {
        publish(a.sums + cell * 3, q.m);
        publish(a.sums + cell * 3 + 1, q.s);
        publish(a.sums + cell * 3 + 2, q.t);
    }
    if constexpr (TOP) rank_list(sh, found, a.k, [&](int place, const Entry<T>& e) { e.publish(a.best + cell * a.k + place); });
    if (!last_to_arrive(a.counters + r * a.counter_step, (unsigned)a.segments, &sh.arrived)) return;
    constexpr int EACH = kList / kThreads;
    Entry<T> mine[EACH];
    if constexpr (TOP) {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int i = tid + n * kThreads;
            mine[n] = i < a.segments * a.k ? Entry<T>::observe(a.best + r * a.segments * a.k + i) : Entry<T>::none();
            sh.list[i] = mine[n];
        }
        if (tid == 0) sh.count = 0;
    }
    Sums<T> all;
    if ((tid & 63) < a.segments) {
        const T* p = a.sums + (r * a.segments + (tid & 63)) * 3;
        all.m = observe(p), all.s = observe(p + 1), all.t = observe(p + 2);
    }
    all.over_wave();
    const RowResult<T> done = result_of(all.m, all.s);
    if (tid == 0) write_row(a, r, done, all.s, all.t, token, own);
    if constexpr (TOP) {
        __syncthreads();
        if (a.k <= kByHeads) {
            // The segments' lists are in order: a lane stands at the head of one, and the best head is next (5 of 1x50257: 7.9 us, as below 8.7; 20: 11.5, below 10.3)
            if (tid >= 64) return;
            int at = 0;
            Entry<T> head = tid < a.segments ? sh.list[tid * a.k] : Entry<T>::none(), kept = Entry<T>::none();
            for (int n = 0; n < a.k; ++n) {
                const Entry<T> best = best_of_lanes<64>(head);
                if (n == tid) kept = best;
                if (tid < a.segments && !best.better(head)) head = ++at < a.k ? sh.list[tid * a.k + at] : Entry<T>::none();
            }
            if (tid < a.k) write_alternative(a, r, x, done, tid, kept);
            return;
        }
        // the k-th best of 64 entries from the front of the lists (k of any entries would do) bounds the k best of all
        if (tid < 64) {
            const int segments = a.segments, place = tid / segments, from = tid - place * segments;
            const Entry<T> e = place < a.k ? sh.list[from * a.k + place] : Entry<T>::none();
            const Entry<T> kth = kth_of_wave(e, a.k);
            if (tid == 0) sh.bound = kth;
        }
        __syncthreads();
        const Entry<T> bound = sh.bound;
#pragma unroll
        for (int n = 0; n < EACH; ++n)
            if (!bound.better(mine[n])) sh.list[atomicAdd(&sh.count, 1)] = mine[n];
        __syncthreads();
        rank_list(sh, sh.count, a.k, [&](int place, const Entry<T>& e) { write_alternative(a, r, x, done, place, e); });
    }
}

// One workgroup per row, or per segment of a row: a thread walks its groups once with running sums, which are rescaled when the maximum rises (once per four
// groups). For the alternatives it keeps the best group of each quarter of its walk. What passes the bound that the best groups give lies in the few quarters whose own best
// passes it; their groups are read again: a line of the cache for 16 bytes each time, which is why they are quarters (8192x32000 with 5 alternatives read 1.15 times the
// logits with whole walks, 184 us). Bound by memory: 8192x32000 175 us (6.0 TB/s), with 5, 20 and 64 alternatives 182, 190 and 222 us. One reading with running sums
// instead of a maximum first and the sums after it: the row is larger than what the registers of a workgroup hold.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void log_prob_long(LogProbArgs<T> a) {
    constexpr int N = Vec<T>::N, U = 4, STEP = U * kThreads, PARTS = TOP ? kParts : 1;
    __shared__ Shared<T, TOP> sh;
    const int tid = threadIdx.x;
    const long r = blockIdx.x / (unsigned)a.segments;
    const int segment = (int)(blockIdx.x - (unsigned)r * (unsigned)a.segments);
    const T* x = a.logits + r * a.stride;
    const int groups = groups_of<T>(a.vocab), begin = segment * a.per, end = min(groups, begin + a.per), whole = min(end, a.vocab / N);
    const int span = ((end - begin - 1) / (STEP * PARTS) + 1) * STEP;  // groups of the segment in a part, whole steps of all threads
    const int token = a.tokens[r];
    const T own = token >= 0 && token < a.vocab ? x[token] : T(0);
    Sums<T> q;
    T top[PARTS];
    int top_group[PARTS];
    int j = begin + tid;
    typename Vec<T>::type next[U];
    auto ask = [&](int from) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = *reinterpret_cast<const typename Vec<T>::type*>(x + (long)(from + u * kThreads) * N);
    };
    if (j + STEP - kThreads < whole) ask(j);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        top[part] = -INFINITY;
        top_group[part] = begin + tid + part * span;
        const int limit = PARTS == 1 ? whole : (int)min((long)whole, (long)begin + tid + (part + 1L) * span);  // (a step ends below it or begins at it)
        for (; j + STEP - kThreads < whole && j < limit; j += STEP) {
            typename Vec<T>::type v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = next[u];
            if (j + 2 * STEP - kThreads < whole) ask(j + STEP);  // (under way while these are worked on)
            T high = q.m;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                T g = v[u][0];
#pragma unroll
                for (int i = 1; i < N; ++i) g = Max()(g, v[u][i]);
                high = Max()(high, g);
                if (TOP && g > top[part]) top[part] = g, top_group[part] = j + u * kThreads;
            }
            q.raise(high);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i) q.add(v[u][i]);
        }
    }
    // (what is left is less than a step and lies in one part)
    const int rest = (j - begin - tid) / span;
    for (; j < end; j += kThreads) {
        T v[N];
        load_group(x, j * N, a.vocab, T(-INFINITY), v);
        T g = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) g = Max()(g, v[i]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
            if (TOP && part == rest && g > top[part]) top[part] = g, top_group[part] = j;
        q.raise(Max()(q.m, g));
#pragma unroll
        for (int i = 0; i < N; ++i) q.add(v[i]);
    }
    over_block(q, sh);
    int found = 0;
    if constexpr (TOP) {
        Entry<T> best[PARTS], mine = Entry<T>::none();
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            best[part] = (long)begin + tid + (long)part * span < end ? Entry<T>::of(top[part], top_group[part]) : Entry<T>::none();
            mine = Entry<T>::either(best[part].better(mine), best[part], mine);
        }
        const Entry<T> bound = find_bound(mine, a.k, sh);
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
            if (!bound.better(best[part])) sh.unit[atomicAdd(&sh.units, 1)] = (unsigned short)(part * kThreads + tid);
        __syncthreads();
        const int walks = span / kThreads, all = sh.units * walks;
        for (int i = tid; i < all; i += kThreads) {
            const int n = i / walks, unit = sh.unit[n];
            const long g = (long)begin + (unit & (kThreads - 1)) + (long)(unit / kThreads) * span + (i - n * walks) * kThreads;
            if (g >= end) continue;
            T v[N];
            load_group(x, (int)g * N, a.vocab, T(-INFINITY), v);
            collect(v, (int)g, a.vocab, bound, sh);
        }
        __syncthreads();
        found = sh.count;
        if (found > kList) {
            one_by_one(a, x, begin, end, sh);
            found = a.k;
        }
    }
    finish(a, r, segment, x, q, found, token, own, sh);
}

// Segments that a workgroup holds in registers, E groups to a thread: all of them are loaded at once and nothing is read again. 65536x3000 128 us (6.2 TB/s), with 5
// alternatives 187; 32768x8000 170 and 181 us. A single row of 50257 in 24 segments takes 7.0 us with 5 alternatives and 10.2 with 20, 4.6 without: a chain of one reading,
// the folds, the bound, two trips to memory for what the segments found and its ranking.
template <typename T, bool TOP, int E>
__global__ __launch_bounds__(kThreads) void log_prob_segments(LogProbArgs<T> a) {
    constexpr int N = Vec<T>::N;
    __shared__ Shared<T, TOP> sh;
    const int tid = threadIdx.x;
    const long r = blockIdx.x / (unsigned)a.segments;
    const int segment = (int)(blockIdx.x - (unsigned)r * (unsigned)a.segments);
    const T* x = a.logits + r * a.stride;
    const int begin = segment * a.per, end = min(groups_of<T>(a.vocab), begin + a.per);
    typename Vec<T>::type asked[E];
    T v[E][N];
    auto at = [&](int e) { return begin + tid + e * kThreads < end ? (begin + tid + e * kThreads) * N : a.vocab; };
#pragma unroll
    for (int e = 0; e < E; ++e) asked[e] = ask_group<true>(x, at(e), a.vocab);
#pragma unroll
    for (int e = 0; e < E; ++e) take_group<true>(asked[e], at(e), a.vocab, T(-INFINITY), v[e]);
    const int token = a.tokens[r];
    const T own = token >= 0 && token < a.vocab ? x[token] : T(0);
    Sums<T> q;
    T top = -INFINITY, high = q.m;
    int top_group = begin + tid;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        T g = v[e][0];
#pragma unroll
        for (int i = 1; i < N; ++i) g = Max()(g, v[e][i]);
        high = Max()(high, g);
        if (TOP && g > top) top = g, top_group = begin + tid + e * kThreads;
    }
    q.m = high;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < N; ++i) q.add(v[e][i]);
    over_block(q, sh);
    int found = 0;
    if constexpr (TOP) {
        const Entry<T> bound = find_bound(begin + tid < end ? Entry<T>::of(top, top_group) : Entry<T>::none(), a.k, sh);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int g = begin + tid + e * kThreads;
            if (g < end) collect(v[e], g, a.vocab, bound, sh);
        }
        __syncthreads();
        found = sh.count;
        if (found > kList) {
            one_by_one(a, x, begin, end, sh);
            found = a.k;
        }
    }
    finish(a, r, segment, x, q, found, token, own, sh);
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
        // (the weight first: an exponent whose weight is small or 0 would carry a large gradient past the type's range)
        const T d = x - lse, w = Real<T>::weight(d);
        return (c == token ? g : T(0)) - (w * g + (w * h) * (Max()(d, Real<T>::under) + entropy));
    }
};

// The gradient is a map once a row's lse is known: one reading, one writing, bound by memory. LANES lanes to a row: 51200x97 9.2 us (4.3 TB/s, an odd length costs lanes
// and whole lines), 65536x613 57 us (5.7 TB/s)
template <typename T, int LANES, int E, bool PAST>
__global__ __launch_bounds__(kThreads) void log_prob_backward_short(LogProbBackwardArgs<T> a) {
    constexpr int N = Vec<T>::N;
    const int l = threadIdx.x % LANES;
    const long r = (long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (r >= a.rows) return;
    const T* x = a.logits + r * a.stride;
    typename Vec<T>::type g[E];
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = ask_group<(LANES > 8)>(x, (l + e * LANES) * N, a.vocab);
    const RowGradient<T> q(a, r);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = (l + e * LANES) * N;
        T v[N];
        take_group<(LANES > 8)>(g[e], c, a.vocab, T(-INFINITY), v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = q.of(v[i], c + i);
        store_group<PAST>(a.d_logits + r * a.vocab, c, a.vocab, v);
    }
}

// a workgroup to a piece of a row, four groups to a thread: 8192x32000 393 us (5.3 TB/s, above a plain copy of that size)
template <typename T, bool PAST>
__global__ __launch_bounds__(kThreads) void log_prob_backward_long(LogProbBackwardArgs<T> a) {
    constexpr int N = Vec<T>::N, U = 4;
    const long r = blockIdx.x / (unsigned)a.pieces;
    const int piece = (int)(blockIdx.x - (unsigned)r * (unsigned)a.pieces);
    const T* x = a.logits + r * a.stride;
    const RowGradient<T> q(a, r);
    const int first = (piece * U * kThreads + (int)threadIdx.x) * N;  // (the last group of the longest row ends at 2^31 - 1)
    typename Vec<T>::type g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) g[u] = ask_group<true>(x, (int)min((long)first + u * kThreads * N, (long)a.vocab), a.vocab);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long c = (long)first + u * kThreads * N;
        if (c >= a.vocab) break;
        T v[N];
        take_group<true>(g[u], (int)c, a.vocab, T(-INFINITY), v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = q.of(v[i], (int)c + i);
        store_group<PAST>(a.d_logits + r * a.vocab, (int)c, a.vocab, v);
    }
}

// lanes and groups per lane that hold a row of `groups` groups, up to `most` of them; false: none
template <int MOST, typename F>
bool short_rows(int groups, F launch) {
    auto with = [&](auto lanes, auto e) {
        launch(lanes, e);
        return true;
    };
    if (groups <= 8) return with(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    if (groups <= 16) return with(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    if (groups <= 32) return with(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    if (groups <= 64) return with(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (groups <= 128) return with(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    if (groups <= 256) return with(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    if constexpr (MOST > 256) {
        if (groups <= 512) return with(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    }
    return false;
}

// Workgroups of a launch: HIP takes fewer than 2^32 threads along an axis. More rows take several launches, of which a failed one is the last.
constexpr long kMostBlocks = 1L << 23;
static_assert(kMostBlocks * kThreads < 1L << 32, "threads of a launch");

template <typename T>
int forward(LogProbArgs<T> all) {
    const char* what = "dali_hip_token_log_probs";
    const int groups = groups_of<T>(all.vocab);
    // A wave per row up to 256 groups, and to 512 where there are rows enough for all waves, a workgroup above. Wave and workgroup, with 5 alternatives (us): 256x2000 5.9 and
    // 4.8, 1023x2000 6.0 and 6.1, 8192x2000 18 and 23, 65536x2000 107 and 164; above 512 groups 65536x3000 234 and 187.
    const bool is_short = groups <= 256 || (groups <= 512 && all.rows >= 1024);
    for (long done = 0; done < all.rows;) {
        LogProbArgs<T> a = all;
        a.rows = std::min(all.rows - done, kMostBlocks);
        a.logits += done * a.stride;
        a.tokens += done;
        a.log_probs += done, a.entropy += done, a.lse += done;
        if (a.k) a.top += done * a.k, a.top_tokens += done * a.k;
        done += a.rows;
        a.segments = 1;
        a.per = groups;
        if (is_short) {
            short_rows<512>(groups, [&](auto lanes, auto e) {
                constexpr int LANES = decltype(lanes)::value, E = decltype(e)::value, per = kThreads / LANES;
                const dim3 grid((unsigned)((a.rows + per - 1) / per));
                if (a.k) hipLaunchKernelGGL((log_prob_short<T, LANES, E, true>), grid, dim3(kThreads), 0, stream(), a);
                else hipLaunchKernelGGL((log_prob_short<T, LANES, E, false>), grid, dim3(kThreads), 0, stream(), a);
            });
            if (launched(what)) return DALI_HIP_ERROR;
            continue;
        }
        // Few long rows are cut into segments of at least 512 groups, two or three for a thread, 512 workgroups or so together. The segments' alternatives are joined in one list,
        // and a lane of one wave stands for a segment. Cut and whole, with 5 alternatives (us): 8x32000 7.3 and 9.1, 64x32000 8.1 and 9.1, 130x32000 10.8 and 9.1, 100x8000
        // 7.7 and 6.3, 130x100000 15.2 and 16.9, 250x200000 42.2 and 45.9.
        const bool cuts = (a.rows <= 128 && groups >= 4096) || (a.rows <= 256 && groups >= 16384);
        const long cut = cuts ? std::min({512L / a.rows, (long)groups / 512, (long)kList / std::max(a.k, 1), (long)kMerge}) : 1;
        if (cut > 1) {
            a.segments = (int)cut;
            a.per = (groups + a.segments - 1) / a.segments;
            a.segments = (groups + a.per - 1) / a.per;
            a.counters = (unsigned*)workspace();
            a.counter_step = counter_step(a.rows);
            a.best = (Entry<T>*)(workspace() + kWorkspaceCounterBytes);
            a.sums = (T*)(a.best + a.rows * a.segments * a.k);
        }
        const dim3 grid((unsigned)(a.rows * a.segments));
        auto launch = [&](auto top) {
            constexpr bool TOP = decltype(top)::value;
            auto held = [&](auto e) {
                if (a.per > decltype(e)::value * kThreads) return false;
                hipLaunchKernelGGL((log_prob_segments<T, TOP, decltype(e)::value>), grid, dim3(kThreads), 0, stream(), a);
                return true;
            };
            if (held(std::integral_constant<int, 2>()) || held(std::integral_constant<int, 3>()) || held(std::integral_constant<int, 4>()) ||
                held(std::integral_constant<int, 5>()) || held(std::integral_constant<int, 6>()) || held(std::integral_constant<int, 8>()))
                return;
            hipLaunchKernelGGL((log_prob_long<T, TOP>), grid, dim3(kThreads), 0, stream(), a);
        };
        if (a.k) launch(std::true_type());
        else launch(std::false_type());
        if (launched(what)) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
}

template <typename T>
int backward(LogProbBackwardArgs<T> all) {
    const bool past = past_caches(2.0 * sizeof(T) * all.rows * all.vocab);
    const int groups = groups_of<T>(all.vocab);
    const long pieces = ((long)groups + 4 * kThreads - 1) / (4 * kThreads);
    for (long done = 0; done < all.rows;) {
        LogProbBackwardArgs<T> a = all;
        a.rows = std::min(all.rows - done, std::max(1L, kMostBlocks / pieces));
        a.logits += done * a.stride;
        a.d_logits += done * a.vocab;
        a.tokens += done;
        a.d_log_probs += done, a.lse += done;
        if (a.d_entropy) a.d_entropy += done, a.entropy += done;
        done += a.rows;
        a.pieces = (int)pieces;
        const bool is_short = short_rows<256>(groups, [&](auto lanes, auto e) {
            constexpr int per = kThreads / decltype(lanes)::value;
            either_way(past, [&](auto p) {
                hipLaunchKernelGGL((log_prob_backward_short<T, decltype(lanes)::value, decltype(e)::value, decltype(p)::value>), dim3((unsigned)((a.rows + per - 1) / per)),
                                   dim3(kThreads), 0, stream(), a);
            });
        });
        if (!is_short)
            either_way(past, [&](auto p) { hipLaunchKernelGGL((log_prob_backward_long<T, decltype(p)::value>), dim3((unsigned)(a.rows * pieces)), dim3(kThreads), 0, stream(), a); });
        if (launched("dali_hip_token_log_probs_backward")) return DALI_HIP_ERROR;
    }
    return DALI_HIP_OK;
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
    if (off_elements({logits, log_probs, entropy, lse, top_log_probs}, size) || off_elements({tokens, top_tokens}, 4)) return fail("%s: an address is off its type's size", what);
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
    if (off_elements({d_log_probs, d_entropy, logits, lse, entropy, d_logits}, size) || off_elements({tokens}, 4)) return fail("%s: an address is off its type's size", what);
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT)
        return backward<float>({(const float*)d_log_probs, (const float*)d_entropy, (const float*)logits, (const float*)lse, (const float*)entropy, tokens, (float*)d_logits,
                                (long)rows, (long)stride, vocab, 1});
    return backward<double>({(const double*)d_log_probs, (const double*)d_entropy, (const double*)logits, (const double*)lse, (const double*)entropy, tokens, (double*)d_logits,
                             (long)rows, (long)stride, vocab, 1});
}
