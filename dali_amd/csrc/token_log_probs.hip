// Log probabilities of given tokens under softmax(logits), row by row, with the entropy of the row and its best alternatives; and the gradient.
//
//   m = max x,  S = sum e^(x - m),  T = sum e^(x - m) (x - m)
//   lse = m + ln S,  log p(t) = x_t - lse,  entropy = -sum p ln p = ln S - T / S
//   d x = d log p(t) (delta_t - p) - d entropy p (ln p + entropy)
//
// A value of -inf (or far below m) has weight 0 and adds nothing to the entropy. A row of -inf alone has lse = -inf, entropy 0 and no gradient.
// A NaN or +inf makes its row's results NaN. A token outside [0, vocab) stands for none: its log probability is 0 and has no gradient.
#include <algorithm>

#include "row_math.h"

namespace dali_hip {
namespace {

constexpr int kThreads = 256;

// x - m is at most 0; a weight that underflows must not meet an infinite exponent
template <typename T>
__device__ __forceinline__ T lowest() {
    return sizeof(T) == 4 ? T(-1e30f) : T(-1e300);
}

template <typename T>
struct LogProbArgs {
    const T* logits;
    const int* tokens;
    T *log_probs, *entropy, *lse, *top;
    int* top_tokens;
    long rows, stride;
    int vocab, k;
};

// of two entries the better: the larger value, the lower position among equals
template <typename T>
__device__ __forceinline__ bool better(T v, int i, T w, int j) {
    return v > w || (v == w && i < j);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void log_prob_rows(LogProbArgs<T> a) {
    __shared__ T scratch[kThreads / 64];
    __shared__ int positions[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the best entry that all threads hold
    auto best_of_all = [&](T& v, int& i) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const T w = __shfl_xor(v, d, 64);
            const int j = __shfl_xor(i, d, 64);
            if (better(w, j, v, i)) v = w, i = j;
        }
        __syncthreads();
        if (lane == 0) scratch[wave] = v, positions[wave] = i;
        __syncthreads();
        v = scratch[0], i = positions[0];
        for (int w = 1; w < kThreads / 64; ++w)
            if (better(scratch[w], positions[w], v, i)) v = scratch[w], i = positions[w];
    };
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = a.logits + r * a.stride;
        T lse = 0;
        {
            T m = -INFINITY;
            int at = a.vocab;
            for (int c = threadIdx.x; c < a.vocab; c += kThreads)
                if (better(x[c], c, m, at)) m = x[c], at = c;
            best_of_all(m, at);
            const T base = m == T(-INFINITY) ? T(0) : m;
            T s = 0, t = 0;
            for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
                const T d = x[c] - base, e = exp(d);
                s += e;
                t += e * fmax(d, lowest<T>());
            }
            s = block_sum<kThreads>(s, scratch);
            t = block_sum<kThreads>(t, scratch);
            const T ln = log(s);
            lse = base + ln;
            if (threadIdx.x == 0) {
                const int token = a.tokens[r];
                a.lse[r] = lse;
                a.entropy[r] = s == T(0) ? T(0) : ln - t / s;
                a.log_probs[r] = token < 0 || token >= a.vocab ? T(0) : s == T(0) ? T(-INFINITY) : (x[token] - base) - ln;
            }
        }
        // the alternatives, one after the other: the best of what comes after the one before (NaN ranks as -inf)
        T last = INFINITY;
        int last_at = -1;
        for (int n = 0; n < a.k; ++n) {
            T v = -INFINITY;
            int at = a.vocab;
            for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
                const T w = x[c] == x[c] ? x[c] : T(-INFINITY);
                if (better(last, last_at, w, c) && better(w, c, v, at)) v = w, at = c;
            }
            best_of_all(v, at);
            if (threadIdx.x == 0) {
                a.top[r * a.k + n] = lse == T(-INFINITY) ? T(-INFINITY) : x[at] - lse;
                a.top_tokens[r * a.k + n] = at;
            }
            last = v;
            last_at = at;
        }
        __syncthreads();
    }
}

template <typename T>
struct LogProbBackwardArgs {
    const T *d_log_probs, *d_entropy, *logits, *lse, *entropy;
    const int* tokens;
    T* d_logits;
    long rows, stride;
    int vocab;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void log_prob_backward_rows(LogProbBackwardArgs<T> a) {
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = a.logits + r * a.stride;
        T* out = a.d_logits + r * a.vocab;
        const int token = a.tokens[r];
        const bool none = token < 0 || token >= a.vocab, nothing = a.lse[r] == T(-INFINITY);
        const T lse = nothing ? T(0) : a.lse[r], g = none || nothing ? T(0) : a.d_log_probs[r];
        const T h = a.d_entropy ? a.d_entropy[r] : T(0), entropy = a.d_entropy ? a.entropy[r] : T(0);
        for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
            const T d = x[c] - lse, p = exp(d);
            out[c] = (c == token ? g : T(0)) - p * (g + h * (fmax(d, lowest<T>()) + entropy));
        }
    }
}

template <typename T>
int forward(LogProbArgs<T> a) {
    hipLaunchKernelGGL(log_prob_rows<T>, dim3((unsigned)std::min(a.rows, 65536L)), dim3(kThreads), 0, stream(), a);
    return launched("dali_hip_token_log_probs");
}

template <typename T>
int backward(LogProbBackwardArgs<T> a) {
    hipLaunchKernelGGL(log_prob_backward_rows<T>, dim3((unsigned)std::min(a.rows, 65536L)), dim3(kThreads), 0, stream(), a);
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
                                (long)rows, (long)stride, vocab});
    return backward<double>({(const double*)d_log_probs, (const double*)d_entropy, (const double*)logits, (const double*)lse, (const double*)entropy, tokens, (double*)d_logits,
                             (long)rows, (long)stride, vocab});
}
