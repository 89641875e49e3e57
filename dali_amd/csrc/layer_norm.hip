// Layer normalisation along the last axis and its gradient.
//
//   mean = sum(x) / n,  rstd = 1 / sqrt(sum((x - mean)^2) / n + epsilon),  y = (x - mean) rstd gamma + beta
//   u = (x - mean) rstd,  a = dy gamma,  dx = rstd (a - mean(a) - u mean(a u)),  dgamma = sum over rows of dy u,  dbeta = that of dy
//
// Sums are held in the operands' own type (32 bits or more). The variance is the mean of squared distances from the mean, with the mean's own
// rounding error taken out again (x - mean sums to delta n where the mean is off by delta): rows far from zero keep their digits.
#include <algorithm>

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

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_rows(NormArgs<T> a) {
    __shared__ T scratch[kThreads / 64];
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = a.x + r * a.stride;
        T s = 0;
        for (int c = threadIdx.x; c < a.width; c += kThreads) s += x[c];
        const T near = block_sum<kThreads>(s, scratch) / a.width;
        T off = 0, sq = 0;
        for (int c = threadIdx.x; c < a.width; c += kThreads) {
            const T d = x[c] - near;
            off += d;
            sq += d * d;
        }
        off = block_sum<kThreads>(off, scratch) / a.width;
        sq = block_sum<kThreads>(sq, scratch) / a.width - off * off;
        const T rstd = T(1) / sqrt((sq > 0 || sq != sq ? sq : T(0)) + a.epsilon);
        T* y = a.y + r * a.width;
        for (int c = threadIdx.x; c < a.width; c += kThreads) {
            const T u = ((x[c] - near) - off) * rstd;
            y[c] = u * (a.gamma ? a.gamma[c] : T(1)) + (a.beta ? a.beta[c] : T(0));
        }
        if (threadIdx.x == 0) {
            a.mean[r] = near + off;
            a.rstd[r] = rstd;
        }
    }
}

template <typename T>
struct NormBackwardArgs {
    const T *dy, *x, *mean, *rstd, *gamma;
    T *dx, *dgamma, *dbeta;
    T* partial;  // [parts][2][width]
    long rows, dy_stride, x_stride;
    int width, parts;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_backward_rows(NormBackwardArgs<T> a) {
    __shared__ T scratch[kThreads / 64];
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = a.x + r * a.x_stride, *dy = a.dy + r * a.dy_stride;
        const T mean = a.mean[r], rstd = a.rstd[r];
        T level = 0, along = 0;
        for (int c = threadIdx.x; c < a.width; c += kThreads) {
            const T g = dy[c] * (a.gamma ? a.gamma[c] : T(1));
            level += g;
            along += g * ((x[c] - mean) * rstd);
        }
        level = block_sum<kThreads>(level, scratch) / a.width;
        along = block_sum<kThreads>(along, scratch) / a.width;
        T* dx = a.dx + r * a.width;
        for (int c = threadIdx.x; c < a.width; c += kThreads) {
            const T g = dy[c] * (a.gamma ? a.gamma[c] : T(1));
            dx[c] = rstd * ((g - level) - (x[c] - mean) * rstd * along);
        }
    }
}

// columns of one strip over one part of the rows, then the parts in order
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_weights(NormBackwardArgs<T> a) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.width) return;
    T g = 0, b = 0;
    for (long r = blockIdx.y; r < a.rows; r += a.parts) {
        const T d = a.dy[r * a.dy_stride + c];
        g += d * ((a.x[r * a.x_stride + c] - a.mean[r]) * a.rstd[r]);
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

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_fold(NormBackwardArgs<T> a) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.width) return;
    T g = 0, b = 0;
    for (int i = 0; i < a.parts; ++i) {
        g += a.partial[(long)i * 2 * a.width + c];
        b += a.partial[(long)i * 2 * a.width + a.width + c];
    }
    a.dgamma[c] = g;
    a.dbeta[c] = b;
}

template <typename T>
int forward(NormArgs<T> a) {
    hipLaunchKernelGGL(norm_rows<T>, dim3((unsigned)std::min(a.rows, 65536L)), dim3(kThreads), 0, stream(), a);
    return launched("dali_hip_layer_norm");
}

template <typename T>
int backward(NormBackwardArgs<T> a) {
    // (the weights first: dx may take the place of x or dy)
    if (a.dgamma) {
        const long fit = (long)(kWorkspacePartialBytes / (2 * sizeof(T) * (size_t)a.width));
        a.parts = (int)std::max(1L, std::min({64L, a.rows, fit}));
        a.partial = (T*)(workspace() + kWorkspaceCounterBytes);
        const dim3 grid((a.width + kThreads - 1) / kThreads, a.parts);
        hipLaunchKernelGGL(norm_weights<T>, grid, dim3(kThreads), 0, stream(), a);
        if (a.parts > 1) hipLaunchKernelGGL(norm_fold<T>, dim3(grid.x), dim3(kThreads), 0, stream(), a);
    }
    if (a.rows > 0) hipLaunchKernelGGL(norm_backward_rows<T>, dim3((unsigned)std::min(a.rows, 65536L)), dim3(kThreads), 0, stream(), a);
    return launched("dali_hip_layer_norm_backward");
}

}  // namespace
}  // namespace dali_hip

using namespace dali_hip;

extern "C" int dali_hip_layer_norm(int dtype, int64_t rows, int width, const void* x, int64_t x_stride, const void* gamma, const void* beta, double epsilon, void* y,
                                   void* mean, void* rstd) {
    const char* what = "dali_hip_layer_norm";
    if (!is_real(dtype)) return fail("%s: dtype %d is neither float nor double", what, dtype);
    if (rows < 0 || width < 1) return fail("%s: %lld rows of %d values", what, (long long)rows, width);
    if (!(epsilon >= 0) || epsilon > 1e30) return fail("%s: epsilon must be a number that is not negative (got %g)", what, epsilon);
    if (rows == 0) return DALI_HIP_OK;
    if (!x || !y || !mean || !rstd) return fail("%s: NULL argument", what);
    const size_t size = dtype == DALI_HIP_FLOAT ? 4 : 8;
    if (check_spans(what, {Span("y", y, rows * width, size), Span("mean", mean, rows, size), Span("rstd", rstd, rows, size)},
                    {Span("x", x, rows, width, x_stride, size), Span("gamma", gamma, width, size), Span("beta", beta, width, size)}, 1))
        return DALI_HIP_ERROR;
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
    if (ensure_init()) return DALI_HIP_ERROR;
    if (dtype == DALI_HIP_FLOAT)
        return backward<float>({(const float*)dy, (const float*)x, (const float*)mean, (const float*)rstd, (const float*)gamma, (float*)dx, (float*)dgamma, (float*)dbeta, nullptr,
                                (long)rows, (long)dy_stride, (long)x_stride, width, 1});
    return backward<double>({(const double*)dy, (const double*)x, (const double*)mean, (const double*)rstd, (const double*)gamma, (double*)dx, (double*)dgamma, (double*)dbeta,
                             nullptr, (long)rows, (long)dy_stride, (long)x_stride, width, 1});
}
