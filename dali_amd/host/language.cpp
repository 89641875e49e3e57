// Operators that language models are trained, scored and answered with, over the library's own kernels: layer normalisation, log probabilities of
// tokens, clipping by the global norm. They are evaluated when called, as the composites of array.cpp are, write into new arrays or into
// destinations that the caller keeps, and record themselves like any other launch.
#include "../../include/dali_hip.h"
#include "jit_internal.h"

namespace dali {
namespace {

// the operand as rows along its last axis: a view whose rows are dense and evenly spaced is read where it lies, anything else is laid out first
struct Rows {
    Array array;
    int64_t rows = 1, stride = 0;
    int width = 0;
};

Rows as_rows(const Array& a) {
    a.eval();
    const std::vector<int>& shape = a.shape();
    Rows r;
    r.array = a;
    r.width = shape.back();
    for (size_t i = 0; i + 1 < shape.size(); ++i) r.rows *= shape[i];
    r.stride = r.width;
    if (a.contiguous_memory()) return r;
    const std::vector<int> st = a.normalized_strides();
    bool dense = r.width == 1 || st.back() == 1, first = true;
    int64_t next = 0;  // the stride that the axis in front has to have
    for (int i = (int)shape.size() - 2; i >= 0 && dense; --i) {
        if (shape[i] == 1) continue;
        if (first) r.stride = st[i];
        else dense = st[i] == next;
        first = false;
        next = (int64_t)st[i] * shape[i];
    }
    if (!dense) {
        r.array = a.ascontiguousarray();
        r.stride = r.width;
    }
    return r;
}

Array dense(const Array& a) {
    a.eval();
    return a.contiguous_memory() ? a : a.ascontiguousarray();
}

bool is_real(const Array& a) { return a.dtype() == DTYPE_FLOAT || a.dtype() == DTYPE_DOUBLE; }

std::vector<int> leading(const Array& a) { return std::vector<int>(a.shape().begin(), a.shape().end() - 1); }

void check_shape(const char* what, const char* name, const Array& a, const std::vector<int>& shape, DType dtype) {
    DALI_ASSERT(a.shape() == shape && a.dtype() == dtype,
                make_message(what, ": ", name, " must be ", dtype_to_cpp_name(dtype), " of shape ", shape_str(shape), ", got ", dtype_to_cpp_name(a.dtype()), " of shape ",
                             shape_str(a.shape())));
}

// the array that receives a result: the caller's, or a new one
Array destination(const char* what, const char* name, const Array& given, const std::vector<int>& shape, DType dtype) {
    if (given.is_stateless()) return Array(shape, dtype);
    check_shape(what, name, given, shape, dtype);
    DALI_ASSERT(given.is_buffer() && given.contiguous_memory(), make_message(what, ": the destination of ", name, " must be a dense buffer"));
    return given;
}

const void* read(const Array& a) { return a.is_stateless() ? nullptr : a.device_ptr(); }
// (what a destination held stays if the call is refused)
void* write(const Array& a) { return a.is_stateless() ? nullptr : a.device_ptr(memory::AM_MUTABLE); }

// Issues the launch now and, while a recording is open, on every replay. `keep`: makes the list of all arrays that it reads, and of those that it writes.
template <typename Launch, typename Keep>
void issue(const char* kind, const Launch& launch, const Keep& keep) {
    DALI_SCOPE(kind);
    check_hip(launch(), kind);
    jit_stats().kernels_launched++;
    jit_stats().last_kernel_kinds = kind;
    if (!g_recording) return;
    std::vector<Array> reads, writes;
    keep(reads, writes);
    for (const Array& a : writes)
        if (!a.is_stateless()) note_recorded_write(a.expression()->memory);
    g_recording->push_back([kind, reads, writes, launch]() { check_hip(launch(), kind); });
}

}  // namespace

namespace op {

LayerNorm layer_norm(const Array& x, const Array& gamma, const Array& beta, double epsilon, const LayerNorm& out) {
    const char* what = "layer_norm";
    DALI_ASSERT(x.ndim() >= 1 && is_real(x) && x.shape().back() >= 1, make_message(what, ": x must be float or double and have a last axis that is not empty"));
    const DType dtype = x.dtype();
    const std::vector<int> vector = {x.shape().back()};
    if (!gamma.is_stateless()) check_shape(what, "gamma", gamma, vector, dtype);
    if (!beta.is_stateless()) check_shape(what, "beta", beta, vector, dtype);
    LayerNorm r = {destination(what, "y", out.y, x.shape(), dtype), destination(what, "mean", out.mean, leading(x), dtype),
                   destination(what, "rstd", out.rstd, leading(x), dtype)};
    const Rows in = as_rows(x);
    const Array g = gamma.is_stateless() ? gamma : dense(gamma), b = beta.is_stateless() ? beta : dense(beta);
    if (g_dry_run) return r;
    const void *xp = read(in.array), *gp = read(g), *bp = read(b);
    void *yp = write(r.y), *mp = write(r.mean), *sp = write(r.rstd);
    const int64_t rows = in.rows, stride = in.stride;
    const int width = in.width;
    issue(
        what, [=]() { return dali_hip_layer_norm(dtype, rows, width, xp, stride, gp, bp, epsilon, yp, mp, sp); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {in.array, g, b}, writes = {r.y, r.mean, r.rstd}; });
    return r;
}

LayerNormGradient layer_norm_backward(const Array& dy, const Array& x, const Array& mean, const Array& rstd, const Array& gamma, const LayerNormGradient& out) {
    const char* what = "layer_norm_backward";
    DALI_ASSERT(x.ndim() >= 1 && is_real(x) && x.shape().back() >= 1, make_message(what, ": x must be float or double and have a last axis that is not empty"));
    const DType dtype = x.dtype();
    const std::vector<int> vector = {x.shape().back()};
    check_shape(what, "dy", dy, x.shape(), dtype);
    check_shape(what, "mean", mean, leading(x), dtype);
    check_shape(what, "rstd", rstd, leading(x), dtype);
    const bool weights = !gamma.is_stateless();
    if (weights) check_shape(what, "gamma", gamma, vector, dtype);
    DALI_ASSERT(weights || (out.gamma.is_stateless() && out.beta.is_stateless()), make_message(what, ": without gamma there are no gradients of weights to write"));
    LayerNormGradient r;
    r.x = destination(what, "dx", out.x, x.shape(), dtype);
    if (weights) {
        r.gamma = destination(what, "dgamma", out.gamma, vector, dtype);
        r.beta = destination(what, "dbeta", out.beta, vector, dtype);
    }
    const Rows gy = as_rows(dy), in = as_rows(x);
    const Array m = dense(mean), s = dense(rstd), g = weights ? dense(gamma) : gamma;
    if (g_dry_run) return r;
    const void *dyp = read(gy.array), *xp = read(in.array), *mp = read(m), *sp = read(s), *gp = read(g);
    void *dxp = write(r.x), *dgp = write(r.gamma), *dbp = write(r.beta);
    const int64_t rows = in.rows, x_stride = in.stride, dy_stride = gy.stride;
    const int width = in.width;
    issue(
        what, [=]() { return dali_hip_layer_norm_backward(dtype, rows, width, dyp, dy_stride, xp, x_stride, mp, sp, gp, dxp, dgp, dbp); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {gy.array, in.array, m, s, g}, writes = {r.x, r.gamma, r.beta}; });
    return r;
}

TokenLogProbs token_log_probs(const Array& logits, const Array& tokens, int k, const TokenLogProbs& out) {
    const char* what = "token_log_probs";
    DALI_ASSERT(logits.ndim() >= 1 && is_real(logits) && logits.shape().back() >= 1,
                make_message(what, ": logits must be float or double and have a last axis that is not empty"));
    const DType dtype = logits.dtype();
    const std::vector<int> rows_shape = leading(logits);
    check_shape(what, "tokens", tokens, rows_shape, DTYPE_INT32);
    DALI_ASSERT(k >= 0 && k <= DALI_HIP_MAX_ALTERNATIVES && k <= logits.shape().back(),
                make_message(what, ": k must be from 0 to ", std::min(DALI_HIP_MAX_ALTERNATIVES, logits.shape().back()), " here (got ", k, ")"));
    DALI_ASSERT(k > 0 || (out.top_log_probs.is_stateless() && out.top_tokens.is_stateless()), make_message(what, ": with k = 0 there are no alternatives to write"));
    TokenLogProbs r;
    r.log_probs = destination(what, "log_probs", out.log_probs, rows_shape, dtype);
    r.entropy = destination(what, "entropy", out.entropy, rows_shape, dtype);
    r.lse = destination(what, "lse", out.lse, rows_shape, dtype);
    if (k) {
        std::vector<int> top = logits.shape();
        top.back() = k;
        r.top_log_probs = destination(what, "top_log_probs", out.top_log_probs, top, dtype);
        r.top_tokens = destination(what, "top_tokens", out.top_tokens, top, DTYPE_INT32);
    }
    const Rows in = as_rows(logits);
    const Array t = dense(tokens);
    if (g_dry_run) return r;
    const void *xp = read(in.array), *tp = read(t);
    void *pp = write(r.log_probs), *ep = write(r.entropy), *lp = write(r.lse), *vp = write(r.top_log_probs), *ip = write(r.top_tokens);
    const int64_t rows = in.rows, stride = in.stride;
    const int vocab = in.width;
    issue(
        what, [=]() { return dali_hip_token_log_probs(dtype, rows, vocab, xp, stride, (const int32_t*)tp, k, pp, ep, lp, vp, (int32_t*)ip); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {in.array, t}, writes = {r.log_probs, r.entropy, r.lse, r.top_log_probs, r.top_tokens}; });
    return r;
}

Array token_log_probs_backward(const Array& d_log_probs, const Array& d_entropy, const Array& logits, const Array& tokens, const Array& lse, const Array& entropy,
                               const Array& out) {
    const char* what = "token_log_probs_backward";
    DALI_ASSERT(logits.ndim() >= 1 && is_real(logits) && logits.shape().back() >= 1,
                make_message(what, ": logits must be float or double and have a last axis that is not empty"));
    const DType dtype = logits.dtype();
    const std::vector<int> rows_shape = leading(logits);
    check_shape(what, "d_log_probs", d_log_probs, rows_shape, dtype);
    check_shape(what, "tokens", tokens, rows_shape, DTYPE_INT32);
    check_shape(what, "lse", lse, rows_shape, dtype);
    const bool with_entropy = !d_entropy.is_stateless();
    if (with_entropy) {
        check_shape(what, "d_entropy", d_entropy, rows_shape, dtype);
        DALI_ASSERT(!entropy.is_stateless(), make_message(what, ": the gradient of the entropy needs the entropy"));
        check_shape(what, "entropy", entropy, rows_shape, dtype);
    }
    const Array r = destination(what, "d_logits", out, logits.shape(), dtype);
    const Rows in = as_rows(logits);
    const Array g = dense(d_log_probs), t = dense(tokens), l = dense(lse), h = with_entropy ? dense(d_entropy) : Array(), e = with_entropy ? dense(entropy) : Array();
    if (g_dry_run) return r;
    const void *gp = read(g), *hp = read(h), *xp = read(in.array), *tp = read(t), *lp = read(l), *ep = read(e);
    void* rp = write(r);
    const int64_t rows = in.rows, stride = in.stride;
    const int vocab = in.width;
    issue(
        what, [=]() { return dali_hip_token_log_probs_backward(dtype, rows, vocab, gp, hp, xp, stride, (const int32_t*)tp, lp, ep, rp); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {in.array, g, t, l, h, e}, writes = {r}; });
    return r;
}

static Array norm_of(const char* what, const std::vector<Array>& arrays, double max_norm, const std::vector<Array>* clipped, const Array& out) {
    DALI_ASSERT(!arrays.empty(), make_message(what, ": needs at least one array"));
    const size_t count = arrays.size();
    const DType dtype = arrays[0].dtype();
    std::vector<Array> laid_out;  // of arrays that are not dense
    std::vector<void*> pointers(2 * count);
    std::vector<int64_t> sizes(count);
    for (const Array& a : arrays) DALI_ASSERT(is_real(a) && a.dtype() == dtype, make_message(what, ": the arrays must be float or double, all of one type"));
    const Array norm = destination(what, "the norm", out, {}, dtype);
    if (g_dry_run) return norm;
    for (size_t i = 0; i < count; ++i) {
        const Array a = dense(arrays[i]);
        sizes[i] = a.number_of_elements();
        pointers[i] = a.device_ptr();
        if (a.state_ != arrays[i].state_) laid_out.push_back(a);
    }
    if (clipped)
        for (size_t i = 0; i < count; ++i) pointers[count + i] = write((*clipped)[i]);
    void* np = write(norm);
    const bool clip = clipped != nullptr;
    issue(
        what,
        [dtype, count, pointers, sizes, max_norm, clip, np]() {
            return dali_hip_clip_by_global_norm(dtype, (int)count, pointers.data(), clip ? pointers.data() + count : nullptr, sizes.data(), max_norm, np);
        },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) {
            reads = arrays;
            reads.insert(reads.end(), laid_out.begin(), laid_out.end());
            if (clipped) writes = *clipped;
            writes.push_back(norm);
        });
    return norm;
}

Array global_norm(const std::vector<Array>& arrays, const Array& out) { return norm_of("global_norm", arrays, 0.0, nullptr, out); }

ClippedArrays clip_by_global_norm(const std::vector<Array>& arrays, double max_norm, const ClippedArrays& out) {
    const char* what = "clip_by_global_norm";
    DALI_ASSERT(max_norm >= 0, make_message(what, ": max_norm must not be negative (got ", max_norm, ")"));
    DALI_ASSERT(out.arrays.empty() || out.arrays.size() == arrays.size(),
                make_message(what, ": ", arrays.size(), " arrays and ", out.arrays.size(), " destinations"));
    ClippedArrays r;
    for (size_t i = 0; i < arrays.size(); ++i)
        r.arrays.push_back(destination(what, "an array", out.arrays.empty() ? Array() : out.arrays[i], arrays[i].shape(), arrays[i].dtype()));
    r.norm = norm_of(what, arrays, max_norm, &r.arrays, out.norm);
    return r;
}

}  // namespace op
}  // namespace dali
