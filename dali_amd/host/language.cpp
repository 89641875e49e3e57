// Operators that language models are trained, scored and answered with, over the library's own kernels: layer normalisation, log probabilities of
// tokens, clipping by the global norm, embedding rows, attention to an encoder's states, cross entropy of a projection. They are evaluated when called, as the composites of array.cpp are, write into new arrays or into
// destinations that the caller keeps, and record themselves like any other launch.
#include <array>
#include <cmath>

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

void check_scale(const char* what, double scale, DType dtype) {
    DALI_ASSERT(std::isfinite(dtype == DTYPE_FLOAT ? (double)(float)scale : scale),
                make_message(what, ": the scale must be finite (got ", scale, " for ", dtype_to_cpp_name(dtype), ")"));
}

// what an entry of the library keeps beside its operands for the time of a call (or as long as a recording holds it)
template <typename Bytes>
Array workspace(const char* what, const Bytes& bytes) {
    size_t n = 0;
    check_hip(bytes(&n), what);
    if (n == 0) return Array();
    DALI_ASSERT(n / 8 < 2147483647u, make_message(what, ": a workspace of ", n, " bytes"));
    return Array({(int)(n / 8) + 1}, DTYPE_DOUBLE);
}

// the operand [batch, rows, heads, width] with the strides of its first three axes: a view whose last axis is dense is read where it lies
struct Heads {
    Array array;
    std::array<int64_t, 3> strides;
};

Heads as_heads(const Array& a) {
    a.eval();
    Heads h;
    h.array = a;
    const std::vector<int>& shape = a.shape();
    if (!a.contiguous_memory()) {
        const std::vector<int> st = a.normalized_strides();
        if (shape[3] == 1 || st[3] == 1) {
            h.strides = {st[0], st[1], st[2]};
            return h;
        }
        h.array = a.ascontiguousarray();
    }
    h.strides = {(int64_t)shape[1] * shape[2] * shape[3], (int64_t)shape[2] * shape[3], shape[3]};
    return h;
}

// a matrix as the products take it: rows `stride` apart, or (by_columns) its transposition's
struct Projection {
    Array array;
    int64_t stride = 0;
    bool by_columns = false;
};

Projection as_projection(const Array& w) {
    w.eval();
    Projection p;
    p.array = w;
    const int rows = w.shape()[0], cols = w.shape()[1];
    p.stride = cols;
    if (w.contiguous_memory()) return p;
    const std::vector<int> st = w.normalized_strides();
    if (st[1] == 1 && st[0] >= cols) {
        p.stride = st[0];
    } else if (st[0] == 1 && st[1] >= rows) {
        p.by_columns = true;
        p.stride = st[1];
    } else {
        p.array = w.ascontiguousarray();
    }
    return p;
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

Array embedding(const Array& table, const Array& tokens, double scale, const Array& out) {
    const char* what = "embedding";
    DALI_ASSERT(table.ndim() == 2 && is_real(table) && table.shape()[0] >= 1 && table.shape()[1] >= 1,
                make_message(what, ": the table must be a float or double matrix that is not empty"));
    DALI_ASSERT(tokens.dtype() == DTYPE_INT32, make_message(what, ": tokens must be int"));
    check_scale(what, scale, table.dtype());
    const DType dtype = table.dtype();
    std::vector<int> shape = tokens.shape();
    shape.push_back(table.shape()[1]);
    const Array y = destination(what, "y", out, shape, dtype);
    const Rows in = as_rows(table);
    const Array t = dense(tokens);
    if (g_dry_run) return y;
    const void *xp = read(in.array), *tp = read(t);
    void* yp = write(y);
    const int64_t count = t.number_of_elements(), stride = in.stride;
    const int rows = table.shape()[0], width = in.width;
    issue(
        what, [=]() { return dali_hip_embedding(dtype, count, rows, width, xp, stride, (const int32_t*)tp, scale, yp); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {in.array, t}, writes = {y}; });
    return y;
}

Array embedding_backward(const Array& dy, const Array& tokens, int rows, double scale, const Array& out) {
    const char* what = "embedding_backward";
    DALI_ASSERT(dy.ndim() >= 1 && is_real(dy) && dy.shape().back() >= 1, make_message(what, ": dy must be float or double and have a last axis that is not empty"));
    check_shape(what, "tokens", tokens, leading(dy), DTYPE_INT32);
    DALI_ASSERT(rows >= 1, make_message(what, ": a table has at least one row (got ", rows, ")"));
    check_scale(what, scale, dy.dtype());
    const DType dtype = dy.dtype();
    const int width = dy.shape().back();
    const Array r = destination(what, "dtable", out, {rows, width}, dtype);
    const Rows in = as_rows(dy);
    const Array t = dense(tokens);
    const int64_t count = t.number_of_elements(), stride = in.stride;
    const Array space = workspace(what, [&](size_t* n) { return dali_hip_embedding_backward_workspace(dtype, count, rows, width, n); });
    if (g_dry_run) return r;
    const void *xp = count ? read(in.array) : nullptr, *tp = count ? read(t) : nullptr;
    void *rp = write(r), *sp = write(space);
    issue(
        what, [=]() { return dali_hip_embedding_backward(dtype, count, rows, width, xp, stride, (const int32_t*)tp, scale, rp, sp); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {in.array, t}, writes = {r, space}; });
    return r;
}

// what both directions of attention ask of their operands; the sizes that the entries take
struct AttentionSizes {
    DType dtype;
    int batch, queries, keys, heads, kv_heads, width;
    AttentionSizes(const char* what, const Array& q, const Array& k, const Array& v, const Array& counts, double scale) {
        DALI_ASSERT(q.ndim() == 4 && is_real(q), make_message(what, ": queries must be float or double of shape [batch, positions, heads, width]"));
        dtype = q.dtype();
        batch = q.shape()[0], queries = q.shape()[1], heads = q.shape()[2], width = q.shape()[3];
        DALI_ASSERT(width >= 1 && width <= DALI_HIP_MAX_HEAD_WIDTH, make_message(what, ": heads are from 1 to ", DALI_HIP_MAX_HEAD_WIDTH, " wide (got ", width, ")"));
        DALI_ASSERT(k.ndim() == 4 && k.dtype() == dtype && k.shape()[0] == batch && k.shape()[3] == width,
                    make_message(what, ": keys must be ", dtype_to_cpp_name(dtype), " of shape [", batch, ", states, shared heads, ", width, "], got ", dtype_to_cpp_name(k.dtype()), " of shape ",
                                 shape_str(k.shape())));
        keys = k.shape()[1], kv_heads = k.shape()[2];
        check_shape(what, "values", v, k.shape(), dtype);
        DALI_ASSERT(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, make_message(what, ": ", heads, " heads cannot share ", kv_heads));
        if (!counts.is_stateless()) check_shape(what, "key_counts", counts, {batch}, DTYPE_INT32);
        check_scale(what, scale, dtype);
    }
};

Attention cross_attention(const Array& queries, const Array& keys, const Array& values, const Array& key_counts, double scale, const Attention& out) {
    const char* what = "cross_attention";
    const AttentionSizes z(what, queries, keys, values, key_counts, scale);
    const std::vector<int> rows = leading(queries);
    Attention r = {destination(what, "y", out.y, queries.shape(), z.dtype), destination(what, "lse", out.lse, rows, z.dtype)};
    const Heads q = as_heads(queries), k = as_heads(keys), v = as_heads(values);
    const Array n = key_counts.is_stateless() ? key_counts : dense(key_counts);
    const Array space = workspace(
        what, [&](size_t* bytes) { return dali_hip_cross_attention_workspace(z.dtype, z.batch, z.queries, z.keys, z.heads, z.kv_heads, z.width, 0, bytes); });
    if (g_dry_run) return r;
    const void *qp = read(q.array), *kp = read(k.array), *vp = read(v.array), *np = read(n);
    void *yp = write(r.y), *lp = write(r.lse), *sp = write(space);
    const auto qs = q.strides, ks = k.strides, vs = v.strides;
    issue(
        what,
        [=]() {
            return dali_hip_cross_attention(z.dtype, z.batch, z.queries, z.keys, z.heads, z.kv_heads, z.width, qp, qs.data(), kp, ks.data(), vp, vs.data(),
                                            (const int32_t*)np, scale, yp, lp, sp);
        },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {q.array, k.array, v.array, n}, writes = {r.y, r.lse, space}; });
    return r;
}

AttentionGradient cross_attention_backward(const Array& dy, const Array& queries, const Array& keys, const Array& values, const Array& y, const Array& lse,
                                           const Array& key_counts, double scale, const AttentionGradient& out) {
    const char* what = "cross_attention_backward";
    const AttentionSizes z(what, queries, keys, values, key_counts, scale);
    check_shape(what, "dy", dy, queries.shape(), z.dtype);
    check_shape(what, "y", y, queries.shape(), z.dtype);
    check_shape(what, "lse", lse, leading(queries), z.dtype);
    AttentionGradient r = {destination(what, "d_queries", out.queries, queries.shape(), z.dtype), destination(what, "d_keys", out.keys, keys.shape(), z.dtype),
                           destination(what, "d_values", out.values, keys.shape(), z.dtype)};
    const Heads g = as_heads(dy), q = as_heads(queries), k = as_heads(keys), v = as_heads(values);
    const Array yd = dense(y), l = dense(lse), n = key_counts.is_stateless() ? key_counts : dense(key_counts);
    const Array space = workspace(
        what, [&](size_t* bytes) { return dali_hip_cross_attention_workspace(z.dtype, z.batch, z.queries, z.keys, z.heads, z.kv_heads, z.width, 1, bytes); });
    if (g_dry_run) return r;
    const void *gp = read(g.array), *qp = read(q.array), *kp = read(k.array), *vp = read(v.array), *yp = read(yd), *lp = read(l), *np = read(n);
    void *dqp = write(r.queries), *dkp = write(r.keys), *dvp = write(r.values), *sp = write(space);
    const auto gs = g.strides, qs = q.strides, ks = k.strides, vs = v.strides;
    issue(
        what,
        [=]() {
            return dali_hip_cross_attention_backward(z.dtype, z.batch, z.queries, z.keys, z.heads, z.kv_heads, z.width, gp, gs.data(), qp, qs.data(), kp, ks.data(), vp,
                                                     vs.data(), yp, lp, (const int32_t*)np, scale, dqp, dkp, dvp, sp);
        },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) {
            reads = {g.array, q.array, k.array, v.array, yd, l, n}, writes = {r.queries, r.keys, r.values, space};
        });
    return r;
}

// rows of x as a product takes them: whole rows one after the other
static Rows as_whole_rows(const Array& x) {
    Rows r = as_rows(x);
    if (r.rows > 1 && r.stride < r.width) {
        r.array = x.ascontiguousarray();
        r.stride = r.width;
    }
    return r;
}

static void check_projection(const char* what, const Array& x, const Array& w, const Array& targets, const Array& bias) {
    DALI_ASSERT(x.ndim() >= 1 && is_real(x) && x.shape().back() >= 1, make_message(what, ": x must be float or double and have a last axis that is not empty"));
    const int inputs = x.shape().back();
    DALI_ASSERT(w.ndim() == 2 && w.dtype() == x.dtype() && w.shape()[0] == inputs && w.shape()[1] >= 1,
                make_message(what, ": w must be ", dtype_to_cpp_name(x.dtype()), " of shape [", inputs, ", vocabulary], got ", dtype_to_cpp_name(w.dtype()), " of shape ",
                             shape_str(w.shape())));
    check_shape(what, "targets", targets, leading(x), DTYPE_INT32);
    if (!bias.is_stateless()) check_shape(what, "bias", bias, {w.shape()[1]}, x.dtype());
}

ProjectedCrossEntropy projected_cross_entropy(const Array& x, const Array& w, const Array& targets, const Array& bias, const ProjectedCrossEntropy& out) {
    const char* what = "projected_cross_entropy";
    check_projection(what, x, w, targets, bias);
    const DType dtype = x.dtype();
    ProjectedCrossEntropy r = {destination(what, "losses", out.losses, leading(x), dtype), destination(what, "lse", out.lse, leading(x), dtype)};
    const Rows in = as_whole_rows(x);
    const Projection p = as_projection(w);
    const Array t = dense(targets), b = bias.is_stateless() ? bias : dense(bias);
    const int64_t rows = in.rows, stride = in.stride, w_stride = p.stride;
    const int inputs = in.width, vocab = w.shape()[1], by_columns = p.by_columns;
    const Array space =
        workspace(what, [&](size_t* n) { return dali_hip_projected_cross_entropy_workspace(dtype, rows, inputs, vocab, 0, !b.is_stateless(), n); });
    if (g_dry_run) return r;
    const void *xp = read(in.array), *wp = read(p.array), *tp = read(t), *bp = read(b);
    void *op = write(r.losses), *lp = write(r.lse), *sp = write(space);
    issue(
        what,
        [=]() { return dali_hip_projected_cross_entropy(dtype, rows, inputs, vocab, xp, stride, wp, w_stride, by_columns, bp, (const int32_t*)tp, op, lp, sp); },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {in.array, p.array, t, b}, writes = {r.losses, r.lse, space}; });
    return r;
}

ProjectedCrossEntropyGradient projected_cross_entropy_backward(const Array& d_losses, const Array& x, const Array& w, const Array& targets, const Array& lse,
                                                               const Array& bias, const ProjectedCrossEntropyGradient& out) {
    const char* what = "projected_cross_entropy_backward";
    check_projection(what, x, w, targets, bias);
    const DType dtype = x.dtype();
    check_shape(what, "d_losses", d_losses, leading(x), dtype);
    check_shape(what, "lse", lse, leading(x), dtype);
    DALI_ASSERT(!bias.is_stateless() || out.bias.is_stateless(), make_message(what, ": without bias there is no gradient of it to write"));
    const Projection p = as_projection(w);
    ProjectedCrossEntropyGradient r;
    r.x = destination(what, "dx", out.x, x.shape(), dtype);
    bool dw_by_columns = p.by_columns;
    if (out.w.is_stateless()) {
        r.w = p.by_columns ? Array({w.shape()[1], w.shape()[0]}, dtype).transpose() : Array(w.shape(), dtype);
    } else {
        check_shape(what, "dw", out.w, w.shape(), dtype);
        dw_by_columns = out.w.is_buffer() && !out.w.contiguous_memory() && out.w.transpose().contiguous_memory();
        r.w = dw_by_columns ? out.w : destination(what, "dw", out.w, w.shape(), dtype);
    }
    if (!bias.is_stateless()) r.bias = destination(what, "dbias", out.bias, {w.shape()[1]}, dtype);
    const Rows in = as_whole_rows(x);
    const Array g = dense(d_losses), t = dense(targets), l = dense(lse), b = bias.is_stateless() ? bias : dense(bias);
    const int64_t rows = in.rows, stride = in.stride, w_stride = p.stride;
    const int inputs = in.width, vocab = w.shape()[1], by_columns = p.by_columns, dw_columns = dw_by_columns;
    const Array space =
        workspace(what, [&](size_t* n) { return dali_hip_projected_cross_entropy_workspace(dtype, rows, inputs, vocab, 1, !b.is_stateless(), n); });
    if (g_dry_run) return r;
    const void *gp = read(g), *xp = read(in.array), *wp = read(p.array), *tp = read(t), *lp = read(l), *bp = read(b);
    void *dxp = write(r.x), *dwp = write(r.w), *dbp = write(r.bias), *sp = write(space);
    issue(
        what,
        [=]() {
            return dali_hip_projected_cross_entropy_backward(dtype, rows, inputs, vocab, gp, xp, stride, wp, w_stride, by_columns, bp, (const int32_t*)tp, lp, dxp, dwp,
                                                             dw_columns, dbp, sp);
        },
        [&](std::vector<Array>& reads, std::vector<Array>& writes) { reads = {g, in.array, p.array, t, l, b}, writes = {r.x, r.w, r.bias, space}; });
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
