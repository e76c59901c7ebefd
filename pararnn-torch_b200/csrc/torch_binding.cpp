// PyTorch binding of the token-model operators: allocation, the current stream and the autograd nodes
// in C++ over the C ABI.  These operators are short (tens of microseconds), and a backward node in
// Python costs about as much again on the host: a group norm forward + backward took 135 us of host
// time through ctypes and Python nodes against 85 us on the GPU.  Argument checks that need names and
// shapes are in attn_ops.py and token_ops.py; this file trusts them.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/pararnn_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int code(const Tensor& t) { return t.scalar_type() == at::kFloat ? PRB_F32 : PRB_BF16; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
prb_stream_t stream(const Tensor& t) {
    return reinterpret_cast<prb_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}
void check(int rc, const char* what) {
    if (rc == PRB_OK) return;
    const char* why = prb_error_string(rc);
    if (rc == PRB_ERR_BAD_ARG || rc == PRB_ERR_UNSUPPORTED || rc == PRB_ERR_TOO_LARGE)
        TORCH_CHECK_VALUE(false, what, ": ", why, " (code ", rc, ")");
    TORCH_CHECK(false, what, ": ", why, " (code ", rc, ")");
}
void once(const char* name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the gradient of ", name,
                " cannot be differentiated again (create_graph=True)");
}
// the C ABI counts rows, heads and slots in 32 bits
void narrow(std::initializer_list<int64_t> sizes, const char* what) {
    for (const int64_t n : sizes) TORCH_CHECK_VALUE(n < (1ll << 31), what, " must fit in 32 bits, got ", n);
}
Tensor scratch(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
// A kernel has written `t` through its pointer: autograd is told, so that a node which saved `t` refuses its
// backward pass instead of reading the new values.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor plain(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor aligned(const Tensor& t) {
    Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

// ------------------------------------------------------------------------------- linear attention

// `t` where the kernels can address it (unit channel stride, no broadcast axes, for bf16 16-byte aligned
// rows), else a contiguous copy
Tensor heads(const Tensor& t, prb_heads& h) {
    Tensor c = t;
    bool copy = t.stride(3) != 1 && t.size(3) > 1;
    for (int i = 0; i < 3; ++i)
        copy |= t.size(i) > 1 && (t.stride(i) == 0 || (t.scalar_type() == at::kBFloat16 && t.stride(i) % 8 != 0));
    if (copy && !t.is_contiguous()) c = t.contiguous();
    if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16) c = c.clone(at::MemoryFormat::Contiguous);
    // an axis of length 1 may carry any stride
    auto st = [&](int i) { return (long long)(c.size(i) > 1 ? c.stride(i) : c.size(3)); };
    h = prb_heads{c.data_ptr(), st(0), st(1), st(2)};
    return c;
}

// A bounded wait of an earlier sweep on the current device ran out: told by whatever call of the family comes next,
// so that a model without any other check of the device hears of it.
void reported(const Tensor& t) {
    const int rc = prb_linear_attention_poll(1);
    TORCH_CHECK(rc == PRB_OK, "pararnn_b200: a bounded device-side wait ran out in an earlier linear attention call on ",
                t.device(), " (status ", rc, "); the results of that call are not valid");
}

struct AttnCall {
    int rows, time, n_seq, longest, hq, hkv, dk, dv, dtype;
    bool packed;
    size_t bytes(bool backward) const {
        return prb_linear_attention_workspace_bytes(rows, time, n_seq, longest, hq, hkv, dk, dv, dtype, packed, backward);
    }
};
AttnCall attn_call(const Tensor& q, const Tensor& k, const Tensor& v, bool packed, int64_t n_seq, int64_t longest) {
    narrow({q.size(0), q.size(1), q.size(2), k.size(2), n_seq}, "batch, time and heads");
    return AttnCall{(int)q.size(0), (int)q.size(1), (int)n_seq,     (int)longest, (int)q.size(2),
                    (int)k.size(2), (int)q.size(3), (int)v.size(3), code(q),      packed};
}

// cu: int32 offsets on the device.  sparse: they may leave tokens out, whose outputs are zeros
std::tuple<Tensor, Tensor> attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay,
                                         const OptTensor& state_, const OptTensor& cu_, int64_t n_seq,
                                         int64_t longest, double scale, bool want_state, bool sparse) {
    const AttnCall c = attn_call(q, k, v, cu_.has_value(), n_seq, longest);
    const c10::cuda::CUDAGuard guard(q.device());
    reported(q);
    const Tensor state = plain(get(state_)), cu = get(cu_);
    prb_heads hq, hk, hv;
    const Tensor qc = heads(q, hq), kc = heads(k, hk), vc = heads(v, hv);
    Tensor out = at::empty({c.rows, c.time, c.hq, c.dv}, q.options());
    if (sparse) out.zero_();
    Tensor last = want_state ? at::empty({c.n_seq, c.hkv, c.dk, c.dv}, q.options().dtype(at::kFloat)) : Tensor();
    const size_t n = c.bytes(false);
    const Tensor ws = scratch(n, q);
    check(prb_linear_attention(&hq, &hk, &hv, (const float*)ptr(decay), (const float*)ptr(state), (const int*)ptr(cu),
                               ptr(out), (float*)ptr(last), c.rows, c.time, c.n_seq, c.longest, c.hq, c.hkv, c.dk, c.dv,
                               c.dtype, (float)scale, ptr(ws), n, stream(q)),
          "linear_attention_fused");
    return {out, last};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attention_bwd(const Tensor& q, const Tensor& k, const Tensor& v,
                                                         const Tensor& decay, const Tensor& grad_,
                                                         const OptTensor& state_, const OptTensor& grad_state_,
                                                         const OptTensor& cu_, int64_t n_seq, int64_t longest,
                                                         double scale, bool want_state, bool sparse) {
    const AttnCall c = attn_call(q, k, v, cu_.has_value(), n_seq, longest);
    const c10::cuda::CUDAGuard guard(q.device());
    reported(q);
    const Tensor state = plain(get(state_)), gs = plain(get(grad_state_)), cu = get(cu_);
    prb_heads hq, hk, hv, hg;
    const Tensor qc = heads(q, hq), kc = heads(k, hk), vc = heads(v, hv), gc = heads(grad_.to(q.scalar_type()), hg);
    Tensor g_q = at::empty({c.rows, c.time, c.hq, c.dk}, q.options());
    Tensor g_k = at::empty({c.rows, c.time, c.hkv, c.dk}, q.options());
    Tensor g_v = at::empty({c.rows, c.time, c.hkv, c.dv}, q.options());
    if (sparse) g_q.zero_(), g_k.zero_(), g_v.zero_();
    Tensor g_s = want_state ? at::empty({c.n_seq, c.hkv, c.dk, c.dv}, q.options().dtype(at::kFloat)) : Tensor();
    const size_t n = c.bytes(true);
    const Tensor ws = scratch(n, q);
    check(prb_bwd_linear_attention(&hq, &hk, &hv, &hg, (const float*)ptr(decay), (const float*)ptr(state),
                                   (const float*)ptr(gs), (const int*)ptr(cu), ptr(g_q), ptr(g_k), ptr(g_v),
                                   (float*)ptr(g_s), c.rows, c.time, c.n_seq, c.longest, c.hq, c.hkv, c.dk, c.dv,
                                   c.dtype, (float)scale, ptr(ws), n, stream(q)),
          "linear_attention_reverse_vjp");
    return {g_q, g_k, g_v, g_s};
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& decay, const OptTensor& state, const OptTensor& cu, int64_t n_seq,
                                 int64_t longest, double scale, bool want_state, bool sparse) {
        auto [out, last] = attention_fwd(q, k, v, decay, state, cu, n_seq, longest, scale, want_state, sparse);
        ctx->save_for_backward({q, k, v, decay, get(state), get(cu)});
        ctx->saved_data["n_seq"] = n_seq;
        ctx->saved_data["longest"] = longest;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["sparse"] = sparse;
        ctx->set_materialize_grads(false);
        if (!last.defined()) return {out};
        return {out, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("linear_attention");
        const variable_list s = ctx->get_saved_variables();
        variable_list r(11);
        const Tensor gs = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !gs.defined()) return r;
        const Tensor& q = s[0];
        const Tensor g = grads[0].defined() ? grads[0] : at::zeros({q.size(0), q.size(1), q.size(2), s[2].size(3)}, q.options());
        auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        const bool want = s[4].defined() && ctx->needs_input_grad(4);
        auto [g_q, g_k, g_v, g_s] =
            attention_bwd(q, s[1], s[2], s[3], g, opt(s[4]), opt(gs), opt(s[5]), ctx->saved_data["n_seq"].toInt(),
                          ctx->saved_data["longest"].toInt(), ctx->saved_data["scale"].toDouble(), want,
                          ctx->saved_data["sparse"].toBool());
        if (ctx->needs_input_grad(0)) r[0] = g_q;
        if (ctx->needs_input_grad(1)) r[1] = g_k;
        if (ctx->needs_input_grad(2)) r[2] = g_v;
        if (want) r[4] = g_s;
        return r;
    }
};
std::tuple<Tensor, Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay,
                                     const OptTensor& state, const OptTensor& cu, int64_t n_seq, int64_t longest,
                                     double scale, bool want_state, bool sparse) {
    variable_list r =
        AttentionNode::apply(q, k, v, decay, state, cu, n_seq, longest, scale, want_state, sparse);
    return {r[0], r.size() > 1 ? r[1] : Tensor()};
}

// Memory that a call writes must hold nothing else that it reads or writes: other CTAs (heads, slices of the value
// channels, the one that applies a repeated slot's rows) may still be at it.
void apart(const Tensor& w, const char* w_name, const Tensor& t, const char* name) {
    // a tensor that is not contiguous is copied before the launch
    if (!t.defined() || !t.is_contiguous() || t.numel() == 0 || w.numel() == 0) return;
    const uintptr_t w0 = reinterpret_cast<uintptr_t>(w.data_ptr()), t0 = reinterpret_cast<uintptr_t>(t.data_ptr());
    TORCH_CHECK_VALUE(w0 + w.nbytes() <= t0 || t0 + t.nbytes() <= w0, w_name, " must not share memory with ", name);
}

void attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& state,
                    const OptTensor& table_, double scale, const Tensor& out) {
    narrow({q.size(0), q.size(1), k.size(1), state.size(0)}, "rows, heads and slots");
    apart(out, "out", q, "q");
    apart(out, "out", k, "k");
    // a value is read by the CTA that writes the output in its place, so out may be v where the heads are the same
    if (out.data_ptr() != v.data_ptr() || q.size(1) != k.size(1)) apart(out, "out", v, "v");
    apart(out, "out", decay, "log_decay");
    apart(out, "out", state, "state");
    apart(out, "out", get(table_), "block_table");
    apart(state, "state", q, "q");
    apart(state, "state", k, "k");
    apart(state, "state", v, "v");
    apart(state, "state", decay, "log_decay");
    apart(state, "state", get(table_), "block_table");
    const c10::cuda::CUDAGuard guard(q.device());
    reported(q);
    const Tensor qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous(), table = plain(get(table_));
    check(prb_linear_attention_step(ptr(qc), ptr(kc), ptr(vc), (const float*)ptr(decay), (float*)ptr(state), ptr(table),
                                    table.defined() && table.scalar_type() == at::kLong, ptr(out), (int)q.size(0),
                                    (int)state.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), (int)v.size(2),
                                    code(q), (float)scale, stream(q)),
          "linear_attention_step");
    written(state);
    written(out);
}

// ------------------------------------------------------------------------------------- group norm

void norm_sizes(const Tensor& x, int64_t& n, int64_t& c, int64_t& p) {
    n = x.size(0), c = x.size(-1), p = x.numel() / (n * c);
    TORCH_CHECK_VALUE(c < (1ll << 31) && p < (1ll << 31), "channels and positions must fit in 32 bits");
}
int weight_code(const Tensor& w, const Tensor& b) { return w.defined() ? code(w) : b.defined() ? code(b) : PRB_F32; }

std::tuple<Tensor, Tensor> norm_fwd(const Tensor& x, int64_t groups, const OptTensor& w_, const OptTensor& b_,
                                    double eps, int64_t act, bool want_stats) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xc = aligned(x), w = plain(get(w_)), b = plain(get(b_));
    int64_t n, c, p;
    norm_sizes(x, n, c, p);
    Tensor y = at::empty_like(xc);
    Tensor stats = want_stats ? at::empty({n, groups, 2}, x.options().dtype(at::kFloat)) : Tensor();
    const size_t need = prb_group_norm_workspace_bytes(n, (int)p, (int)c, (int)groups, code(x), 0);
    const Tensor ws = scratch(need, x);
    check(prb_group_norm(ptr(xc), ptr(w), ptr(b), ptr(y), (float*)ptr(stats), n, (int)p, (int)c, (int)groups, (float)eps,
                         (int)act, code(x), weight_code(w, b), ptr(ws), need, stream(x)),
          "group_norm_fused");
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> norm_bwd(const Tensor& x, const Tensor& gy_, const Tensor& stats_, int64_t groups,
                                            const OptTensor& w_, const OptTensor& b_, int64_t act, bool want_params) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xc = aligned(x), gy = aligned(gy_.to(x.scalar_type())), w = plain(get(w_)), b = plain(get(b_)),
                 stats = stats_.contiguous();
    int64_t n, c, p;
    norm_sizes(x, n, c, p);
    Tensor gx = at::empty_like(xc);
    Tensor gw = w.defined() && want_params ? at::empty_like(w) : Tensor();
    Tensor gb = b.defined() && want_params ? at::empty_like(b) : Tensor();
    const size_t need = prb_group_norm_workspace_bytes(n, (int)p, (int)c, (int)groups, code(x), 1);
    const Tensor ws = scratch(need, x);
    check(prb_bwd_group_norm(ptr(xc), ptr(gy), ptr(w), ptr(b), (const float*)ptr(stats), ptr(gx), ptr(gw), ptr(gb), n,
                             (int)p, (int)c, (int)groups, (int)act, code(x), weight_code(w, b), ptr(ws), need,
                             stream(x)),
          "group_norm_vjp");
    return {gx, gw, gb};
}

struct NormNode : torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b,
                          int64_t groups, double eps, int64_t act) {
        auto [y, stats] = norm_fwd(x, groups, w, b, eps, act, true);
        ctx->save_for_backward({x, get(w), get(b), stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("group_norm");
        const variable_list s = ctx->get_saved_variables();
        auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        // edges count the tensors that were given: without a weight the bias is edge 1
        const bool has_w = s[1].defined(), nw = has_w && ctx->needs_input_grad(1),
                   nb = s[2].defined() && ctx->needs_input_grad(has_w ? 2 : 1);
        auto [gx, gw, gb] = norm_bwd(s[0], grads[0], s[3], ctx->saved_data["groups"].toInt(), opt(s[1]), opt(s[2]),
                                     ctx->saved_data["act"].toInt(), nw || nb);
        variable_list r(6);
        if (ctx->needs_input_grad(0)) r[0] = gx;
        if (nw) r[1] = gw;
        if (nb) r[2] = gb;
        return r;
    }
};
Tensor norm(const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t groups, double eps, int64_t act) {
    return NormNode::apply(x, w, b, groups, eps, act);
}

// -------------------------------------------------------------------------------------- embedding

Tensor embed_fwd(const Tensor& ids, const Tensor& table, double scale) {
    const c10::cuda::CUDAGuard guard(table.device());
    TORCH_CHECK_VALUE(table.size(0) < (1ll << 31) && table.size(1) < (1ll << 31), "weight's sizes must fit in 32 bits");
    const Tensor idc = ids.contiguous(), w = table.contiguous();
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(w.size(1));
    Tensor out = at::empty(shape, w.options());
    if (ids.numel() == 0) return out;
    check(prb_embedding(ptr(idc), ids.scalar_type() == at::kLong, ptr(w), ptr(out), ids.numel(), (int)w.size(0),
                        (int)w.size(1), code(w), (float)scale, stream(w)),
          "embedding_fused");
    return out;
}
Tensor embed_bwd(const Tensor& ids, const Tensor& grad, int64_t vocab, double scale) {
    const c10::cuda::CUDAGuard guard(grad.device());
    const Tensor idc = ids.contiguous(), g = grad.contiguous();
    const int64_t c = g.size(-1);
    TORCH_CHECK_VALUE(vocab < (1ll << 31) && c < (1ll << 31), "vocab and channels must fit in 32 bits");
    if (ids.numel() == 0) return at::zeros({vocab, c}, g.options());
    Tensor out = at::empty({vocab, c}, g.options());
    const size_t need = prb_bwd_embedding_workspace_bytes(ids.numel(), (int)vocab, (int)c);
    const Tensor ws = scratch(need, g);
    check(prb_bwd_embedding(ptr(idc), ids.scalar_type() == at::kLong, ptr(g), ptr(out), ids.numel(), (int)vocab, (int)c,
                            code(g), (float)scale, ptr(ws), need, stream(g)),
          "embedding_vjp");
    return out;
}
struct EmbedNode : torch::autograd::Function<EmbedNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale) {
        ctx->save_for_backward({ids});
        ctx->saved_data["vocab"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["type"] = (int64_t)table.scalar_type();
        return embed_fwd(ids, table, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("embedding");
        const Tensor g = grads[0].to((at::ScalarType)ctx->saved_data["type"].toInt());
        return {Tensor(), embed_bwd(ctx->get_saved_variables()[0], g, ctx->saved_data["vocab"].toInt(),
                                    ctx->saved_data["scale"].toDouble()),
                Tensor()};
    }
};
Tensor embed(const Tensor& ids, const Tensor& table, double scale) { return EmbedNode::apply(ids, table, scale); }

}  // namespace

TORCH_LIBRARY(pararnn_b200_native, m) {
    m.def("attention_fwd(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor? state, Tensor? cu, int n_seq, int longest, "
          "float scale, bool want_state, bool sparse) -> (Tensor, Tensor)", attention_fwd);
    m.def("attention_bwd(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor grad, Tensor? state, Tensor? grad_state, "
          "Tensor? cu, int n_seq, int longest, float scale, bool want_state, bool sparse) -> "
          "(Tensor, Tensor, Tensor, Tensor)", attention_bwd);
    m.def("attention(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor? state, Tensor? cu, int n_seq, int longest, "
          "float scale, bool want_state, bool sparse) -> (Tensor, Tensor)", attention);
    m.def("attention_step(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor(a!) state, Tensor? table, float scale, "
          "Tensor(b!) out) -> ()", attention_step);
    m.def("norm_fwd(Tensor x, int groups, Tensor? w, Tensor? b, float eps, int act, bool want_stats) -> (Tensor, Tensor)",
          norm_fwd);
    m.def("norm_bwd(Tensor x, Tensor gy, Tensor stats, int groups, Tensor? w, Tensor? b, int act, bool want_params) -> "
          "(Tensor, Tensor, Tensor)", norm_bwd);
    m.def("norm(Tensor x, Tensor? w, Tensor? b, int groups, float eps, int act) -> Tensor", norm);
    m.def("embed_fwd(Tensor ids, Tensor table, float scale) -> Tensor", embed_fwd);
    m.def("embed_bwd(Tensor ids, Tensor grad, int vocab, float scale) -> Tensor", embed_bwd);
    m.def("embed(Tensor ids, Tensor table, float scale) -> Tensor", embed);
}
