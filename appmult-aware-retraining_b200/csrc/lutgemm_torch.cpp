// The head norms, attention and log probabilities as PyTorch operators with autograd, over the library's C interface.
//
// In C++ because these calls are short: a training pass of one small layer through a Python autograd function took the host 175 us for
// 45 us of kernels (the backward pass crosses into Python on another thread), and callers with many small layers would wait for
// the host.  The module holds no state; every call checks its arguments, runs on the current stream of its operands' device and
// raises what the library refuses.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "lutgemm.h"

namespace {

using at::Tensor;
using MaybeTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int status, const char *what) {
    TORCH_CHECK(status == LUTGEMM_OK, what, " failed with status ", status, ": ", lutgemm_status_string(status));
}

int dtype_of(const Tensor &x) {
    return x.scalar_type() == at::kFloat ? LUTGEMM_F32 : x.scalar_type() == at::kBFloat16 ? LUTGEMM_BF16 : LUTGEMM_F16;
}
bool has_kernels(const Tensor &x) {
    return x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf;
}

void check_heads(const Tensor &x, const char *name) {
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDAtensor");
    TORCH_CHECK(has_kernels(x), name, " must be of type torch.float32, torch.bfloat16 or torch.float16");
    TORCH_CHECK(x.dim() == 4, name, " must be [B, T, heads, D], got ", x.sizes());
}
void check_like(const Tensor &x, const char *name, const Tensor &like) {
    check_heads(x, name);
    TORCH_CHECK(x.scalar_type() == like.scalar_type() && x.device() == like.device(), name, " must be of type ", like.scalar_type(), " on ",
                like.device());
}
void check_side(const Tensor &x, const char *name, at::ScalarType type, at::IntArrayRef shape, const Tensor &like) {
    TORCH_CHECK(x.scalar_type() == type, name, " must be of type ", type);
    TORCH_CHECK(x.device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(x.sizes() == shape, name, " has shape ", x.sizes(), ", expected ", shape);
}

// x as the kernels read it: by the strides of its first three axes
Tensor rows(const Tensor &x) { return x.stride(3) == 1 || x.size(3) == 1 ? x : x.contiguous(); }
// the same where 16-bit operands are read by bulk copies: a copy of one that lies on other boundaries or repeats itself
Tensor vectors(const Tensor &x) {
    if (x.scalar_type() == at::kFloat) return rows(x);
    bool fits = (x.stride(3) == 1 || x.size(3) == 1) && !(reinterpret_cast<uintptr_t>(x.const_data_ptr()) & 15);
    for (int i = 0; i < 3; ++i) fits = fits && (x.size(i) == 1 || (x.stride(i) > 0 && x.stride(i) % 8 == 0));
    return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}
template <typename T = void>
T *data(const MaybeTensor &x) {
    return x.has_value() && x->defined() ? static_cast<T *>(x->data_ptr()) : nullptr;
}
MaybeTensor maybe(const Tensor &x) { return x.defined() ? MaybeTensor(x) : c10::nullopt; }
Tensor or_undefined(const MaybeTensor &x) { return x.has_value() ? *x : Tensor(); }
bool wants_grad(const MaybeTensor &x) { return x.has_value() && x->defined() && x->requires_grad(); }
Tensor scratch(size_t bytes, const Tensor &like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void *stream_of(const Tensor &x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }
// a tangent that forward-mode differentiation has given a tensor would be lost: the result's derivative would be taken for zero
void no_tangents(const char *what, std::initializer_list<const Tensor *> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *x : inputs)
        TORCH_CHECK(!x || !x->defined() || !x->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}
const Tensor *given(const MaybeTensor &x) { return x.has_value() ? &*x : nullptr; }
void no_second_derivative(const char *what, const variable_list &grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative (create_graph=True)");
    for (const Tensor &g : grads) no_tangents(what, {&g});
}
#define STRIDES(x) (long)(x).stride(0), (long)(x).stride(1), (long)(x).stride(2)

// ---- norm_rotate ---------------------------------------------------------------------------------------------------------
std::pair<Tensor, Tensor> norm_forward(const Tensor &q, const Tensor &k, const MaybeTensor &qw, const MaybeTensor &kw, const Tensor &cos,
                                       const Tensor &sin, const MaybeTensor &positions, bool interleaved, double eps) {
    Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), q.options());
    if (q.size(0) * q.size(1) > 0) {
        const c10::cuda::CUDAGuard guard(q.device());
        check(lutgemm_norm_rotate(q.data_ptr(), STRIDES(q), k.data_ptr(), STRIDES(k), data<float>(qw), data<float>(kw), cos.data_ptr<float>(),
                                  sin.data_ptr<float>(), (int)cos.size(0), data<int>(positions), qo.data_ptr(), ko.data_ptr(), dtype_of(q),
                                  (int)q.size(0), (int)q.size(1), (int)q.size(2), (int)k.size(2), (int)q.size(3), (int)(2 * cos.size(1)),
                                  interleaved, (float)eps, stream_of(q)),
              "norm_rotate");
    }
    return {qo, ko};
}

struct NormRotate : torch::autograd::Function<NormRotate> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const MaybeTensor &qw, const MaybeTensor &kw,
                                 const Tensor &cos, const Tensor &sin, const MaybeTensor &positions, bool interleaved, double eps) {
        ctx->save_for_backward({q, k, or_undefined(qw), or_undefined(kw), cos, sin, or_undefined(positions)});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["eps"] = eps;
        const auto out = norm_forward(q, k, qw, kw, cos, sin, positions, interleaved, eps);
        return {out.first, out.second};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        no_second_derivative("norm_rotate", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &cos = saved[4], &sin = saved[5];
        const MaybeTensor qw = maybe(saved[2]), kw = maybe(saved[3]), positions = maybe(saved[6]);
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dqw, dkw;
        if (wants_grad(qw)) dqw = at::empty(qw->sizes(), qw->options());
        if (wants_grad(kw)) dkw = at::empty(kw->sizes(), kw->options());
        if (q.size(0) * q.size(1) > 0) {
            const Tensor gq = rows(grads[0]), gk = rows(grads[1]);
            const c10::cuda::CUDAGuard guard(q.device());
            const size_t bytes = dqw.defined() || dkw.defined() ? lutgemm_norm_rotate_backward_scratch_bytes((int)q.size(3)) : 0;
            const Tensor work = scratch(bytes, q);
            check(lutgemm_norm_rotate_backward(gq.data_ptr(), STRIDES(gq), gk.data_ptr(), STRIDES(gk), q.data_ptr(), STRIDES(q), k.data_ptr(),
                                               STRIDES(k), data<float>(qw), data<float>(kw), cos.data_ptr<float>(), sin.data_ptr<float>(),
                                               (int)cos.size(0), data<int>(positions), dq.data_ptr(), dk.data_ptr(), data<float>(maybe(dqw)),
                                               data<float>(maybe(dkw)), dtype_of(q), (int)q.size(0), (int)q.size(1), (int)q.size(2),
                                               (int)k.size(2), (int)q.size(3), (int)(2 * cos.size(1)), ctx->saved_data["interleaved"].toBool(),
                                               (float)ctx->saved_data["eps"].toDouble(), data(maybe(work)), bytes, stream_of(q)),
                  "norm_rotate (backward)");
        } else {
            if (dqw.defined()) dqw.zero_();
            if (dkw.defined()) dkw.zero_();
        }
        return {dq, dk, dqw, dkw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::pair<Tensor, Tensor> norm_rotate(const Tensor &q, const Tensor &k, const MaybeTensor &q_weight, const MaybeTensor &k_weight,
                                      const MaybeTensor &cos_table, const MaybeTensor &sin_table, const MaybeTensor &places,
                                      const std::string &layout, double eps) {
    check_heads(q, "q");
    check_like(k, "k", q);
    no_tangents("norm_rotate", {&q, &k, given(q_weight), given(k_weight), given(cos_table), given(sin_table)});
    const int64_t B = q.size(0), T = q.size(1), D = q.size(3);
    TORCH_CHECK(k.size(0) == B && k.size(1) == T && k.size(3) == D, "k has shape ", k.sizes(), ", expected [", B, ", ", T, ", heads, ", D, "]");
    TORCH_CHECK(q.size(2) > 0 && k.size(2) > 0 && D > 0 && D % 2 == 0 && D <= 256, "heads must be at least one of an even size up to 256, got ",
                q.size(2), " and ", k.size(2), " of ", D);
    TORCH_CHECK(B <= 0x7fffffffLL && T <= 0x7fffffffLL && q.size(2) <= 0x7fffffffLL && k.size(2) <= 0x7fffffffLL, "q or k is too large");
    TORCH_CHECK_VALUE(layout == "half" || layout == "interleaved", "layout must be 'half' or 'interleaved', got ", layout);
    TORCH_CHECK(cos_table.has_value() == sin_table.has_value(), "cos and sin belong together");
    Tensor cos, sin;
    MaybeTensor positions;
    if (cos_table.has_value()) {
        cos = *cos_table;
        sin = *sin_table;
        TORCH_CHECK(cos.dim() == 2 && 2 * cos.size(1) <= D, "cos must be [positions, at most ", D / 2, "], got ", cos.sizes());
        check_side(cos, "cos", at::kFloat, cos.sizes(), q);
        check_side(sin, "sin", at::kFloat, cos.sizes(), q);
        TORCH_CHECK(!at::GradMode::is_enabled() || !(cos.requires_grad() || sin.requires_grad()), "cos and sin have no gradient");
        TORCH_CHECK(cos.size(0) <= 0x7fffffffLL, "cos and sin have too many positions");
        cos = cos.contiguous();
        sin = sin.contiguous();
        if (places.has_value()) {
            // (64-bit places beyond 32 bits are beyond any table)
            const Tensor at32 = places->scalar_type() == at::kLong ? places->clamp(-1, 0x7fffffff).to(at::kInt) : *places;
            check_side(at32, "positions", at::kInt, {B, T}, q);
            positions = at32.contiguous();
        } else {
            TORCH_CHECK(cos.size(0) >= T, "cos and sin have ", cos.size(0), " positions, the rows ", T);
        }
    } else {
        cos = sin = at::empty({T, 0}, q.options().dtype(at::kFloat));
    }
    MaybeTensor weights[2] = {q_weight, k_weight};
    for (int i = 0; i < 2; ++i) {
        if (!weights[i].has_value()) continue;
        check_side(*weights[i], i ? "k_weight" : "q_weight", has_kernels(*weights[i]) ? weights[i]->scalar_type() : at::kFloat, {D}, q);
        weights[i] = weights[i]->to(at::kFloat).contiguous();
    }
    const Tensor qr = rows(q), kr = rows(k);
    const bool interleaved = layout == "interleaved";
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || wants_grad(weights[0]) || wants_grad(weights[1]))) {
        const variable_list out = NormRotate::apply(qr, kr, weights[0], weights[1], cos, sin, positions, interleaved, eps);
        return {out[0], out[1]};
    }
    return norm_forward(qr, kr, weights[0], weights[1], cos, sin, positions, interleaved, eps);
}

// ---- attention ----------------------------------------------------------------------------------------------------------
struct Masks {
    double scale, cap;
    bool causal;
    MaybeTensor slopes, prefix, doc_q, doc_k;
};
#define MASKS(m)                                                                                                                          \
    (float)(m).scale, (float)(m).cap, data<float>((m).slopes), (m).causal, data<int>((m).prefix), data<int>((m).doc_q),                 \
        (m).doc_q ? (long)(m).doc_q->stride(0) : 0, data<int>((m).doc_k), (m).doc_k ? (long)(m).doc_k->stride(0) : 0

struct AttentionResult {
    Tensor out, rest, lse;  // rest (16-bit operands, for a backward pass): what the rounding of out leaves
};
AttentionResult attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Masks &m, bool training) {
    const int B = (int)q.size(0), Tq = (int)q.size(1), H = (int)q.size(2), D = (int)q.size(3), Tk = (int)k.size(1), G = (int)k.size(2);
    AttentionResult r;
    r.out = at::empty(q.sizes(), q.options());
    r.lse = at::empty({B, G, (int64_t)Tq * (H / G)}, q.options().dtype(at::kFloat));
    const int dtype = dtype_of(q);
    if (training && dtype != LUTGEMM_F32) r.rest = at::empty(q.sizes(), q.options());
    const c10::cuda::CUDAGuard guard(q.device());
    const size_t bytes = lutgemm_attention_scratch_bytes(dtype, B, Tq, Tk, H, G, D, m.doc_k.has_value());
    const Tensor work = scratch(bytes, q);
    check(lutgemm_attention(q.data_ptr(), STRIDES(q), k.data_ptr(), STRIDES(k), v.data_ptr(), STRIDES(v), r.out.data_ptr(), data(maybe(r.rest)),
                            r.lse.data_ptr<float>(), dtype, B, Tq, Tk, H, G, D, MASKS(m), data(maybe(work)), bytes, stream_of(q)),
          "attention");
    return r;
}

struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, double scale, double cap,
                          const MaybeTensor &slopes, bool causal, const MaybeTensor &prefix, const MaybeTensor &doc_q, const MaybeTensor &doc_k) {
        const AttentionResult r = attention_forward(q, k, v, Masks{scale, cap, causal, slopes, prefix, doc_q, doc_k}, true);
        ctx->save_for_backward({q, k, v, r.out, r.rest, r.lse, or_undefined(slopes), or_undefined(prefix), or_undefined(doc_q), or_undefined(doc_k)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["cap"] = cap;
        ctx->saved_data["causal"] = causal;
        return r.out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        no_second_derivative("attention", grads);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], go = vectors(grads[0]);
        const Masks m{ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(), ctx->saved_data["causal"].toBool(), maybe(s[6]),
                      maybe(s[7]), maybe(s[8]), maybe(s[9])};
        const int B = (int)q.size(0), Tq = (int)q.size(1), H = (int)q.size(2), D = (int)q.size(3), Tk = (int)k.size(1), G = (int)k.size(2);
        const int dtype = dtype_of(q);
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dv = at::empty(v.sizes(), q.options());
        const c10::cuda::CUDAGuard guard(q.device());
        const size_t bytes = lutgemm_attention_backward_scratch_bytes(dtype, B, Tq, Tk, H, G, D, m.doc_k.has_value());
        const Tensor work = scratch(bytes, q);
        check(lutgemm_attention_backward(go.data_ptr(), STRIDES(go), q.data_ptr(), STRIDES(q), k.data_ptr(), STRIDES(k), v.data_ptr(), STRIDES(v),
                                         s[3].data_ptr(), data(maybe(s[4])), s[5].data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                         dtype, B, Tq, Tk, H, G, D, MASKS(m), data(maybe(work)), bytes, stream_of(q)),
              "attention (backward)");
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// no queries or no keys: zeros, whose gradients are zeros
struct NothingToSee : torch::autograd::Function<NothingToSee> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v) {
        ctx->save_for_backward({q, k, v});
        return at::zeros(q.sizes(), q.options());
    }
    static variable_list backward(AutogradContext *ctx, variable_list) {
        variable_list grads;
        for (const Tensor &x : ctx->get_saved_variables()) grads.push_back(at::zeros(x.sizes(), x.options()));
        return grads;
    }
};

Tensor attention(const Tensor &q, const Tensor &k, const Tensor &v, c10::optional<double> given_scale, double cap, MaybeTensor slopes, bool causal,
                 MaybeTensor prefix, MaybeTensor documents, MaybeTensor query_documents) {
    check_heads(q, "q");
    check_like(k, "k", q);
    check_like(v, "v", q);
    no_tangents("attention", {&q, &k, &v, given(slopes)});
    const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), D = q.size(3), Tk = k.size(1), G = k.size(2);
    TORCH_CHECK(k.size(0) == B && k.size(3) == D && k.sizes() == v.sizes(), "k and v must both be [", B, ", Tk, heads, ", D, "], got ", k.sizes(),
                " and ", v.sizes());
    TORCH_CHECK(G > 0 && H > 0 && H % G == 0 && H / G <= 64, "q's ", H, " heads must be a multiple of the ", G,
                " heads of k and v, at most 64 to one");
    TORCH_CHECK(D > 0 && D % 8 == 0 && D <= 128, "the size of a head must be a multiple of 8 up to 128, got ", D);
    const double scale = given_scale.has_value() ? *given_scale : 1.0 / std::sqrt((double)D);
    TORCH_CHECK_VALUE(cap >= 0.0 && std::isfinite(cap) && std::isfinite(scale), "cap must not be negative, cap and scale must be finite, got ",
                      cap, " and ", scale);
    if (slopes.has_value()) {
        check_side(*slopes, "slopes", at::kFloat, {H}, q);
        TORCH_CHECK(!at::GradMode::is_enabled() || !slopes->requires_grad(), "slopes have no gradient");
        slopes = slopes->contiguous();
    }
    if (prefix.has_value()) {
        TORCH_CHECK(causal, "prefix belongs to causal attention");
        check_side(*prefix, "prefix", at::kInt, {B}, q);
        prefix = prefix->contiguous();
    }
    TORCH_CHECK(!query_documents.has_value() || documents.has_value(), "query_documents belong to documents");
    if (documents.has_value()) {
        const auto along = [](const Tensor &x) { return x.stride(1) == 1 || x.size(1) <= 1 ? x : x.contiguous(); };
        check_side(*documents, "documents", at::kInt, {B, Tk}, q);
        documents = along(*documents);
        if (query_documents.has_value()) {
            check_side(*query_documents, "query_documents", at::kInt, {B, Tq}, q);
            query_documents = along(*query_documents);
        } else {
            TORCH_CHECK(Tq <= Tk, "more queries than keys need query_documents");
            query_documents = documents->narrow(1, Tk - Tq, Tq);
        }
    }
    TORCH_CHECK(B <= 65535 && G <= 65535 && H <= 0x7fffffffLL && Tq * (H / G) <= 0x7fffff00LL && Tk <= 0x7fffff00LL, "q or k has too many rows or heads");
    if (B * Tq == 0 || Tk == 0) return NothingToSee::apply(q, k, v);
    const Tensor qv = vectors(q), kv = vectors(k), vv = vectors(v);
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return Attention::apply(qv, kv, vv, scale, cap, slopes, causal, prefix, query_documents, documents);
    return attention_forward(qv, kv, vv, Masks{scale, cap, causal, slopes, prefix, query_documents, documents}, false).out;
}

// ---- token_logprobs -------------------------------------------------------------------------------------------------------
variable_list logprobs_forward(const Tensor &logits, const Tensor &targets, int64_t top, int64_t ignore) {
    const int64_t N = logits.size(0), C = logits.size(1);
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor logp = at::empty({N}, f32), entropy = at::empty({N}, f32), top_logp = at::empty({N, top}, f32),
           top_index = at::empty({N, top}, logits.options().dtype(at::kLong)), stats = at::empty({N, 3}, f32);
    if (N > 0) {
        const c10::cuda::CUDAGuard guard(logits.device());
        const size_t bytes = lutgemm_token_logprobs_scratch_bytes((long)N, (int)C, (int)top);
        const Tensor work = scratch(bytes, logits);
        check(lutgemm_token_logprobs(logits.data_ptr(), dtype_of(logits), (long)logits.stride(0), (long)N, (int)C,
                                     reinterpret_cast<const long long *>(targets.data_ptr<int64_t>()), (long long)ignore, (int)top,
                                     logp.data_ptr<float>(), entropy.data_ptr<float>(), stats.data_ptr<float>(), top_logp.data_ptr<float>(),
                                     reinterpret_cast<long long *>(top_index.data_ptr<int64_t>()), data(maybe(work)), bytes, stream_of(logits)),
              "token_logprobs");
    }
    return {logp, entropy, top_logp, top_index, stats};
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &targets, int64_t top, int64_t ignore) {
        variable_list out = logprobs_forward(logits, targets, top, ignore);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({logits, targets, out[4]});
        ctx->saved_data["ignore"] = ignore;
        out.pop_back();
        ctx->mark_non_differentiable({out[2], out[3]});
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        no_second_derivative("token_logprobs", grads);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &logits = s[0];
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        Tensor grad = at::empty(logits.sizes(), logits.options());
        if (logits.size(0) > 0) {
            const Tensor gl = grads[0].defined() ? grads[0].contiguous() : grads[0], ge = grads[1].defined() ? grads[1].contiguous() : grads[1];
            const c10::cuda::CUDAGuard guard(logits.device());
            check(lutgemm_token_logprobs_backward(logits.data_ptr(), dtype_of(logits), (long)logits.stride(0), (long)logits.size(0),
                                                  (int)logits.size(1), reinterpret_cast<const long long *>(s[1].data_ptr<int64_t>()),
                                                  (long long)ctx->saved_data["ignore"].toInt(), s[2].data_ptr<float>(), data<float>(maybe(gl)),
                                                  data<float>(maybe(ge)), grad.data_ptr(), stream_of(logits)),
                  "token_logprobs (backward)");
        }
        return {grad, Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor &logits, const Tensor &targets, int64_t top, int64_t ignore) {
    TORCH_CHECK(logits.is_cuda(), "logits must be a CUDAtensor");
    TORCH_CHECK(has_kernels(logits), "logits must be of type torch.float32, torch.bfloat16 or torch.float16");
    no_tangents("token_logprobs", {&logits});
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0 && logits.size(-1) <= 0x7fffffffLL, "logits must be [..., classes], got ", logits.sizes());
    TORCH_CHECK(targets.scalar_type() == at::kLong && targets.device() == logits.device(), "targets must be of type torch.int64 on ",
                logits.device());
    const int64_t C = logits.size(-1);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK(targets.sizes() == lead, "targets have shape ", targets.sizes(), ", expected ", lead);
    TORCH_CHECK_VALUE(top >= 0 && top <= std::min<int64_t>(32, C), "top must lie between 0 and ", std::min<int64_t>(32, C), ", got ", top);
    const bool matrix = logits.dim() == 2;
    Tensor x = matrix ? logits : logits.reshape({-1, C});
    if (C > 1 && x.stride(1) != 1) x = x.contiguous();
    const Tensor t = (matrix ? targets : targets.reshape({-1})).contiguous();
    const variable_list out = at::GradMode::is_enabled() && x.requires_grad() ? TokenLogprobs::apply(x, t, top, ignore)
                                                                             : logprobs_forward(x, t, top, ignore);
    if (matrix) return {out[0], out[1], out[2], out[3]};
    auto answers = lead.vec();
    answers.push_back(top);
    return {out[0].view(lead), out[1].view(lead), out[2].view(answers), out[3].view(answers)};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    const auto free = py::call_guard<py::gil_scoped_release>();
    m.def("norm_rotate", &norm_rotate, free);
    m.def("attention", &attention, free);
    m.def("token_logprobs", &token_logprobs, free);
}
