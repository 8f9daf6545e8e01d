// d1ops: the Python calls of libd1ops.so on torch tensors (module _d1ops).
//
// A call on a small minibatch is a few microseconds of GPU work, less than its argument checks and
// three allocations take in Python (11 us a call there, 6 here, 3 of them the launch itself). Checks, outputs
// and scratch memory are therefore made here; the kernels and their C ABI know nothing of torch. Argument errors
// are ValueError before any launch. The caller has made the tensors' device the current one and gives its stream.
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/d1ops.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

[[noreturn]] void refuse(const std::string &why) { throw py::value_error(why); }

void check(int code, const char *what) {
    if (code) throw std::runtime_error(std::string(what) + " failed with code " + std::to_string(code));
}

std::string describe(const Tensor &t) {
    return std::string(c10::toString(t.scalar_type())) + " of " + c10::str(t.sizes()) + " on " + t.device().str();
}

int type_of(at::ScalarType t) {
    return t == at::kFloat ? D1_FP32 : t == at::kBFloat16 ? D1_BF16 : t == at::kHalf ? D1_FP16 : -1;
}

// Forward-mode tangents are lost in a kernel call, so they are refused here. Inside an autograd function's forward torch
// hides them and refuses by itself.
void no_tangent(const Tensor &t, const char *name) {
    if (!t._fw_grad(0).defined()) return;
    PyErr_SetString(PyExc_NotImplementedError, (std::string(name) + " has a forward-mode tangent: the operators have none").c_str());
    throw py::error_already_set();
}

// torch.jit.trace would record that outputs are made, but not what fills them. Only the forward of an autograd function
// may run in one, which records the function as a whole.
void no_trace(const char *name) {
    if (torch::jit::tracer::isTracing())
        throw std::runtime_error(std::string(name) + " cannot be part of a trace (token_logprobs and layer_norm can)");
}

int rows_type(const Tensor &x, const char *name) {
    no_tangent(x, name);
    if (!x.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor (there is no CPU fallback)");
    const int code = type_of(x.scalar_type());
    if (code < 0) refuse(std::string(name) + " must be fp32, bf16 or fp16, not " + c10::toString(x.scalar_type()));
    if (x.dim() == 0 || x.size(-1) == 0) refuse(std::string(name) + " must have a last dimension of at least one element");
    return code;
}

// x as [rows, width] with adjacent elements in a row, a view where its strides allow it
Tensor as_rows(const Tensor &x) {
    const int64_t width = x.size(-1);
    Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / width, width});
    return width > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

// t as a contiguous tensor of that type and shape on x's device
Tensor like(const Tensor &t, at::IntArrayRef shape, at::ScalarType type, const Tensor &x, const char *name) {
    no_tangent(t, name);
    if (t.scalar_type() != type || t.sizes() != shape || t.device() != x.device())
        refuse(std::string(name) + " must be " + c10::toString(type) + " of " + c10::str(shape) + " on " + x.device().str() +
               ", not " + describe(t));
    return t.contiguous();
}

void *ptr(const Tensor &t) { return t.data_ptr(); }
void *ptr(const Maybe &t) { return t ? t->data_ptr() : nullptr; }
Tensor scratch(int64_t bytes, const Tensor &x) { return at::empty({bytes}, x.options().dtype(at::kByte)); }
// The kernels write through raw pointers, which torch does not see: a caller's tensor that a call has changed gets a new
// version, as from any operation in place, for autograd's check of saved tensors and for what is kept by version
// (Policy.packed). Tensors made under inference mode have none.
void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- tokens

struct TokenArgs {
    int code;
    Tensor rows, tokens;
    Maybe mask;
    int64_t mask_stride = 0;
    int64_t n, vocab;
};

TokenArgs token_args(const Tensor &logits, const Tensor &tokens, const Maybe &mask) {
    TokenArgs a;
    a.code = rows_type(logits, "logits");
    a.vocab = logits.size(-1);
    if (a.vocab > D1_TOKENS_MAX_VOCAB) refuse("logits: at most " + std::to_string(D1_TOKENS_MAX_VOCAB) + " entries a row");
    a.tokens = like(tokens, logits.sizes().slice(0, logits.dim() - 1), at::kLong, logits, "tokens");
    a.rows = as_rows(logits);
    a.n = a.rows.size(0);
    if (mask) {
        if ((mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte) || mask->device() != logits.device())
            refuse("mask must be bool or uint8 on the device of the logits");
        if (mask->sizes() == logits.sizes()) {
            a.mask = as_rows(*mask);
            a.mask_stride = a.mask->stride(0);
        } else if (mask->dim() == 1 && mask->size(0) == a.vocab) {
            a.mask = mask->contiguous();
        } else {
            refuse("mask must have the shape of the logits or of one row, not " + c10::str(mask->sizes()));
        }
    }
    return a;
}

py::tuple tokens_fwd(const Tensor &logits, const Tensor &tokens, const Maybe &mask, int64_t top, int64_t stream) {
    const TokenArgs a = token_args(logits, tokens, mask);
    if (top < 0 || top > D1_TOKENS_MAX_TOP || top > a.vocab)
        refuse("top must be 0 to " + std::to_string(D1_TOKENS_MAX_TOP) + " and at most the number of entries, not " + std::to_string(top));
    const auto fp32 = logits.options().dtype(at::kFloat);
    std::vector<int64_t> shape(a.tokens.sizes().begin(), a.tokens.sizes().end());
    const Tensor logp = at::empty(shape, fp32), entropy = at::empty(shape, fp32);
    shape.push_back(2);
    const Tensor stats = at::empty(shape, fp32);
    Maybe ids, top_logp, work;
    if (top) {
        shape.back() = top;
        ids = at::empty(shape, logits.options().dtype(at::kLong));
        top_logp = at::empty(shape, fp32);
    }
    const int64_t need = d1_tokens_work_bytes(a.n, (int)a.vocab, (int)top);
    if (need > 0) work = scratch(need, logits);
    check(d1_tokens_fwd(ptr(a.rows), a.code, a.n, (int)a.vocab, a.rows.stride(0), (const int64_t *)ptr(a.tokens),
                        (const uint8_t *)ptr(a.mask), a.mask_stride, (int)top, (float *)ptr(logp), (float *)ptr(entropy),
                        (float *)ptr(stats), (int64_t *)ptr(ids), (float *)ptr(top_logp), ptr(work), need, (void *)stream),
          "d1_tokens_fwd");
    return py::make_tuple(logp, entropy, ids, top_logp, stats);
}

Tensor tokens_bwd(const Tensor &logits, const Tensor &tokens, const Tensor &stats_, const Tensor &entropy_, const Maybe &dlogp_,
                  const Maybe &dentropy_, const Maybe &mask, int64_t stream) {
    no_trace("token_logprobs_bwd");
    const TokenArgs a = token_args(logits, tokens, mask);
    const auto shape = a.tokens.sizes();
    std::vector<int64_t> two(shape.begin(), shape.end());
    two.push_back(2);
    const Tensor stats = like(stats_, two, at::kFloat, logits, "result.stats");
    const Tensor entropy = like(entropy_, shape, at::kFloat, logits, "result.entropy");
    Maybe dlogp, dentropy;
    if (dlogp_) dlogp = like(*dlogp_, shape, at::kFloat, logits, "dlogp");
    if (dentropy_) dentropy = like(*dentropy_, shape, at::kFloat, logits, "dentropy");
    const Tensor out = at::empty(logits.sizes(), logits.options());
    check(d1_tokens_bwd(ptr(a.rows), a.code, a.n, (int)a.vocab, a.rows.stride(0), (const int64_t *)ptr(a.tokens),
                        (const uint8_t *)ptr(a.mask), a.mask_stride, (const float *)ptr(stats), (const float *)ptr(entropy),
                        (const float *)ptr(dlogp), (const float *)ptr(dentropy), ptr(out), (void *)stream),
          "d1_tokens_bwd");
    return out;
}

// ---- layer norm

struct NormArgs {
    int code, wcode;
    Tensor rows;
    Maybe weight, bias;
    int64_t n, width;
};

NormArgs norm_args(const Tensor &x, const Maybe &weight, const Maybe &bias) {
    NormArgs a;
    a.code = a.wcode = rows_type(x, "x");
    a.width = x.size(-1);
    if (a.width > D1_NORM_MAX_WIDTH) refuse("x: rows of at most " + std::to_string(D1_NORM_MAX_WIDTH) + " elements");
    if (weight || bias) {
        const at::ScalarType type = (weight ? *weight : *bias).scalar_type();
        if (type != x.scalar_type() && type != at::kFloat)
            refuse(std::string("weight and bias must be fp32 or of x's type, not ") + c10::toString(type));
        a.wcode = type_of(type);
        if (weight) a.weight = like(*weight, {a.width}, type, x, "weight");
        if (bias) a.bias = like(*bias, {a.width}, type, x, "bias");
    }
    a.rows = as_rows(x);
    a.n = a.rows.size(0);
    return a;
}

py::tuple norm_fwd(const Tensor &x, const Maybe &weight, const Maybe &bias, double eps, int64_t stream) {
    const NormArgs a = norm_args(x, weight, bias);
    const Tensor y = at::empty(x.sizes(), x.options());
    const auto fp32 = x.options().dtype(at::kFloat);
    const auto shape = x.sizes().slice(0, x.dim() - 1);
    const Tensor mean = at::empty(shape, fp32), rstd = at::empty(shape, fp32);
    check(d1_norm_fwd(ptr(a.rows), a.code, a.n, (int)a.width, a.rows.stride(0), ptr(a.weight), ptr(a.bias), a.wcode, (float)eps,
                      ptr(y), (float *)ptr(mean), (float *)ptr(rstd), (void *)stream),
          "d1_norm_fwd");
    return py::make_tuple(y, mean, rstd);
}

py::tuple norm_fwd_alone(const Tensor &x, const Maybe &weight, const Maybe &bias, double eps, int64_t stream) {
    no_trace("layer_norm_fwd");
    return norm_fwd(x, weight, bias, eps, stream);
}

py::tuple norm_bwd(const Tensor &dy, const Tensor &x, const Maybe &weight, const Maybe &bias, const Tensor &mean_, const Tensor &rstd_,
                   int64_t stream) {
    no_trace("layer_norm_bwd");
    const NormArgs a = norm_args(x, weight, bias);
    no_tangent(dy, "dy");
    if (dy.sizes() != x.sizes() || dy.scalar_type() != x.scalar_type() || dy.device() != x.device())
        refuse("dy must be like x, " + describe(x) + ", not " + describe(dy));
    const Tensor drows = as_rows(dy);
    const auto shape = x.sizes().slice(0, x.dim() - 1);
    const Tensor mean = like(mean_, shape, at::kFloat, x, "mean"), rstd = like(rstd_, shape, at::kFloat, x, "rstd");
    const Tensor dx = at::empty(x.sizes(), x.options());
    Maybe dw, db, work;
    if (a.weight) dw = at::empty({a.width}, a.weight->options());
    if (a.bias) db = at::empty({a.width}, a.bias->options());
    const int64_t need = dw || db ? d1_norm_work_bytes(a.n, (int)a.width, a.code) : 0;
    if (need > 0) work = scratch(need, x);
    check(d1_norm_bwd(ptr(drows), drows.stride(0), ptr(a.rows), a.code, a.n, (int)a.width, a.rows.stride(0), ptr(a.weight), a.wcode,
                      (const float *)ptr(mean), (const float *)ptr(rstd), ptr(dx), ptr(dw), ptr(db), ptr(work), need, (void *)stream),
          "d1_norm_bwd");
    return py::make_tuple(dx, dw, db);
}

// ---- AdamW

using Tensors = std::vector<Tensor>;

void adamw_step(const Tensors &params, const Tensors &grads, const Tensors &exp_avg, const Tensors &exp_avg_sq, const Tensor &step,
                const std::vector<double> &lr, const std::vector<double> &weight_decay, double beta1, double beta2, double eps,
                double max_norm, const std::optional<std::vector<Maybe>> &copies, const std::optional<Tensors> &m_exps,
                const std::optional<Tensors> &v_exps, const std::optional<std::vector<int64_t>> &counters,
                const std::optional<std::vector<int64_t>> &lags, uint64_t seed, const Maybe &other, int64_t stream) {
    no_trace("adamw_step");
    const size_t count = params.size();
    const bool eight = m_exps.has_value();
    auto same = [&](size_t n, const char *name) {
        if (n != count) refuse(std::string(name) + ": " + std::to_string(n) + " for " + std::to_string(count) + " parameters");
    };
    same(grads.size(), "grads");
    same(exp_avg.size(), "exp_avg");
    same(exp_avg_sq.size(), "exp_avg_sq");
    same(lr.size(), "lr");
    same(weight_decay.size(), "weight_decay");
    if (copies) same(copies->size(), "copies");
    if (counters) same(counters->size(), "counters");
    if (lags) same(lags->size(), "lags");
    if (eight) {
        same(m_exps->size(), "exps[0]");
        same(v_exps->size(), "exps[1]");
    }
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && max_norm >= 0))
        refuse("betas must be in [0, 1), eps and max_grad_norm not negative");
    if (step.scalar_type() != at::kInt || step.dim() != 1 || step.size(0) != 8 || !step.is_cuda() || !step.is_contiguous())
        refuse("step must be a contiguous int32 CUDA tensor of 8 elements");
    if (other && (other->scalar_type() != at::kInt || other->dim() != 1 || other->size(0) != 8 || !other->is_contiguous() ||
                  other->device() != step.device() || ptr(*other) == ptr(step)))
        refuse("the other step's counts must be a contiguous int32 tensor of 8 elements on " + step.device().str() + ", not this one's");
    const at::ScalarType moment = eight ? at::kByte : at::kFloat;
    std::vector<D1AdamWTensor> table(count);
    Tensors held;            // contiguous gradients, until the launches that read them are queued
    for (size_t i = 0; i < count; i++) {
        const Tensor &p = params[i], &m = exp_avg[i], &v = exp_avg_sq[i];
        Tensor g = grads[i];
        const int64_t n = p.numel();
        auto fail = [&](const std::string &why) { refuse("tensor " + std::to_string(i) + ": " + why); };
        no_tangent(p, "parameter");
        no_tangent(g, "gradient");
        const int ptype = type_of(p.scalar_type()), gtype = type_of(g.scalar_type());
        if (!(ptype == D1_FP32 || ptype == D1_BF16) || !(gtype == D1_FP32 || gtype == D1_BF16))
            fail("parameter and gradient must be fp32 or bf16, not " + describe(p) + " and " + describe(g));
        if (m.scalar_type() != moment || v.scalar_type() != moment || g.numel() != n || m.numel() != n || v.numel() != n)
            fail(std::string("the gradient must have the size of the parameter, the moments too, in ") + c10::toString(moment));
        if (p.device() != step.device() || g.device() != step.device() || m.device() != step.device() || v.device() != step.device())
            fail("parameter, gradient and moments must be on " + step.device().str());
        if (!p.is_contiguous() || !m.is_contiguous() || !v.is_contiguous()) fail("parameter and moments must be contiguous");
        if (!(lr[i] >= 0 && weight_decay[i] >= 0)) fail("lr and weight_decay must not be negative");
        if (!g.is_contiguous()) {
            g = g.contiguous();
            held.push_back(g);
        }
        D1AdamWTensor &t = table[i];
        t = D1AdamWTensor{};
        t.p = ptr(p);
        t.g = ptr(g);
        t.m = ptr(m);
        t.v = ptr(v);
        t.n = n;
        t.lr = lr[i];
        t.weight_decay = weight_decay[i];
        t.ptype = (uint8_t)ptype;
        t.gtype = (uint8_t)gtype;
        if (counters) t.counter = (*counters)[i];
        if (lags) {
            if ((*lags)[i] < 0 || (*lags)[i] > INT32_MAX) fail("a lag must be 0 to 2^31 - 1");
            t.lag = (int32_t)(*lags)[i];
        }
        if (copies && (*copies)[i]) {
            const Tensor &c = *(*copies)[i];
            if (c.scalar_type() != at::kBFloat16 || c.numel() != n || !c.is_contiguous() || c.device() != step.device() || ptype != D1_FP32)
                fail("a copy is contiguous bf16 of the size of an fp32 parameter");
            t.copy = ptr(c);
        }
        if (eight) {
            for (const Tensor *e : {&(*m_exps)[i], &(*v_exps)[i]})
                if (e->scalar_type() != at::kByte || e->numel() != (n + D1_ADAMW_BLOCK - 1) / D1_ADAMW_BLOCK || !e->is_contiguous() ||
                    e->device() != step.device())
                    fail("exponents are contiguous uint8, one for each " + std::to_string(D1_ADAMW_BLOCK) + " elements");
            t.m_exp = (uint8_t *)ptr((*m_exps)[i]);
            t.v_exp = (uint8_t *)ptr((*v_exps)[i]);
        }
    }
    D1AdamW h{};
    h.beta1 = beta1;
    h.beta2 = beta2;
    h.eps = eps;
    h.max_norm = max_norm;
    h.seed = seed;
    h.bits = eight ? 8 : 32;
    const int64_t need = d1_adamw_work_bytes(table.data(), (int)count, &h);
    check(need < 0 ? (int)need : 0, "d1_adamw_work_bytes");
    Maybe work;
    if (need) work = scratch(need, step);
    check(d1_adamw_step_with(table.data(), (int)count, &h, (int32_t *)ptr(step), (int32_t *)ptr(other), ptr(work), need, (void *)stream),
          "d1_adamw_step_with");
    for (size_t i = 0; i < count; i++) {
        for (const Tensor *t : {&params[i], &exp_avg[i], &exp_avg_sq[i]}) written(*t);
        if (copies && (*copies)[i]) written(*(*copies)[i]);
        if (eight) {
            written((*m_exps)[i]);
            written((*v_exps)[i]);
        }
    }
    written(step);
    if (other) written(*other);
}

Tensor adamw_read(const Tensor &code, const Tensor &exp, bool is_signed, const Maybe &out_, int64_t stream) {
    no_trace("read_moment");
    const int64_t n = code.numel();
    if (code.scalar_type() != at::kByte || exp.scalar_type() != at::kByte || !code.is_cuda() || exp.device() != code.device() ||
        !code.is_contiguous() || !exp.is_contiguous() || exp.numel() != (n + D1_ADAMW_BLOCK - 1) / D1_ADAMW_BLOCK)
        refuse("code and exp must be contiguous uint8 CUDA tensors, one exponent for each " + std::to_string(D1_ADAMW_BLOCK) + " codes");
    if (out_ && (out_->scalar_type() != at::kFloat || out_->numel() != n || !out_->is_contiguous() || out_->device() != code.device()))
        refuse("out must be contiguous fp32 of the size of the codes, on their device");
    const Tensor out = out_ ? *out_ : at::empty(code.sizes(), code.options().dtype(at::kFloat));
    check(d1_adamw_read((const uint8_t *)ptr(code), (const uint8_t *)ptr(exp), n, is_signed, (float *)ptr(out), (void *)stream),
          "d1_adamw_read");
    written(out);
    return out;
}

// ---- the policy loss

// t as an input of [rows, length] tokens, a view where its strides allow it; what it refers to is put into `held`
D1LossInput loss_input(const Tensor &t, const Tensor &logp, int64_t rows, int64_t length, const char *name, Tensors &held) {
    no_tangent(t, name);
    const int code = type_of(t.scalar_type());
    if (code < 0 || t.sizes() != logp.sizes() || t.device() != logp.device())
        refuse(std::string(name) + " must be fp32, bf16 or fp16 of " + c10::str(logp.sizes()) + " on " + logp.device().str() + ", not " +
               describe(t));
    D1LossInput in{};
    in.type = code;
    if (t.dim() <= 2) {
        in.row = t.dim() == 2 ? t.stride(0) : length;
        in.step = t.stride(-1);
        in.data = t.data_ptr();
        held.push_back(t);
    } else {
        const Tensor r = t.reshape({rows, length});
        in.row = r.stride(0);
        in.step = r.stride(1);
        in.data = r.data_ptr();
        held.push_back(r);
    }
    return in;
}

// -> (terms [8], each of them, dlogp, dentropy, dvalues); a gradient that is not asked for is None. grads: a bit for each of them, and 8
// for all in fp32
py::tuple policy_loss(const Tensor &logp, const Tensor &old_logp, const Tensor &advantages, const Maybe &ref_logp, const Maybe &entropy,
                      const Maybe &values, const Maybe &returns, const Maybe &old_values, const Maybe &mask, double clip_low,
                      double clip_high, double kl_coef, double value_coef, double value_clip, double entropy_coef, bool sequence, int64_t grads,
                      int64_t stream) {
    no_trace("policy_loss");
    if (!logp.is_cuda()) refuse("logp must be a CUDA tensor (there is no CPU fallback)");
    if (logp.dim() == 0) refuse("logp must have at least one dimension");
    if (values.has_value() != returns.has_value()) refuse("values and returns come together");
    if (!(clip_low >= 0 && clip_low <= 1 && clip_high >= 0)) refuse("clip must be (0 to 1, 0 or more)");
    if (!(value_clip >= 0)) refuse("value_clip must not be negative");
    if (value_clip > 0 && values && !old_values) refuse("value_clip needs old_values");
    for (double c : {kl_coef, value_coef, entropy_coef})
        if (!std::isfinite(c)) refuse("coefficients must be finite");
    Tensors held;
    D1PolicyLoss h{};
    h.length = logp.size(-1);
    h.rows = h.length ? logp.numel() / h.length : 0;
    auto given = [&](const Tensor &t, const char *name) { return loss_input(t, logp, h.rows, h.length, name, held); };
    h.logp = given(logp, "logp");
    h.old_logp = given(old_logp, "old_logp");
    if (advantages.sizes() == logp.sizes()) {
        h.advantages = given(advantages, "advantages");
    } else {                 // one a sequence
        no_tangent(advantages, "advantages");
        const int code = type_of(advantages.scalar_type());
        if (code < 0 || advantages.sizes() != logp.sizes().slice(0, logp.dim() - 1) || advantages.device() != logp.device())
            refuse("advantages must be fp32, bf16 or fp16 of " + c10::str(logp.sizes()) + " or without its last dimension on " +
                   logp.device().str() + ", not " + describe(advantages));
        held.push_back(advantages.dim() == 1 ? advantages : advantages.reshape({h.rows}));
        h.advantages = {held.back().data_ptr(), held.back().stride(0), 0, code, 0};
    }
    if (ref_logp) h.ref_logp = given(*ref_logp, "ref_logp");
    if (entropy) h.entropy = given(*entropy, "entropy");
    if (values) {
        h.values = given(*values, "values");
        h.returns = given(*returns, "returns");
        if (old_values) h.old_values = given(*old_values, "old_values");
    }
    if (mask) {
        if ((mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte) || mask->sizes() != logp.sizes() ||
            mask->device() != logp.device())
            refuse("mask must be bool or uint8 of " + c10::str(logp.sizes()) + " on " + logp.device().str() + ", not " + describe(*mask));
        held.push_back(mask->dim() == 2 ? *mask : mask->reshape({h.rows, h.length}));
        h.mask = {held.back().data_ptr(), held.back().stride(0), held.back().stride(1), 0, 0};
    }
    h.clip_low = clip_low;
    h.clip_high = clip_high;
    h.value_clip = value_clip;
    h.kl_coef = kl_coef;
    h.value_coef = value_coef;
    h.entropy_coef = entropy_coef;
    h.sequence = sequence;
    h.fp32_grads = grads >> 3 & 1;
    const at::AutoDispatchBelowADInplaceOrView below;        // ten small tensors and views that autograd need not see
    const Tensor terms = at::empty({8}, logp.options().dtype(at::kFloat));
    Maybe dlogp, dentropy, dvalues, work;
    auto gradient = [&](const Tensor &of) { return at::empty(logp.sizes(), h.fp32_grads ? of.options().dtype(at::kFloat) : of.options()); };
    if (grads & 1) dlogp = gradient(logp);
    if ((grads & 2) && entropy) dentropy = gradient(*entropy);
    if ((grads & 4) && values) dvalues = gradient(*values);
    const int64_t need = d1_policy_loss_work_bytes(&h);
    check(need < 0 ? (int)need : 0, "d1_policy_loss_work_bytes");
    if (need) work = scratch(need, logp);
    check(d1_policy_loss(&h, (float *)ptr(terms), ptr(dlogp), ptr(dentropy), ptr(dvalues), ptr(work), need, (void *)stream),
          "d1_policy_loss");
    return py::make_tuple(terms, terms.unbind(0), dlogp, dentropy, dvalues);
}

// policy_loss's gradients, kept in fp32, times a number on the device, rounded to `types`, in tensors of their own: a graph that
// is kept, or a pass that is captured and replayed, finds them as they were
std::vector<Maybe> scale_grads(const Tensor &by, const std::vector<Maybe> &grads, const std::vector<at::ScalarType> &types, int64_t stream) {
    no_tangent(by, "the loss's gradient");
    if (by.scalar_type() != at::kFloat || by.numel() != 1 || !by.is_cuda()) refuse("the loss's gradient must be one fp32 number");
    std::vector<Maybe> out(grads.size());
    for (size_t i = 0; i < grads.size(); i++)
        if (grads[i]) {
            out[i] = at::empty(grads[i]->sizes(), grads[i]->options().dtype(types[i]));
            check(d1_scale_to((const float *)ptr(grads[i]), ptr(out[i]), type_of(types[i]), grads[i]->numel(), (const float *)ptr(by),
                              (void *)stream), "d1_scale_to");
        }
    return out;
}

// ---- the gated recurrence

struct ScanArgs {
    D1Scan h{};
    Tensor x, gate;
    Maybe state, reset;
    std::vector<int64_t> cells;          // the state's shape
};

// [steps, rows, width] or [steps, width], adjacent channels
Tensor scan_sequence(const Tensor &t, const Tensor &x, const char *name) {
    no_tangent(t, name);
    if (t.sizes() != x.sizes() || t.scalar_type() != x.scalar_type() || t.device() != x.device())
        refuse(std::string(name) + " must be like x, " + describe(x) + ", not " + describe(t));
    return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t;
}
int64_t row_stride(const Tensor &t) { return t.dim() == 3 ? t.stride(1) : 0; }

ScanArgs scan_args(const Tensor &x, const Tensor &gate, const Maybe &state, const Maybe &reset) {
    ScanArgs a;
    if (!x.is_cuda()) refuse("x must be a CUDA tensor (there is no CPU fallback)");
    a.h.type = type_of(x.scalar_type());
    if (a.h.type < 0) refuse(std::string("x must be fp32, bf16 or fp16, not ") + c10::toString(x.scalar_type()));
    if (x.dim() != 2 && x.dim() != 3) refuse("x must be [steps, rows, width] or [steps, width], not " + c10::str(x.sizes()));
    if (x.size(-1) > D1_SCAN_MAX_WIDTH || x.size(0) > D1_SCAN_MAX_STEPS) refuse("x: too many steps or channels");
    a.x = scan_sequence(x, x, "x");
    a.gate = scan_sequence(gate, x, "gate");
    a.cells.assign(x.sizes().begin() + 1, x.sizes().end());
    a.h.steps = x.size(0);
    a.h.rows = x.dim() == 3 ? x.size(1) : 1;
    a.h.width = (int32_t)x.size(-1);
    if (state) {
        a.state = like(*state, a.cells, at::kFloat, x, "state");
        a.h.state = (const float *)ptr(a.state);
    }
    if (reset) {
        if ((reset->scalar_type() != at::kBool && reset->scalar_type() != at::kByte) || reset->device() != x.device() ||
            reset->sizes() != x.sizes().slice(0, x.dim() - 1))
            refuse("reset must be bool or uint8 of " + c10::str(x.sizes().slice(0, x.dim() - 1)) + " on " + x.device().str() + ", not " +
                   describe(*reset));
        a.reset = reset;
        a.h.reset = (const uint8_t *)ptr(a.reset);
        a.h.reset_t = reset->stride(0);
        a.h.reset_n = reset->dim() == 2 ? reset->stride(1) : 0;
    }
    a.h.x = ptr(a.x);
    a.h.x_t = a.x.stride(0);
    a.h.x_n = row_stride(a.x);
    a.h.gate = ptr(a.gate);
    a.h.gate_t = a.gate.stride(0);
    a.h.gate_n = row_stride(a.gate);
    return a;
}

// an output like a sequence: its strides where they leave channels adjacent and no two elements on one place
Tensor scan_like(const Tensor &t) {
    const Tensor out = at::empty_like(t);
    return t.size(-1) > 1 && out.stride(-1) != 1 ? at::empty(t.sizes(), t.options()) : out;
}

// -> (h, last, marks); marks only where `keep` asks for them and a backward pass needs them
py::tuple scan_fwd(const Tensor &x, const Tensor &gate, const Maybe &state, const Maybe &reset, bool keep, int64_t stream) {
    no_trace("gated_scan");
    ScanArgs a = scan_args(x, gate, state, reset);
    const auto fp32 = x.options().dtype(at::kFloat);
    const Tensor h = scan_like(a.x);
    if (a.h.steps == 0) return py::make_tuple(h, a.state ? a.state->clone() : at::zeros(a.cells, fp32), Maybe());
    const Tensor last = at::empty(a.cells, fp32);
    Maybe marks, work;
    const int64_t count = keep ? d1_scan_marks(&a.h) : 0;
    check(count < 0 ? (int)count : 0, "d1_scan_marks");
    if (count) {
        marks = at::empty({count, a.h.rows * a.h.width}, fp32);
        a.h.marks = (float *)ptr(marks);
    }
    const int64_t need = d1_scan_work_bytes(&a.h);
    check(need < 0 ? (int)need : 0, "d1_scan_work_bytes");
    if (need) work = scratch(need, x);
    check(d1_scan_fwd(&a.h, ptr(h), h.stride(0), row_stride(h), (float *)ptr(last), ptr(work), need, (void *)stream), "d1_scan_fwd");
    return py::make_tuple(h, last, marks);
}

py::tuple scan_bwd(const Maybe &dh_, const Maybe &dlast_, const Tensor &x, const Tensor &gate, const Maybe &state, const Maybe &reset,
                   const Maybe &marks, int64_t stream) {
    no_trace("gated_scan_bwd");
    ScanArgs a = scan_args(x, gate, state, reset);
    const Tensor dh = dh_ ? scan_sequence(*dh_, x, "dh") : at::zeros(x.sizes(), x.options());
    Maybe dlast, dstate, work;
    if (dlast_) dlast = like(*dlast_, a.cells, at::kFloat, x, "dlast");
    const Tensor dx = scan_like(a.x), dgate = scan_like(a.gate);
    if (a.h.steps == 0) {
        if (state) dstate = dlast ? dlast->clone() : at::zeros(a.cells, x.options().dtype(at::kFloat));
        return py::make_tuple(dx, dgate, dstate);
    }
    if (state) dstate = at::empty(a.cells, x.options().dtype(at::kFloat));
    const int64_t count = d1_scan_marks(&a.h);
    check(count < 0 ? (int)count : 0, "d1_scan_marks");
    if (count) {
        if (!marks || marks->scalar_type() != at::kFloat || !marks->is_contiguous() || marks->device() != x.device() ||
            marks->numel() != count * a.h.rows * a.h.width)
            refuse("marks must be those of gated_scan_fwd with the same arguments");
        a.h.marks = (float *)ptr(*marks);
    }
    const int64_t need = d1_scan_work_bytes(&a.h);
    check(need < 0 ? (int)need : 0, "d1_scan_work_bytes");
    if (need) work = scratch(need, x);
    check(d1_scan_bwd(&a.h, ptr(dh), dh.stride(0), row_stride(dh), (const float *)ptr(dlast), ptr(dx), dx.stride(0), row_stride(dx),
                      ptr(dgate), dgate.stride(0), row_stride(dgate), (float *)ptr(dstate), ptr(work), need, (void *)stream),
          "d1_scan_bwd");
    return py::make_tuple(dx, dgate, dstate);
}

// ---- orthogonalised updates

D1Muon muon_settings(double a, double b, double c, double eps, int64_t steps, int64_t terms, double momentum, bool nesterov) {
    if (steps < 1 || steps > D1_MUON_MAX_STEPS) refuse("steps must be 1 to " + std::to_string(D1_MUON_MAX_STEPS));
    if (!(eps >= 0)) refuse("eps must not be negative");
    if (!(momentum >= 0 && momentum < 1)) refuse("momentum must be in [0, 1)");
    if (terms != 0 && terms != 1 && terms != 3) refuse("product_bits is None, 16 or 32");
    D1Muon h{};
    h.a = a;
    h.b = b;
    h.c = c;
    h.eps = eps;
    h.momentum = momentum;
    h.steps = (int32_t)steps;
    h.nesterov = nesterov;
    h.terms = (int32_t)terms;
    if (d1_muon_check(&h)) refuse("coefficients: singular values in [0, 1] must stay under 3.8 through all steps");
    return h;
}

Tensor muon_launch(const std::vector<D1MuonTensor> &table, const D1Muon &h, int32_t *ctl, const Maybe &work_, const Tensor &on,
                   int64_t stream) {
    const int64_t need = d1_muon_work_bytes(table.data(), (int)table.size(), &h);
    check(need < 0 ? (int)need : 0, "d1_muon_work_bytes");
    const Tensor work = work_ ? *work_ : scratch(need, on);
    if (work.nbytes() != (size_t)need) refuse("the second part of a step takes the same matrices as its first");
    check(d1_muon_step(table.data(), (int)table.size(), &h, ctl, ptr(work), need, (void *)stream), "d1_muon_step");
    return work;
}

// matrices [..., rows, cols] -> the same, orthogonalised, contiguous and of their types
Tensors orthogonalize(const Tensors &updates, double a, double b, double c, double eps, int64_t steps, int64_t terms, int64_t stream) {
    no_trace("orthogonalize");
    const D1Muon h = muon_settings(a, b, c, eps, steps, terms, 0.0, false);
    Tensors out, held;
    std::vector<D1MuonTensor> table;
    for (const Tensor &u : updates) {
        no_tangent(u, "update");
        const int code = type_of(u.scalar_type());
        if (code < 0 || u.dim() < 2 || !u.is_cuda() || u.device() != updates[0].device())
            refuse("an update must be an fp32, bf16 or fp16 CUDA tensor of two dimensions or more, all on one device, not " + describe(u));
        if (u.size(-1) > D1_MUON_MAX_SIDE || u.size(-2) > D1_MUON_MAX_SIDE)
            refuse("an update has sides of at most " + std::to_string(D1_MUON_MAX_SIDE));
        held.push_back(u.contiguous());
        out.push_back(at::empty(u.sizes(), u.options()));
        const int64_t each = u.size(-1) * u.size(-2), bytes = each * u.element_size();
        for (int64_t i = 0; each && i < u.numel() / each; i++) {
            D1MuonTensor t{};
            t.g = (const char *)ptr(held.back()) + i * bytes;
            t.out = (char *)ptr(out.back()) + i * bytes;
            t.rows = u.size(-2);
            t.cols = u.size(-1);
            t.type = t.gtype = code;
            table.push_back(t);
        }
    }
    if (!table.empty()) muon_launch(table, h, nullptr, {}, updates[0], stream);
    return out;
}

// part 0: a whole step; 1: its norms and whether it is made, -> what part 2 needs; 2: the rest of it
Maybe muon_step(const Tensors &params, const Tensors &grads, const Tensors &momenta, const Tensor &step, const std::vector<double> &lr,
               const std::vector<double> &scale, const std::vector<double> &weight_decay, const std::optional<std::vector<Maybe>> &copies,
               double momentum, bool nesterov, double a, double b, double c, double eps, int64_t steps, int64_t terms, int64_t part,
               const Maybe &work_, int64_t stream) {
    no_trace("muon_step");
    D1Muon h = muon_settings(a, b, c, eps, steps, terms, momentum, nesterov);
    h.part = (int32_t)part;
    const size_t count = params.size();
    auto same = [&](size_t n, const char *name) {
        if (n != count) refuse(std::string(name) + ": " + std::to_string(n) + " for " + std::to_string(count) + " parameters");
    };
    same(grads.size(), "grads");
    same(momenta.size(), "momenta");
    same(lr.size(), "lr");
    same(scale.size(), "scales");
    same(weight_decay.size(), "weight_decay");
    if (copies) same(copies->size(), "copies");
    if (step.scalar_type() != at::kInt || step.dim() != 1 || step.size(0) != 8 || !step.is_cuda() || !step.is_contiguous())
        refuse("step must be a contiguous int32 CUDA tensor of 8 elements");
    std::vector<D1MuonTensor> table(count);
    Tensors held;
    for (size_t i = 0; i < count; i++) {
        const Tensor &p = params[i], &m = momenta[i], &g = grads[i];
        auto fail = [&](const std::string &why) { refuse("matrix " + std::to_string(i) + ": " + why); };
        no_tangent(p, "parameter");
        no_tangent(g, "gradient");
        const int ptype = type_of(p.scalar_type()), gtype = type_of(g.scalar_type());
        if (!(ptype == D1_FP32 || ptype == D1_BF16) || !(gtype == D1_FP32 || gtype == D1_BF16))
            fail("parameter and gradient must be fp32 or bf16, not " + describe(p) + " and " + describe(g));
        if (p.dim() < 2) fail("a parameter must have two dimensions or more, not " + c10::str(p.sizes()));
        if (m.scalar_type() != at::kFloat || m.sizes() != p.sizes() || g.sizes() != p.sizes())
            fail("gradient and momentum (fp32) must have the parameter's shape");
        if (p.device() != step.device() || g.device() != step.device() || m.device() != step.device())
            fail("parameter, gradient and momentum must be on " + step.device().str());
        if (!p.is_contiguous() || !m.is_contiguous()) fail("parameter and momentum must be contiguous");
        if (!(lr[i] >= 0 && weight_decay[i] >= 0 && scale[i] >= 0) || !std::isfinite(lr[i] * scale[i]) || !std::isfinite(lr[i] * weight_decay[i]))
            fail("lr, scale and weight_decay must be finite and not negative");
        held.push_back(g.contiguous());
        D1MuonTensor &t = table[i];
        t = D1MuonTensor{};
        t.g = ptr(held.back());
        t.momentum = (float *)ptr(m);
        t.out = ptr(p);
        t.rows = p.size(0);
        t.cols = t.rows ? p.numel() / t.rows : 0;
        if (t.rows > D1_MUON_MAX_SIDE || t.cols > D1_MUON_MAX_SIDE) fail("a matrix has sides of at most " + std::to_string(D1_MUON_MAX_SIDE));
        t.lr = lr[i];
        t.scale = scale[i];
        t.weight_decay = weight_decay[i];
        t.type = ptype;
        t.gtype = gtype;
        if (copies && (*copies)[i]) {
            const Tensor &c_ = *(*copies)[i];
            if (c_.scalar_type() != at::kBFloat16 || c_.numel() != p.numel() || !c_.is_contiguous() || c_.device() != step.device() ||
                ptype != D1_FP32)
                fail("a copy is contiguous bf16 of the size of an fp32 parameter");
            t.copy = ptr(c_);
        }
    }
    // two of them on one place would step it twice, in any order
    std::vector<std::pair<const char *, const char *>> places;
    auto place = [&](const Tensor &t) {
        if (t.numel()) places.emplace_back((const char *)ptr(t), (const char *)ptr(t) + t.nbytes());
    };
    for (size_t i = 0; i < count; i++) {
        place(params[i]);
        place(momenta[i]);
        if (copies && (*copies)[i]) place(*(*copies)[i]);
    }
    std::sort(places.begin(), places.end());
    for (size_t i = 1; i < places.size(); i++)
        if (places[i].first < places[i - 1].second) refuse("parameters, momenta and copies must not overlap");
    // and a gradient on one of them would be read after it is written (what was copied to be contiguous lies elsewhere)
    for (size_t i = 0; i < count; i++) {
        if (!held[i].numel()) continue;
        const char *begin = (const char *)ptr(held[i]), *end = begin + held[i].nbytes();
        const auto behind = std::lower_bound(places.begin(), places.end(), std::make_pair(end, (const char *)nullptr));
        if (behind != places.begin() && (behind - 1)->second > begin)
            refuse("matrix " + std::to_string(i) + ": its gradient must not overlap parameters, momenta or copies");
    }
    const Tensor work = muon_launch(table, h, (int32_t *)ptr(step), work_, step, stream);
    written(step);
    if (part == 1) return work;
    for (size_t i = 0; i < count; i++) {
        written(params[i]);
        written(momenta[i]);
        if (copies && (*copies)[i]) written(*(*copies)[i]);
    }
    return {};
}

}  // namespace

PYBIND11_MODULE(_d1ops, m) {
    m.def("orthogonalize", &orthogonalize);
    m.def("muon_step", &muon_step);
    m.def("scan_fwd", &scan_fwd);
    m.def("scan_bwd", &scan_bwd);
    m.def("policy_loss", &policy_loss);
    m.def("scale_grads", &scale_grads);
    m.def("tokens_fwd", &tokens_fwd);
    m.def("tokens_bwd", &tokens_bwd);
    m.def("norm_fwd", &norm_fwd);
    m.def("norm_fwd_alone", &norm_fwd_alone);
    m.def("norm_bwd", &norm_bwd);
    m.def("adamw_step", &adamw_step);
    m.def("adamw_read", &adamw_read);
}
