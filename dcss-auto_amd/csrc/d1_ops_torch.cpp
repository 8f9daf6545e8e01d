// d1ops: the Python calls of libd1ops.so on torch tensors (module _d1ops).
//
// A call on a small minibatch is a few microseconds of GPU work, less than its argument checks and
// three allocations take in Python (11 us a call there, 6 here, 3 of them the launch itself). Checks, outputs
// and scratch memory are therefore made here; the kernels and their C ABI know nothing of torch. Argument errors
// are ValueError before any launch. The caller has made the tensors' device the current one and gives its stream.
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <string>
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
                const std::optional<std::vector<int64_t>> &lags, uint64_t seed, int64_t stream) {
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
    check(d1_adamw_step(table.data(), (int)count, &h, (int32_t *)ptr(step), ptr(work), need, (void *)stream), "d1_adamw_step");
    for (size_t i = 0; i < count; i++) {
        for (const Tensor *t : {&params[i], &exp_avg[i], &exp_avg_sq[i]}) written(*t);
        if (copies && (*copies)[i]) written(*(*copies)[i]);
        if (eight) {
            written((*m_exps)[i]);
            written((*v_exps)[i]);
        }
    }
    written(step);
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

}  // namespace

PYBIND11_MODULE(_d1ops, m) {
    m.def("tokens_fwd", &tokens_fwd);
    m.def("tokens_bwd", &tokens_bwd);
    m.def("norm_fwd", &norm_fwd);
    m.def("norm_fwd_alone", &norm_fwd_alone);
    m.def("norm_bwd", &norm_bwd);
    m.def("adamw_step", &adamw_step);
    m.def("adamw_read", &adamw_read);
}
