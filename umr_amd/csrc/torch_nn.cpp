// torch_nn.cpp -- the network-side operators (include/umr_nn.h) as PyTorch operators: schemas, argument checks, device and meta
// implementations, autograd.  Compiled into umr_amd/lib/libumr_torch.so, which links libumr_hip.so; loaded by umr_amd/ops_nn.py.
//
// In C++ and not in Python as the older operators are: these are called for layers of a few hundred columns, whose kernels take some
// microseconds, and an operator with a Python implementation and a Python autograd formula costs 70 - 120 us a call on the host.
//
//   umr::linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act, float slope) -> Tensor
//       weight [N, K]:     x [.., K],    bias [N],    residual [.., N] or [N]             -> [.., N]
//       weight [G, N, K]:  x [.., G, K], bias [G, N], residual [.., G, N] or [G, N]       -> [.., G, N]
//   umr::linear_act_z(...) -> (y, z)     the same below autograd, z as umr_linear_forward keeps it
//   umr::linear_act_backward(grad, x, weight, z, int act, float slope, bool need_x, need_w, need_b, need_r) -> (dx, dw, db, dr),
//       undefined (None) where not needed
//   umr::balance_loss(Tensor scores, Tensor inds, Tensor? mask) -> (loss, counts)
//   umr::balance_loss_coef(...) -> (loss, counts, coef)     below autograd
//   umr::balance_loss_backward(grad, scores, mask, coef) -> Tensor
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/umr_nn.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int type_of(const Tensor &t, const char *who) {
    switch (t.scalar_type()) {
        case at::kFloat: return UMR_F32;
        case at::kBFloat16: return UMR_BF16;
        case at::kHalf: return UMR_F16;
        default: TORCH_CHECK(false, "umr_amd: ", who, ": float32, bfloat16 or float16 expected, got ", t.scalar_type());
    }
}

void on_gpu(const Tensor &t, const Tensor &first, const char *who, const char *name) {
    TORCH_CHECK(t.is_cuda(), "umr_amd: expected a GPU tensor, got ", t.device(), " (no CPU path exists)");
    TORCH_CHECK(t.device() == first.device(), "umr_amd: ", who, ": ", name, " is on ", t.device(), ", not on ", first.device());
}

// Kernels are launched on the current stream of the CURRENT device, as all of this library's: a tensor elsewhere is refused.
void *stream_of(const Tensor &t) {
    const auto current = c10::hip::current_device();
    TORCH_CHECK(t.device().index() == current, "umr_amd: tensors live on cuda:", (int)t.device().index(), " but the current device is cuda:",
                (int)current, "; call torch.cuda.set_device first");
    return (void *)c10::hip::getCurrentHIPStream(current).stream();
}

void check_status(int rc, const char *what) {
    TORCH_CHECK(rc == UMR_OK, "umr_amd: ", what, " failed with status ", rc, rc == UMR_ERR_ARG ? " (rejected arguments)" : " (kernel launch error)");
}

Tensor workspace(size_t bytes, const Tensor &like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void *data_of(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---------------------------------------------------------------------------------------------- linear_act
struct Sizes {
    int64_t M, G, N, K;
    bool heads;
};

// shapes and types; valid for meta tensors too
Sizes linear_sizes(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act, double slope) {
    const char *who = "linear_act";
    TORCH_CHECK(w.dim() == 2 || w.dim() == 3, "umr_amd: linear_act: weight must be [N, K] or [G, N, K], got ", w.sizes());
    Sizes s;
    s.heads = w.dim() == 3;
    s.G = s.heads ? w.size(0) : 1;
    s.N = w.size(-2);
    s.K = w.size(-1);
    TORCH_CHECK(s.G >= 1 && s.G <= 65535, "umr_amd: linear_act: 1 to 65535 heads, got ", s.G);
    TORCH_CHECK(x.dim() >= (s.heads ? 2 : 1) && x.size(-1) == s.K && (!s.heads || x.size(-2) == s.G),
                "umr_amd: linear_act: x ", x.sizes(), " does not fit weight ", w.sizes(), ": expected [.., ", s.heads ? "G, " : "", "K]");
    s.M = 1;
    for (int64_t d = 0; d < x.dim() - (s.heads ? 2 : 1); ++d) s.M *= x.size(d);
    type_of(x, who);
    TORCH_CHECK(w.scalar_type() == x.scalar_type(), "umr_amd: linear_act: weight is ", w.scalar_type(), ", x is ", x.scalar_type());
    if (b) {
        TORCH_CHECK(b->scalar_type() == x.scalar_type(), "umr_amd: linear_act: bias is ", b->scalar_type(), ", x is ", x.scalar_type());
        TORCH_CHECK(b->sizes() == (s.heads ? at::IntArrayRef({s.G, s.N}) : at::IntArrayRef({s.N})), "umr_amd: linear_act: bias ", b->sizes(),
                    " does not fit weight ", w.sizes());
    }
    if (r) {
        TORCH_CHECK(r->scalar_type() == x.scalar_type(), "umr_amd: linear_act: residual is ", r->scalar_type(), ", x is ", x.scalar_type());
        std::vector<int64_t> full(x.sizes().begin(), x.sizes().end());
        full.back() = s.N;
        TORCH_CHECK(r->sizes() == at::IntArrayRef(full) || r->sizes() == (s.heads ? at::IntArrayRef({s.G, s.N}) : at::IntArrayRef({s.N})),
                    "umr_amd: linear_act: residual must be the output's shape ", full, " or one row of it, got ", r->sizes());
    }
    TORCH_CHECK(act >= UMR_ACT_NONE && act <= UMR_ACT_SILU, "umr_amd: linear_act: unknown activation ", act);
    TORCH_CHECK(act != UMR_ACT_LEAKY_RELU || slope >= 0, "umr_amd: linear_act: leaky_relu needs a slope >= 0, got ", slope);
    return s;
}

// A [.., (G,) C] tensor as rows: element strides of a row and of a head.  Copied only where its leading dimensions are not evenly
// spaced or its last one is not contiguous.
struct Rows {
    Tensor t;                   // keeps a copy alive
    int64_t row = 0, head = 0;
    const void *data() const { return t.defined() && t.numel() ? t.const_data_ptr() : nullptr; }
};

bool rows_of(const Tensor &t, bool heads, Rows &out) {
    if (t.size(-1) > 1 && t.stride(-1) != 1) return false;
    int64_t row = -1, span = 0;                                  // span: the stride that the next outer dimension must have
    for (int64_t d = t.dim() - (heads ? 3 : 2); d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (row < 0) row = span = t.stride(d);
        else if (t.stride(d) != span) return false;
        span *= t.size(d);
    }
    out.row = row < 0 ? 0 : row;
    out.head = heads && t.size(-2) > 1 ? t.stride(-2) : 0;
    out.t = t;
    return true;
}

Rows as_rows(const Tensor &t, bool heads) {
    Rows r;
    r.t = t;
    if (t.numel() != 0 && !rows_of(t, heads, r)) TORCH_INTERNAL_ASSERT(rows_of(t.contiguous(), heads, r));
    return r;
}

Rows as_weight(const Tensor &w) {                                // [N, K] or [G, N, K]: row = along N
    Rows r;
    r.t = w.size(-1) > 1 && w.stride(-1) != 1 ? w.contiguous() : w;
    r.row = r.t.size(-2) > 1 ? r.t.stride(-2) : 0;
    r.head = w.dim() == 3 && r.t.size(0) > 1 ? r.t.stride(0) : 0;
    return r;
}

Rows as_residual(const Tensor &r, const Tensor &x, bool heads) {
    if (r.dim() == x.dim()) return as_rows(r, heads);
    Rows o;                                                      // one row for all
    o.t = r.size(-1) > 1 && r.stride(-1) != 1 ? r.contiguous() : r;
    o.head = heads && o.t.size(0) > 1 ? o.t.stride(0) : 0;
    return o;
}

bool kinked(int64_t act) { return act == UMR_ACT_RELU || act == UMR_ACT_LEAKY_RELU; }
at::TensorOptions options_of_z(const Tensor &x, int64_t act) { return kinked(act) ? x.options() : x.options().dtype(at::kFloat); }

std::vector<int64_t> with_last(const Tensor &x, int64_t n) {
    std::vector<int64_t> v(x.sizes().begin(), x.sizes().end());
    v.back() = n;
    return v;
}

Tensor linear_forward(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act, double slope, Tensor *z) {
    const Sizes s = linear_sizes(x, w, b, r, act, slope);
    const char *who = "linear_act";
    on_gpu(x, x, who, "x");
    on_gpu(w, x, who, "weight");
    if (b) on_gpu(*b, x, who, "bias");
    if (r) on_gpu(*r, x, who, "residual");
    void *stream = stream_of(x);
    const int dt = type_of(x, who);
    const Rows xr = as_rows(x, s.heads), wr = as_weight(w);
    const Tensor bias = b ? b->contiguous() : Tensor();
    const Rows rr = r ? as_residual(*r, x, s.heads) : Rows();
    Tensor y = at::empty(with_last(x, s.N), x.options());
    if (z) *z = at::empty(y.sizes(), options_of_z(x, act));
    const size_t bytes = umr_linear_forward_workspace_bytes(s.M, s.N, s.K, (int)s.G, dt);
    const Tensor ws = workspace(bytes, x);
    check_status(umr_linear_forward(xr.data(), xr.row, xr.head, wr.data(), wr.row, wr.head, b && s.N ? bias.const_data_ptr() : nullptr,
                                    rr.data(), rr.row, rr.head, data_of(y), z ? data_of(*z) : nullptr, s.M, s.N, s.K, (int)s.G, dt, (int)act,
                                    (float)slope, data_of(ws), bytes, stream),
                 "umr_linear_forward");
    return y;
}

Tensor linear_act(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act, double slope) {
    return linear_forward(x, w, b, r, act, slope, nullptr);
}
std::tuple<Tensor, Tensor> linear_act_z(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act,
                                        double slope) {
    Tensor z, y = linear_forward(x, w, b, r, act, slope, &z);
    return {y, z};
}

Tensor linear_act_meta(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act, double slope) {
    return at::empty(with_last(x, linear_sizes(x, w, b, r, act, slope).N), x.options());
}
std::tuple<Tensor, Tensor> linear_act_z_meta(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act,
                                             double slope) {
    Tensor y = linear_act_meta(x, w, b, r, act, slope);
    return {y, at::empty(y.sizes(), options_of_z(x, act))};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> linear_act_backward(const Tensor &grad, const Tensor &x, const Tensor &w, const Tensor &z, int64_t act,
                                                               double slope, bool need_x, bool need_w, bool need_b, bool need_r) {
    const char *who = "linear_act_backward";
    const Sizes s = linear_sizes(x, w, {}, {}, act, slope);
    TORCH_CHECK(grad.sizes() == at::IntArrayRef(with_last(x, s.N)) && grad.scalar_type() == x.scalar_type(),
                "umr_amd: linear_act_backward: the gradient must be the output's shape and type, got ", grad.sizes(), " ", grad.scalar_type());
    TORCH_CHECK(act == UMR_ACT_NONE || (z.sizes() == grad.sizes() && z.scalar_type() == c10::typeMetaToScalarType(options_of_z(x, act).dtype())),
                "umr_amd: linear_act_backward: z must be the output's shape, in ", kinked(act) ? "x's type" : "float32", ", got ", z.sizes(), " ", z.scalar_type());
    on_gpu(x, x, who, "x");
    on_gpu(grad, x, who, "grad");
    on_gpu(w, x, who, "weight");
    void *stream = stream_of(x);
    const int dt = type_of(x, who);
    const int G = (int)s.G;
    const auto opt = x.options();
    const Rows gr = as_rows(grad, s.heads);
    const at::IntArrayRef row2 = w.sizes().slice(0, w.dim() - 1);                 // [N] or [G, N]
    Tensor dx, dw, db, dr;
    if (need_x) dx = at::empty(x.sizes(), opt);
    if (need_w) dw = at::empty(w.sizes(), opt);
    if (need_b) db = at::empty(row2, opt);
    if (need_r) dr = at::empty(row2, opt);
    Rows dz = gr;
    const bool derive = act != UMR_ACT_NONE && (need_x || need_w || need_b);
    if (derive || need_b || need_r) {
        Tensor out;
        Tensor zc;
        if (derive) {
            on_gpu(z, x, who, "z");
            zc = z.contiguous();
            out = at::empty(grad.sizes(), opt);
        }
        const size_t bytes = need_b || need_r ? umr_linear_grad_act_workspace_bytes(s.M, s.N, G) : 0;
        const Tensor ws = workspace(bytes, x);
        check_status(umr_linear_grad_act(gr.data(), gr.row, gr.head, data_of(zc), data_of(out),
                                         need_b && s.N ? db.data_ptr() : nullptr, need_r && s.N ? dr.data_ptr() : nullptr, s.M, s.N, G, dt,
                                         derive ? (int)act : UMR_ACT_NONE, (float)slope, data_of(ws), bytes, stream),
                     "umr_linear_grad_act");
        if (derive) dz = as_rows(out, s.heads);
    }
    if (need_x) {
        const Rows wr = as_weight(w);
        const size_t bytes = umr_linear_grad_input_workspace_bytes(s.M, s.N, s.K, G, dt);
        const Tensor ws = workspace(bytes, x);
        check_status(umr_linear_grad_input(dz.data(), dz.row, dz.head, wr.data(), wr.row, wr.head, data_of(dx), s.M, s.N, s.K, G, dt, data_of(ws),
                                           bytes, stream),
                     "umr_linear_grad_input");
    }
    if (need_w) {
        const Rows xr = as_rows(x, s.heads);
        const size_t bytes = umr_linear_grad_weight_workspace_bytes(s.M, s.N, s.K, G, dt);
        const Tensor ws = workspace(bytes, x);
        check_status(umr_linear_grad_weight(dz.data(), dz.row, dz.head, xr.data(), xr.row, xr.head, data_of(dw), s.M, s.N, s.K, G, dt, data_of(ws),
                                            bytes, stream),
                     "umr_linear_grad_weight");
    }
    return {dx, dw, db, dr};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> linear_act_backward_meta(const Tensor &grad, const Tensor &x, const Tensor &w, const Tensor &z, int64_t act,
                                                                    double slope, bool need_x, bool need_w, bool need_b, bool need_r) {
    const auto opt = x.options();
    const at::IntArrayRef row2 = w.sizes().slice(0, w.dim() - 1);
    return {need_x ? at::empty(x.sizes(), opt) : Tensor(), need_w ? at::empty(w.sizes(), opt) : Tensor(), need_b ? at::empty(row2, opt) : Tensor(),
            need_r ? at::empty(row2, opt) : Tensor()};
}

template <class Signature> auto typed(const char *name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

enum { HAS_BIAS = 256, HAS_RESIDUAL = 512, ROW_RESIDUAL = 1024 };       // above the activation, in one saved number

struct LinearAct : public torch::autograd::Function<LinearAct> {
    static Variable forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act,
                            double slope) {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto plain = typed<decltype(linear_act)>("umr::linear_act");
        static const auto with_z = typed<decltype(linear_act_z)>("umr::linear_act_z");
        // act' needs the pre-activation -- or, for the two kinked ones without a residual, only its sign, which is the output's
        Tensor y, z;
        if (act != UMR_ACT_NONE && !(kinked(act) && !r)) std::tie(y, z) = with_z.call(x, w, b, r, act, slope);
        else y = plain.call(x, w, b, r, act, slope);
        ctx->save_for_backward({x, w, act == UMR_ACT_NONE ? Tensor() : z.defined() ? z : y});
        ctx->saved_data["act"] = act | (b ? HAS_BIAS : 0) | (r ? HAS_RESIDUAL : 0) | (r && r->dim() != x.dim() ? ROW_RESIDUAL : 0);
        ctx->saved_data["slope"] = slope;
        return y;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        static const auto op = typed<decltype(linear_act_backward)>("umr::linear_act_backward");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &g = grads[0];
        const int64_t kept = ctx->saved_data["act"].toInt(), act = kept & 255;
        const bool has_b = kept & HAS_BIAS, row = kept & ROW_RESIDUAL;
        // needs_input_grad counts the tensors that were passed, in their order
        const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = has_b && ctx->needs_input_grad(2),
                   nr = (kept & HAS_RESIDUAL) && ctx->needs_input_grad(has_b ? 3 : 2);
        Tensor dx, dw, db, dr;
        if (nx || nw || nb || (nr && row))
            std::tie(dx, dw, db, dr) = op.call(g, x, w, act == UMR_ACT_NONE ? g : saved[2], act, ctx->saved_data["slope"].toDouble(), nx, nw, nb, nr && row);
        return {dx, dw, db, nr ? (row ? dr : g) : Tensor(), Tensor(), Tensor()};
    }
};

// A tangent (torch.autograd.forward_ad, torch.func.jvp) needs no requires_grad and passes no_grad: refused wherever one arrives,
// or the result would come without it.
void no_tangent(const char *name, std::initializer_list<const Tensor *> inputs) {
    for (const Tensor *t : inputs)
        TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), "umr_amd: ", name, " has no forward-mode derivative");
}
const Tensor *given(const optional<Tensor> &t) { return t ? &*t : nullptr; }

bool tracked(const Tensor &a) { return a.requires_grad(); }
bool tracked(const optional<Tensor> &a) { return a && a->requires_grad(); }

Tensor linear_act_autograd(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act, double slope) {
    no_tangent("linear_act", {&x, &w, given(b), given(r)});
    if (at::GradMode::is_enabled() && (tracked(x) || tracked(w) || tracked(b) || tracked(r))) return LinearAct::apply(x, w, b, r, act, slope);
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = typed<decltype(linear_act)>("umr::linear_act");
    return op.call(x, w, b, r, act, slope);
}

// Under torch.autocast every tensor is cast to its type, as torch's own linear layer does.  (balance_loss takes scores of any type.)
Tensor linear_act_autocast(const Tensor &x, const Tensor &w, const optional<Tensor> &b, const optional<Tensor> &r, int64_t act, double slope) {
    c10::impl::ExcludeDispatchKeyGuard below(c10::DispatchKey::AutocastCUDA);
    static const auto op = typed<decltype(linear_act)>("umr::linear_act");
    const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
    const auto cast = [&](const auto &t) { return at::autocast::cached_cast(type, t, at::kCUDA); };
    return op.call(cast(x), cast(w), cast(b), cast(r), act, slope);
}

// ---------------------------------------------------------------------------------------------- balance_loss
void balance_sizes(const Tensor &z, const Tensor &inds, const optional<Tensor> &mask) {
    type_of(z, "balance_loss");
    TORCH_CHECK(z.dim() == 2 && z.size(1) >= 1 && z.size(1) <= UMR_BALANCE_MAX_CHOICES, "umr_amd: balance_loss: scores must be [T, E] with 1 <= E <= ",
                UMR_BALANCE_MAX_CHOICES, ", got ", z.sizes());
    TORCH_CHECK(inds.dim() == 2 && inds.size(0) == z.size(0) && inds.size(1) >= 1 && inds.scalar_type() == at::kLong,
                "umr_amd: balance_loss: inds must be [T, k] int64 with k >= 1, got ", inds.sizes(), " ", inds.scalar_type());
    TORCH_CHECK(!mask || (mask->dim() == 1 && mask->size(0) == z.size(0) && mask->scalar_type() == at::kBool),
                "umr_amd: balance_loss: mask must be [T] bool");
}

std::tuple<Tensor, Tensor, Tensor> balance_loss_coef(const Tensor &z_, const Tensor &inds_, const optional<Tensor> &mask_) {
    const char *who = "balance_loss";
    balance_sizes(z_, inds_, mask_);
    on_gpu(z_, z_, who, "scores");
    on_gpu(inds_, z_, who, "inds");
    if (mask_) on_gpu(*mask_, z_, who, "mask");
    void *stream = stream_of(z_);
    const Tensor z = z_.contiguous(), inds = inds_.contiguous(), mask = mask_ ? mask_->contiguous() : Tensor();
    const int64_t T = z.size(0), E = z.size(1);
    Tensor loss = at::empty({}, z.options().dtype(at::kFloat)), counts = at::empty({E}, z.options().dtype(at::kLong));
    Tensor coef = at::empty({E + 1}, z.options().dtype(at::kFloat));
    const size_t bytes = umr_balance_workspace_bytes(T, (int)E);
    const Tensor ws = workspace(bytes, z);
    check_status(umr_balance_forward(z.const_data_ptr(), (const long long *)inds.const_data_ptr(),
                                     mask.defined() ? (const unsigned char *)mask.const_data_ptr() : nullptr, (float *)loss.data_ptr(),
                                     (long long *)counts.data_ptr(), (float *)coef.data_ptr(), T, (int)E, (int)std::min<int64_t>(inds.size(1), INT32_MAX),
                                     type_of(z, who), data_of(ws), bytes, stream),
                 "umr_balance_forward");
    return {loss, counts, coef};
}

std::tuple<Tensor, Tensor, Tensor> balance_loss_coef_meta(const Tensor &z, const Tensor &inds, const optional<Tensor> &mask) {
    balance_sizes(z, inds, mask);
    const auto f = z.options().dtype(at::kFloat);
    return {at::empty({}, f), at::empty({z.size(1)}, z.options().dtype(at::kLong)), at::empty({z.size(1) + 1}, f)};
}

Tensor balance_loss_backward(const Tensor &grad, const Tensor &z_, const optional<Tensor> &mask_, const Tensor &coef_) {
    const char *who = "balance_loss_backward";
    on_gpu(z_, z_, who, "scores");
    on_gpu(grad, z_, who, "grad");
    on_gpu(coef_, z_, who, "coef");
    if (mask_) on_gpu(*mask_, z_, who, "mask");
    TORCH_CHECK(z_.dim() == 2 && z_.size(1) >= 1 && z_.size(1) <= UMR_BALANCE_MAX_CHOICES && grad.numel() == 1 && grad.scalar_type() == at::kFloat &&
                    coef_.numel() == z_.size(1) + 1 && coef_.scalar_type() == at::kFloat &&
                    (!mask_ || (mask_->numel() == z_.size(0) && mask_->scalar_type() == at::kBool)),
                "umr_amd: balance_loss_backward: arguments do not fit");
    void *stream = stream_of(z_);
    const Tensor z = z_.contiguous(), coef = coef_.contiguous(), mask = mask_ ? mask_->contiguous() : Tensor();
    Tensor dz = at::empty(z.sizes(), z.options());
    check_status(umr_balance_backward(z.const_data_ptr(), mask.defined() ? (const unsigned char *)mask.const_data_ptr() : nullptr,
                                      (const float *)coef.const_data_ptr(), (const float *)grad.const_data_ptr(), dz.data_ptr(), z.size(0),
                                      (int)z.size(1), type_of(z, who), stream),
                 "umr_balance_backward");
    return dz;
}
Tensor balance_loss_backward_meta(const Tensor &, const Tensor &z, const optional<Tensor> &, const Tensor &) { return at::empty(z.sizes(), z.options()); }

struct BalanceLoss : public torch::autograd::Function<BalanceLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &z, const Tensor &inds, const optional<Tensor> &mask) {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = typed<decltype(balance_loss_coef)>("umr::balance_loss_coef");
        auto [loss, counts, coef] = op.call(z, inds, mask);
        ctx->save_for_backward({z, coef, mask ? *mask : Tensor()});
        ctx->mark_non_differentiable({counts});
        return {loss, counts};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        static const auto op = typed<decltype(balance_loss_backward)>("umr::balance_loss_backward");
        const auto saved = ctx->get_saved_variables();
        if (!ctx->needs_input_grad(0)) return {Tensor(), Tensor(), Tensor()};
        return {op.call(grads[0], saved[0], saved[2].defined() ? optional<Tensor>(saved[2]) : optional<Tensor>(), saved[1]), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> balance_loss_autograd(const Tensor &z, const Tensor &inds, const optional<Tensor> &mask) {
    no_tangent("balance_loss", {&z});
    if (at::GradMode::is_enabled() && z.requires_grad()) {
        auto out = BalanceLoss::apply(z, inds, mask);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = typed<decltype(balance_loss_coef)>("umr::balance_loss_coef");
    auto [loss, counts, coef] = op.call(z, inds, mask);
    return {loss, counts};
}
std::tuple<Tensor, Tensor> balance_loss(const Tensor &z, const Tensor &inds, const optional<Tensor> &mask) {
    auto [loss, counts, coef] = balance_loss_coef(z, inds, mask);
    return {loss, counts};
}
std::tuple<Tensor, Tensor> balance_loss_meta(const Tensor &z, const Tensor &inds, const optional<Tensor> &mask) {
    auto [loss, counts, coef] = balance_loss_coef_meta(z, inds, mask);
    return {loss, counts};
}

// The backward operators have no derivative of their own: refused instead of a result that is cut off from the graph.
void once_only(bool any, const char *name) {
    TORCH_CHECK(!(any && at::GradMode::is_enabled()), "umr_amd: ", name, " is not differentiable a second time");
}
std::tuple<Tensor, Tensor, Tensor, Tensor> linear_act_backward_once(const Tensor &grad, const Tensor &x, const Tensor &w, const Tensor &z, int64_t act,
                                                                    double slope, bool nx, bool nw, bool nb, bool nr) {
    no_tangent("the gradient of linear_act", {&grad, &x, &w, &z});
    once_only(tracked(grad) || tracked(x) || tracked(w) || tracked(z), "linear_act");
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = typed<decltype(linear_act_backward)>("umr::linear_act_backward");
    return op.call(grad, x, w, z, act, slope, nx, nw, nb, nr);
}
Tensor balance_loss_backward_once(const Tensor &grad, const Tensor &z, const optional<Tensor> &mask, const Tensor &coef) {
    no_tangent("the gradient of balance_loss", {&grad, &z, &coef});
    once_only(tracked(grad) || tracked(z) || tracked(coef), "balance_loss");
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = typed<decltype(balance_loss_backward)>("umr::balance_loss_backward");
    return op.call(grad, z, mask, coef);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(umr, m) {
    m.def("linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act, float slope) -> Tensor");
    m.def("linear_act_z(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act, float slope) -> (Tensor, Tensor)");
    m.def("linear_act_backward(Tensor grad, Tensor x, Tensor weight, Tensor z, int act, float slope, bool need_x, bool need_w, bool need_b, "
          "bool need_r) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("balance_loss(Tensor scores, Tensor inds, Tensor? mask) -> (Tensor, Tensor)");
    m.def("balance_loss_coef(Tensor scores, Tensor inds, Tensor? mask) -> (Tensor, Tensor, Tensor)");
    m.def("balance_loss_backward(Tensor grad, Tensor scores, Tensor? mask, Tensor coef) -> Tensor");
}
TORCH_LIBRARY_IMPL(umr, CUDA, m) {
    m.impl("linear_act", linear_act);
    m.impl("linear_act_z", linear_act_z);
    m.impl("linear_act_backward", linear_act_backward);
    m.impl("balance_loss", balance_loss);
    m.impl("balance_loss_coef", balance_loss_coef);
    m.impl("balance_loss_backward", balance_loss_backward);
}
TORCH_LIBRARY_IMPL(umr, Meta, m) {
    m.impl("linear_act", linear_act_meta);
    m.impl("linear_act_z", linear_act_z_meta);
    m.impl("linear_act_backward", linear_act_backward_meta);
    m.impl("balance_loss", balance_loss_meta);
    m.impl("balance_loss_coef", balance_loss_coef_meta);
    m.impl("balance_loss_backward", balance_loss_backward_meta);
}
TORCH_LIBRARY_IMPL(umr, AutocastCUDA, m) { m.impl("linear_act", linear_act_autocast); }
TORCH_LIBRARY_IMPL(umr, Autograd, m) {
    m.impl("linear_act", linear_act_autograd);
    m.impl("linear_act_backward", linear_act_backward_once);
    m.impl("balance_loss", balance_loss_autograd);
    m.impl("balance_loss_backward", balance_loss_backward_once);
}

extern "C" const char *umr_torch_build_id(void) { return UMR_SRC_HASH; }
