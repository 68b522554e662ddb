// pss_torch.cpp -- torch binding of the batch-row operators: argument checks, outputs and autograd
// nodes around the C entries of include/pss.h (module _pss_torch; ops.py is the public face).
//
// The rest of the package binds the C ABI with ctypes.  These calls sit inside a training step, where
// a backward pass runs on autograd's own thread: the same node in Python costs 87 us for a forward and
// backward of 64 x 1024 values (39 of them the hand-over to that thread), most of it interpreter work on
// a second core, against 3 us of kernels.
//
// The entries come as addresses from _lib (bind()), so that the library it loaded is the one used.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/pss.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- the C entries -------------------------------------------------------------------------------
#define ENTRIES(F) \
    F(pss_last_error) F(pss_dropout) F(pss_route_workspace) F(pss_route) F(pss_route_grad) F(pss_dispatch) \
    F(pss_combine) F(pss_combine_grad) F(pss_gather_dropout)
struct Entries {
#define FIELD(name) decltype(&::name) name = nullptr;
    ENTRIES(FIELD)
#undef FIELD
} lib;

void bind(const std::map<std::string, uint64_t> &at) {
#define SET(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at(#name));
    ENTRIES(SET)
#undef SET
}

void check(int rc, const char *name) {
    TORCH_CHECK(rc == PSS_OK, name, " failed (code ", rc, "): ", lib.pss_last_error());
}

void *stream_of(const Tensor &t) {
    return (void *)at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// The entries work on memory, which a recorder of torch's own operations does not see: its graph would hold
// the allocation of an output and nothing that fills it.  (torch.compile runs these calls outside its graphs.)
void check_eager() {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    const bool recorded = torch::jit::tracer::isTracing() ||
                          c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                          TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) ||
                          TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) ||
                          TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL);
    TORCH_CHECK(!recorded, "the batch-row operators cannot be traced, exported or run on fake tensors");
}

// ---- arguments -----------------------------------------------------------------------------------
int32_t dtype_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PSS_F32;
        case at::kBFloat16: return PSS_BF16;
        case at::kHalf: return PSS_F16;
        default: return -1;
    }
}

void check_rows(const char *name, const Tensor &t) {
    TORCH_CHECK_TYPE(dtype_of(t) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, name, " must be a dense tensor");
}

void check_like(const char *name, const Tensor &t, const Tensor &like, at::IntArrayRef shape) {
    check_rows(name, t);
    TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type() && t.device() == like.device(), name,
                     " must have the dtype and device of the rows: ", like.scalar_type(), " on ", like.device(), ", got ",
                     t.scalar_type(), " on ", t.device());
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
}

void check_p(double p) { TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p); }

void check_ids(const Tensor &ids, int64_t n, const Tensor &like) {
    if (!ids.defined()) return;
    TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong && ids.device() == like.device(),
                     "rows must be an int, or an int64 tensor on the rows' device");
    TORCH_CHECK_VALUE(ids.numel() == 1 || ids.numel() == n,
                      "rows must hold one id (the first row's) or one per row (", n, "), got ", ids.numel());
}

// (an undefined tensor as an argument of a node's forward is none; needs_input_grad counts those given)
using Opt = std::optional<Tensor>;
Opt opt(const Tensor &t) { return t.defined() ? Opt(t) : Opt(); }
Tensor get(const Opt &t) { return t ? *t : Tensor(); }

// The values as they lie in memory: torch may hold a sign that is still to be applied (the imaginary part of a
// conjugate), which `contiguous` alone leaves as it is.
Tensor plain(const Tensor &t) { return t.resolve_neg().contiguous(); }

// Rows of [.., D], also where D is 0
int64_t rows_of(const Tensor &x) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < x.dim(); i++) n *= x.size(i);
    return n;
}

// Rows [.., D]: as they are where they lie at one distance and a row's values are adjacent, else copied.
struct Rows {
    Tensor t;
    int64_t n, d, ld;
    explicit Rows(const Tensor &x_) {
        const Tensor x = x_.resolve_neg();
        if (x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1)) {
            t = x;
            n = x.size(0);
            d = x.size(1);
            ld = x.stride(0);
        } else {
            t = x.contiguous();
            d = x.dim() ? x.size(-1) : 1;
            n = rows_of(x);
            ld = d;
        }
    }
};

const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const int64_t *ids_ptr(const Tensor &t) { return (const int64_t *)ptr(t); }
int64_t ids_n(const Tensor &t) { return t.defined() ? t.numel() : 0; }

// The gradients of a backward pass that a graph is asked of: differentiating them again is an error (as
// torch's once_differentiable).
variable_list once(const variable_list &in, variable_list out) {
    if (!at::GradMode::is_enabled()) return out;
    bool any = false;
    for (const Tensor &t : in) any |= t.defined() && t.requires_grad();
    if (!any) return out;
    for (Tensor &t : out)
        if (t.defined()) t = t.detach().requires_grad_();
    return torch::autograd::DelayedError("the gradients of the batch-row operators cannot be differentiated again",
                                         (int64_t)out.size())(std::move(out));
}

// ---- dropout -------------------------------------------------------------------------------------
Tensor dropout_run(const Tensor &x, const Tensor &residual, double p, uint64_t key, int64_t row0, const Tensor &ids) {
    check_eager();
    const Rows r(x);
    Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    const Rows q(residual.defined() ? residual : r.t);
    const bool host = x.is_cpu();
    c10::OptionalDeviceGuard guard;
    if (!host) guard.reset_device(x.device());
    check(lib.pss_dropout(r.t.const_data_ptr(), r.ld, residual.defined() ? q.t.const_data_ptr() : nullptr, q.ld,
                          y.data_ptr(), r.n, r.d, dtype_of(x), p, key, row0, ids_ptr(ids), ids_n(ids), host,
                          host ? nullptr : stream_of(x)),
          "pss_dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Opt &residual, double p, int64_t key, int64_t row0,
                          const Opt &ids) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["key"] = key;
        ctx->saved_data["row0"] = row0;
        ctx->saved_data["residual"] = residual.has_value();
        ctx->save_for_backward({get(ids)});
        return dropout_run(x, get(residual), p, (uint64_t)key, row0, get(ids));
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        variable_list out(6);
        if (!g[0].defined()) return out;
        if (ctx->needs_input_grad(0))
            out[0] = dropout_run(g[0], Tensor(), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["key"].toInt(),
                                 ctx->saved_data["row0"].toInt(), ctx->get_saved_variables()[0]);
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = g[0];
        return once(g, std::move(out));
    }
};

Tensor dropout(const Tensor &x, double p, uint64_t key, int64_t row0, const Opt &ids,
               const Opt &residual) {
    check_p(p);
    check_rows("x", x);
    TORCH_CHECK_VALUE(x.dim() > 0, "x must have rows [..., D]");
    TORCH_CHECK_TYPE(x.is_cpu() || x.is_cuda(), "x must be on the CPU or a ROCm GPU");
    if (residual) check_like("residual", *residual, x, x.sizes());
    Tensor i;
    if (ids) {
        check_ids(*ids, rows_of(x), x);
        i = ids->reshape({-1}).contiguous();
    }
    return Dropout::apply(x, residual, p, (int64_t)key, row0, opt(i));
}

// ---- gather with dropout -------------------------------------------------------------------------
// Rows of device-resident files (IndexEngine.gather with p > 0): `device` is the handle's.  No autograd node.
Tensor gather(uint64_t handle, const at::Device &device, int64_t files, const Tensor &data, const Tensor &base_rows_,
              const Tensor &fpos_, const Tensor &off_, const Opt &out_, double p, uint64_t key, int64_t row0,
              const Opt &ids_) {
    check_eager();
    check_p(p);
    TORCH_CHECK_TYPE(dtype_of(data) >= 0, "gather with dropout needs float32, bfloat16 or float16 data, got ",
                     data.scalar_type());
    TORCH_CHECK_VALUE(data.device() == device && data.is_contiguous() && data.dim() > 0,
                      "gather: data must be contiguous rows on the engine's device");
    TORCH_CHECK(!at::GradMode::is_enabled() || !(data.requires_grad() || (out_ && out_->requires_grad())),
                "gather has no gradient: data and out must not require one (index the rows and call ops.dropout, or "
                "gather under torch.no_grad)");
    const Tensor fpos = fpos_.reshape({-1}).contiguous(), off = off_.reshape({-1}).to(at::kInt).contiguous();
    const Tensor base = base_rows_.to(device, at::kLong).contiguous();
    const int64_t n = fpos.numel(), values = data.size(0) ? data.numel() / data.size(0) : 0;
    TORCH_CHECK_VALUE(fpos.scalar_type() == at::kInt && fpos.device() == device && off.device() == device,
                      "gather: file_pos and offset must be int32 on the engine's device");
    TORCH_CHECK_VALUE(off.numel() == n && base.numel() >= files,
                      "gather: file_pos and offset must be of one length, base_rows must have an entry for each of the ",
                      files, " files");
    Tensor out = get(out_), ids = get(ids_);
    if (out.defined()) {
        TORCH_CHECK_VALUE(out.is_contiguous() && !out.is_neg() && out.scalar_type() == data.scalar_type() && out.device() == device &&
                              out.numel() >= n * values,
                          "gather: out must be contiguous, of the data's dtype, on the engine's device");
    } else {
        auto sizes = data.sizes().vec();
        sizes[0] = n;
        out = at::empty(sizes, data.options());
    }
    check_ids(ids, n, data);
    if (ids.defined()) ids = ids.reshape({-1}).contiguous();
    const Tensor rows = data.resolve_neg();
    check(lib.pss_gather_dropout((pss_sampler *)handle, rows.const_data_ptr(), dtype_of(data), values,
                                 base.const_data_ptr<int64_t>(), fpos.const_data_ptr<int32_t>(),
                                 off.const_data_ptr<int32_t>(), n, p, key, row0, ids_ptr(ids), ids_n(ids),
                                 out.data_ptr(), data.is_cpu() ? nullptr : stream_of(data)),
          "pss_gather_dropout");
    if (out_ && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();     // (written in place)
    return out;
}

// ---- routing -------------------------------------------------------------------------------------
struct Route : torch::autograd::Function<Route> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, int64_t k, int64_t score, const Opt &bias,
                                 const Opt &valid, int64_t groups, int64_t top_groups, int64_t group_sum, bool renorm,
                                 double scale) {
        check_eager();
        const Rows r(logits);
        const auto i32 = logits.options().dtype(at::kInt);
        c10::DeviceGuard guard(logits.device());
        Tensor experts = at::empty({r.n, k}, i32), weights = at::empty({r.n, k}, logits.options().dtype(at::kFloat));
        Tensor offsets = at::empty({r.d + 1}, i32), pos = at::empty({r.n, k}, i32), src = at::empty({r.n * k}, i32);
        const int64_t need = lib.pss_route_workspace(r.n, (int32_t)r.d);
        Tensor ws, slopes;
        if (need) ws = at::empty({need}, logits.options().dtype(at::kByte));
        const bool grad = logits.requires_grad();
        if (grad && score == PSS_SIGMOID) slopes = at::empty({r.n, k}, weights.options());
        check(lib.pss_route(r.t.const_data_ptr(), r.ld, r.n, (int32_t)r.d, (int32_t)k, dtype_of(logits), (int32_t)score,
                            (const float *)ptr(get(bias)), (const uint8_t *)ptr(get(valid)), (int32_t)groups,
                            (int32_t)top_groups, (int32_t)group_sum, renorm, scale, experts.data_ptr<int32_t>(),
                            weights.data_ptr<float>(), slopes.defined() ? slopes.data_ptr<float>() : nullptr,
                            offsets.data_ptr<int32_t>(), pos.data_ptr<int32_t>(), src.data_ptr<int32_t>(),
                            need ? ws.data_ptr() : nullptr, need, stream_of(logits)),
              "pss_route");
        ctx->mark_non_differentiable({experts, offsets, pos, src});
        ctx->set_materialize_grads(false);
        if (grad) {
            ctx->saved_data["score"] = score;
            ctx->saved_data["renorm"] = renorm;
            ctx->saved_data["scale"] = scale;
            ctx->saved_data["experts"] = r.d;
            ctx->saved_data["dtype"] = (int64_t)logits.scalar_type();
            ctx->save_for_backward({score == PSS_SOFTMAX && !renorm ? logits : Tensor(), experts, weights, slopes});
        }
        return {experts, weights, offsets, pos, src};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        variable_list out(10);
        if (!g[1].defined() || !ctx->needs_input_grad(0)) return out;
        check_eager();
        const auto saved = ctx->get_saved_variables();
        const Tensor &experts = saved[1], &weights = saved[2], &slopes = saved[3];
        const int64_t n = experts.size(0), k = experts.size(1), e = ctx->saved_data["experts"].toInt();
        const Tensor dw = plain(g[1]);
        c10::DeviceGuard guard(dw.device());
        out[0] = at::empty({n, e}, weights.options().dtype((at::ScalarType)ctx->saved_data["dtype"].toInt()));
        const Rows r(saved[0].defined() ? saved[0] : out[0]);
        check(lib.pss_route_grad(r.t.const_data_ptr(), r.ld, n, (int32_t)e, (int32_t)k, dtype_of(out[0]),
                                 (int32_t)ctx->saved_data["score"].toInt(), ctx->saved_data["renorm"].toBool(),
                                 ctx->saved_data["scale"].toDouble(), experts.const_data_ptr<int32_t>(),
                                 weights.const_data_ptr<float>(), (const float *)ptr(slopes),
                                 dw.const_data_ptr<float>(), out[0].data_ptr(), stream_of(dw)),
              "pss_route_grad");
        return once(g, std::move(out));
    }
};

variable_list route(const Tensor &logits, int64_t k, int64_t score, const Opt &bias,
                    const Opt &valid, int64_t groups, int64_t top_groups, int64_t group_sum, bool renorm,
                    double scale) {
    check_rows("logits", logits);
    TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be [T, E], got ", logits.sizes());
    TORCH_CHECK(logits.is_cuda(), "route needs its logits on a ROCm GPU (no CPU fallback)");
    const int64_t n = logits.size(0), e = logits.size(1);
    // (the entry checks the numbers; here only what would not fit its 32-bit arguments, or an allocation)
    TORCH_CHECK(e <= 1024 && k >= 1 && k <= 16 && k <= e, "route: 1 <= k <= experts, at most 1024 experts, 16 of them for a row");
    for (int64_t v : {groups, top_groups, group_sum}) TORCH_CHECK(v >= 1 && v <= 1024, "route: groups, top_groups or group_sum is out of range");
    Tensor b, v;
    if (bias) {
        TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->device() == logits.device() && bias->dim() == 1 &&
                              bias->size(0) == e,
                          "bias must be float32 [", e, "] on the logits' device");
        b = plain(bias->detach());
    }
    if (valid) {
        TORCH_CHECK_VALUE(valid->scalar_type() == at::kBool && valid->device() == logits.device() && valid->dim() == 1 &&
                              valid->size(0) == n,
                          "valid must be bool [", n, "] on the logits' device");
        v = valid->contiguous();
    }
    return Route::apply(logits, k, score, opt(b), opt(v), groups, top_groups, group_sum, renorm, scale);
}

// ---- dispatch and combine ------------------------------------------------------------------------
// (T, k) of a plan's tensors
std::pair<int64_t, int64_t> check_plan(const Tensor &experts, const Tensor &pos, const Tensor &like) {
    for (const auto &[name, t] : {std::pair<const char *, const Tensor &>("experts", experts), {"pos", pos}})
        TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.device() == like.device() && t.is_contiguous(),
                          "routing.", name, " must be contiguous int32 [T, k] on the rows' device");
    TORCH_CHECK_VALUE(pos.sizes() == experts.sizes(), "routing.pos and routing.experts differ in shape");
    return {pos.size(0), pos.size(1)};
}

Tensor combine_run(const Tensor &y_, const Tensor &experts, const Tensor &pos, const Tensor &w, const Tensor &residual,
                   double p, uint64_t key, int64_t row0, const Tensor &ids) {
    check_eager();
    const Tensor y = plain(y_);
    const int64_t n = pos.size(0), k = pos.size(1), d = y.size(1);
    c10::DeviceGuard guard(y.device());
    Tensor out = at::empty({n, d}, y.options());
    const Rows q(residual.defined() ? residual : y);
    check(lib.pss_combine(y.const_data_ptr(), n, (int32_t)k, d, dtype_of(y), experts.const_data_ptr<int32_t>(),
                          pos.const_data_ptr<int32_t>(), (const float *)ptr(w),
                          residual.defined() ? q.t.const_data_ptr() : nullptr, q.ld, p, key, row0, ids_ptr(ids),
                          ids_n(ids), out.data_ptr(), stream_of(y)),
          "pss_combine");
    return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &experts, const Tensor &pos) {
        check_eager();
        const Rows r(x);
        const int64_t k = pos.size(1);
        c10::DeviceGuard guard(x.device());
        Tensor xs = at::empty({r.n * k, r.d}, x.options());
        check(lib.pss_dispatch(r.t.const_data_ptr(), r.ld, r.n, (int32_t)k, r.d, dtype_of(x),
                               experts.const_data_ptr<int32_t>(), pos.const_data_ptr<int32_t>(), xs.data_ptr(),
                               stream_of(x)),
              "pss_dispatch");
        ctx->save_for_backward({experts, pos});
        return xs;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        variable_list out(3);
        if (!g[0].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        out[0] = combine_run(g[0], saved[0], saved[1], Tensor(), Tensor(), 0.0, 0, 0, Tensor());
        return once(g, std::move(out));
    }
};

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &w, const Opt &residual,
                          const Tensor &experts, const Tensor &pos, double p, int64_t key, int64_t row0, const Opt &ids) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["key"] = key;
        ctx->saved_data["row0"] = row0;
        ctx->saved_data["residual"] = residual.has_value();
        ctx->save_for_backward({y, w, experts, pos, get(ids)});
        return combine_run(y, experts, pos, w, get(residual), p, (uint64_t)key, row0, get(ids));
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        variable_list out(9);
        if (!g[0].defined()) return out;
        const bool want_y = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        if (want_y || want_w) {
            check_eager();
            const auto saved = ctx->get_saved_variables();
            const Tensor y = plain(saved[0]), &w = saved[1], &experts = saved[2], &pos = saved[3], &ids = saved[4];
            const Rows r(g[0]);
            const int64_t n = pos.size(0), k = pos.size(1);
            c10::DeviceGuard guard(y.device());
            if (want_y) out[0] = at::empty(y.sizes(), y.options());
            if (want_w) out[1] = at::empty({n, k}, w.options());
            check(lib.pss_combine_grad(r.t.const_data_ptr(), r.ld, y.const_data_ptr(), n, (int32_t)k, r.d, dtype_of(y),
                                       experts.const_data_ptr<int32_t>(), pos.const_data_ptr<int32_t>(),
                                       w.const_data_ptr<float>(), ctx->saved_data["p"].toDouble(),
                                       (uint64_t)ctx->saved_data["key"].toInt(), ctx->saved_data["row0"].toInt(),
                                       ids_ptr(ids), ids_n(ids), want_y ? out[0].data_ptr() : nullptr,
                                       want_w ? out[1].data_ptr<float>() : nullptr, stream_of(y)),
                  "pss_combine_grad");
        }
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(2)) out[2] = g[0];
        return once(g, std::move(out));
    }
};

Tensor dispatch(const Tensor &x, const Tensor &experts, const Tensor &pos) {
    check_rows("x", x);
    TORCH_CHECK_VALUE(x.dim() == 2 && x.is_cuda(), "x must be [T, D] on a ROCm GPU");
    const auto [n, k] = check_plan(experts, pos, x);
    TORCH_CHECK_VALUE(x.size(0) == n, "the routing is of ", n, " rows, got ", x.size(0));
    (void)k;
    return Dispatch::apply(x, experts, pos);
}

Tensor combine(const Tensor &y, const Tensor &weights, const Tensor &experts, const Tensor &pos,
               const Opt &residual, double p, uint64_t key, int64_t row0, const Opt &ids) {
    check_p(p);
    check_rows("y", y);
    TORCH_CHECK_VALUE(y.dim() == 2 && y.is_cuda(), "y must be [T * k, D] on a ROCm GPU");
    const auto [n, k] = check_plan(experts, pos, y);
    TORCH_CHECK_VALUE(y.size(0) == n * k, "y must have the routing's ", n * k, " rows, got ", y.size(0));
    TORCH_CHECK_VALUE(weights.scalar_type() == at::kFloat && weights.sizes() == pos.sizes() && weights.device() == y.device(),
                      "routing.weights must be float32 [", n, ", ", k, "] on the rows' device");
    if (residual) check_like("residual", *residual, y, {n, y.size(1)});
    Tensor i;
    if (ids) {
        check_ids(*ids, n, y);
        i = ids->reshape({-1}).contiguous();
    }
    return Combine::apply(y, plain(weights), residual, experts, pos, p, (int64_t)key, row0, opt(i));
}

}  // namespace

PYBIND11_MODULE(_pss_torch, m) {
    m.def("bind", &bind);
    m.def("dropout", &dropout);
    m.def("gather", &gather);
    m.def("route", &route);
    m.def("dispatch", &dispatch);
    m.def("combine", &combine);
}
