// The torch side of the calls around the routed experts: argument checks, outputs, streams and gradients in front of the C entry points.
//
// A call through ctypes and a Python autograd function costs the host 10 to 14 us, a backward pass 100; the kernels of a decode step take 2 to 6.  From here
// a call costs 4.5 to 5.5, forward and backward together 50 to 54, of which torch's engine has most (its own exp and the gradient: 49).  Nothing here computes: every function makes its outputs and calls libnestquant_b200.so on the current stream of the
// tensors' device.  Errors are thrown as nestquant_b200.capi.NestQuantError before anything is enqueued.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../include/nestquant_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };

template <class... A>
[[noreturn]] void refuse(const A&... a) { throw Error(c10::str(a...)); }
#define NQ_CHECK(cond, ...) do { if (!(cond)) refuse(__VA_ARGS__); } while (0)

void check(int rc, const char* what)
{
    if (rc != NQ_OK) refuse(what, " failed (", rc, "): ", nq_last_error());
}
int type_of(at::ScalarType t, const char* what)
{
    if (t == at::kFloat) return NQ_F32;
    if (t == at::kHalf) return NQ_F16;
    NQ_CHECK(t == at::kBFloat16, what, ": ", t, " (fp32, fp16 or bf16)");
    return NQ_BF16;
}
void on_gpu(const Tensor& t, int64_t dims, const char* what)
{
    NQ_CHECK(t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.dim() == dims, what, ": expected a CUDA tensor of ", dims, " dimensions");
}
void same_device(const Tensor& a, const Tensor& b, const char* what) { NQ_CHECK(a.device() == b.device(), what, ": tensors on different devices"); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
// t, or a copy, whose rows are contiguous and do not overlap
Tensor strided(const Tensor& t) { return t.numel() == 0 || (t.stride(1) == 1 && t.stride(0) >= t.size(1)) ? t : t.contiguous(); }
int64_t stride_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
bool wants_grad(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }
// forward-mode derivatives are not built; without this a dual tensor's would be lost without a word, as if they were 0
void no_tangent(const Tensor& t, const char* what) { NQ_CHECK(!t._fw_grad(/*level=*/0).defined(), what, ": no forward-mode derivative (unpack the dual tensor)"); }
// gradients that say so when somebody wants to differentiate them
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    const int n = (int)grads.size();
    for (Tensor& g : grads)
        if (g.defined()) g.requires_grad_(true);
    return (*std::make_shared<torch::autograd::DelayedError>("nestquant_b200: gradients of gradients are not built", n))(std::move(grads));
}

// ---- route ----------------------------------------------------------------------------------------------------------------------

struct RouteHow { int64_t topk, score; bool renorm; double scale; at::ScalarType dtype; };

std::tuple<Tensor, Tensor> route_now(const Tensor& logits, const c10::optional<Tensor>& bias, const RouteHow& h)
{
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t T = logits.size(0), E = logits.size(1);
    Tensor sel = at::empty({T, h.topk}, logits.options().dtype(at::kLong)), rw = at::empty({T, h.topk}, logits.options().dtype(h.dtype));
    check(nq_route(logits.data_ptr(), type_of(logits.scalar_type(), "route"), stride_of(logits), bias ? bias->data_ptr<float>() : nullptr, (int)T, (int)E, (int)h.topk,
                   (int)h.score, h.renorm, (float)h.scale, sel.data_ptr<int64_t>(), rw.data_ptr(), type_of(h.dtype, "route"), stream_of(logits)), "route");
    return {sel, rw};
}

struct Route : torch::autograd::Function<Route> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const c10::optional<Tensor>& bias, RouteHow h)
    {
        auto [sel, rw] = route_now(logits, bias, h);
        ctx->save_for_backward({logits, sel});
        ctx->saved_data["topk"] = h.topk;
        ctx->saved_data["score"] = h.score;
        ctx->saved_data["renorm"] = h.renorm;
        ctx->saved_data["scale"] = h.scale;
        ctx->mark_non_differentiable({sel});
        ctx->set_materialize_grads(false);               // (zeros for sel would be a launch)
        return {sel, rw};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        if (!grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
        const variable_list saved = ctx->get_saved_variables();
        const Tensor logits = saved[0].detach(), &sel = saved[1], drw = grads[1].detach().contiguous();
        const c10::cuda::CUDAGuard guard(logits.device());
        Tensor grad = at::empty(logits.sizes(), logits.options());
        check(nq_route_bwd(logits.data_ptr(), type_of(logits.scalar_type(), "route"), stride_of(logits), sel.data_ptr<int64_t>(), drw.data_ptr(),
                           type_of(drw.scalar_type(), "route"), (int)logits.size(0), (int)logits.size(1), (int)ctx->saved_data["topk"].toInt(),
                           (int)ctx->saved_data["score"].toInt(), ctx->saved_data["renorm"].toBool(), (float)ctx->saved_data["scale"].toDouble(), grad.data_ptr(),
                           stream_of(logits)), "route backward");
        return once({grad, Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor> route(const Tensor& logits_, int64_t topk, const std::string& score, const c10::optional<Tensor>& bias, bool renorm, double scale, at::ScalarType dtype)
{
    on_gpu(logits_, 2, "route: logits");
    const int64_t E = logits_.size(1);
    type_of(logits_.scalar_type(), "route: logits");
    type_of(dtype, "route: weights");
    no_tangent(logits_, "route: logits");
    NQ_CHECK(score == "sigmoid" || score == "softmax", "route: score ", score, " (sigmoid, softmax)");
    NQ_CHECK(topk >= 1 && topk <= E && topk <= 32 && E <= 1024, "route: ", topk, " picks of ", E, " experts (to 32 of 1024)");
    NQ_CHECK(logits_.size(0) <= 0x7fffffff, "route: too many tokens");
    if (bias)
    {
        NQ_CHECK(score == "sigmoid", "route: a bias goes with sigmoid scores");
        on_gpu(*bias, 1, "route: bias");
        NQ_CHECK(bias->scalar_type() == at::kFloat && bias->size(0) == E && bias->is_contiguous(), "route: bias, expected contiguous fp32 [", E, "]");
        NQ_CHECK(!wants_grad(*bias), "route: the bias has no gradient (detach it)");
        no_tangent(*bias, "route: bias");
        same_device(logits_, *bias, "route");
    }
    const Tensor logits = strided(logits_);
    const RouteHow h{topk, score == "softmax", renorm, scale, dtype};
    if (!wants_grad(logits)) return route_now(logits, bias, h);
    variable_list r = Route::apply(logits, bias, h);
    return {r[0], r[1]};
}

// ---- rows by expert and back ----------------------------------------------------------------------------------------------------

// The picks of a call sorted by expert: one buffer of int32, start [E + 2], then pos [P], then the sort's scratch.  Expert and token of each place are
// worked out when they are asked for: no call needs them, and in the sort they are scattered stores.
struct Order : torch::CustomClassHolder {
    int64_t T, topk, E;
    Tensor buf;
    int64_t P() const { return T * topk; }
    Tensor start() const { return buf.as_strided({E + 1}, {1}, 0); }
    Tensor pos() const { return buf.as_strided({T, topk}, {topk, 1}, E + 2); }
    Tensor token() const
    {
        const c10::cuda::CUDAGuard guard(buf.device());
        const Tensor picks = at::arange(P(), buf.options());
        return at::empty_like(picks).scatter_(0, pos().flatten().to(at::kLong), at::floor_divide(picks, topk));
    }
    Tensor expert() const
    {
        const c10::cuda::CUDAGuard guard(buf.device());
        return at::bucketize(at::arange(P(), buf.options()), buf.narrow(0, 1, E), /*out_int32=*/true, /*right=*/true);
    }
    const int32_t* live_ptr() const { return buf.data_ptr<int32_t>() + E; }
    const int32_t* pos_ptr() const { return buf.data_ptr<int32_t>() + E + 2; }
};
using OrderPtr = c10::intrusive_ptr<Order>;
// An order that a backward pass needs.  start and pos are views that a caller can write to: one that was written to since is no longer what the forward pass went
// by (torch counts the writes; not to a tensor of inference mode, which cannot be told).
void keep(AutogradContext* ctx, const OrderPtr& o)
{
    ctx->saved_data["order"] = c10::IValue::make_capsule(o);
    ctx->saved_data["version"] = o->buf.is_inference() ? int64_t(-1) : (int64_t)o->buf._version();
}
OrderPtr kept(AutogradContext* ctx, const char* what)
{
    const auto o = c10::static_intrusive_pointer_cast<Order>(ctx->saved_data["order"].toCapsule());
    const int64_t version = ctx->saved_data["version"].toInt();
    NQ_CHECK(version < 0 || version == (int64_t)o->buf._version(), what, ": the order's start or pos was changed behind the backward pass");
    return o;
}

OrderPtr sort_picks(const Tensor& sel_, int64_t E)
{
    on_gpu(sel_, 2, "sort_picks: sel");
    NQ_CHECK(sel_.scalar_type() == at::kLong, "sort_picks: sel, expected int64");
    const int64_t T = sel_.size(0), topk = sel_.size(1);
    NQ_CHECK(E >= 1 && E <= 1024 && topk >= 1 && 2 * T * topk + E + 2 <= 0x7fffffff, "sort_picks: ", T, " x ", topk, " picks of ", E, " experts (to 1024)");
    const int ints = nq_pf_sort_scratch_ints((int)(T * topk), (int)E);
    NQ_CHECK(ints > 0 || T == 0, "sort_picks: counts of ", T, " x ", topk, " picks and ", E, " experts are more than an array can hold");
    const c10::cuda::CUDAGuard guard(sel_.device());
    const Tensor sel = sel_.contiguous();
    auto o = c10::make_intrusive<Order>();
    o->T = T; o->topk = topk; o->E = E;
    o->buf = at::empty({E + 2 + T * topk + std::max(ints, 1)}, sel.options().dtype(at::kInt));
    int32_t *start = o->buf.data_ptr<int32_t>(), *pos = start + E + 2, *scratch = pos + T * topk;
    check(nq_sort_picks(sel.data_ptr<int64_t>(), (int)T, (int)topk, (int)E, nullptr, nullptr, pos, start, scratch, std::max(ints, 1), stream_of(sel)), "sort_picks");
    return o;
}

Tensor dispatch_now(const Tensor& x, const Order& o)
{
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor xs = at::empty({o.P(), x.size(1)}, x.options());
    check(nq_dispatch(x.data_ptr(), type_of(x.scalar_type(), "dispatch"), stride_of(x), o.pos_ptr(), o.live_ptr(), (int)o.T, (int)o.topk, (int)x.size(1), xs.data_ptr(), stream_of(x)),
          "dispatch");
    return xs;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, OrderPtr o)
    {
        keep(ctx, o);
        return dispatch_now(x, *o);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const OrderPtr held = kept(ctx, "dispatch backward");
        const Order& o = *held;
        const Tensor dxs = grads[0].detach().contiguous();
        const c10::cuda::CUDAGuard guard(dxs.device());
        Tensor dx = at::empty({o.T, dxs.size(1)}, dxs.options());
        check(nq_dispatch_bwd(dxs.data_ptr(), type_of(dxs.scalar_type(), "dispatch"), o.pos_ptr(), o.live_ptr(), (int)o.T, (int)o.topk, (int)dxs.size(1), dx.data_ptr(), stream_of(dxs)),
              "dispatch backward");
        return once({dx, Tensor()});
    }
};

Tensor dispatch(const Tensor& x_, const OrderPtr& o)
{
    on_gpu(x_, 2, "dispatch: x");
    type_of(x_.scalar_type(), "dispatch: x");
    no_tangent(x_, "dispatch: x");
    NQ_CHECK(x_.size(0) == o->T && x_.size(1) >= 1 && x_.size(1) <= 0x7fffffff, "dispatch: x ", x_.sizes(), ", an order of ", o->T, " tokens");
    same_device(x_, o->buf, "dispatch");
    const Tensor x = strided(x_);
    return wants_grad(x) ? Dispatch::apply(x, o) : dispatch_now(x, *o);
}

Tensor combine_now(const Tensor& y, const Tensor& rw, const Order& o, at::ScalarType dtype)
{
    const c10::cuda::CUDAGuard guard(y.device());
    Tensor out = at::empty({o.T, y.size(1)}, y.options().dtype(dtype));
    check(nq_combine(y.data_ptr(), type_of(y.scalar_type(), "combine"), rw.data_ptr(), type_of(rw.scalar_type(), "combine"), o.pos_ptr(), o.live_ptr(), (int)o.T, (int)o.topk,
                     (int)y.size(1), out.data_ptr(), type_of(dtype, "combine"), stream_of(y)), "combine");
    return out;
}

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& rw, OrderPtr o, at::ScalarType dtype)
    {
        ctx->save_for_backward({y, rw});
        keep(ctx, o);
        return combine_now(y, rw, *o, dtype);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &y = saved[0], &rw = saved[1], dout = grads[0].detach().contiguous();
        const OrderPtr held = kept(ctx, "combine backward");
        const Order& o = *held;
        const c10::cuda::CUDAGuard guard(y.device());
        Tensor dy, drw;
        if (ctx->needs_input_grad(0)) dy = at::empty(y.sizes(), y.options());
        if (ctx->needs_input_grad(1)) drw = at::empty(rw.sizes(), rw.options());
        check(nq_combine_bwd(dout.data_ptr(), type_of(dout.scalar_type(), "combine"), y.data_ptr(), type_of(y.scalar_type(), "combine"), rw.data_ptr(),
                             type_of(rw.scalar_type(), "combine"), o.pos_ptr(), o.live_ptr(), (int)o.T, (int)o.topk, (int)y.size(1), dy.defined() ? dy.data_ptr() : nullptr,
                             drw.defined() ? drw.data_ptr() : nullptr, stream_of(y)), "combine backward");
        return once({dy, drw, Tensor(), Tensor()});
    }
};

Tensor combine(const Tensor& y_, const OrderPtr& o, const Tensor& rw_, const c10::optional<at::ScalarType>& dtype_)
{
    on_gpu(y_, 2, "combine: y");
    on_gpu(rw_, 2, "combine: rw");
    type_of(y_.scalar_type(), "combine: y");
    type_of(rw_.scalar_type(), "combine: rw");
    no_tangent(y_, "combine: y");
    no_tangent(rw_, "combine: rw");
    const at::ScalarType dtype = dtype_.value_or(y_.scalar_type());
    NQ_CHECK(y_.size(0) == o->P() && y_.size(1) >= 1 && y_.size(1) <= 0x7fffffff && rw_.size(0) == o->T && rw_.size(1) == o->topk, "combine: y ", y_.sizes(), ", rw ", rw_.sizes(),
             ", an order of ", o->T, " x ", o->topk, " picks");
    NQ_CHECK(dtype == y_.scalar_type() || dtype == at::kFloat, "combine: ", y_.scalar_type(), " rows as ", dtype, " (their own type, or fp32)");
    same_device(y_, o->buf, "combine");
    same_device(y_, rw_, "combine");
    const Tensor y = y_.contiguous(), rw = rw_.contiguous();
    return wants_grad(y) || wants_grad(rw) ? Combine::apply(y, rw, o, dtype) : combine_now(y, rw, *o, dtype);
}

// ---- 4-bit products -------------------------------------------------------------------------------------------------------------

// planes of one matrix, or of one per expert (see nq_w4_layout)
struct W4Planes : torch::CustomClassHolder {
    Tensor qw, sc, zp, status;
    int64_t E, N, K, group;
    bool experts;
};
using W4Ptr = c10::intrusive_ptr<W4Planes>;

bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

W4Ptr w4_planes(const Tensor& q_, const Tensor& scales_, const c10::optional<Tensor>& zeros_)
{
    NQ_CHECK(q_.is_cuda() && q_.scalar_type() == at::kByte && scales_.is_cuda() && half_type(scales_.scalar_type()), "W4: q uint8, scales fp16 or bf16, on the GPU");
    NQ_CHECK((q_.dim() == 2 || q_.dim() == 3) && scales_.dim() == q_.dim() && q_.sizes().slice(0, q_.dim() - 1) == scales_.sizes().slice(0, q_.dim() - 1) && q_.numel() && scales_.numel(),
             "W4: q ", q_.sizes(), ", scales ", scales_.sizes(), ": expected [..,N,K/2] and [..,N,K/group]");
    auto w = c10::make_intrusive<W4Planes>();
    w->experts = q_.dim() == 3;
    w->E = w->experts ? q_.size(0) : 1;
    w->N = q_.size(-2);
    w->K = 2 * q_.size(-1);
    w->group = w->K / scales_.size(-1);
    NQ_CHECK((w->group == 32 || w->group == 64 || w->group == 128) && w->group * scales_.size(-1) == w->K, "W4: ", w->K, " columns with ", scales_.size(-1),
             " scales a row: groups are of 32, 64 or 128 columns");
    same_device(q_, scales_, "W4");
    if (zeros_)
    {
        NQ_CHECK(zeros_->is_cuda() && zeros_->scalar_type() == at::kByte && zeros_->sizes() == scales_.sizes(), "W4: zeros, expected uint8 ", scales_.sizes(), " on the GPU");
        same_device(q_, *zeros_, "W4");
    }
    NQ_CHECK(w->N <= 0x7fffffff && w->K <= 0x7fffffff, "W4: too large");
    int64_t units;
    check(nq_w4_units((int)w->E, (int)w->N, (int)w->K, &units), "W4");
    const c10::cuda::CUDAGuard guard(q_.device());
    Tensor q = q_.contiguous();
    if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 2) q = q.clone();       // (read two bytes at a time)
    const Tensor scales = scales_.contiguous(), zeros = zeros_ ? zeros_->contiguous() : Tensor();
    const int64_t per = 16 * (128 / w->group);
    w->qw = at::empty({units * 1024}, q.options());
    w->sc = at::empty({units * per}, scales.options());
    if (zeros.defined()) w->zp = at::empty({units * per}, q.options());
    w->status = at::zeros({1}, q.options().dtype(at::kInt));
    check(nq_w4_layout(q.data_ptr(), scales.data_ptr(), zeros.defined() ? zeros.data_ptr() : nullptr, (int)w->E, (int)w->N, (int)w->K, (int)w->group, w->qw.data_ptr(), w->sc.data_ptr(),
                       zeros.defined() ? w->zp.data_ptr() : nullptr, stream_of(q)), "W4");
    return w;
}

Tensor w4_matmul(const W4Ptr& w, const Tensor& x_, const c10::optional<Tensor>& start, const c10::optional<at::ScalarType>& dtype_)
{
    on_gpu(x_, 2, "W4: x");
    const at::ScalarType own = x_.scalar_type(), dtype = dtype_.value_or(own);
    NQ_CHECK(half_type(own) && x_.size(1) == w->K && (dtype == own || dtype == at::kFloat), "W4: x ", x_.sizes(), " of ", own, " as ", dtype, ", a matrix of ", w->K,
             " columns (x fp16 or bf16, result in x's own type or fp32)");
    same_device(x_, w->qw, "W4: x and the weights");
    NQ_CHECK(!wants_grad(x_), "W4: no gradient (detach x, or call under torch.no_grad)");
    no_tangent(x_, "W4: x");
    NQ_CHECK(w->experts == start.has_value(), "W4: start goes with one matrix per expert, and only with that");
    if (start)
    {
        on_gpu(*start, 1, "W4: start");
        NQ_CHECK(start->scalar_type() == at::kInt && start->is_contiguous() && start->numel() > w->E, "W4: start, expected contiguous int32 [", w->E + 1, "]");
        same_device(x_, *start, "W4");
    }
    const int64_t T = x_.size(0);
    NQ_CHECK(T <= 0x7fffffff, "W4: too many rows");
    const c10::cuda::CUDAGuard guard(x_.device());
    Tensor x = x_;
    int64_t rows = T > 1 ? x.stride(0) : w->K;
    if (x.stride(1) != 1 || rows < w->K || rows % 8 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16)
    {
        x = x.clone(at::MemoryFormat::Contiguous);       // rows that the kernel reads start on 16 bytes
        rows = w->K;
    }
    Tensor out = at::empty({T, w->N}, x.options().dtype(dtype));
    check(nq_w4_matmul(x.data_ptr(), type_of(own, "W4"), rows, w->qw.data_ptr(), w->sc.data_ptr(), type_of(w->sc.scalar_type(), "W4"), w->zp.defined() ? w->zp.data_ptr() : nullptr,
                       start ? start->data_ptr<int32_t>() : nullptr, (int)T, (int)w->E, (int)w->N, (int)w->K, (int)w->group, out.data_ptr(), type_of(dtype, "W4"), w->N,
                       w->status.data_ptr<int32_t>(), stream_of(x)), "W4");
    return out;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m)
{
    static py::object error = py::module_::import("nestquant_b200.capi").attr("NestQuantError");
    py::register_exception_translator([](std::exception_ptr p) {
        try { if (p) std::rethrow_exception(p); }
        catch (const Error& e) { PyErr_SetString(error.ptr(), e.what()); }
    });
    py::class_<Order, OrderPtr>(m, "Order",
        "The picks of a call sorted by expert (sort_picks).  int32 tensors on the device: start [E+1], first place of each expert's picks (start[E]: where the\n"
        "picks without an expert begin); pos [T,topk], place of each pick; expert [P] (E: none) and token [P] of each place, P = T * topk.  start and pos are the\n"
        "order itself: a backward pass raises if they were written to since the forward pass.")
        .def_readonly("T", &Order::T).def_readonly("topk", &Order::topk).def_readonly("E", &Order::E).def_property_readonly("P", &Order::P)
        .def_property_readonly("start", &Order::start).def_property_readonly("pos", &Order::pos)
        .def_property_readonly("expert", &Order::expert).def_property_readonly("token", &Order::token);
    py::class_<W4Planes, W4Ptr>(m, "W4Planes")
        .def_readonly("qw", &W4Planes::qw).def_readonly("sc", &W4Planes::sc).def_readonly("status", &W4Planes::status)
        .def_property_readonly("zp", [](const W4Planes& w) { return w.zp.defined() ? c10::optional<Tensor>(w.zp) : c10::nullopt; })
        .def_readonly("E", &W4Planes::E).def_readonly("N", &W4Planes::N).def_readonly("K", &W4Planes::K).def_readonly("group", &W4Planes::group).def_readonly("experts", &W4Planes::experts);
    m.def("route", &route);
    m.def("sort_picks", &sort_picks);
    m.def("dispatch", &dispatch);
    m.def("combine", &combine);
    m.def("w4_planes", &w4_planes);
    m.def("w4_matmul", &w4_matmul);
}
