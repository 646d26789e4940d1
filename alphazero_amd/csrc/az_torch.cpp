// az_torch.cpp -- autograd functions over the C ABI, and what else is asked of tensors at every step, for calls whose launches
// are shorter than Python's way to them: a step of the group norm at the shipped batch of 128 is 18 us on the device; its
// autograd function written in Python took 73 to 115 us a call on the host, this one 42 to 70 (of which the engine's own
// threads are 30).  Host code only; the entry points of libazhip.so are handed over as addresses (alphazero_amd/_lib.py), so
// that both sides use one library.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include "../../include/azhip.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct {
    decltype(&az_last_error) last_error;
    decltype(&az_group_norm_workspace_bytes) group_norm_workspace_bytes;
    decltype(&az_group_norm_act) group_norm_act;
    decltype(&az_group_norm_act_backward) group_norm_act_backward;
} az;

void check(int rc) { TORCH_CHECK(rc == 0, az.last_error()); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int32_t type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return AZ_F32;
        case at::kBFloat16: return AZ_BF16;
        case at::kHalf: return AZ_F16;
        default: TORCH_CHECK_TYPE(false, "float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

// channels last, without a copy where it is that already
Tensor last(const Tensor& t) { return t.dim() == 2 ? t.contiguous() : t.contiguous(at::MemoryFormat::ChannelsLast); }

// The kernels read memory only; what else a tensor can carry must not be lost without a word.
void plain(const Tensor& t) {
    if (!t.defined()) return;
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "group_norm_act has no forward-mode derivative on the GPU");
    TORCH_CHECK_NOT_IMPLEMENTED(t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch(),
                                "group_norm_act takes tensors with memory of their own on the GPU: no vmap, no functorch transforms");
}

// A launch goes past torch's dispatcher: a tracer would record the allocation of the result and nothing that fills it.
void untraced() {
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY) &&
                                    !TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::FAKE) &&
                                    !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
                                "group_norm_act cannot be traced on the GPU (torch.jit.trace, make_fx, torch.export, fake tensors)");
}

// `t` is what a kernel that goes by `like` takes it for
void same(const Tensor& t, const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == like.device(),
                "group_norm_act: a saved tensor came back as another one (", t.scalar_type(), t.sizes(), " on ", t.device(), "; it was ",
                type, sizes, " on ", like.device(), ")");
}

az_group_norm descriptor(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, double eps, int64_t act) {
    const int64_t cells = x.dim() == 4 ? x.size(2) * x.size(3) : 1;
    TORCH_CHECK_VALUE(x.size(0) <= INT32_MAX && cells <= INT32_MAX && x.size(1) <= INT32_MAX, "tensor too large");
    az_group_norm g{};
    g.batch = (int32_t)x.size(0); g.cells = (int32_t)cells; g.channels = (int32_t)x.size(1); g.groups = (int32_t)groups;
    g.dtype = type_of(x);
    g.param_dtype = weight.defined() ? type_of(weight) : bias.defined() ? type_of(bias) : AZ_F32;
    g.act = (int32_t)act; g.eps = eps;
    return g;
}

// one for each call, from torch's allocator: calls on several streams or in several captured graphs share nothing
Tensor workspace(const az_group_norm& g, int backward, const Tensor& x, int64_t& bytes) {
    bytes = az.group_norm_workspace_bytes(&g, backward);
    TORCH_CHECK(bytes >= 0, az.last_error());
    return bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor();
}

Tensor group_norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, const az_group_norm& g,
                          const Tensor& stats) {
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x);
    int64_t bytes;
    const Tensor ws = workspace(g, 0, x, bytes);
    check(az.group_norm_act(&g, ptr(x), ptr(weight), ptr(bias), ptr(residual), ptr(y), (double*)ptr(stats), ptr(ws), bytes, stream_of(x)));
    return y;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_,
                          const std::optional<Tensor>& residual_, int64_t groups, double eps, int64_t act) {
        const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
        const az_group_norm g = descriptor(x, weight, bias, groups, eps, act);
        const Tensor stats = at::empty({x.size(0), groups, 2}, x.options().dtype(at::kDouble).memory_format(at::MemoryFormat::Contiguous));
        Tensor y = group_norm_forward(x, weight, bias, residual, g, stats);
        ctx->save_for_backward({x, weight, bias, residual, stats});
        ctx->saved_data["groups"] = groups; ctx->saved_data["eps"] = eps; ctx->saved_data["act"] = act;
        int64_t needs = 0;
        const Tensor* leaves[] = {&x, &weight, &bias, &residual};
        for (int i = 0; i < 4; ++i) needs |= (int64_t)(leaves[i]->defined() && leaves[i]->requires_grad()) << i;
        ctx->saved_data["needs"] = needs;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &stats_ = saved[4], &dy_ = dys[0];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        const int64_t needs = ctx->saved_data["needs"].toInt();
        variable_list grads(7);
        {
            untraced();
            plain(dy_);
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(dy_.device());
            // a saved-tensor hook may have given the values back in another order of memory, or other tensors altogether
            const Tensor &x_ = saved[0], &w_ = saved[1], &b_ = saved[2], &r_ = saved[3];
            const int64_t channels = dy_.size(1);
            same(x_, dy_, dy_.sizes(), dy_.scalar_type());
            if (r_.defined()) same(r_, dy_, dy_.sizes(), dy_.scalar_type());
            for (const Tensor* t : {&w_, &b_})
                if (t->defined()) same(*t, dy_, {channels}, t->scalar_type() == at::kFloat ? at::kFloat : dy_.scalar_type());
            TORCH_CHECK(!w_.defined() || !b_.defined() || w_.scalar_type() == b_.scalar_type(), "group_norm_act: weight and bias of two types were saved");
            same(stats_, dy_, {dy_.size(0), groups, 2}, at::kDouble);
            const Tensor x = last(x_), residual = r_.defined() ? last(r_) : r_, weight = w_.defined() ? w_.contiguous() : w_,
                         bias = b_.defined() ? b_.contiguous() : b_, stats = stats_.contiguous(), dy = last(dy_);
            const az_group_norm g = descriptor(x, weight, bias, groups, ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt());
            const Tensor* inputs[] = {&x, &weight, &bias, &residual};
            for (int i = 0; i < 4; ++i)
                if (needs >> i & 1) grads[i] = at::empty_like(*inputs[i]);
            int64_t bytes;
            const Tensor ws = workspace(g, 1, x, bytes);
            check(az.group_norm_act_backward(&g, ptr(dy), ptr(x), ptr(weight), ptr(bias), ptr(residual), (const double*)ptr(stats),
                                             ptr(grads[0]), ptr(grads[1]), ptr(grads[2]), ptr(grads[3]), ptr(ws), bytes, stream_of(x)));
        }
        if (at::GradMode::is_enabled()) {
            // create_graph: whoever differentiates these gradients is told
            for (Tensor& t : grads)
                if (t.defined())
                    t = std::make_shared<torch::autograd::DelayedError>("group_norm_act: trying to differentiate twice", 1)->apply({t.requires_grad_()})[0];
        }
        return grads;
    }
};

// x and residual channels last, every argument checked (norm.py)
Tensor group_norm_act(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                      const std::optional<Tensor>& residual, int64_t groups, double eps, int64_t act) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    untraced();
    for (const Tensor* t : {&x, &w, &b, &r}) plain(*t);
    const bool grad = at::GradMode::is_enabled() &&
                      (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()) || (r.defined() && r.requires_grad()));
    if (grad) return GroupNormAct::apply(x, weight, bias, residual, groups, eps, act);
    return group_norm_forward(x, w, b, r, descriptor(x, w, b, groups, eps, act), Tensor());
}

// What FlatAdamW asks before every step: are the parameters and their gradients still where it put them?  (300 tensors: 3 us;
// the same question in Python 20.)
struct Places {
    std::vector<Tensor> params, grads;
    std::vector<void*> at;
    Places(std::vector<Tensor> p, std::vector<Tensor> g) : params(std::move(p)), grads(std::move(g)) {
        TORCH_CHECK_VALUE(params.size() == grads.size(), "a gradient for each parameter");
        for (const Tensor& t : params) at.push_back(t.data_ptr());
    }
    bool in_place() const {
        for (size_t i = 0; i < params.size(); ++i)
            if (params[i].data_ptr() != at[i] || !params[i].grad().is_same(grads[i])) return false;
        return true;
    }
};

void bind(const std::vector<uintptr_t>& entries) {
    TORCH_CHECK(entries.size() == 4, "four entry points");
    az.last_error = reinterpret_cast<decltype(az.last_error)>(entries[0]);
    az.group_norm_workspace_bytes = reinterpret_cast<decltype(az.group_norm_workspace_bytes)>(entries[1]);
    az.group_norm_act = reinterpret_cast<decltype(az.group_norm_act)>(entries[2]);
    az.group_norm_act_backward = reinterpret_cast<decltype(az.group_norm_act_backward)>(entries[3]);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("bind", &bind);
    pybind11::class_<Places>(m, "Places").def(pybind11::init<std::vector<Tensor>, std::vector<Tensor>>()).def("in_place", &Places::in_place);
    m.def("group_norm_act", &group_norm_act, pybind11::call_guard<pybind11::gil_scoped_release>());
}
