// train_ops_bind.cpp — the training operators as C++ autograd functions, bound to Python. The kernels stay behind the C ABI of
// libsdfx_hip.so (include/sdfx.h); this file allocates, keeps what a backward pass needs and calls it on the current stream. It exists for
// latency: a backward pass that runs Python code on autograd's thread costs 70 us more than its kernels, which is most of a small call (GEGLU
// of 128 x 10240, forward and backward: 120 us from Python, 45 us from here).
// The library's entry points arrive as addresses (bind()), so that the library that _sdfx.py opened is the one that runs.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>
#include <unordered_map>

#include "../../include/sdfx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&sdfx_last_error) last_error = nullptr;
    decltype(&sdfx_attention_train_scratch_bytes) attention_scratch = nullptr;
    decltype(&sdfx_attention_train_forward) attention_forward = nullptr;
    decltype(&sdfx_attention_train_backward) attention_backward = nullptr;
    decltype(&sdfx_group_norm_train_scratch_bytes) norm_scratch = nullptr;
    decltype(&sdfx_group_norm_train_forward) norm_forward = nullptr;
    decltype(&sdfx_group_norm_train_backward) norm_backward = nullptr;
    decltype(&sdfx_geglu_train_forward) geglu_forward = nullptr;
    decltype(&sdfx_geglu_train_backward) geglu_backward = nullptr;
} api;

template <typename F> void take(F& f, const std::unordered_map<std::string, uint64_t>& m, const char* name) {
    const auto it = m.find(name);
    TORCH_CHECK(it != m.end() && it->second, "sdfx: no address of ", name);
    f = reinterpret_cast<F>(it->second);
}
void bind(const std::unordered_map<std::string, uint64_t>& m) {
    take(api.last_error, m, "sdfx_last_error");
    take(api.attention_scratch, m, "sdfx_attention_train_scratch_bytes");
    take(api.attention_forward, m, "sdfx_attention_train_forward");
    take(api.attention_backward, m, "sdfx_attention_train_backward");
    take(api.norm_scratch, m, "sdfx_group_norm_train_scratch_bytes");
    take(api.norm_forward, m, "sdfx_group_norm_train_forward");
    take(api.norm_backward, m, "sdfx_group_norm_train_backward");
    take(api.geglu_forward, m, "sdfx_geglu_train_forward");
    take(api.geglu_backward, m, "sdfx_geglu_train_backward");
}
void check(int rc) { TORCH_CHECK(rc == 0, "sdfx error ", rc, ": ", api.last_error()); }

sdfx_stream_t stream_of(const Tensor& t) {          // the current stream of the tensor's device
    return reinterpret_cast<sdfx_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}
const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float* scratch_of(uint64_t bytes, const Tensor& like, Tensor& keep) {
    if (bytes == 0) return nullptr;
    keep = at::empty({(int64_t)((bytes + 7) / 8)}, like.options().dtype(at::kDouble));
    return static_cast<float*>(keep.mutable_data_ptr());
}
Tensor dense16(const Tensor& t, at::MemoryFormat f) {
    const Tensor c = t.contiguous(f);
    return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone(f) : c;
}
// A saved tensor as it comes back: hooks on saved tensors may have moved it into another layout (copied), but its size, type and device are what
// the kernels' addresses are formed from.
void same(const Tensor& t, const char* what, at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device, what, ": a hook on saved tensors returned ",
                t.defined() ? t.toString() : std::string("nothing"), " ", t.defined() ? t.sizes() : at::IntArrayRef(), " where ", type, " ", sizes, " on ",
                device, " was saved");
}
Tensor back(const Tensor& t, const char* what, at::IntArrayRef sizes, at::ScalarType type, const at::Device& device,
            at::MemoryFormat f = at::MemoryFormat::Contiguous) {
    same(t, what, sizes, type, device);
    return dense16(t, f);
}
// gradients that raise when they are differentiated again
variable_list once(variable_list v) {
    if (!at::GradMode::is_enabled()) return v;
    variable_list fake;
    for (auto& t : v) {
        if (t.defined()) t = t.detach().requires_grad_(true);
        fake.push_back(t);
    }
    return torch::autograd::DelayedError("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)v.size())
        .apply(std::move(fake));
}
uint32_t u(int64_t v) { return (uint32_t)v; }

// ---- attention --------------------------------------------------------------------------------------------------------------------
struct Strides { uint64_t s[3]; };
Strides strides(const Tensor& t) { return {{(uint64_t)t.stride(0), (uint64_t)t.stride(2), (uint64_t)t.stride(1)}}; }    // batch, token, head
Tensor rows16(const Tensor& t) {          // as the kernels read it, or a copy
    const bool ok = t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 && t.stride(2) < (1 << 24) &&
                    reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    return ok ? t : at::empty(t.sizes(), t.options()).copy_(t);          // (contiguous() returns a dense tensor as it is, misaligned or with odd strides of its axes of one)
}
struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0, const std::optional<Tensor>& mask0, bool causal,
                          double scale, bool keep) {
        const c10::DeviceGuard guard(q0.device());
        const Tensor q = rows16(q0), k = rows16(k0), v = rows16(v0), mask = mask0 ? mask0->contiguous() : Tensor();
        const int64_t B = q.size(0), H = q.size(1), Nq = q.size(2), d = q.size(3), Hk = k.size(1), Nk = k.size(2);
        const Tensor o = at::empty({B, Nq, H * d}, q.options());
        Tensor lo, lse, scratch;
        if (keep) {
            lo = at::empty(o.sizes(), o.options().dtype(at::kShort));
            lse = at::empty({B, H, Nq}, q.options().dtype(at::kFloat));
        }
        float* sp = scratch_of(api.attention_scratch(u(B), u(H), u(Hk), u(Nq), u(Nk), u(d), 0), q, scratch);
        const Strides qs = strides(q), ks = strides(k), vs = strides(v);
        check(api.attention_forward(in(q), in(k), in(v), in(mask), u(B), u(H), u(Hk), u(Nq), u(Nk), u(d), qs.s, ks.s, vs.s, (float)scale, causal,
                                    q.scalar_type() == at::kBFloat16, out(o), out(lo), static_cast<float*>(out(lse)), sp, stream_of(q)));
        if (keep) {
            ctx->save_for_backward({q, k, v, mask, o, lo, lse});
            ctx->saved_data["dims"] = std::vector<int64_t>{B, H, Hk, Nq, Nk, d};
            ctx->saved_data["causal"] = causal;
            ctx->saved_data["scale"] = scale;
        }
        return o;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        const at::Device dev = g[0].device();
        const at::ScalarType type = g[0].scalar_type();
        const c10::DeviceGuard guard(dev);
        const auto dims = ctx->saved_data["dims"].toIntVector();
        const int64_t B = dims[0], H = dims[1], Hk = dims[2], Nq = dims[3], Nk = dims[4], d = dims[5];
        Tensor dq, dk, dv, scratch;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            same(s[0], "attention", {B, H, Nq, d}, type, dev);
            same(s[1], "attention", {B, Hk, Nk, d}, type, dev);
            same(s[2], "attention", {B, Hk, Nk, d}, type, dev);
            const Tensor q = rows16(s[0]), k = rows16(s[1]), v = rows16(s[2]), o = back(s[4], "attention", {B, Nq, H * d}, type, dev),
                         lo = back(s[5], "attention", {B, Nq, H * d}, at::kShort, dev), lse = back(s[6], "attention", {B, H, Nq}, at::kFloat, dev),
                         mask = s[3].defined() ? back(s[3], "attention", {B, Nk}, at::kBool, dev) : Tensor();
            const Tensor dy = dense16(g[0], at::MemoryFormat::Contiguous);
            if (ctx->needs_input_grad(0)) dq = at::empty({B, Nq, H, d}, q.options());
            if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
                dk = at::empty({B, Nk, Hk, d}, q.options());
                dv = at::empty({B, Nk, Hk, d}, q.options());
            }
            float* sp = scratch_of(api.attention_scratch(u(B), u(H), u(Hk), u(Nq), u(Nk), u(d), 1), q, scratch);
            const Strides qs = strides(q), ks = strides(k), vs = strides(v);
            check(api.attention_backward(in(q), in(k), in(v), in(mask), in(o), in(lo), static_cast<const float*>(in(lse)), in(dy), u(B), u(H), u(Hk),
                                         u(Nq), u(Nk), u(d), qs.s, ks.s, vs.s, (float)ctx->saved_data["scale"].toDouble(),
                                         ctx->saved_data["causal"].toBool(), q.scalar_type() == at::kBFloat16, out(dq), out(dk), out(dv), sp,
                                         stream_of(q)));
            for (Tensor* t : {&dq, &dk, &dv})
                if (t->defined()) *t = t->transpose(1, 2);
        }
        variable_list r = once({dq, dk, dv});
        r.resize(7);
        return r;
    }
};
Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask, bool causal, double scale) {
    const bool keep = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    return Attention::apply(q, k, v, mask, causal, scale, keep);
}

// ---- group norm -------------------------------------------------------------------------------------------------------------------
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kHalf ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }

struct Norm : torch::autograd::Function<Norm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x0, const std::optional<Tensor>& pre0, const Tensor& w0, const Tensor& b0, int64_t G, double eps,
                          bool act, bool eight, bool keep) {
        const c10::DeviceGuard guard(x0.device());
        const Tensor x = dense16(x0, at::MemoryFormat::ChannelsLast), pre = pre0 ? dense16(*pre0, at::MemoryFormat::Contiguous) : Tensor(),
                     w = dense16(w0, at::MemoryFormat::Contiguous), b = dense16(b0, at::MemoryFormat::Contiguous);
        const int64_t N = x.size(0), C = x.size(1), HW = x.size(2) * x.size(3);
        const Tensor y = at::empty_like(x), stats = at::empty({N, G, 2}, x.options().dtype(at::kFloat));
        Tensor saved, scratch;
        if (eight && keep) saved = at::empty({x.numel() + x.numel() / 32}, x.options().dtype(at::kByte));
        float* sp = scratch_of(api.norm_scratch(u(N), u(HW), u(C), u(G)), x, scratch);
        check(api.norm_forward(in(x), in(pre), in(w), in(b), u(N), u(HW), u(C), u(G), (float)eps, act, dtype_of(x), w.scalar_type() == at::kFloat, out(y),
                               out(saved), static_cast<float*>(out(stats)), sp, stream_of(x)));
        if (keep) {
            ctx->save_for_backward({saved.defined() ? saved : x, pre, w, b, stats});
            ctx->saved_data["shape"] = x.sizes();
            ctx->saved_data["G"] = G;
            ctx->saved_data["flags"] = (int64_t)(act ? 1 : 0) | (saved.defined() ? 2 : 0) | (w.scalar_type() == at::kFloat ? 4 : 0);
        }
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        const at::Device dev = g[0].device();
        const at::ScalarType type = g[0].scalar_type();
        const c10::DeviceGuard guard(dev);
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const int64_t N = shape[0], C = shape[1], HW = shape[2] * shape[3], G = ctx->saved_data["G"].toInt(), flags = ctx->saved_data["flags"].toInt();
        Tensor dx, dpre, dw, db, scratch;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            const Tensor dy = dense16(g[0], at::MemoryFormat::ChannelsLast);
            const int64_t n = N * HW * C;
            const Tensor x = (flags & 2) ? back(s[0], "group_norm_act", {n + n / 32}, at::kByte, dev)
                                         : back(s[0], "group_norm_act", shape, type, dev, at::MemoryFormat::ChannelsLast);
            const Tensor w = back(s[2], "group_norm_act", {C}, (flags & 4) ? at::kFloat : type, dev), b = back(s[3], "group_norm_act", {C}, w.scalar_type(), dev),
                         stats = back(s[4], "group_norm_act", {N, G, 2}, at::kFloat, dev),
                         pre = s[1].defined() ? back(s[1], "group_norm_act", {N, C}, type, dev) : Tensor();
            const size_t e = pre.defined() ? 1 : 0;                 // (an absent `pre` has no edge)
            if (ctx->needs_input_grad(0)) dx = at::empty_like(dy);
            if (e && ctx->needs_input_grad(1)) dpre = at::empty_like(pre);
            if (ctx->needs_input_grad(1 + e)) dw = at::empty_like(w);
            if (ctx->needs_input_grad(2 + e)) db = at::empty_like(b);
            float* sp = scratch_of(api.norm_scratch(u(N), u(HW), u(C), u(G)), dy, scratch);
            check(api.norm_backward(in(x), (flags & 2) != 0, in(pre), in(dy), in(w), in(b), static_cast<const float*>(in(stats)), u(N), u(HW), u(C), u(G),
                                    flags & 1, dtype_of(dy), w.scalar_type() == at::kFloat, out(dx), out(dpre), out(dw), out(db), sp, stream_of(dy)));
        }
        variable_list r = once({dx, dpre, dw, db});
        r.resize(9);
        return r;
    }
};
Tensor group_norm(const Tensor& x, const std::optional<Tensor>& pre, const Tensor& w, const Tensor& b, int64_t G, double eps, bool act, bool eight) {
    const bool keep = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || b.requires_grad() || (pre && pre->requires_grad()));
    return Norm::apply(x, pre, w, b, G, eps, act, eight, keep);
}

// ---- GEGLU ------------------------------------------------------------------------------------------------------------------------
struct Geglu : torch::autograd::Function<Geglu> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x0, bool eight, bool keep) {
        const c10::DeviceGuard guard(x0.device());
        const Tensor x = dense16(x0, at::MemoryFormat::Contiguous);
        const int64_t n = x.size(-1) / 2, rows = x.numel() / (2 * n);
        std::vector<int64_t> shape = x.sizes().vec();
        shape.back() = n;
        const Tensor y = at::empty(shape, x.options());
        Tensor saved;
        if (eight && keep) saved = at::empty({x.numel() + x.numel() / 32}, x.options().dtype(at::kByte));
        check(api.geglu_forward(in(x), (uint64_t)rows, u(n), dtype_of(x), out(y), out(saved), stream_of(x)));
        if (keep) {
            ctx->save_for_backward({saved.defined() ? saved : x});
            ctx->saved_data["eight"] = saved.defined();
        }
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        const at::Device dev = g[0].device();
        const c10::DeviceGuard guard(dev);
        const bool eight = ctx->saved_data["eight"].toBool();
        Tensor dx;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            const Tensor dy = dense16(g[0], at::MemoryFormat::Contiguous);
            const int64_t n = dy.size(-1);
            std::vector<int64_t> shape = dy.sizes().vec();
            shape.back() = 2 * n;
            const int64_t all = 2 * dy.numel();
            const Tensor x = eight ? back(s[0], "geglu", {all + all / 32}, at::kByte, dev) : back(s[0], "geglu", shape, dy.scalar_type(), dev);
            dx = at::empty(shape, dy.options());
            check(api.geglu_backward(in(x), eight, in(dy), (uint64_t)(dy.numel() / n), u(n), dtype_of(dy), out(dx), stream_of(dy)));
        }
        variable_list r = once({dx});
        r.resize(3);
        return r;
    }
};
Tensor geglu(const Tensor& x, bool eight) { return Geglu::apply(x, eight, at::GradMode::is_enabled() && x.requires_grad()); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("bind", &bind);
    m.def("attention", &attention, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("group_norm", &group_norm, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("geglu", &geglu, pybind11::call_guard<pybind11::gil_scoped_release>());
}
