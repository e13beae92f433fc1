// torch binding of the feature operators: argument checks, allocation and
// autograd around the C-ABI calls of include/dot_b200.h, in C++ because a small
// training call is bound by the host (as Python autograd Functions over ctypes a
// norm's forward and backward took 121 us, 73 here with the same kernels and 68
// since the parameters' gradients need no launch of their own).
//
// Semantics and messages are those documented in dot_b200/norm.py and
// dot_b200/rotary.py, whose functions call these.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/dot_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int feature_dtype(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return DOT_F32;
        case at::kBFloat16: return DOT_BF16;
        case at::kHalf: return DOT_F16;
        default: return -1;
    }
}

// A failed C-ABI call as the Python exception that dot_b200._lib.check raises.
void check(int rc, const char* what) {
    if (rc == DOT_OK) return;
    const char* msg = dot_last_error();
    TORCH_CHECK_NOT_IMPLEMENTED(rc != DOT_ERR_UNSUPPORTED, what, ": ", msg);
    TORCH_CHECK_VALUE(rc != DOT_ERR_INVALID, what, ": ", msg);
    TORCH_CHECK(false, what, " failed (", rc, "): ", msg);
}

// What would pass these operators by without a word is refused: a tangent of forward-mode
// differentiation would be dropped, and a trace would keep the allocation of the outputs
// but not the launch that fills them.
template <typename... Ts>
void refuse_modes(const char* what, const Ts&... inputs) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "dot_b200: ", what,
                                " cannot be recorded by torch.jit.trace");
    const bool tangent = ((inputs.defined() && inputs._fw_grad(/*level=*/0).defined()) || ...);
    TORCH_CHECK_NOT_IMPLEMENTED(!tangent, "dot_b200: ", what, " has no forward-mode derivative");
}

// The address of a tensor that may be left out.  One that is there but has no memory (torch's
// tensors of zeros without storage, fake ones) must not pass for one that is not.
void* out(const Tensor& t) {
    if (!t.defined()) return nullptr;
    void* p = t.data_ptr();
    TORCH_CHECK_VALUE(p != nullptr || t.numel() == 0, "dot_b200: a tensor without memory");
    return p;
}
const void* ptr(const Tensor& t) { return out(t); }

// The values as they are in memory: a view that torch negates when it is read is copied.
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

optional<Tensor> present(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

void* current_stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// ---- group norm ---------------------------------------------------------------

// x [N, *S, C] read in place where its channels are consecutive and its
// positions lie at one stride, else a copy.
struct Rows {
    Tensor t;
    int64_t N, S, C, batch = 0, pos = 0;
    explicit Rows(const Tensor& x_in) : t(plain(x_in)), N(t.size(0)), S(1), C(t.size(-1)) {
        const Tensor x = t;
        const int64_t dims = x.dim();
        for (int64_t d = 1; d < dims - 1; ++d) S *= x.size(d);
        if (x.numel() == 0) return;
        bool ok = C == 1 || x.stride(-1) == 1, any = false;
        int64_t next = 0;   // the stride that continues the axes seen so far
        for (int64_t d = dims - 2; ok && d >= 1; --d) {
            if (x.size(d) == 1) continue;
            if (!any)
                pos = x.stride(d);
            else
                ok = x.stride(d) == next;
            any = true;
            next = x.stride(d) * x.size(d);
        }
        if (ok) {
            batch = x.stride(0);
        } else {
            t = x.contiguous();
            batch = S * C;
            pos = C;
        }
    }
};

struct NormOptions {
    int64_t groups;
    double eps;
    int64_t activation;
};

// y and the statistics, which begin the one buffer that also holds the workspace.
std::pair<Tensor, Tensor> norm_forward(const Tensor& x_in, const Tensor& w, const Tensor& b, const Tensor& lengths,
                                       const NormOptions& o) {
    const Rows r(x_in);
    const c10::cuda::CUDAGuard guard(x_in.device());
    Tensor y = dense_like(x_in);
    const size_t at = (size_t(r.N) * size_t(o.groups) * 8 + 255) / 256 * 256;
    const size_t ws = dot_group_norm_fwd_workspace_bytes(r.N, r.S, r.C, o.groups);
    Tensor stats = at::empty({int64_t((at + ws) / 4)}, x_in.options().dtype(at::kFloat));
    char* base = static_cast<char*>(stats.data_ptr());
    const Tensor& p = w.defined() ? w : b;
    check(dot_group_norm_fwd(r.t.data_ptr(), feature_dtype(x_in.scalar_type()), r.batch, r.pos, ptr(w), ptr(b),
                             p.defined() ? feature_dtype(p.scalar_type()) : DOT_F32,
                             static_cast<const int32_t*>(ptr(lengths)), r.N, r.S, r.C, o.groups, float(o.eps),
                             int(o.activation), y.data_ptr(), reinterpret_cast<float*>(base), base + at, ws,
                             current_stream(x_in)),
          "dot_group_norm_fwd");
    return {y, stats};
}

struct NormFn : torch::autograd::Function<NormFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                          const optional<Tensor>& bias, const optional<Tensor>& len, int64_t groups, double eps,
                          int64_t activation) {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()), lengths = len.value_or(Tensor());
        auto [y, stats] = norm_forward(x, w, b, lengths, {groups, eps, activation});
        ctx->save_for_backward({x, w, b, lengths, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["activation"] = activation;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &lengths = saved[3], &stats = saved[4];
        refuse_modes("the backward of group_norm_act", grads[0]);
        const int64_t groups = ctx->saved_data["groups"].toInt(), act = ctx->saved_data["activation"].toInt();
        const Rows r(x), g(grads[0]);
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor dx, dw, db;
        size_t input = 0;   // inputs are counted without those that are not there
        if (ctx->needs_input_grad(input++)) dx = dense_like(x);
        if (w.defined() && ctx->needs_input_grad(input++)) dw = dense_like(w);
        if (b.defined() && ctx->needs_input_grad(input++)) db = dense_like(b);
        const size_t ws_bytes = dot_group_norm_bwd_workspace_bytes(r.N, r.S, r.C, groups);
        Tensor ws = at::empty({int64_t(ws_bytes)}, x.options().dtype(at::kByte));
        const Tensor& p = w.defined() ? w : b;
        check(dot_group_norm_bwd(r.t.data_ptr(), feature_dtype(x.scalar_type()), r.batch, r.pos, g.t.data_ptr(),
                                 g.batch, g.pos, ptr(w), ptr(b),
                                 p.defined() ? feature_dtype(p.scalar_type()) : DOT_F32,
                                 static_cast<const int32_t*>(ptr(lengths)), r.N, r.S, r.C, groups, int(act),
                                 static_cast<const float*>(stats.data_ptr()), out(dx), out(dw), out(db),
                                 ws.data_ptr(), ws_bytes, current_stream(x)),
              "dot_group_norm_bwd");
        if (at::GradMode::is_enabled()) {   // recorded: a second differentiation has to fail, not to give zero
            variable_list outs;
            for (Tensor* t : {&dx, &dw, &db})
                if (t->defined()) outs.push_back(t->detach().set_requires_grad(true));
            auto refuse = std::make_shared<torch::autograd::DelayedError>(
                "dot_b200: group_norm_act is once differentiable", int64_t(outs.size()));
            outs = (*refuse)(std::move(outs));
            size_t k = 0;
            for (Tensor* t : {&dx, &dw, &db})
                if (t->defined()) *t = outs[k++];
        }
        return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor norm_param(const optional<Tensor>& p, const Tensor& x, const char* name) {
    if (!p.has_value()) return Tensor();
    const int64_t C = x.size(-1);
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == C, name, " must have shape [", C, "]");
    TORCH_CHECK_VALUE(p->device() == x.device(), name, " must be on ", x.device());
    return plain(p->contiguous());
}

Tensor group_norm_act(const Tensor& x, int64_t groups, const optional<Tensor>& weight, const optional<Tensor>& bias,
                      double eps, int64_t activation, const optional<Tensor>& lengths_in) {
    refuse_modes("group_norm_act", x, weight.value_or(Tensor()), bias.value_or(Tensor()));
    TORCH_CHECK(x.is_cuda(), "dot_b200: x must be a CUDA tensor (dot_b200 runs on NVIDIA GPUs only)");
    TORCH_CHECK_VALUE(x.dim() >= 2, "x must be [N, ..., C]");
    TORCH_CHECK_NOT_IMPLEMENTED(feature_dtype(x.scalar_type()) >= 0, "x must be float32, bfloat16 or float16, got ",
                                x.scalar_type());
    const int64_t C = x.size(-1);
    TORCH_CHECK_VALUE(groups >= 1 && C % groups == 0, "num_groups (", groups,
                      ") must be >= 1 and divide the channels (", C, ")");
    TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0");
    Tensor w = norm_param(weight, x, "weight"), b = norm_param(bias, x, "bias"), lengths;
    const Tensor& p = w.defined() ? w : b;
    if (p.defined() && (feature_dtype(p.scalar_type()) < 0 || (b.defined() && b.scalar_type() != p.scalar_type()))) {
        // the kernels read both parameters as one type
        if (w.defined()) w = w.to(at::kFloat);
        if (b.defined()) b = b.to(at::kFloat);
    }
    if (lengths_in.has_value()) {
        TORCH_CHECK_VALUE(lengths_in->dim() == 1 && lengths_in->size(0) == x.size(0), "lengths must be [N]");
        TORCH_CHECK_VALUE(lengths_in->scalar_type() == at::kInt, "lengths must be int32");
        lengths = lengths_in->to(x.device()).contiguous();
    }
    if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) ||
                                       (b.defined() && b.requires_grad())))
        return NormFn::apply(x, present(w), present(b), present(lengths), groups, eps, activation);
    return norm_forward(x, w, b, lengths, {groups, eps, activation}).first;
}

// ---- rotary ---------------------------------------------------------------------

int position_dtype(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return DOT_F32;
        case at::kInt: return DOT_I32;
        case at::kLong: return DOT_I64;
        default: return -1;
    }
}

// q [B,L,Hq,D] and/or k [B,L,Hk,D] (either may be undefined) turned by the
// angles of positions [B or 1, L, A] and freqs [P,A].
std::pair<Tensor, Tensor> turn(const Tensor& q_in, const Tensor& k_in, const Tensor& positions_in,
                               const Tensor& freqs_in, bool interleaved, bool inverse) {
    const Tensor& ref = q_in.defined() ? q_in : k_in;
    const c10::cuda::CUDAGuard guard(ref.device());
    const Tensor positions = plain(positions_in), freqs = plain(freqs_in);
    const int64_t D = ref.size(3);
    Tensor q, k, qo, ko;
    int64_t qs[3] = {}, ks[3] = {}, ps[3];
    auto take = [&](const Tensor& in, Tensor& t, Tensor& o, int64_t* s) {
        if (!in.defined()) return;
        t = plain(in);
        if (D > 1 && t.stride(3) != 1) t = t.contiguous();   // elements of a head are consecutive
        o = dense_like(in);
        for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
    };
    take(q_in, q, qo, qs);
    take(k_in, k, ko, ks);
    for (int i = 0; i < 3; ++i) ps[i] = positions.stride(i);
    if (positions.size(0) != ref.size(0)) ps[0] = 0;
    check(dot_rotary(ptr(q), qs, q.defined() ? q.size(2) : 0, ptr(k), ks, k.defined() ? k.size(2) : 0,
                     feature_dtype(ref.scalar_type()), ptr(positions), position_dtype(positions.scalar_type()),
                     ps, static_cast<const float*>(ptr(freqs)), ref.size(0), ref.size(1), D, freqs.size(0),
                     int(freqs.size(1)), interleaved, inverse, out(qo), out(ko), current_stream(ref)),
          "dot_rotary");
    return {qo, ko};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
    static variable_list forward(AutogradContext* ctx, const optional<Tensor>& q_in, const optional<Tensor>& k_in,
                                 const Tensor& positions, const Tensor& freqs, bool interleaved, bool inverse) {
        const Tensor q = q_in.value_or(Tensor()), k = k_in.value_or(Tensor());
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, freqs});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        auto [qo, ko] = turn(q, k, positions, freqs, interleaved, inverse);
        variable_list outs;
        if (qo.defined()) outs.push_back(qo);
        if (ko.defined()) outs.push_back(ko);
        ctx->saved_data["has_q"] = q.defined();
        ctx->saved_data["has_k"] = k.defined();
        return outs;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const bool interleaved = ctx->saved_data["interleaved"].toBool();
        const bool inverse = ctx->saved_data["inverse"].toBool();
        Tensor dq, dk;
        size_t input = 0;   // inputs and outputs are counted without those that are not there
        if (ctx->saved_data["has_q"].toBool()) {
            if (ctx->needs_input_grad(input)) dq = grads[input];
            ++input;
        }
        if (ctx->saved_data["has_k"].toBool() && ctx->needs_input_grad(input)) dk = grads[input];
        variable_list all(6);
        if (!dq.defined() && !dk.defined()) return all;
        refuse_modes("the backward of rotary", dq, dk);
        // the turn is orthogonal: its backward is the turn by -angle
        if (at::GradMode::is_enabled()) {
            variable_list outs = RotaryFn::apply(present(dq), present(dk), saved[0], saved[1], interleaved, !inverse);
            size_t i = 0;
            if (dq.defined()) all[0] = outs[i++];
            if (dk.defined()) all[1] = outs[i];
        } else {
            std::tie(all[0], all[1]) = turn(dq, dk, saved[0], saved[1], interleaved, !inverse);
        }
        return all;
    }
};

void check_heads(const Tensor& x, const char* name) {
    TORCH_CHECK(x.is_cuda(), "dot_b200: ", name, " must be a CUDA tensor (dot_b200 runs on NVIDIA GPUs only)");
    TORCH_CHECK_VALUE(x.dim() >= 3, name, " must be [..., tokens, heads, head_dim]");
    TORCH_CHECK_NOT_IMPLEMENTED(feature_dtype(x.scalar_type()) >= 0, name,
                                " must be float32, bfloat16 or float16, got ", x.scalar_type());
}

Tensor as_4d(const Tensor& x) {
    if (x.dim() == 4) return x;
    if (x.dim() == 3) return x.unsqueeze(0);
    int64_t B = 1;
    for (int64_t d = 0; d < x.dim() - 3; ++d) B *= x.size(d);
    return x.reshape({B, x.size(-3), x.size(-2), x.size(-1)});
}

std::pair<Tensor, optional<Tensor>> rotary(const Tensor& q, const Tensor& positions_in, const Tensor& freqs_in,
                                           const optional<Tensor>& k_in, bool interleaved) {
    refuse_modes("rotary", q, k_in.value_or(Tensor()), positions_in, freqs_in);
    check_heads(q, "q");
    const int64_t dims = q.dim(), lead = dims - 2, L = q.size(-3), D = q.size(-1);
    Tensor k;
    if (k_in.has_value()) {
        k = *k_in;
        check_heads(k, "k");
        TORCH_CHECK_VALUE(k.dim() == dims && k.sizes().slice(0, lead) == q.sizes().slice(0, lead) && k.size(-1) == D,
                          "k must have q's shape except for the number of heads");
        TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.device() == q.device(),
                          "k must have q's dtype and device");
    }
    TORCH_CHECK_VALUE(freqs_in.dim() == 2 && freqs_in.scalar_type() == at::kFloat, "freqs must be float32 [P, A]");
    TORCH_CHECK_VALUE(position_dtype(positions_in.scalar_type()) >= 0, "positions must be int32, int64 or float32");
    TORCH_CHECK_VALUE(positions_in.device() == q.device() && freqs_in.device() == q.device(),
                      "positions and freqs must be on q's device");
    TORCH_CHECK_VALUE(!positions_in.requires_grad() && !freqs_in.requires_grad(),
                      "positions and freqs are not differentiable here: detach them");
    const int64_t P = freqs_in.size(0), A = freqs_in.size(1);
    TORCH_CHECK_VALUE(A >= 1 && A <= 4, "freqs must have 1 to 4 axes");
    TORCH_CHECK_VALUE(2 * P <= D, "freqs must hold at most D/2 pairs");
    Tensor positions = positions_in;
    const bool full = positions.dim() == lead + 1 && positions.size(-1) == A &&
                      positions.sizes().slice(0, lead) == q.sizes().slice(0, lead);
    if (!full) {
        TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(0) == L && positions.size(1) == A,
                          "positions must be [*, L, A] with q's leading axes, or [L, A]");
        positions = positions.unsqueeze(0);
    } else if (lead != 2) {
        int64_t B = 1;
        for (int64_t d = 0; d < lead - 1; ++d) B *= q.size(d);
        positions = positions.reshape({B, L, A});
    }
    const Tensor freqs = freqs_in.contiguous();
    const Tensor q4 = as_4d(q), k4 = k.defined() ? as_4d(k) : Tensor();
    Tensor qo, ko;
    if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
        variable_list outs = RotaryFn::apply(present(q4), present(k4), positions, freqs, interleaved, false);
        qo = outs[0];
        if (k.defined()) ko = outs[1];
    } else {
        std::tie(qo, ko) = turn(q4, k4, positions, freqs, interleaved, false);
    }
    if (dims != 4) {
        qo = qo.view(q.sizes());
        if (k.defined()) ko = ko.view(k.sizes());
    }
    return {qo, k.defined() ? optional<Tensor>(ko) : std::nullopt};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "torch binding of dot_b200's feature operators";
    m.def("group_norm_act", &group_norm_act, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("rotary", &rotary, pybind11::call_guard<pybind11::gil_scoped_release>());
}
