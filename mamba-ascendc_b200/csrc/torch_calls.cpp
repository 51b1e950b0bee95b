// The operators around a selective state space layer as calls on torch tensors: checks, allocation, argument records and
// autograd nodes in front of the C ABI (include/ssd_b200.h).  A generation step takes the GPU 2 to 10 us; built and launched
// from Python through ctypes a call took the host 20 us, and an autograd node in Python about 100.
//
// Every function takes what its Python counterpart takes and answers None where the arguments are not what the operator
// takes; the Python function then says which, in the package's own words.  The library's functions come from Python
// (`bind`), so that one shared object, the one the ctypes binding loaded, serves both.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <limits>
#include <optional>
#include <string>

#include "../../include/ssd_b200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

namespace {

struct Library {
    decltype(&ssd_error_string) error_string;
    decltype(&ssd_rms_norm_fwd) norm_fwd;
    decltype(&ssd_rms_norm_work_bytes) norm_work;
    decltype(&ssd_rms_norm_bwd) norm_bwd;
    decltype(&ssd_short_conv_fwd) conv_fwd;
    decltype(&ssd_short_conv_work_bytes) conv_work;
    decltype(&ssd_short_conv_bwd) conv_bwd;
    decltype(&ssd_short_conv_step) conv_step;
    decltype(&ssd_selective_scan_work_bytes) scan_work;
    decltype(&ssd_selective_scan_checkpoint_bytes) scan_checkpoints;
    decltype(&ssd_selective_scan_fwd) scan_fwd;
    decltype(&ssd_selective_scan_grad_work_bytes) scan_grad_work;
    decltype(&ssd_selective_scan_bwd) scan_bwd;
    decltype(&ssd_selective_scan_step) scan_step;
} lib;

void bind(const py::dict& addresses) {
    const auto take = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::decay_t<decltype(f)>>(addresses[name].cast<uintptr_t>());
    };
    take(lib.error_string, "ssd_error_string");
    take(lib.norm_fwd, "ssd_rms_norm_fwd");
    take(lib.norm_work, "ssd_rms_norm_work_bytes");
    take(lib.norm_bwd, "ssd_rms_norm_bwd");
    take(lib.conv_fwd, "ssd_short_conv_fwd");
    take(lib.conv_work, "ssd_short_conv_work_bytes");
    take(lib.conv_bwd, "ssd_short_conv_bwd");
    take(lib.conv_step, "ssd_short_conv_step");
    take(lib.scan_work, "ssd_selective_scan_work_bytes");
    take(lib.scan_checkpoints, "ssd_selective_scan_checkpoint_bytes");
    take(lib.scan_fwd, "ssd_selective_scan_fwd");
    take(lib.scan_grad_work, "ssd_selective_scan_grad_work_bytes");
    take(lib.scan_bwd, "ssd_selective_scan_bwd");
    take(lib.scan_step, "ssd_selective_scan_step");
}

void check(int code, const char* op) {
    TORCH_CHECK(code == SSD_OK, op, ": ", lib.error_string(code), " (code ", code, ")");
}

// A size as the records have it.
int32_t number(int64_t size, const char* op) {
    check(size <= std::numeric_limits<int32_t>::max() ? SSD_OK : SSD_ERR_RANGE, op);
    return static_cast<int32_t>(size);
}

// ---- what a tensor is
int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SSD_F32;
        case at::kBFloat16: return SSD_BF16;
        case at::kHalf: return SSD_F16;
        default: return -1;
    }
}
// (inside a function transform a tensor has no storage of its own)
bool dense(const Tensor& t) { return t.has_storage() && t.is_cuda() && t.layout() == at::kStrided; }
// columns side by side
bool rowwise(const Tensor& t) { return t.dim() > 0 && (t.stride(-1) == 1 || t.size(-1) <= 1); }
bool activation(const Tensor& t, const Tensor& like) {
    return dense(t) && t.scalar_type() == like.scalar_type() && t.device() == like.device() && rowwise(t);
}
bool whole(const Tensor& t, at::IntArrayRef sizes, const Tensor& like) {
    return dense(t) && t.device() == like.device() && t.sizes() == sizes && t.is_contiguous();
}
bool f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
bool parameter(const Tensor& t, at::IntArrayRef sizes, const Tensor& like) {
    return (f32(t) || t.scalar_type() == like.scalar_type()) && whole(t, sizes, like);
}
const Tensor& of(const Maybe& t) {
    static const Tensor none;
    return t.has_value() ? *t : none;
}
void* ptr(const Tensor& t) {
    // what a call allocates, and gradients that come in, can be tensors of a transform as well
    TORCH_CHECK(!t.defined() || t.has_storage(), "ascend_kernel: cannot run inside a function transform (vmap, grad, jvp)");
    return t.defined() ? t.data_ptr() : nullptr;
}
template <class T>
T* ptr_as(const Tensor& t) { return static_cast<T*>(ptr(t)); }
ssd_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor empty(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().requires_grad(false)); }
Tensor empty_f32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
Tensor scratch(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}
template <class... T>
bool wants_grad(const T&... t) {
    return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}
// Whether a forward-mode derivative is being taken with respect to one of them, which the kernels would lose.
template <class... T>
bool has_tangent(const T&... t) {
    return ((t.defined() && t._fw_grad(/*level=*/0).defined()) || ...);
}
void check_upstream(const Tensor& dout, const Tensor& other, const char* op) {
    TORCH_CHECK(!has_tangent(dout, other), op, ": its gradients have no forward-mode derivatives");
}
Tensor side_by_side(const Tensor& t) { return rowwise(t) ? t : t.contiguous(); }

// Gradients that are differentiated again: the error that the framework raises for nodes that cannot be.
variable_list once(const variable_list& upstream, variable_list grads) {
    bool again = false;
    for (const Tensor& t : upstream) again |= t.defined() && t.requires_grad();
    if (!at::GradMode::is_enabled() || !again) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(grads.size()));
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    return (*error)(std::move(grads));
}

// A node takes an argument that may be missing as an optional; only those that are there have an edge to their gradient.
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
struct Edges {
    AutogradContext* ctx;
    size_t next = 0;
    bool wanted(bool present) { return present && ctx->needs_input_grad(next++); }
};

// A batch without tokens or rows, or without channels: nothing is launched and the states pass through.  (Packed sequences
// without tokens are launched.)
bool empty_call(const Tensor& x, const Tensor& cu) { return x.numel() == 0 && (!cu.defined() || x.size(-1) == 0); }
// Its gradients: zeros for what the call takes beside the initial state, in their order, and that of the initial state.
variable_list unmoved(Edges& edges, std::initializer_list<Tensor> taken, const Tensor& initial, const Tensor& dfinal) {
    variable_list grads;
    for (const Tensor& t : taken) grads.push_back(edges.wanted(t.defined()) ? at::zeros_like(t, at::MemoryFormat::Contiguous) : Tensor());
    const bool want_initial = edges.wanted(initial.defined());
    grads.push_back(!want_initial ? Tensor() : dfinal.defined() ? dfinal.clone() : at::zeros_like(initial));
    return grads;
}

// ---- slots of a cache
bool cache(const Tensor& state, at::IntArrayRef inner, at::ScalarType type, const Tensor& x) {
    if (!dense(state) || state.device() != x.device() || state.scalar_type() != type ||
        state.dim() != static_cast<int64_t>(inner.size()) + 1)
        return false;
    int64_t want = 1;
    for (int64_t d = inner.size(); d > 0; --d) {
        if (state.size(d) != inner[d - 1] || (state.size(d) > 1 && state.stride(d) != want)) return false;
        want *= state.size(d);
    }
    return state.size(0) <= 1 || state.stride(0) >= want;
}
bool slot_numbers(const Tensor& slots, const Tensor& x, const Tensor& state) {
    if (!slots.defined()) return state.size(0) == x.size(0);
    return slots.scalar_type() == at::kInt && whole(slots, {x.size(0)}, x);
}
// Rows run at the same time, so a row's new state must not lie on what another row (or the row itself, elsewhere) reads: slot i of
// `out` may share memory with slot i of `state` if they are the same, and with no other.
bool apart(const Tensor& state, const Tensor& out) {
    const int64_t count = state.size(0), bytes = state.element_size();
    const int64_t inner = count > 0 ? state.numel() / count * bytes : 0;
    if (inner == 0) return true;
    const int64_t step = count > 1 ? state.stride(0) * bytes : inner, step_out = count > 1 ? out.stride(0) * bytes : inner;
    const int64_t first = reinterpret_cast<intptr_t>(state.data_ptr()), first_out = reinterpret_cast<intptr_t>(out.data_ptr());
    if (first + (count - 1) * step + inner <= first_out || first_out + (count - 1) * step_out + inner <= first) return true;
    const int64_t distance = first_out - first;
    if (step == step_out) {  // from each slot the same way to the next ones of the other
        const int64_t rest = (distance % step + step) % step;
        return distance == 0 || (rest >= inner && step - rest >= inner);
    }
    for (int64_t i = 0; i < count; ++i) {
        const int64_t at = distance + i * step_out, k = at < 0 ? 0 : at / step;  // slot i of out lies at or behind slot k
        for (int64_t near = k; near < std::min(k + 2, count); ++near)
            if (at < near * step + inner && near * step < at + inner && !(near == i && at == i * step)) return false;
    }
    return true;
}
// The slots are written through their pointer, so the framework is told that the tensor (and what it is a view of) changed: what
// was saved of it for a backward pass is an error there.  Tensors of inference mode have no version and are never saved.
void changed(const Tensor& state) {
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}
bool packing(const Tensor& cu, const Tensor& x) {
    return cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.numel() >= 2 && whole(cu, cu.sizes(), x) && x.size(0) == 1;
}

// ============================================================ norm
// Rows of a tensor [..., width] at one distance, or none.
std::optional<int64_t> row_stride(const Tensor& t) {
    int64_t stride = 0, rows = 0;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (rows == 0) {
            stride = t.stride(d);
            rows = t.size(d);
        } else {
            if (t.stride(d) != stride * rows) return std::nullopt;
            rows *= t.size(d);
        }
    }
    return stride;
}
Tensor as_rows(const Tensor& t) { return row_stride(t) ? t : t.contiguous(); }

bool norm_takes(const Tensor& x, const Tensor& weight, const Tensor& residual) {
    if (!dense(x) || dtype_of(x) < 0 || !rowwise(x)) return false;
    const int64_t width = x.size(-1);
    if (width < 1 || width > 16384 || !parameter(weight, {width}, x)) return false;
    return !residual.defined() || (dense(residual) && residual.device() == x.device() &&
                                   (f32(residual) || residual.scalar_type() == x.scalar_type()) &&
                                   residual.sizes() == x.sizes() && rowwise(residual));
}
SsdNormArgs norm_args(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
    SsdNormArgs a{};
    a.x = ptr(x);
    a.residual = ptr(residual);
    a.weight = ptr(weight);
    a.width = static_cast<int32_t>(x.size(-1));
    a.rows = x.numel() / a.width;
    a.x_stride = *row_stride(x);
    a.residual_stride = residual.defined() ? *row_stride(residual) : 0;
    a.dtype = dtype_of(x);
    a.residual_f32 = residual.defined() && f32(residual);
    a.weight_f32 = f32(weight);
    a.eps = static_cast<float>(eps);
    return a;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list call(const Tensor& x_in, const Tensor& weight, const Tensor& residual_in, double eps, Tensor* rstd) {
        const Tensor x = as_rows(x_in), residual = residual_in.defined() ? as_rows(residual_in) : residual_in;
        const c10::cuda::CUDAGuard guard(x.device());
        SsdNormArgs a = norm_args(x, weight, residual, eps);
        Tensor out = empty(x.sizes(), x), stream;
        if (residual.defined()) stream = empty(x.sizes(), residual);
        if (rstd != nullptr) *rstd = empty_f32({a.rows}, x);
        a.out = ptr(out);
        a.stream = ptr(stream);
        a.rstd = rstd ? ptr_as<float>(*rstd) : nullptr;
        check(lib.norm_fwd(&a, stream_of(x)), "rms_norm");
        return residual.defined() ? variable_list{out, stream} : variable_list{out};
    }
    // Keeps the row's 1 / rms and what its sum is formed of: the fp32 stream, or x and a residual in fewer bits (the stream
    // is rounded then, and the gradient of the weight would carry that rounding).
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& maybe_residual,
                                 double eps) {
        const Tensor& residual = of(maybe_residual);
        ctx->set_materialize_grads(false);
        Tensor rstd;
        variable_list outputs = call(x, weight, residual, eps, &rstd);
        if (!residual.defined())
            ctx->save_for_backward({weight, rstd, x, Tensor()});
        else if (f32(residual))
            ctx->save_for_backward({weight, rstd, outputs[1], Tensor()});
        else
            ctx->save_for_backward({weight, rstd, residual, x});
        ctx->saved_data["types"] = c10::IValue(std::vector<int64_t>{static_cast<int64_t>(x.scalar_type()), residual.defined()});
        return outputs;
    }
    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor weight = saved[0], rstd = saved[1], stream = as_rows(saved[2]);
        const Tensor addend = saved[3].defined() ? as_rows(saved[3]) : saved[3];
        const auto types = ctx->saved_data["types"].toIntVector();
        const auto x_type = static_cast<at::ScalarType>(types[0]);
        const bool has_residual = types[1] != 0;
        Tensor dout = upstream[0], dstream = upstream.size() > 1 ? upstream[1] : Tensor();
        if (!dout.defined() && !dstream.defined()) return variable_list(4);
        check_upstream(dout, dstream, "rms_norm");
        const c10::cuda::CUDAGuard guard(stream.device());
        const auto options = stream.options().dtype(x_type).requires_grad(false);
        dout = dout.defined() ? as_rows(side_by_side(dout)) : at::zeros(stream.sizes(), options);
        if (dstream.defined()) dstream = as_rows(side_by_side(dstream));
        const bool want_x = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
        const bool want_residual = has_residual && ctx->needs_input_grad(2);
        Tensor dx = at::empty(stream.sizes(), options), dresidual, dweight, work;
        if (want_residual && stream.scalar_type() != x_type) dresidual = empty(stream.sizes(), stream);
        SsdNormGradArgs g{};
        g.width = static_cast<int32_t>(stream.size(-1));
        g.rows = stream.numel() / g.width;
        g.dtype = dtype_of(dx);
        if (want_weight) {
            dweight = empty(weight.sizes(), weight);
            work = scratch(lib.norm_work(g.rows, g.width, g.dtype), stream);
        }
        g.dout = ptr(dout);
        g.dstream = ptr(dstream);
        g.stream = ptr(stream);
        g.addend = ptr(addend);
        g.weight = ptr(weight);
        g.rstd = ptr_as<float>(rstd);
        g.dx = ptr(dx);
        g.dresidual = ptr(dresidual);
        g.dweight = ptr(dweight);
        g.work = ptr_as<float>(work);
        g.dout_stride = *row_stride(dout);
        g.dstream_stride = dstream.defined() ? *row_stride(dstream) : 0;
        g.stream_stride = *row_stride(stream);
        g.addend_stride = addend.defined() ? *row_stride(addend) : 0;
        g.residual_f32 = f32(stream);
        g.weight_f32 = f32(weight);
        check(lib.norm_bwd(&g, stream_of(stream)), "rms_norm");
        // one tensor for x and a residual of the same type, as the gradient of an addition is
        if (want_residual && !dresidual.defined()) dresidual = dx;
        return once(upstream, {want_x ? dx : Tensor(), dweight, dresidual, Tensor()});
    }
};

std::optional<variable_list> rms_norm_call(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
    if (!norm_takes(x, weight, residual) || has_tangent(x, weight, residual)) return std::nullopt;
    if (x.numel() == 0) {
        const Tensor stream = residual.defined() ? residual + x.to(residual.scalar_type()) : x;
        const Tensor out = stream.to(x.scalar_type()) * weight.to(x.scalar_type());
        return residual.defined() ? variable_list{out, stream} : variable_list{out};
    }
    if (wants_grad(x, weight, residual)) return NormNode::apply(x, weight, maybe(residual), eps);
    return NormNode::call(x, weight, residual, eps, nullptr);
}
std::optional<variable_list> rms_norm_quant_call(const Tensor& x_in, const Tensor& weight, const Tensor& residual_in, double eps,
                                                 int64_t group, const Tensor& scale) {
    if (!norm_takes(x_in, weight, residual_in) || wants_grad(x_in, weight, residual_in) ||
        has_tangent(x_in, weight, residual_in, scale))
        return std::nullopt;
    const int64_t width = x_in.size(-1);
    if (group != 0 && ((group != 32 && group != 64 && group != 128) || width % group != 0)) return std::nullopt;
    if (scale.defined() && (group != 0 || !f32(scale) || scale.numel() != 1 || !whole(scale, scale.sizes(), x_in))) return std::nullopt;
    const c10::cuda::CUDAGuard guard(x_in.device());
    std::vector<int64_t> sizes = x_in.sizes().vec();
    const Tensor q = at::empty(sizes, x_in.options().dtype(at::kFloat8_e4m3fn).requires_grad(false));
    sizes.back() = group ? width / group : 1;
    const Tensor scales = scale.defined() ? scale : empty_f32(sizes, x_in);
    Tensor stream;
    if (residual_in.defined()) stream = empty(x_in.sizes(), residual_in);
    if (x_in.numel() > 0) {
        const Tensor x = as_rows(x_in), residual = residual_in.defined() ? as_rows(residual_in) : residual_in;
        SsdNormArgs a = norm_args(x, weight, residual, eps);
        a.q = ptr(q);
        a.stream = ptr(stream);
        a.group = static_cast<int32_t>(group);
        if (scale.defined())
            a.static_scale = ptr(scale);
        else
            a.scales = ptr_as<float>(scales);
        check(lib.norm_fwd(&a, stream_of(x)), "rms_norm_quant");
    }
    return stream.defined() ? variable_list{q, scales, stream} : variable_list{q, scales};
}

// ============================================================ short convolution
bool filter_takes(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    const int64_t channels = x.size(-1);
    return weight.dim() == 2 && weight.size(1) >= 2 && weight.size(1) <= 4 && parameter(weight, {channels, weight.size(1)}, x) &&
           (!bias.defined() || (bias.scalar_type() == weight.scalar_type() && whole(bias, {channels}, x)));
}
SsdConvArgs conv_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& initial, const Tensor& cu, bool silu) {
    SsdConvArgs a{};
    a.x = ptr(x);
    a.weight = ptr(weight);
    a.bias = ptr(bias);
    a.initial_state = ptr(initial);
    a.cu_seqlens = ptr_as<int32_t>(cu);
    a.tokens = x.size(1);
    a.batch_stride = x.stride(0);
    a.token_stride = x.stride(1);
    a.rows = number(cu.defined() ? cu.numel() - 1 : x.size(0), "short_conv");
    a.channels = number(x.size(2), "short_conv");
    a.width = static_cast<int32_t>(weight.size(1));
    a.dtype = dtype_of(x);
    a.weight_f32 = f32(weight);
    a.silu = silu;
    return a;
}

struct ConvNode : torch::autograd::Function<ConvNode> {
    static variable_list call(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& initial, const Tensor& cu,
                              bool silu, bool want_final) {
        const c10::cuda::CUDAGuard guard(x.device());
        SsdConvArgs a = conv_args(x, weight, bias, initial, cu, silu);
        Tensor out = empty(x.sizes(), x), final;
        if (want_final) final = empty({a.rows, a.width - 1, a.channels}, x);
        a.out = ptr(out);
        a.final_state = ptr(final);
        if (!empty_call(x, cu))
            check(lib.conv_fwd(&a, stream_of(x)), "short_conv");
        else if (want_final)
            initial.defined() ? final.copy_(initial) : final.zero_();
        return want_final ? variable_list{out, final} : variable_list{out};
    }
    // Keeps its inputs; backward forms the sum in front of the activation again.
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias,
                                 const Maybe& initial, const Maybe& cu, bool silu, bool want_final) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, weight, of(bias), of(initial), of(cu)});
        ctx->saved_data["silu"] = silu;
        return call(x, weight, of(bias), of(initial), of(cu), silu, want_final);
    }
    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &initial = saved[3], &cu = saved[4];
        Tensor dout = upstream[0], dfinal = upstream.size() > 1 ? upstream[1] : Tensor();
        if (!dout.defined() && !dfinal.defined()) return variable_list(7);
        check_upstream(dout, dfinal, "short_conv");
        const c10::cuda::CUDAGuard guard(x.device());
        dout = dout.defined() ? dout.contiguous() : at::zeros(x.sizes(), x.options().requires_grad(false));
        if (dfinal.defined()) dfinal = dfinal.contiguous();
        if (empty_call(x, cu)) {
            Edges edges{ctx};
            variable_list grads = unmoved(edges, {x, weight, bias}, initial, dfinal);
            grads.resize(7);
            return once(upstream, std::move(grads));
        }
        Edges edges{ctx};
        const bool want_x = edges.wanted(true), want_weight = edges.wanted(true), want_bias = edges.wanted(bias.defined());
        const bool want_initial = edges.wanted(initial.defined());
        SsdConvGradArgs g{};
        g.forward = conv_args(x, weight, bias, initial, cu, ctx->saved_data["silu"].toBool());
        Tensor dx = empty(x.sizes(), x), dinitial, dweight, dbias, work;
        if (want_initial) dinitial = empty(initial.sizes(), initial);
        if (want_weight || want_bias) {
            dweight = empty(weight.sizes(), weight);
            if (want_bias) dbias = empty(bias.sizes(), bias);
            work = scratch(lib.conv_work(&g.forward), x);
        }
        g.dout = ptr(dout);
        g.dfinal = ptr(dfinal);
        g.dx = ptr(dx);
        g.dinitial = ptr(dinitial);
        g.dweight = ptr(dweight);
        g.dbias = ptr(dbias);
        g.work = ptr_as<float>(work);
        check(lib.conv_bwd(&g, stream_of(x)), "short_conv");
        return once(upstream, {want_x ? dx : Tensor(), want_weight ? dweight : Tensor(), dbias, dinitial, Tensor(), Tensor(), Tensor()});
    }
};

std::optional<variable_list> short_conv_call(const Tensor& x, const Tensor& weight, const Tensor& bias, bool silu,
                                             const Tensor& initial, const Tensor& cu, bool want_final) {
    if (!dense(x) || dtype_of(x) < 0 || x.dim() != 3 || !rowwise(x) || !filter_takes(x, weight, bias) ||
        has_tangent(x, weight, bias, initial))
        return std::nullopt;
    if (cu.defined() && !packing(cu, x)) return std::nullopt;
    const int64_t rows = cu.defined() ? cu.numel() - 1 : x.size(0), channels = x.size(2), held = weight.size(1) - 1;
    if (initial.defined() && (initial.scalar_type() != x.scalar_type() || !whole(initial, {rows, held, channels}, x)))
        return std::nullopt;
    if (wants_grad(x, weight, bias, initial)) return ConvNode::apply(x, weight, maybe(bias), maybe(initial), maybe(cu), silu, want_final);
    return ConvNode::call(x, weight, bias, initial, cu, silu, want_final);
}

std::optional<variable_list> short_conv_step_call(const Tensor& x, const Tensor& state, const Tensor& weight, const Tensor& bias,
                                                  bool silu, const Tensor& slots, const Tensor& state_out) {
    if (!dense(x) || dtype_of(x) < 0 || x.dim() != 2 || !rowwise(x) || !filter_takes(x, weight, bias) ||
        wants_grad(x, state, weight, bias, state_out) || has_tangent(x, state, weight, bias, state_out))
        return std::nullopt;
    const int64_t inner[2] = {weight.size(1) - 1, x.size(1)};
    const Tensor& next = state_out.defined() ? state_out : state;
    if (!cache(state, inner, x.scalar_type(), x) || !slot_numbers(slots, x, state)) return std::nullopt;
    if (state_out.defined() &&
        (!cache(state_out, inner, x.scalar_type(), x) || state_out.size(0) != state.size(0) || !apart(state, state_out)))
        return std::nullopt;
    const c10::cuda::CUDAGuard guard(x.device());
    if (x.numel() == 0 || state.size(0) == 0) return variable_list{at::zeros(x.sizes(), x.options().requires_grad(false))};
    const Tensor out = empty(x.sizes(), x);
    SsdConvStepArgs a{};
    a.x = ptr(x);
    a.weight = ptr(weight);
    a.bias = ptr(bias);
    a.state = ptr(state);
    a.slots = ptr_as<int32_t>(slots);
    a.state_out = ptr(next);
    a.out = ptr(out);
    a.x_stride = x.stride(0);
    a.state_stride = state.stride(0);
    a.state_out_stride = next.stride(0);
    a.rows = number(x.size(0), "short_conv_step");
    a.slot_count = number(state.size(0), "short_conv_step");
    a.channels = number(x.size(1), "short_conv_step");
    a.width = static_cast<int32_t>(weight.size(1));
    a.dtype = dtype_of(x);
    a.weight_f32 = f32(weight);
    a.silu = silu;
    check(lib.conv_step(&a, stream_of(x)), "short_conv_step");
    changed(next);
    return variable_list{out};
}

// ============================================================ selective scan
// `lead`: dimensions in front of the channels
bool scan_takes(int64_t lead, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& D,
                const Tensor& z, const Tensor& bias) {
    if (!dense(x) || dtype_of(x) < 0 || x.dim() != lead + 1 || !rowwise(x)) return false;
    if (!activation(dt, x) || dt.sizes() != x.sizes() || (z.defined() && (!activation(z, x) || z.sizes() != x.sizes()))) return false;
    if (!activation(B, x) || !activation(C, x) || B.dim() != lead + 2 || B.sizes() != C.sizes()) return false;
    for (int64_t d = 0; d < lead; ++d)
        if (B.size(d) != x.size(d)) return false;
    const int64_t channels = x.size(-1), groups = B.size(-2), n = B.size(-1);
    if (groups == 0 || channels % groups != 0 || n < 1 || n > 128) return false;
    return f32(A) && whole(A, {channels, n}, x) && (!D.defined() || (f32(D) && whole(D, {channels}, x))) &&
           (!bias.defined() || (f32(bias) && whole(bias, {channels}, x)));
}
SsdScanArgs scan_args(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& D,
                      const Tensor& z, const Tensor& bias, const Tensor& initial, const Tensor& cu, bool softplus) {
    SsdScanArgs a{};
    a.x = ptr(x);
    a.dt = ptr(dt);
    a.z = ptr(z);
    a.bm = ptr(B);
    a.cm = ptr(C);
    a.A = ptr_as<float>(A);
    a.D = ptr_as<float>(D);
    a.dt_bias = ptr_as<float>(bias);
    a.initial_state = ptr_as<float>(initial);
    a.cu_seqlens = ptr_as<int32_t>(cu);
    a.tokens = x.size(1);
    for (int d = 0; d < 2; ++d) {
        a.x_strides[d] = x.stride(d);
        a.dt_strides[d] = dt.stride(d);
        a.z_strides[d] = z.defined() ? z.stride(d) : 0;
    }
    for (int d = 0; d < 3; ++d) {
        a.b_strides[d] = B.stride(d);
        a.c_strides[d] = C.stride(d);
    }
    a.rows = number(cu.defined() ? cu.numel() - 1 : x.size(0), "selective_scan");
    a.channels = number(x.size(2), "selective_scan");
    a.dstate = static_cast<int32_t>(A.size(1));
    a.groups = number(B.size(2), "selective_scan");
    a.dtype = dtype_of(x);
    a.softplus = softplus;
    return a;
}

struct ScanNode : torch::autograd::Function<ScanNode> {
    static variable_list call(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& D,
                              const Tensor& z, const Tensor& bias, const Tensor& initial, const Tensor& cu, bool softplus,
                              bool want_final, Tensor* checkpoints) {
        const c10::cuda::CUDAGuard guard(x.device());
        SsdScanArgs a = scan_args(x, dt, A, B, C, D, z, bias, initial, cu, softplus);
        Tensor out = empty(x.sizes(), x), final;
        if (want_final) final = empty_f32({a.rows, a.channels, a.dstate}, x);
        if (empty_call(x, cu)) {
            if (want_final) initial.defined() ? final.copy_(initial) : final.zero_();
            return want_final ? variable_list{out, final} : variable_list{out};
        }
        if (checkpoints != nullptr) {
            *checkpoints = empty_f32({static_cast<int64_t>(lib.scan_checkpoints(&a) / sizeof(float))}, x);
            a.checkpoints = ptr_as<float>(*checkpoints);
        }
        const Tensor work = scratch(lib.scan_work(&a), x);
        a.out = ptr(out);
        a.final_state = ptr_as<float>(final);
        a.work = ptr_as<float>(work);
        check(lib.scan_fwd(&a, stream_of(x)), "selective_scan");
        return want_final ? variable_list{out, final} : variable_list{out};
    }
    // Keeps its inputs and the states at every 64th token; backward forms what lies between again.
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                                 const Tensor& C, const Maybe& D, const Maybe& z, const Maybe& bias, const Maybe& initial,
                                 const Maybe& cu, bool softplus, bool want_final) {
        ctx->set_materialize_grads(false);
        Tensor checkpoints;
        variable_list outputs = call(x, dt, A, B, C, of(D), of(z), of(bias), of(initial), of(cu), softplus, want_final, &checkpoints);
        ctx->save_for_backward({x, dt, A, B, C, of(D), of(z), of(bias), of(initial), of(cu), checkpoints});
        ctx->saved_data["softplus"] = softplus;
        return outputs;
    }
    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &A = s[2], &D = s[5], &z = s[6], &bias = s[7], &initial = s[8];
        Tensor dout = upstream[0], dfinal = upstream.size() > 1 ? upstream[1] : Tensor();
        if (!dout.defined() && !dfinal.defined()) return variable_list(12);
        check_upstream(dout, dfinal, "selective_scan");
        const c10::cuda::CUDAGuard guard(x.device());
        dout = dout.defined() ? dout.contiguous() : at::zeros(x.sizes(), x.options().requires_grad(false));
        if (dfinal.defined()) dfinal = dfinal.contiguous();
        if (empty_call(x, s[9])) {
            Edges edges{ctx};
            variable_list grads = unmoved(edges, {x, s[1], A, s[3], s[4], D, z, bias}, initial, dfinal);
            grads.resize(12);
            return once(upstream, std::move(grads));
        }
        SsdScanGradArgs g{};
        g.forward = scan_args(x, s[1], A, s[3], s[4], D, z, bias, initial, s[9], ctx->saved_data["softplus"].toBool());
        g.forward.checkpoints = ptr_as<float>(s[10]);
        const auto like = [&](const Tensor& t) { return t.defined() ? empty(t.sizes(), t) : Tensor(); };
        Edges edges{ctx};
        bool wanted[9];
        for (int i = 0; i < 9; ++i) wanted[i] = edges.wanted(s[i].defined());
        variable_list grads = {like(x), like(s[1]), like(A), like(s[3]), like(s[4]), like(D), like(z), like(bias)};
        grads.push_back(wanted[8] ? like(initial) : Tensor());
        const Tensor work = scratch(lib.scan_grad_work(&g.forward), x);
        g.dout = ptr(dout);
        g.dfinal = ptr_as<float>(dfinal);
        g.dx = ptr(grads[0]);
        g.ddt = ptr(grads[1]);
        g.dA = ptr_as<float>(grads[2]);
        g.dbm = ptr(grads[3]);
        g.dcm = ptr(grads[4]);
        g.dD = ptr_as<float>(grads[5]);
        g.dz = ptr(grads[6]);
        g.d_dt_bias = ptr_as<float>(grads[7]);
        g.dinitial = ptr_as<float>(grads[8]);
        g.work = ptr_as<float>(work);
        check(lib.scan_bwd(&g, stream_of(x)), "selective_scan");
        for (size_t i = 0; i < grads.size(); ++i)
            if (!wanted[i]) grads[i] = Tensor();
        grads.resize(12);
        return once(upstream, std::move(grads));
    }
};

std::optional<variable_list> selective_scan_call(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                                 const Tensor& D, const Tensor& z, const Tensor& bias, bool softplus,
                                                 const Tensor& initial, const Tensor& cu, bool want_final) {
    if (!scan_takes(2, x, dt, A, B, C, D, z, bias) || (cu.defined() && !packing(cu, x)) ||
        has_tangent(x, dt, A, B, C, D, z, bias, initial))
        return std::nullopt;
    const int64_t rows = cu.defined() ? cu.numel() - 1 : x.size(0), channels = x.size(2), n = A.size(1);
    if (initial.defined() && (!f32(initial) || !whole(initial, {rows, channels, n}, x))) return std::nullopt;
    if (wants_grad(x, dt, A, B, C, D, z, bias, initial))
        return ScanNode::apply(x, dt, A, B, C, maybe(D), maybe(z), maybe(bias), maybe(initial), maybe(cu), softplus, want_final);
    return ScanNode::call(x, dt, A, B, C, D, z, bias, initial, cu, softplus, want_final, nullptr);
}

std::optional<variable_list> selective_scan_step_call(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                                                      const Tensor& C, const Tensor& state, const Tensor& D, const Tensor& z,
                                                      const Tensor& bias, bool softplus, const Tensor& slots,
                                                      const Tensor& state_out) {
    if (!scan_takes(1, x, dt, A, B, C, D, z, bias) || wants_grad(x, dt, A, B, C, D, z, bias, state, state_out) ||
        has_tangent(x, dt, A, B, C, D, z, bias, state, state_out))
        return std::nullopt;
    const int64_t inner[2] = {x.size(1), A.size(1)};
    const Tensor& next = state_out.defined() ? state_out : state;
    if (!cache(state, inner, at::kFloat, x) || !slot_numbers(slots, x, state)) return std::nullopt;
    if (state_out.defined() &&
        (!cache(state_out, inner, at::kFloat, x) || state_out.size(0) != state.size(0) || !apart(state, state_out)))
        return std::nullopt;
    const c10::cuda::CUDAGuard guard(x.device());
    if (x.numel() == 0 || state.size(0) == 0) return variable_list{at::zeros(x.sizes(), x.options().requires_grad(false))};
    const Tensor out = empty(x.sizes(), x);
    SsdScanStepArgs a{};
    a.x = ptr(x);
    a.dt = ptr(dt);
    a.z = ptr(z);
    a.bm = ptr(B);
    a.cm = ptr(C);
    a.A = ptr_as<float>(A);
    a.D = ptr_as<float>(D);
    a.dt_bias = ptr_as<float>(bias);
    a.state = ptr_as<float>(state);
    a.slots = ptr_as<int32_t>(slots);
    a.state_out = ptr_as<float>(next);
    a.out = ptr(out);
    a.x_stride = x.stride(0);
    a.dt_stride = dt.stride(0);
    a.z_stride = z.defined() ? z.stride(0) : 0;
    for (int d = 0; d < 2; ++d) {
        a.b_strides[d] = B.stride(d);
        a.c_strides[d] = C.stride(d);
    }
    a.state_stride = state.stride(0);
    a.state_out_stride = next.stride(0);
    a.rows = number(x.size(0), "selective_scan_step");
    a.slot_count = number(state.size(0), "selective_scan_step");
    a.channels = number(x.size(1), "selective_scan_step");
    a.dstate = static_cast<int32_t>(A.size(1));
    a.groups = number(B.size(1), "selective_scan_step");
    a.dtype = dtype_of(x);
    a.softplus = softplus;
    check(lib.scan_step(&a, stream_of(x)), "selective_scan_step");
    changed(next);
    return variable_list{out};
}

// None, a tensor, or a tuple of them; the interpreter's lock is not held meanwhile.
template <class F>
py::object answer(F call) {
    std::optional<variable_list> got;
    {
        const py::gil_scoped_release unlocked;
        got = call();
    }
    if (!got) return py::none();
    if (got->size() == 1) return py::cast((*got)[0]);
    py::tuple tuple(got->size());
    for (size_t i = 0; i < got->size(); ++i) tuple[i] = py::cast((*got)[i]);
    return tuple;
}

}  // namespace

PYBIND11_MODULE(_calls, m) {
    m.def("bind", &bind);
    m.def("rms_norm", [](const Tensor& x, const Tensor& weight, const Maybe& residual, double eps) {
        return answer([&] { return rms_norm_call(x, weight, of(residual), eps); });
    });
    m.def("rms_norm_quant", [](const Tensor& x, const Tensor& weight, const Maybe& residual, double eps, int64_t group,
                               const Maybe& scale) {
        return answer([&] { return rms_norm_quant_call(x, weight, of(residual), eps, group, of(scale)); });
    });
    m.def("short_conv", [](const Tensor& x, const Tensor& weight, const Maybe& bias, bool silu, const Maybe& initial, const Maybe& cu,
                           bool want_final) {
        return answer([&] { return short_conv_call(x, weight, of(bias), silu, of(initial), of(cu), want_final); });
    });
    m.def("short_conv_step", [](const Tensor& x, const Tensor& state, const Tensor& weight, const Maybe& bias, bool silu,
                                const Maybe& slots, const Maybe& state_out) {
        return answer([&] { return short_conv_step_call(x, state, weight, of(bias), silu, of(slots), of(state_out)); });
    });
    m.def("selective_scan", [](const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D,
                               const Maybe& z, const Maybe& bias, bool softplus, const Maybe& initial, const Maybe& cu,
                               bool want_final) {
        return answer([&] {
            return selective_scan_call(x, dt, A, B, C, of(D), of(z), of(bias), softplus, of(initial), of(cu), want_final);
        });
    });
    m.def("selective_scan_step", [](const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                    const Tensor& state, const Maybe& D, const Maybe& z, const Maybe& bias, bool softplus,
                                    const Maybe& slots, const Maybe& state_out) {
        return answer([&] {
            return selective_scan_step_call(x, dt, A, B, C, state, of(D), of(z), of(bias), softplus, of(slots), of(state_out));
        });
    });
}
