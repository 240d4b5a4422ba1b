// aimet_amd/_native.so: layer norm and linear (miq_layer_norm_*, miq_linear_* of libmiq) as functions of torch tensors,
// with their backward passes as autograd nodes.
//
// The same could be written in Python over ctypes, as the rest of the package is.  A training step of a small layer is
// bound by the host, though: with Python nodes one norm, forward and backward, took 125 us of host time for 25 us of
// kernels, most of it because the backward pass runs in another thread, which first has to get the interpreter back.
// These nodes never enter the interpreter.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/library.h>

#include "../../include/miq.h"

namespace
{
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ----------------------------------------------------------------------------------------------------- arguments
// Every tensor that is defined lives on x's GPU and has x's type
void require_like(const Tensor& x, std::initializer_list<std::pair<const char*, const Tensor*>> others)
{
    TORCH_CHECK(x.is_cuda(), "aimet_amd kernels run on the GPU only; got a tensor on ", x.device());
    TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, "unsupported dtype ",
                x.scalar_type(), ": float32 and bfloat16 are implemented");
    for (const auto& [name, t] : others)
    {
        if (!t->defined())
            continue;
        TORCH_CHECK(t->is_cuda(), "aimet_amd kernels run on the GPU only; got a tensor on ", t->device());
        TORCH_CHECK(t->device() == x.device(), "tensors are on different devices: ", t->device(), " vs ", x.device());
        TORCH_CHECK(t->scalar_type() == x.scalar_type(), name, " is ", t->scalar_type(), " but the input is ",
                    x.scalar_type(), ": one type is expected");
    }
}

void check(int status)
{
    TORCH_CHECK(status == MIQ_OK, "libmiq status ", status, ": ", miq_last_error());
}

void* stream_of(const Tensor& x)
{
    return c10::hip::getCurrentHIPStream(x.get_device()).stream();
}

template <typename P>
P* data(const Tensor& t)
{
    return t.defined() ? static_cast<P*>(t.data_ptr()) : nullptr;
}

// t's values, row after row in memory (a lazily negated tensor, as the imaginary part of a conjugate is, holds others)
Tensor contiguous(const Tensor& t)
{
    return !t.defined() ? t : t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous();
}

void no_forward_mode(std::initializer_list<const Tensor*> tensors)
{
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(),
                    "aimet_amd kernels are not differentiated in forward mode: got a dual tensor");
}

// make_fx records torch's own operators below autograd, where nothing of a call here but its allocations goes by
void no_proxies()
{
    TORCH_CHECK(!c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                "aimet_amd kernels cannot be recorded into a graph of torch's operators");
}

bool traced()
{
    return at::tracer::impl::is_dispatch_enabled();
}

// what neither make_fx nor torch.jit.trace may record: the backward passes, and the functions that give or take statistics
void not_recorded()
{
    no_proxies();
    TORCH_CHECK(!traced(), "only layer_norm() and linear() of aimet_amd are recorded by a trace, no backward pass and nothing below them");
}

bool is_bf16(const Tensor& x)
{
    return x.scalar_type() == at::kBFloat16;
}

// ----------------------------------------------------------------------------------------------------- layer norm
int64_t rows_of(const Tensor& x, int64_t width)
{
    TORCH_CHECK(width >= 1 && x.numel() % width == 0, "a tensor of ", x.numel(), " elements has no rows of ", width);
    return x.numel() / width;
}

// x, weight and bias contiguous; stats: undefined, or receives float32 [2, rows]
Tensor layer_norm_fwd(const Tensor& x, int64_t width, const Tensor& weight, const Tensor& bias, double eps,
                      Tensor* stats)
{
    require_like(x, {{"weight", &weight}, {"bias", &bias}});
    const int64_t rows = rows_of(x, width);
    TORCH_CHECK(!weight.defined() || weight.numel() == width, "weight has ", weight.numel(), " elements, a row has ", width);
    TORCH_CHECK(!bias.defined() || bias.numel() == width, "bias has ", bias.numel(), " elements, a row has ", width);
    const c10::DeviceGuard guard(x.device());
    const Tensor xc = contiguous(x), w = contiguous(weight), b = contiguous(bias);
    Tensor y        = at::empty(x.sizes(), xc.options());
    float* mean     = nullptr;
    if (stats)
    {
        *stats = at::empty({2, rows}, xc.options().dtype(at::kFloat));
        mean   = data<float>(*stats);
    }
    float* rstd = mean ? mean + rows : nullptr;
    if (is_bf16(x))
        check(miq_layer_norm_fwd_bf16(data<uint16_t>(xc), data<uint16_t>(w), data<uint16_t>(b), rows, width, (float) eps,
                                      data<uint16_t>(y), mean, rstd, stream_of(x)));
    else
        check(miq_layer_norm_fwd_f32(data<float>(xc), data<float>(w), data<float>(b), rows, width, (float) eps,
                                     data<float>(y), mean, rstd, stream_of(x)));
    return y;
}

struct NormGrads
{
    Tensor x, weight, bias;
};

NormGrads layer_norm_bwd(const Tensor& x, const Tensor& grad, int64_t width, const Tensor& weight, const Tensor& stats,
                         bool want_x, bool want_weight, bool want_bias)
{
    require_like(x, {{"grad", &grad}, {"weight", &weight}});
    const int64_t rows = rows_of(x, width);
    TORCH_CHECK(grad.numel() == x.numel(), "x has ", x.numel(), " and grad ", grad.numel(), " elements");
    TORCH_CHECK(stats.defined() && stats.device() == x.device() && stats.scalar_type() == at::kFloat &&
                    stats.sizes() == at::IntArrayRef({2, rows}) && stats.is_contiguous(),
                "stats is not what layer_norm_fwd returned for these rows");
    TORCH_CHECK(!weight.defined() || weight.numel() == width, "weight has ", weight.numel(), " elements, a row has ", width);
    const c10::DeviceGuard guard(x.device());
    const Tensor xc = contiguous(x), g = contiguous(grad), w = contiguous(weight);
    NormGrads out;
    Tensor workspace;
    if (want_x)
        out.x = at::empty(x.sizes(), xc.options());
    if (want_weight)
        out.weight = at::empty({width}, xc.options());
    if (want_bias)
        out.bias = at::empty({width}, xc.options());
    if (want_weight || want_bias)
        workspace = at::empty({miq_layer_norm_bwd_workspace_bytes(rows, width)}, xc.options().dtype(at::kByte));
    const float* mean = data<float>(stats);
    if (is_bf16(x))
        check(miq_layer_norm_bwd_bf16(data<uint16_t>(xc), data<uint16_t>(g), data<uint16_t>(w), mean, mean + rows, rows,
                                      width, data<uint16_t>(out.x), data<uint16_t>(out.weight), data<uint16_t>(out.bias),
                                      data<void>(workspace), stream_of(x)));
    else
        check(miq_layer_norm_bwd_f32(data<float>(xc), data<float>(g), data<float>(w), mean, mean + rows, rows, width,
                                     data<float>(out.x), data<float>(out.weight), data<float>(out.bias),
                                     data<void>(workspace), stream_of(x)));
    return out;
}

// ---------------------------------------------------------------------------------------------------------- linear
int64_t linear_rows(const Tensor& x, const Tensor& weight)
{
    TORCH_CHECK(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1), "an input of shape ", x.sizes(),
                " does not go with a weight of shape ", weight.sizes(), ": [..., in] and [out, in] are expected");
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
        rows *= x.size(i);
    return rows;
}

bool at16(std::initializer_list<const Tensor*> tensors)
{
    uintptr_t bits = 0;
    for (const Tensor* t : tensors)
        bits |= reinterpret_cast<uintptr_t>(t->data_ptr());
    return bits % 16 == 0;
}

// saved: null, or receives what linear_bwd needs (undefined for activation 0)
Tensor linear_fwd(const Tensor& x, const Tensor& weight, const Tensor& bias, int activation, const Tensor& residual,
                  Tensor* saved)
{
    require_like(x, {{"weight", &weight}, {"bias", &bias}, {"residual", &residual}});
    const int64_t rows = linear_rows(x, weight), in = weight.size(1), out = weight.size(0);
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = out;
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == out), "bias has shape ", bias.sizes(), ", [", out,
                "] is expected");
    TORCH_CHECK(!residual.defined() || residual.sizes() == at::IntArrayRef(shape), "residual has shape ",
                residual.sizes(), ", ", at::IntArrayRef(shape), " is expected");
    const c10::DeviceGuard guard(x.device());
    const bool bf16 = is_bf16(x);
    const Tensor xc = contiguous(x), w = contiguous(weight), b = contiguous(bias), r = contiguous(residual);
    Tensor y = at::empty(shape, xc.options()), workspace;
    if (saved && activation)
        *saved = at::empty(shape, xc.options().dtype(bf16 ? at::kHalf : at::kFloat));
    const int64_t bytes = miq_linear_workspace_bytes(rows, in, out, activation, bf16, 0, at16({&xc, &w}));
    if (bytes)
        workspace = at::empty({bytes}, xc.options().dtype(at::kByte));
    if (bf16)
        check(miq_linear_fwd_bf16(data<uint16_t>(xc), data<uint16_t>(w), data<uint16_t>(b), data<uint16_t>(r), rows, in,
                                  out, activation, data<uint16_t>(y), saved ? data<uint16_t>(*saved) : nullptr,
                                  data<void>(workspace), bytes, stream_of(x)));
    else
        check(miq_linear_fwd_f32(data<float>(xc), data<float>(w), data<float>(b), data<float>(r), rows, in, out,
                                 activation, data<float>(y), saved ? data<float>(*saved) : nullptr,
                                 data<void>(workspace), bytes, stream_of(x)));
    return y;
}

struct LinearGrads
{
    Tensor x, weight, bias;
};

LinearGrads linear_bwd(const Tensor& grad, const Tensor& saved, const Tensor& x, const Tensor& weight, int activation,
                       bool want_x, bool want_weight, bool want_bias)
{
    require_like(x, {{"weight", &weight}, {"grad", &grad}});
    const int64_t rows = linear_rows(x, weight), in = weight.size(1), out = weight.size(0);
    const bool bf16 = is_bf16(x);
    TORCH_CHECK(grad.numel() == rows * out, "grad has ", grad.numel(), " elements, the output ", rows * out);
    TORCH_CHECK(!activation || (saved.defined() && saved.device() == x.device() && saved.is_contiguous() &&
                                saved.scalar_type() == (bf16 ? at::kHalf : at::kFloat) && saved.numel() == rows * out),
                "saved is not what linear_fwd returned for these shapes");
    const c10::DeviceGuard guard(x.device());
    const Tensor g = contiguous(grad), xc = contiguous(x), w = contiguous(weight);
    LinearGrads to;
    Tensor workspace;
    if (want_x)
        to.x = at::empty(x.sizes(), xc.options());
    if (want_weight)
        to.weight = at::empty({out, in}, xc.options());
    if (want_bias)
        to.bias = at::empty({out}, xc.options());
    const int64_t bytes = miq_linear_workspace_bytes(rows, in, out, activation, bf16, 1, at16({&g, &xc, &w}));
    if (bytes)
        workspace = at::empty({bytes}, xc.options().dtype(at::kByte));
    const Tensor z = activation ? saved : Tensor();
    if (bf16)
        check(miq_linear_bwd_bf16(data<uint16_t>(g), data<uint16_t>(z), data<uint16_t>(xc), data<uint16_t>(w), rows, in,
                                  out, activation, data<uint16_t>(to.x), data<uint16_t>(to.weight),
                                  data<uint16_t>(to.bias), data<void>(workspace), bytes, stream_of(x)));
    else
        check(miq_linear_bwd_f32(data<float>(g), data<float>(z), data<float>(xc), data<float>(w), rows, in, out,
                                 activation, data<float>(to.x), data<float>(to.weight), data<float>(to.bias),
                                 data<void>(workspace), bytes, stream_of(x)));
    return to;
}

// ------------------------------------------------------------------------------------------------- autograd nodes
// The gradients are not differentiable themselves: under create_graph they come out as what raises when differentiated
variable_list not_twice(variable_list grads)
{
    if (!at::GradMode::is_enabled())
        return grads;
    variable_list defined;
    for (const Tensor& t : grads)
        if (t.defined())
            defined.push_back(t);
    if (defined.empty())
        return grads;
    for (Tensor& t : defined)
        t.requires_grad_();
    torch::autograd::DelayedError error("trying to differentiate twice a function of aimet_amd that is differentiable once",
                                        (int64_t) defined.size());
    const variable_list marked = error.apply(std::move(defined));
    size_t k = 0;
    for (Tensor& t : grads)
        if (t.defined())
            t = marked[k++];
    return grads;
}

// A leaf's gradient is accumulated on the stream of the first graph that is still alive.  Where that is an eager one of the
// default stream, a backward pass under capture would have the default stream wait for a captured one, which ends the
// process: refused beforehand.  Only leaves that this pass wants a gradient of are looked at, also those behind the casts that
// autocast makes here.
void refuse_eager_leaves_under_capture()
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None)
        return;
    const auto node = torch::autograd::get_current_node();
    if (!node)
        return;
    for (size_t i = 0; i < node->num_outputs(); ++i)
    {
        if (!node->task_should_compute_output(i))
            continue;
        torch::autograd::Node* next = node->next_edge(i).function.get();
        while (next->name() == "ToCopyBackward0" && next->num_outputs() == 1 && next->task_should_compute_output(0))
            next = next->next_edge(0).function.get();
        if (next->name() != "torch::autograd::AccumulateGrad")
            continue;
        const std::optional<c10::Stream> stream = next->stream();
        TORCH_CHECK(!stream || stream->id() != 0, "a backward pass cannot be captured into a graph while an eager autograd graph "
                    "of the same leaves, made on the default stream, is alive: delete its outputs first");
    }
}

// A node has an edge for every tensor it was given, and none for those it was not
std::optional<Tensor> given(const Tensor& t)
{
    return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode>
{
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_,
                          const std::optional<Tensor>& bias_, int64_t width, double eps)
    {
        const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
        Tensor stats;
        const Tensor xc = contiguous(x);
        Tensor y        = layer_norm_fwd(xc, width, weight, bias, eps, &stats);
        ctx->save_for_backward({xc, weight, stats});
        ctx->saved_data["width"] = width;
        if (weight.defined())
            ctx->saved_data["weight_shape"] = weight.sizes().vec();
        if (bias.defined())
            ctx->saved_data["bias_shape"] = bias.sizes().vec();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        not_recorded();
        refuse_eager_leaves_under_capture();
        const bool twice = at::GradMode::is_enabled();
        variable_list out(5);
        {
            const at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            size_t edge      = 0;
            const bool x     = ctx->needs_input_grad(edge++);
            const bool w     = ctx->saved_data.count("weight_shape") && ctx->needs_input_grad(edge++);
            const bool b     = ctx->saved_data.count("bias_shape") && ctx->needs_input_grad(edge++);
            NormGrads g = layer_norm_bwd(saved[0], grads[0], ctx->saved_data["width"].toInt(), saved[1], saved[2], x, w, b);
            out[0] = g.x;
            if (g.weight.defined())
                out[1] = g.weight.view(ctx->saved_data["weight_shape"].toIntVector());
            if (g.bias.defined())
                out[2] = g.bias.view(ctx->saved_data["bias_shape"].toIntVector());
        }
        return twice ? not_twice(std::move(out)) : out;
    }
};

struct LinearNode : torch::autograd::Function<LinearNode>
{
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                          const std::optional<Tensor>& bias_, const std::optional<Tensor>& residual_, int64_t activation,
                          bool products)
    {
        const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
        // `products`: x, weight or bias want a gradient, not the residual alone
        Tensor saved;
        const Tensor xc = contiguous(x), w = contiguous(weight);
        Tensor y        = linear_fwd(xc, w, bias, (int) activation, residual, products ? &saved : nullptr);
        if (products)
            ctx->save_for_backward({xc, w, saved});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["bias"]       = bias.defined();
        ctx->saved_data["residual"]   = residual.defined();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        not_recorded();
        refuse_eager_leaves_under_capture();
        const bool twice = at::GradMode::is_enabled();
        variable_list out(6);
        size_t edge         = 0;
        const bool x        = ctx->needs_input_grad(edge++), weight = ctx->needs_input_grad(edge++);
        const bool bias     = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(edge++);
        const bool residual = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge++);
        if (x || weight || bias)
        {
            const at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            LinearGrads g = linear_bwd(grads[0], saved[2], saved[0], saved[1],
                                       (int) ctx->saved_data["activation"].toInt(), x, weight, bias);
            out[0] = g.x, out[1] = g.weight, out[2] = g.bias;
        }
        if (twice)
            out = not_twice(std::move(out));
        if (residual)
            out[3] = grads[0];
        return out;
    }
};

bool differentiates(std::initializer_list<const Tensor*> tensors)
{
    if (!at::GradMode::is_enabled())
        return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad())
            return true;
    return false;
}

Tensor cast(const Tensor& t, at::ScalarType type)
{
    return t.defined() && t.is_floating_point() && t.scalar_type() != at::kDouble && t.scalar_type() != type ? t.to(type) : t;
}

Tensor layer_norm(const Tensor& x_, at::IntArrayRef shape, const Tensor& weight_, const Tensor& bias_, double eps)
{
    Tensor x = x_, weight = weight_, bias = bias_;
    const int64_t dims = (int64_t) shape.size();
    TORCH_CHECK(dims >= 1 && x.dim() >= dims && x.sizes().slice(x.dim() - dims) == shape, "normalized_shape ", shape,
                " is not the end of the input's shape ", x.sizes());
    TORCH_CHECK(!weight.defined() || weight.sizes() == shape, "weight has shape ", weight.sizes(), ", ", shape,
                " is expected");
    TORCH_CHECK(!bias.defined() || bias.sizes() == shape, "bias has shape ", bias.sizes(), ", ", shape, " is expected");
    if (at::autocast::is_autocast_enabled(at::kCUDA))
        x = cast(x, at::kFloat), weight = cast(weight, at::kFloat), bias = cast(bias, at::kFloat);
    no_forward_mode({&x, &weight, &bias});
    no_proxies();
    int64_t width = 1;
    for (const int64_t d : shape)
        width *= d;
    if (differentiates({&x, &weight, &bias}))
        return LayerNormNode::apply(x, given(weight), given(bias), width, eps);
    return layer_norm_fwd(x, width, weight, bias, eps, nullptr);
}

Tensor linear(const Tensor& x_, const Tensor& weight_, const Tensor& bias_, int64_t activation, const Tensor& residual_)
{
    Tensor x = x_, weight = weight_, bias = bias_, residual = residual_;
    if (at::autocast::is_autocast_enabled(at::kCUDA))
    {
        const at::ScalarType type = at::autocast::get_autocast_dtype(at::kCUDA);
        x = cast(x, type), weight = cast(weight, type), bias = cast(bias, type), residual = cast(residual, type);
    }
    no_forward_mode({&x, &weight, &bias, &residual});
    no_proxies();
    if (differentiates({&x, &weight, &bias, &residual}))
        return LinearNode::apply(x, weight, given(bias), given(residual), activation,
                                 differentiates({&x, &weight, &bias}));
    return linear_fwd(x, weight, bias, (int) activation, residual, nullptr);
}

// ------------------------------------------------------------------------------------------------------- tracing
// torch.jit.trace records what goes through the dispatcher.  Of the calls above that is only the allocation of the result, so
// a traced model would return memory that nobody wrote.  While a trace is on, layer_norm() and linear() therefore go through
// the dispatcher as well, as operators of their own; at other times they do not pay for it.
Tensor layer_norm_operator(const Tensor& input, at::IntArrayRef shape, const std::optional<Tensor>& weight,
                           const std::optional<Tensor>& bias, double eps)
{
    return layer_norm(input, shape, weight.value_or(Tensor()), bias.value_or(Tensor()), eps);
}

Tensor linear_operator(const Tensor& input, const Tensor& weight, const std::optional<Tensor>& bias, int64_t activation,
                       const std::optional<Tensor>& residual)
{
    return linear(input, weight, bias.value_or(Tensor()), activation, residual.value_or(Tensor()));
}

Tensor recorded_layer_norm(const Tensor& x, at::IntArrayRef shape, const Tensor& weight, const Tensor& bias, double eps)
{
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("aimet_amd::layer_norm", "")
                               .typed<decltype(layer_norm_operator)>();
    return op.call(x, shape, given(weight), given(bias), eps);
}

Tensor recorded_linear(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t activation, const Tensor& residual)
{
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("aimet_amd::linear", "")
                               .typed<decltype(linear_operator)>();
    return op.call(x, weight, given(bias), activation, given(residual));
}

// ---------------------------------------------------------------------------------------------- Python's side of it
// Arguments come by position, in full: the functions of the package that call these have names and defaults.
Tensor tensor_at(PyObject* const* args, int i, const char* name, bool optional)
{
    if (optional && args[i] == Py_None)
        return Tensor();
    TORCH_CHECK_TYPE(THPVariable_Check(args[i]), name, " must be a tensor, not ", Py_TYPE(args[i])->tp_name);
    return THPVariable_Unpack(args[i]);
}

int64_t integer(PyObject* o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred())
        throw python_error();
    return v;
}

double real(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred())
        throw python_error();
    return v;
}

PyObject* wrapped(const Tensor& t)
{
    if (!t.defined())
        Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}

PyObject* tuple_of(std::initializer_list<Tensor> tensors)
{
    THPObjectPtr out(PyTuple_New((Py_ssize_t) tensors.size()));
    if (!out)
        throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor& t : tensors)
        PyTuple_SET_ITEM(out.get(), i++, wrapped(t));
    return out.release();
}

void expect(Py_ssize_t got, Py_ssize_t want)
{
    TORCH_CHECK_TYPE(got == want, want, " arguments are expected, not ", got);
}

PyObject* py_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    expect(n, 5);
    c10::SmallVector<int64_t, 4> shape;
    if (PyLong_Check(args[1]))
        shape.push_back(integer(args[1]));
    else
    {
        THPObjectPtr items(PySequence_Fast(args[1], "normalized_shape must be an integer or a sequence of them"));
        if (!items)
            throw python_error();
        for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(items.get()); ++i)
            shape.push_back(integer(PySequence_Fast_GET_ITEM(items.get(), i)));
    }
    return wrapped((traced() ? recorded_layer_norm : layer_norm)(tensor_at(args, 0, "input", false), shape,
                                                                 tensor_at(args, 2, "weight", true),
                                                                 tensor_at(args, 3, "bias", true), real(args[4])));
    END_HANDLE_TH_ERRORS
}

PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    expect(n, 5);
    return wrapped((traced() ? recorded_linear : linear)(tensor_at(args, 0, "input", false), tensor_at(args, 1, "weight", false),
                                                         tensor_at(args, 2, "bias", true), integer(args[3]),
                                                         tensor_at(args, 4, "residual", true)));
    END_HANDLE_TH_ERRORS
}

PyObject* py_layer_norm_fwd(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    expect(n, 6);
    not_recorded();
    const at::NoGradGuard no_grad;
    Tensor stats;
    const Tensor y = layer_norm_fwd(tensor_at(args, 0, "x", false), integer(args[1]), tensor_at(args, 2, "weight", true),
                                    tensor_at(args, 3, "bias", true), real(args[4]),
                                    PyObject_IsTrue(args[5]) ? &stats : nullptr);
    return tuple_of({y, stats});
    END_HANDLE_TH_ERRORS
}

PyObject* py_layer_norm_bwd(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    expect(n, 8);
    not_recorded();
    const at::NoGradGuard no_grad;
    const NormGrads g = layer_norm_bwd(tensor_at(args, 0, "x", false), tensor_at(args, 1, "grad", false), integer(args[2]),
                                       tensor_at(args, 3, "weight", true), tensor_at(args, 4, "stats", false),
                                       PyObject_IsTrue(args[5]), PyObject_IsTrue(args[6]), PyObject_IsTrue(args[7]));
    return tuple_of({g.x, g.weight, g.bias});
    END_HANDLE_TH_ERRORS
}

PyObject* py_linear_fwd(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    expect(n, 6);
    not_recorded();
    const at::NoGradGuard no_grad;
    Tensor saved;
    const Tensor y = linear_fwd(tensor_at(args, 0, "x", false), tensor_at(args, 1, "weight", false),
                                tensor_at(args, 2, "bias", true), (int) integer(args[3]),
                                tensor_at(args, 4, "residual", true), PyObject_IsTrue(args[5]) ? &saved : nullptr);
    return tuple_of({y, saved});
    END_HANDLE_TH_ERRORS
}

PyObject* py_linear_bwd(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    expect(n, 8);
    not_recorded();
    const at::NoGradGuard no_grad;
    const LinearGrads g = linear_bwd(tensor_at(args, 0, "grad", false), tensor_at(args, 1, "saved", true),
                                     tensor_at(args, 2, "x", false), tensor_at(args, 3, "weight", false),
                                     (int) integer(args[4]), PyObject_IsTrue(args[5]), PyObject_IsTrue(args[6]),
                                     PyObject_IsTrue(args[7]));
    return tuple_of({g.x, g.weight, g.bias});
    END_HANDLE_TH_ERRORS
}

PyCFunction as_method(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t))
{
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f));
}
}   // namespace

TORCH_LIBRARY(aimet_amd, m)
{
    m.def("layer_norm(Tensor input, int[] normalized_shape, Tensor? weight, Tensor? bias, float eps) -> Tensor",
          layer_norm_operator);
    m.def("linear(Tensor input, Tensor weight, Tensor? bias, int activation, Tensor? residual) -> Tensor", linear_operator);
}

PyMODINIT_FUNC PyInit__native()
{
    static PyMethodDef methods[] = {{"layer_norm", as_method(py_layer_norm), METH_FASTCALL, nullptr},
                                    {"linear", as_method(py_linear), METH_FASTCALL, nullptr},
                                    {"layer_norm_fwd", as_method(py_layer_norm_fwd), METH_FASTCALL, nullptr},
                                    {"layer_norm_bwd", as_method(py_layer_norm_bwd), METH_FASTCALL, nullptr},
                                    {"linear_fwd", as_method(py_linear_fwd), METH_FASTCALL, nullptr},
                                    {"linear_bwd", as_method(py_linear_bwd), METH_FASTCALL, nullptr},
                                    {nullptr, nullptr, 0, nullptr}};
    static PyModuleDef module    = {PyModuleDef_HEAD_INIT, "_native",
                                    "Layer norm and linear of libmiq as functions of torch tensors", -1, methods};
    return PyModule_Create(&module);
}
