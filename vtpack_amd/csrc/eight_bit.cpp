// The operators on blocks of 8-bit numbers as torch calls them: autograd nodes of the Linear, GELU and LayerNorm that keep their input in
// blocks.  Host code only, see training.cpp.
#include "training.h"

namespace {

using namespace vtdge_training;

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t last_of(const Tensor &x) { return x.size(-1); }
int64_t rows_in(const Tensor &x) { return x.size(-1) > 0 ? x.numel() / x.size(-1) : 0; }
// include/vtdge.h; the same without a library call
int64_t blocks_bytes(int64_t rows, int64_t n) { return rows * (up(n, 128) + up((n + 127) / 128, 4)); }

// x [..., n] as rows of memory, n dense elements each, in place where it lies so (and holds its numbers, not their negation)
Tensor flat(const Tensor &x)
{
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Tensor x_ = x.is_neg() ? x.resolve_neg() : x;
    Tensor t = x_.dim() == 2 ? x_ : x_.reshape({rows_in(x), last_of(x)});
    const bool dense = t.size(1) == 1 || t.stride(1) == 1, apart = t.size(0) <= 1 || t.stride(0) >= t.size(1);
    return dense && apart ? t : t.contiguous();
}
Tensor flat_vector(const Tensor &t)
{
    const at::AutoDispatchBelowADInplaceOrView plain;
    return (t.is_neg() ? t.resolve_neg() : t).contiguous();
}
at::DimVector with_last(const Tensor &x, int64_t n)
{
    at::DimVector d(x.sizes().begin(), x.sizes().end());
    d.back() = n;
    return d;
}
bool activation(const Tensor &t)
{
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.dim() >= 1 && t.size(-1) > 0 &&
           (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16);
}
// blocks that hooks on saved tensors may have brought back
void need_blocks(const OperandChecks &check, const Tensor &blocks, const Tensor &like, int64_t rows, int64_t n)
{
    check.need(plain_beside(blocks, like, at::kByte) && blocks.dim() == 1 && blocks.numel() == blocks_bytes(rows, n) && (uintptr_t)blocks.data_ptr() % 128 == 0,
               "the blocks kept have to be those of the forward call");
}
void need_gradient(const OperandChecks &check, const Tensor &grad, at::ScalarType type)
{
    check.need(grad.is_cuda() && grad.layout() == at::kStrided && grad.scalar_type() == type, "the gradient has to be strided, of the result's type, on its GPU");
}

// ------------------------------------------------------------------------------------------------ Linear
struct Linear8Backward : torch::autograd::Node {
    SavedVariable x_blocks, w_blocks;               // undefined where no gradient reads them
    int64_t rows, out, width; at::ScalarType type; at::DimVector sizes; bool has_bias;

    variable_list apply(variable_list &&grads) override
    {
        no_second_order("linear_8bit");
        std::lock_guard<std::mutex> hold(mutex_);
        const Tensor x = x_blocks.unpack(), w = w_blocks.unpack();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const OperandChecks check{"linear_8bit"};
        need_gradient(check, grads[0], type);
        const c10::DeviceGuard guard(grads[0].device());
        const Tensor g = flat(grads[0]);
        variable_list o(3);
        if (task_should_compute_output(0)) o[0] = fresh(g, sizes, type);
        if (task_should_compute_output(1)) o[1] = fresh(g, {out, width}, type);
        if (has_bias && task_should_compute_output(2)) o[2] = fresh(g, {out}, type);
        if (rows == 0) {
            for (Tensor &t : o)
                if (t.defined()) t.zero_();
            return o;
        }
        if (o[0].defined()) need_blocks(check, w, g, out, width);
        if (o[1].defined()) need_blocks(check, x, g, rows, width);
        const int64_t pitch = pitch_of(g);
        const int dtype = code_of(g);
        const bool lies = dtype == VTDGE_BF16 && out % 64 == 0 && pitch % 8 == 0 && pitch < (1 << 22) && (uintptr_t)g.data_ptr() % 16 == 0;
        const int how = (lies ? VTDGE_8BIT_GRADIENT_LIES : 0) | (o[0].defined() ? 0 : VTDGE_8BIT_NO_DX) | (o[1].defined() ? 0 : VTDGE_8BIT_NO_DWEIGHT) |
                        (o[2].defined() ? 0 : VTDGE_8BIT_NO_DBIAS);
        const int64_t bytes = bytes_of<5>({rows, out, width, how, dtype}, [&] { return lib.linear_8bit_backward_workspace(rows, out, width, how, dtype); });
        const Tensor ws = bytes > 0 ? fresh(g, {bytes}, at::kByte) : Tensor();
        must(lib.linear_8bit_backward(g.data_ptr(), pitch, o[1].defined() ? x.data_ptr() : nullptr, o[0].defined() ? w.data_ptr() : nullptr, rows, out, width,
                                      at_of(ws), bytes, at_of(o[0]), at_of(o[1]), at_of(o[2]), dtype, stream_of(g)),
             "vtdge_linear_8bit_backward");
        return o;
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> hold(mutex_);
        x_blocks.reset_data(), w_blocks.reset_data();
    }
    std::string name() const override { return "Linear8bitBackward"; }
};

// weight [out, width], or undefined with its blocks in w_blocks
Tensor linear_8bit(const Tensor &x, const Tensor &weight, Tensor w_blocks, int64_t out, const Tensor &bias, int act)
{
    no_forward_mode("linear_8bit", {&x, &weight, &bias});
    const bool trains = torch::autograd::compute_requires_grad(x, weight, bias);
    if (trains && act != VTDGE_ACT_NONE) throw std::runtime_error("linear_8bit: an activation with gradients is an operator of its own, as gelu_8bit");
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = rows_in(x), width = last_of(x);
    if (trains && rows > VTDGE_MAX_ROWS_8BIT) throw std::runtime_error("linear_8bit: gradients of " + std::to_string(rows) + " rows, up to " + std::to_string(VTDGE_MAX_ROWS_8BIT) + " are supported");
    const Tensor y = fresh(x, with_last(x, out), x.scalar_type());
    Tensor x_blocks;
    if (rows > 0) {
        const Tensor xf = flat(x), wf = weight.defined() ? flat(weight) : Tensor(), b = bias.defined() ? flat_vector(bias) : Tensor();
        if (trains && weight.defined() && weight.requires_grad()) x_blocks = fresh(x, {blocks_bytes(rows, width)}, at::kByte);
        if (trains && weight.defined() && x.requires_grad()) w_blocks = fresh(x, {blocks_bytes(out, width)}, at::kByte);
        const int dtype = code_of(x);
        const int how = (!wf.defined() ? VTDGE_8BIT_WEIGHT_GIVEN : w_blocks.defined() ? VTDGE_8BIT_WEIGHT_KEPT : 0) | (x_blocks.defined() ? VTDGE_8BIT_X_KEPT : 0);
        const int64_t bytes = bytes_of<5>({rows, out, width, how, dtype}, [&] { return lib.linear_8bit_workspace(rows, out, width, how, dtype); });
        const Tensor ws = bytes > 0 ? fresh(x, {bytes}, at::kByte) : Tensor();
        must(lib.linear_8bit(xf.data_ptr(), pitch_of(xf), at_of(wf), wf.defined() ? pitch_of(wf) : 0, at_of(w_blocks), at_of(b), y.data_ptr(), at_of(x_blocks),
                             rows, out, width, act, at_of(ws), bytes, dtype, stream_of(x)),
             "vtdge_linear_8bit");
    }
    if (trains) {
        auto node = std::shared_ptr<Linear8Backward>(new Linear8Backward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
        node->x_blocks = SavedVariable(x_blocks, false), node->w_blocks = SavedVariable(x.requires_grad() ? w_blocks : Tensor(), false);
        node->rows = rows, node->out = out, node->width = width, node->type = x.scalar_type(), node->has_bias = bias.defined();
        node->sizes = at::DimVector(x.sizes().begin(), x.sizes().end());
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ------------------------------------------------------------------------------------------------ GELU
struct Gelu8Backward : torch::autograd::Node {
    SavedVariable blocks;
    at::ScalarType type; at::DimVector sizes;

    variable_list apply(variable_list &&grads) override
    {
        no_second_order("gelu_8bit");
        std::lock_guard<std::mutex> hold(mutex_);
        const Tensor b = blocks.unpack();
        if (!grads[0].defined()) return {Tensor()};
        const OperandChecks check{"gelu_8bit"};
        need_gradient(check, grads[0], type);
        const c10::DeviceGuard guard(grads[0].device());
        const Tensor g = flat(grads[0]), dx = fresh(g, sizes, type);
        if (g.numel() == 0) return {dx};
        need_blocks(check, b, g, g.size(0), g.size(1));
        must(lib.gelu_8bit_backward(g.data_ptr(), pitch_of(g), g.size(0), g.size(1), b.data_ptr(), dx.data_ptr(), code_of(g), stream_of(g)),
             "vtdge_gelu_8bit_backward");
        return {dx};
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> hold(mutex_);
        blocks.reset_data();
    }
    std::string name() const override { return "Gelu8bitBackward"; }
};
Tensor gelu_8bit(const Tensor &x)
{
    no_forward_mode("gelu_8bit", {&x});
    const c10::DeviceGuard guard(x.device());
    const bool trains = torch::autograd::compute_requires_grad(x);
    const int64_t rows = rows_in(x), n = last_of(x);
    const Tensor y = fresh(x, x.sizes(), x.scalar_type()), blocks = trains ? fresh(x, {blocks_bytes(rows, n)}, at::kByte) : Tensor();
    if (rows > 0) {
        const Tensor xf = flat(x);
        must(lib.gelu_8bit(xf.data_ptr(), pitch_of(xf), rows, n, y.data_ptr(), at_of(blocks), code_of(x), stream_of(x)), "vtdge_gelu_8bit");
    }
    if (trains) {
        auto node = std::shared_ptr<Gelu8Backward>(new Gelu8Backward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->blocks = SavedVariable(blocks, false), node->type = x.scalar_type(), node->sizes = at::DimVector(x.sizes().begin(), x.sizes().end());
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ------------------------------------------------------------------------------------------------ LayerNorm
struct LayerNorm8Backward : torch::autograd::Node {
    SavedVariable blocks, rstd, weight;
    at::ScalarType type; at::DimVector sizes;

    variable_list apply(variable_list &&grads) override
    {
        no_second_order("layer_norm_8bit");
        std::lock_guard<std::mutex> hold(mutex_);
        const Tensor b = blocks.unpack(), r = rstd.unpack(), w_ = weight.unpack();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const OperandChecks check{"layer_norm_8bit"};
        need_gradient(check, grads[0], type);
        const c10::DeviceGuard guard(grads[0].device());
        const Tensor g = flat(grads[0]);
        const int64_t rows = g.size(0), n = sizes.back();
        variable_list o(3);
        if (task_should_compute_output(0)) o[0] = fresh(g, sizes, type);
        for (int i = 1; i < 3; i++)
            if (task_should_compute_output(i)) o[i] = fresh(g, {n}, type);
        if (rows == 0) {
            for (Tensor &t : o)
                if (t.defined()) t.zero_();
            return o;
        }
        need_blocks(check, b, g, rows, n);
        check.need(plain_beside(r, g, at::kFloat) && r.dim() == 1 && r.size(0) == rows, "rstd has to be that of the forward call");
        check.need(w_.defined() && w_.device() == g.device() && w_.scalar_type() == type && w_.dim() == 1 && w_.size(0) == n, "weight has to be that of the forward call");
        const Tensor w = flat_vector(w_);
        const int64_t bytes = bytes_of<2>({rows, n}, [&] { return lib.layernorm_8bit_backward_workspace(rows, n); });
        const Tensor ws = fresh(g, {bytes}, at::kByte);
        must(lib.layernorm_8bit_backward(g.data_ptr(), pitch_of(g), w.data_ptr(), b.data_ptr(), r.data_ptr<float>(), rows, n, ws.data_ptr(), bytes, at_of(o[0]),
                                         at_of(o[1]), at_of(o[2]), code_of(g), stream_of(g)),
             "vtdge_layernorm_8bit_backward");
        return o;
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> hold(mutex_);
        blocks.reset_data(), rstd.reset_data(), weight.reset_data();
    }
    std::string name() const override { return "LayerNorm8bitBackward"; }
};
Tensor layer_norm_8bit(const Tensor &x, const Tensor &weight, const Tensor &bias, double eps)
{
    no_forward_mode("layer_norm_8bit", {&x, &weight, &bias});
    const c10::DeviceGuard guard(x.device());
    const bool trains = torch::autograd::compute_requires_grad(x, weight, bias);
    const int64_t rows = rows_in(x), n = last_of(x);
    const Tensor y = fresh(x, x.sizes(), x.scalar_type());
    Tensor blocks, rstd;
    if (trains) blocks = fresh(x, {blocks_bytes(rows, n)}, at::kByte), rstd = fresh(x, {rows}, at::kFloat);
    if (rows > 0) {
        const Tensor xf = flat(x), w = flat_vector(weight), b = flat_vector(bias);
        must(lib.layernorm_8bit(xf.data_ptr(), pitch_of(xf), w.data_ptr(), b.data_ptr(), (float)eps, rows, n, y.data_ptr(), at_of(blocks), (float *)at_of(rstd),
                                code_of(x), stream_of(x)),
             "vtdge_layernorm_8bit");
    }
    if (trains) {
        auto node = std::shared_ptr<LayerNorm8Backward>(new LayerNorm8Backward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
        node->blocks = SavedVariable(blocks, false), node->rstd = SavedVariable(rstd, false), node->weight = SavedVariable(weight, false);
        node->type = x.scalar_type(), node->sizes = at::DimVector(x.sizes().begin(), x.sizes().end());
        torch::autograd::set_history(y, node);
    }
    return y;
}

bool vector_beside(const Tensor &t, const Tensor &x, int64_t n)
{
    return t.defined() && t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.layout() == at::kStrided && t.dim() == 1 && t.size(0) == n;
}
bool blocks_beside(const Tensor &t, const Tensor &x, int64_t rows, int64_t n)
{
    return plain_beside(t, x, at::kByte) && t.dim() == 1 && t.numel() == blocks_bytes(rows, n) && (uintptr_t)t.data_ptr() % 128 == 0;
}

}  // namespace

// Each answers None to operands that are not the kernels', for its caller to say what is wrong with them.
namespace vtdge_training {

// (x [..., n]) -> the buffer of its blocks
PyObject *py_quantize_blocks(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 1, [&]() -> PyObject * {
        no_tracing("quantize_blocks");
        if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
        const Tensor x = tensor(a[0]);
        if (!activation(x)) Py_RETURN_NONE;
        Tensor blocks;
        {
            const NoGil no;
            const c10::DeviceGuard guard(x.device());
            const int64_t rows = rows_in(x), width = last_of(x);
            blocks = fresh(x, {blocks_bytes(rows, width)}, at::kByte);
            if (rows > 0) {
                const Tensor xf = flat(x);
                must(lib.quantize_blocks(xf.data_ptr(), pitch_of(xf), rows, width, blocks.data_ptr(), code_of(x), stream_of(x)), "vtdge_quantize_blocks");
            }
        }
        return wrap(blocks);
    });
}
// (buffer, sizes of the numbers, whether in float32) -> the numbers
PyObject *py_dequantize_blocks(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 3, [&]() -> PyObject * {
        no_tracing("dequantize");
        const Tensor blocks = tensor(a[0]);
        if (!PyTuple_Check(a[1])) throw std::runtime_error("dequantize: expected a tuple of sizes");
        at::DimVector sizes;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[1]); i++) sizes.push_back(whole(PyTuple_GET_ITEM(a[1], i)));
        const at::ScalarType type = whole(a[2]) != 0 ? at::kFloat : at::kBFloat16;
        int64_t rows = 1;
        for (size_t i = 0; i + 1 < sizes.size(); i++) rows *= sizes[i];
        const OperandChecks check{"dequantize"};
        check.need(blocks.defined() && blocks.is_cuda() && !sizes.empty() && sizes.back() > 0, "blocks have to be on a GPU");
        need_blocks(check, blocks, blocks, rows, sizes.back());
        Tensor out;
        {
            const NoGil no;
            const c10::DeviceGuard guard(blocks.device());
            out = fresh(blocks, sizes, type);
            if (rows > 0) must(lib.dequantize_blocks(blocks.data_ptr(), rows, sizes.back(), out.data_ptr(), code_of(out), stream_of(out)), "vtdge_dequantize_blocks");
        }
        return wrap(out);
    });
}
// (x, weight or the buffer of its blocks, its rows or None with a weight, bias or None, act)
PyObject *py_linear_8bit(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 5, [&]() -> PyObject * {
        no_tracing("linear_8bit");
        if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || (a[3] != Py_None && !THPVariable_Check(a[3]))) Py_RETURN_NONE;
        const Tensor x = tensor(a[0]), w = tensor(a[1]), b = tensor(a[3]);
        if (!activation(x)) Py_RETURN_NONE;
        const bool kept = a[2] != Py_None;
        int64_t out;
        if (kept) {
            out = whole(a[2]);
            if (out < 1 || !blocks_beside(w, x, out, last_of(x))) Py_RETURN_NONE;
        } else {
            if (!w.defined() || w.device() != x.device() || w.scalar_type() != x.scalar_type() || w.layout() != at::kStrided || w.dim() != 2 ||
                w.size(1) != last_of(x) || w.size(0) < 1)
                Py_RETURN_NONE;
            out = w.size(0);
        }
        if (b.defined() && !vector_beside(b, x, out)) Py_RETURN_NONE;
        const int act = (int)whole(a[4]);
        Tensor y;
        {
            const NoGil no;
            y = linear_8bit(x, kept ? Tensor() : w, kept ? w : Tensor(), out, b, act);
        }
        return wrap(y);
    });
}
PyObject *py_gelu_8bit(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 1, [&]() -> PyObject * {
        no_tracing("gelu_8bit");
        if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
        const Tensor x = tensor(a[0]);
        if (!activation(x)) Py_RETURN_NONE;
        Tensor y;
        {
            const NoGil no;
            y = gelu_8bit(x);
        }
        return wrap(y);
    });
}
// (x, weight, bias, eps)
PyObject *py_layer_norm_8bit(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 4, [&]() -> PyObject * {
        no_tracing("layer_norm_8bit");
        for (int i = 0; i < 3; i++)
            if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
        if (!PyFloat_Check(a[3])) Py_RETURN_NONE;
        const Tensor x = tensor(a[0]), w = tensor(a[1]), b = tensor(a[2]);
        const double eps = real(a[3]);
        if (!activation(x) || last_of(x) > VTDGE_MAX_NORM_8BIT || !vector_beside(w, x, last_of(x)) || !vector_beside(b, x, last_of(x)) || !(eps >= 0)) Py_RETURN_NONE;
        Tensor y;
        {
            const NoGil no;
            y = layer_norm_8bit(x, w, b, eps);
        }
        return wrap(y);
    });
}

}  // namespace vtdge_training
