// The operators of a training step as torch calls them: cross entropy and balance of gates as autograd nodes, the checks of an
// AdamW step.  Host code only; the kernels are behind the C entry points of vtdge.h, whose addresses `bind` takes.
//
// Why this is native: small calls of these operators are bound by the host.  A backward pass runs in the engine's own thread, whose
// core comes out of its sleep for it, and what Python does there (the interpreter lock, four allocations, 24 arguments) took 32 of
// the 122 us of a DeiT-S classifier's loss with its gradients (73 so); a step over 200 weights looked at some 1000 objects, 77 us beside the
// 31 us of its kernels (9 so).
#include "training.h"

namespace {

using namespace vtdge_training;

// ------------------------------------------------------------------------------------------------ cross entropy
enum Reduction { NONE, MEAN, SUM };
constexpr int64_t KEEP_LAID_OUT = 320 << 20;    // bytes

struct Rows {
    int64_t rows, classes; int width, dtype, lie;   // (a width beyond 32 bits is the largest one within, which the library refuses)
    Rows(const Tensor &x, const Tensor &w)
        : rows(x.size(0)), classes(w.size(0)), width((int)std::min<int64_t>(x.size(1), INT32_MAX)), dtype(code_of(x)),
          lie((lies(x) ? VTDGE_CE_X_LIES : 0) + (lies(w) ? VTDGE_CE_WEIGHT_LIES : 0)) {}
    // whether the kernels read an operand where it lies
    bool lies(const Tensor &t) const
    {
        const int64_t pitch = pitch_of(t);
        return dtype == VTDGE_BF16 && width % 64 == 0 && pitch % 8 == 0 && pitch < (1 << 22) && (uintptr_t)t.data_ptr() % 16 == 0;
    }
    int64_t workspace(bool backward, bool keeps) const
    {
        const int how = lie + (backward ? VTDGE_CE_BACKWARD : 0) + (keeps ? VTDGE_CE_KEEPS : 0);
        return bytes_of<5>({rows, classes, width, dtype, how}, [&] { return lib.cross_entropy_workspace(rows, classes, width, dtype, how); });
    }
    // Operands that do not lie as the kernels read them are laid out in the workspace, with the logits in fp32.  It is kept for the
    // gradients (fp32 1 x 363 x 25766: 20 us of 136 for laying them out again) up to this size, so that no more memory waits between
    // the calls; behind it all is worked out again.
    bool keeps() const { return (dtype != VTDGE_BF16 || width % 64 != 0) && lib.cross_entropy_laid_out(rows, classes, width, dtype) <= KEEP_LAID_OUT; }
};

struct Forward {
    Tensor loss, stats, laid_out;
};
Forward cross_entropy(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &target, int64_t ignore, double smoothing, int reduction,
                      bool for_gradients)
{
    const c10::DeviceGuard guard(x.device());
    const Rows s(x, w);
    const bool keeps = for_gradients && s.keeps();
    Tensor ws = fresh(x, {s.workspace(false, keeps)}, at::kByte);
    // the rows' largest logits, 1 / sums, 1 / the number of rows that count, the rows' losses; the loss is memory of its own, for a
    // caller to change in place
    const Tensor stats = fresh(x, {3 * s.rows + 1}, at::kFloat);
    const Tensor loss = reduction == NONE ? fresh(x, {s.rows}, at::kFloat) : fresh(x, {}, at::kFloat);
    float *const at = stats.data_ptr<float>(), *const out = loss.data_ptr<float>();
    must(lib.cross_entropy(x.data_ptr(), pitch_of(x), w.data_ptr(), pitch_of(w), at_of(bias), target.data_ptr<int64_t>(), s.rows, s.classes, s.width,
                           ignore, (float)smoothing, ws.data_ptr(), ws.numel(), keeps, reduction == NONE ? out : at + 2 * s.rows + 1, at, at + s.rows,
                           reduction == NONE ? nullptr : out, reduction == MEAN ? at + 2 * s.rows : nullptr, s.dtype, stream_of(x)),
         "vtdge_cross_entropy");
    return {loss, stats, keeps ? ws : Tensor()};
}

std::array<Tensor, 3> cross_entropy_backward(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &target, const Tensor &stats,
                                             const Tensor &laid_out, const Tensor &grad, int64_t ignore, double smoothing, int reduction,
                                             std::array<bool, 3> needs)
{
    const c10::DeviceGuard guard(x.device());
    const Rows s(x, w);
    const Tensor ws = fresh(x, {s.workspace(true, laid_out.defined())}, at::kByte);
    std::array<Tensor, 3> out;
    if (needs[0]) out[0] = fresh(x, {s.rows, s.width}, x.scalar_type());
    if (needs[1]) out[1] = fresh(x, {s.classes, s.width}, x.scalar_type());
    if (needs[2] && bias.defined()) out[2] = fresh(x, {s.classes}, x.scalar_type());
    const float *const at = stats.data_ptr<float>();
    must(lib.cross_entropy_backward(x.data_ptr(), pitch_of(x), w.data_ptr(), pitch_of(w), at_of(bias), target.data_ptr<int64_t>(), at, at + s.rows,
                                    grad.data_ptr<float>(), (int)grad.dim(), reduction == MEAN ? at + 2 * s.rows : nullptr, s.rows, s.classes,
                                    s.width, ignore, (float)smoothing, at_of(laid_out), ws.data_ptr(), ws.numel(), at_of(out[0]), at_of(out[1]),
                                    at_of(out[2]), s.dtype, stream_of(x)),
         "vtdge_cross_entropy_backward");
    return out;
}

struct Operands : OperandChecks {
    void loss(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &t, double smoothing, int64_t reduction) const
    {
        need(rows_of_any_place(x), "x has to be [rows, width] of float32 or bfloat16 with dense rows");
        need(rows_of_any_place(w) && w.device() == x.device() && w.scalar_type() == x.scalar_type() && w.size(1) == x.size(1),
             "weight has to be [classes, width] beside x, of its type, with dense rows");
        need(!b.defined() || (plain_beside(b, x, x.scalar_type()) && b.dim() == 1 && b.size(0) == w.size(0)), "bias has to be [classes] beside x, of its type, dense");
        need(plain_beside(t, x, at::kLong) && t.dim() == 1 && t.size(0) == x.size(0), "target has to be int64 [rows] beside x, dense");
        need(smoothing >= 0 && smoothing <= 1, "label_smoothing has to be 0 .. 1");
        need(reduction >= NONE && reduction <= SUM, "no such reduction");
    }
    void loss_gradients(const Tensor &x, const Tensor &w, const Tensor &stats, const Tensor &laid_out, const Tensor &grad, int64_t reduction) const
    {
        need(plain_beside(stats, x, at::kFloat) && stats.dim() == 1 && stats.size(0) == 3 * x.size(0) + 1, "stats has to be that of the forward call");
        need(!laid_out.defined() ||
                 (plain_beside(laid_out, x, at::kByte) && laid_out.numel() >= lib.cross_entropy_laid_out(x.size(0), w.size(0), Rows(x, w).width, code_of(x))),
             "laid_out has to be that of the forward call");
        need(plain_beside(grad, x, at::kFloat) && (grad.dim() == 0 || (grad.dim() == 1 && reduction == NONE && grad.size(0) == x.size(0))),
             "grad has to be float32 beside x: a scalar, or with a loss for each row a value for each");
    }
    void gate(const Tensor &g, const Tensor &m) const
    {
        need(rows_of_any_place(g) && g.size(1) <= VTDGE_MAX_EXPERTS, "gate has to be [tokens, 1 .. 512] of float32 or bfloat16 with dense rows");
        need(!m.defined() || ((plain_beside(m, g, at::kBool) || plain_beside(m, g, at::kByte)) && m.dim() == 1 && m.size(0) == g.size(0)),
             "mask has to be [tokens] of bytes beside the gate, dense");
    }
    void gate_gradients(const Tensor &g, const Tensor &share, const Tensor &grad) const
    {
        need(plain_beside(share, g, at::kFloat) && share.dim() == 1 && share.size(0) == lib.gate_balance_workspace(g.size(0), (int)g.size(1)) / 4 + g.size(1) + 1,
             "share has to be that of the forward call");
        need(plain_beside(grad, g, at::kFloat) && grad.dim() == 0, "grad has to be a float32 scalar beside the gate");
    }
};

// The backward node of a loss, with what it reads as members.
struct LinearCrossEntropyBackward : torch::autograd::Node {
    SavedVariable x, w, bias, target, stats, laid_out;      // (the last two for hooks on saved tensors to see: up to 320 MB)
    int64_t ignore; double smoothing; int reduction;

    variable_list apply(variable_list &&grads) override
    {
        no_second_order("linear_cross_entropy");
        std::lock_guard<std::mutex> hold(mutex_);
        const Tensor x_ = x.unpack(), w_ = w.unpack(), b_ = bias.unpack(), t_ = target.unpack(), s_ = stats.unpack(), l_ = laid_out.unpack();
        Tensor grad = grads[0];
        if (!grad.defined()) return {Tensor(), Tensor(), Tensor()};
        // the same for every row, as a sum over the losses leaves it: one value
        if (grad.dim() == 1) grad = grad.stride(0) == 0 ? grad.select(0, 0) : grad.contiguous();
        // (hooks on saved tensors may have brought others)
        const Operands check{{"linear_cross_entropy"}};
        check.loss(x_, w_, b_, t_, smoothing, reduction);
        check.loss_gradients(x_, w_, s_, l_, grad, reduction);
        check.on_gpu(x_);
        const auto out = cross_entropy_backward(x_, w_, b_, t_, s_, l_, grad, ignore, smoothing, reduction,
                                                {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)});
        return {out[0], out[1], out[2]};
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> hold(mutex_);
        x.reset_data(), w.reset_data(), bias.reset_data(), target.reset_data();
        stats.reset_data(), laid_out.reset_data();
    }
    std::string name() const override { return "LinearCrossEntropyBackward"; }
};
Tensor linear_cross_entropy(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &target, int64_t ignore, double smoothing, int reduction)
{
    no_forward_mode("linear_cross_entropy", {&x, &w, &bias});
    const bool trains = torch::autograd::compute_requires_grad(x, w, bias);
    Forward f = cross_entropy(x, w, bias, target, ignore, smoothing, reduction, trains);
    if (trains) {
        auto node = std::shared_ptr<LinearCrossEntropyBackward>(new LinearCrossEntropyBackward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, bias));
        node->x = SavedVariable(x, false), node->w = SavedVariable(w, false), node->bias = SavedVariable(bias, false);
        node->target = SavedVariable(target, false);
        node->stats = SavedVariable(f.stats, false), node->laid_out = SavedVariable(f.laid_out, false);
        node->ignore = ignore, node->smoothing = smoothing, node->reduction = reduction;
        torch::autograd::set_history(f.loss, node);
    }
    return f.loss;
}

// ------------------------------------------------------------------------------------------------ balance of gates
std::array<Tensor, 3> gate_balance(const Tensor &gate, const Tensor &indices, const Tensor &mask, int top_k)
{
    const c10::DeviceGuard guard(gate.device());
    const int64_t tokens = gate.size(0);
    const int experts = (int)gate.size(1);
    // share: fp32 [experts + 1], behind the sums of the workgroups
    const int64_t size = bytes_of<2>({tokens, experts}, [&] { return lib.gate_balance_workspace(tokens, experts); });
    const Tensor share = fresh(gate, {size / 4 + experts + 1}, at::kFloat), loss = fresh(gate, {}, at::kFloat), counts = fresh(gate, {experts}, at::kLong);
    float *const at = share.data_ptr<float>();
    must(lib.gate_balance(gate.data_ptr(), pitch_of(gate), (const int64_t *)at_of(indices), (const unsigned char *)at_of(mask), tokens, experts,
                          top_k, at, size, loss.data_ptr<float>(), counts.data_ptr<int64_t>(), at + size / 4, code_of(gate), stream_of(gate)),
         "vtdge_gate_balance");
    return {loss, counts, share};
}
Tensor gate_balance_backward(const Tensor &gate, const Tensor &mask, const Tensor &share, const Tensor &grad)
{
    const c10::DeviceGuard guard(gate.device());
    const int experts = (int)gate.size(1);
    const Tensor out = fresh(gate, {gate.size(0), experts}, gate.scalar_type());
    must(lib.gate_balance_backward(gate.data_ptr(), pitch_of(gate), (const unsigned char *)at_of(mask),
                                   share.data_ptr<float>() + share.numel() - experts - 1, grad.data_ptr<float>(), out.data_ptr(), gate.size(0),
                                   experts, code_of(gate), stream_of(gate)),
         "vtdge_gate_balance_backward");
    return out;
}

struct GateBalanceBackward : torch::autograd::Node {
    SavedVariable gate, mask, share;

    variable_list apply(variable_list &&grads) override
    {
        no_second_order("gate_balance");
        std::lock_guard<std::mutex> hold(mutex_);
        const Tensor gate_ = gate.unpack(), mask_ = mask.unpack(), share_ = share.unpack();
        if (!grads[0].defined()) return {Tensor()};
        const Operands check{{"gate_balance"}};
        check.gate(gate_, mask_);
        check.gate_gradients(gate_, share_, grads[0]);
        check.on_gpu(gate_);
        return {gate_balance_backward(gate_, mask_, share_, grads[0])};
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> hold(mutex_);
        gate.reset_data(), mask.reset_data(), share.reset_data();
    }
    std::string name() const override { return "GateBalanceBackward"; }
};
std::array<Tensor, 2> balance(const Tensor &gate, const Tensor &indices, const Tensor &mask, int top_k)
{
    no_forward_mode("gate_balance", {&gate});
    auto out = gate_balance(gate, indices, mask, top_k);
    if (torch::autograd::compute_requires_grad(gate)) {
        auto node = std::shared_ptr<GateBalanceBackward>(new GateBalanceBackward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(gate));
        node->gate = SavedVariable(gate, false), node->mask = SavedVariable(mask, false);
        node->share = SavedVariable(out[2], false);
        torch::autograd::set_history(out[0], node);
    }
    return {out[0], out[1]};
}

// ------------------------------------------------------------------------------------------------ AdamW
// Weights of one type, device and count of steps, with the table the library reads.  Every step looks again at all that a program can
// put in another's place: the weights and their storage, their states and the tensors in them, the gradients.
struct Batch {
    std::vector<PyObject *> params, states, moments, keys;      // moments: keys.size() of them for each state; all held
    std::vector<vtdge_adamw_tensor> table;      // addresses of memory that is theirs; a step looks whether it still is
    at::ScalarType type, types[4];              // of the weights; of the moments
    ~Batch() { clear(); }
    void clear()
    {
        std::vector<PyObject *> all;
        for (auto *list : {&params, &states, &moments, &keys}) {
            all.insert(all.end(), list->begin(), list->end());
            list->clear();
        }
        for (PyObject *o : all) Py_DECREF(o);
    }
};
// The object that Python holds, which the garbage collector sees through: weights may refer to the optimizer that has it.
struct BatchObject {
    PyObject_HEAD
    Batch *batch;
};
int batch_traverse(PyObject *self, visitproc visit, void *arg)
{
    Batch &b = *reinterpret_cast<BatchObject *>(self)->batch;
    for (auto *list : {&b.params, &b.states, &b.moments, &b.keys})
        for (PyObject *o : *list) Py_VISIT(o);
    return 0;
}
int batch_clear(PyObject *self)
{
    reinterpret_cast<BatchObject *>(self)->batch->clear();
    return 0;
}
void batch_dealloc(PyObject *self)
{
    PyObject_GC_UnTrack(self);
    delete reinterpret_cast<BatchObject *>(self)->batch;
    PyObject_GC_Del(self);
}
PyTypeObject *batch_type()
{
    static PyTypeObject type = {PyVarObject_HEAD_INIT(nullptr, 0)};
    if (type.tp_name == nullptr) {
        type.tp_name = "vtpack_amd._training.Batch";
        type.tp_doc = "The weights of an AdamW step, ready for it.";
        type.tp_basicsize = sizeof(BatchObject);
        type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_GC;
        type.tp_traverse = batch_traverse, type.tp_clear = batch_clear, type.tp_dealloc = batch_dealloc;
    }
    return &type;
}

std::vector<PyObject *> held(PyObject *list)
{
    std::vector<PyObject *> out;
    if (!PyList_Check(list)) throw std::runtime_error("adamw_batch: expected lists");
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); i++) {
        out.push_back(PyList_GET_ITEM(list, i));
        Py_INCREF(out.back());
    }
    return out;
}
bool same(const std::vector<PyObject *> &kept, PyObject *list)
{
    if (!PyList_Check(list) || PyList_GET_SIZE(list) != (Py_ssize_t)kept.size()) return false;
    for (size_t i = 0; i < kept.size(); i++)
        if (PyList_GET_ITEM(list, i) != kept[i]) return false;
    return true;
}
// Everything as it was, and a gradient for every weight that can be read as it lies; its address into the table then.
bool ready(Batch &b, PyObject *params, PyObject *state)
{
    if (b.params.empty() || !same(b.params, params)) return false;
    // states lie in the order of their weights, other groups' between them
    Py_ssize_t at = 0;
    PyObject *key, *value;
    size_t met = 0;
    while (met < b.params.size() && PyDict_Next(state, &at, &key, &value))
        if (key == b.params[met] && value != b.states[met++]) return false;
    if (met < b.params.size()) return false;
    const size_t of = b.keys.size();
    for (size_t i = 0; i < b.params.size(); i++) {
        vtdge_adamw_tensor &row = b.table[i];
        const void *const lies[4] = {row.exp_avg, row.exp_avg_sq, row.exp_avg_scale, row.exp_avg_sq_scale};
        for (size_t k = 0; k < of; k++) {
            PyObject *const m = b.moments[i * of + k];
            if (PyDict_GetItem(b.states[i], b.keys[k]) != m) return false;
            const Tensor &t = THPVariable_Unpack(m);
            if (t.data_ptr() != lies[k] || !t.is_cuda() || t.numel() != (k < 2 ? row.n : (row.n + 255) / 256) || t.scalar_type() != b.types[k] || !t.is_contiguous()) return false;
        }
        const Tensor &p = THPVariable_Unpack(b.params[i]), &g = p.grad();
        if (p.data_ptr() != row.param || !p.is_cuda() || p.numel() != row.n || p.scalar_type() != b.type || !p.is_contiguous() || !g.defined() ||
            g.layout() != at::kStrided || g.scalar_type() != b.type || g.device() != p.device() || g.sizes() != p.sizes() || !g.is_contiguous())
            return false;
        row.grad = g.data_ptr();
    }
    return true;
}

// ------------------------------------------------------------------------------------------------ for Python
PyObject *py_bind(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return call(args, n, 2, [&]() -> PyObject * {
#define VT_BIND(name)                                                                    \
    {                                                                                    \
        PyObject *const o = PyDict_GetItemString(args[0], "vtdge_" #name);               \
        if (o == nullptr) throw std::runtime_error("bind: no address of vtdge_" #name);  \
        lib.name = reinterpret_cast<decltype(lib.name)>((uintptr_t)whole(o));            \
    }
        VT_FUNCTIONS(VT_BIND)
#undef VT_BIND
        Py_INCREF(args[1]);
        error_type = args[1];
        Py_RETURN_NONE;
    });
}

// Operands as the kernels take them.  The entry points below answer None to any other, for their callers to bring them into this
// form or to say what is wrong with them.
bool number(PyObject *o) { return PyLong_Check(o) || PyFloat_Check(o); }

// (x, weight, bias or None, target, ignore_index, label_smoothing, reduction's code)
PyObject *py_linear_cross_entropy(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 7, [&]() -> PyObject * {
        no_tracing("linear_cross_entropy");
        for (int i = 0; i < 4; i++)
            if (!THPVariable_Check(a[i]) && !(i == 2 && a[i] == Py_None)) Py_RETURN_NONE;
        if (!PyLong_Check(a[4]) || !number(a[5]) || !PyLong_Check(a[6])) Py_RETURN_NONE;
        const Tensor x = tensor(a[0]), w = tensor(a[1]), b = tensor(a[2]), t = tensor(a[3]);
        const int64_t ignore = whole(a[4]), reduction = whole(a[6]);
        const double smoothing = real(a[5]);
        if (!plain_rows(x) || !plain_rows(w) || w.device() != x.device() || w.scalar_type() != x.scalar_type() || w.size(1) != x.size(1) ||
            !plain_beside(t, x, at::kLong) || t.dim() != 1 || t.size(0) != x.size(0) ||
            (b.defined() && (!plain_beside(b, x, x.scalar_type()) || b.dim() != 1 || b.size(0) != w.size(0))) || !(smoothing >= 0 && smoothing <= 1))
            Py_RETURN_NONE;
        Tensor loss;
        {
            const NoGil no;
            loss = linear_cross_entropy(x, w, b, t, ignore, smoothing, (int)reduction);
        }
        return wrap(loss);
    });
}
std::array<Tensor, 4> of_loss(const Operands &check, PyObject *const *a, double smoothing, int64_t reduction)
{
    const std::array<Tensor, 4> t = {operand(check, a[0], "x has to be a tensor"), operand(check, a[1], "weight has to be a tensor"),
                                     operand(check, a[2], "bias has to be a tensor or None"), operand(check, a[3], "target has to be a tensor")};
    check.loss(t[0], t[1], t[2], t[3], smoothing, reduction);
    return t;
}
PyObject *py_cross_entropy(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 7, [&] {
        const Operands check{{"cross_entropy"}};
        const int64_t ignore = whole(a[4]), reduction = whole(a[6]);
        const double smoothing = real(a[5]);
        const auto [x, w, b, t] = of_loss(check, a, smoothing, reduction);
        check.on_gpu(x);
        Forward f;
        {
            const NoGil no;
            f = cross_entropy(x, w, b, t, ignore, smoothing, (int)reduction, true);
        }
        return tuple({f.loss, f.stats, f.laid_out});
    });
}
PyObject *py_cross_entropy_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 13, [&] {
        const Operands check{{"cross_entropy_backward"}};
        const int64_t ignore = whole(a[7]), reduction = whole(a[9]);
        const double smoothing = real(a[8]);
        const std::array<bool, 3> needs = {whole(a[10]) != 0, whole(a[11]) != 0, whole(a[12]) != 0};
        const auto [x, w, b, t] = of_loss(check, a, smoothing, reduction);
        const Tensor stats = operand(check, a[4], "stats has to be a tensor"), laid_out = operand(check, a[5], "laid_out has to be a tensor or None"),
                     grad = operand(check, a[6], "grad has to be a tensor");
        check.loss_gradients(x, w, stats, laid_out, grad, reduction);
        check.on_gpu(x);
        std::array<Tensor, 3> out;
        {
            const NoGil no;
            out = cross_entropy_backward(x, w, b, t, stats, laid_out, grad, ignore, smoothing, (int)reduction, needs);
        }
        return tuple({out[0], out[1], out[2]});
    });
}
// (gate, indices [tokens, k] or None, mask or None, top_k)
PyObject *py_balance(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 4, [&]() -> PyObject * {
        no_tracing("gate_balance");
        for (int i = 0; i < 3; i++)
            if (!THPVariable_Check(a[i]) && !(i > 0 && a[i] == Py_None)) Py_RETURN_NONE;
        if (!PyLong_Check(a[3])) Py_RETURN_NONE;
        const Tensor gate = tensor(a[0]), indices = tensor(a[1]), mask = tensor(a[2]);
        const int64_t top_k = whole(a[3]);
        if (!plain_rows(gate) || gate.size(1) > 512 || top_k < 1 || top_k > 512 || (!indices.defined() && top_k > gate.size(1)) ||
            (indices.defined() && (!plain_beside(indices, gate, at::kLong) || indices.dim() != 2 || indices.size(0) != gate.size(0) ||
                                   indices.size(1) != top_k)) ||
            (mask.defined() && (!plain_beside(mask, gate, at::kBool) || mask.dim() != 1 || mask.size(0) != gate.size(0))))
            Py_RETURN_NONE;
        std::array<Tensor, 2> out;
        {
            const NoGil no;
            out = balance(gate, indices, mask, (int)top_k);
        }
        return tuple({out[0], out[1]});
    });
}
PyObject *py_gate_balance(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 4, [&] {
        const Operands check{{"gate_balance"}};
        const int64_t top_k = whole(a[3]);
        const Tensor gate = operand(check, a[0], "gate has to be a tensor"), indices = operand(check, a[1], "indices have to be a tensor or None"),
                     mask = operand(check, a[2], "mask has to be a tensor or None");
        check.gate(gate, mask);
        check.need(top_k >= 1 && top_k <= (indices.defined() ? VTDGE_MAX_EXPERTS : gate.size(1)), "top_k has to be 1 .. the number of logits");
        check.need(!indices.defined() || (plain_beside(indices, gate, at::kLong) && indices.dim() == 2 && indices.size(0) == gate.size(0) && indices.size(1) == top_k),
                   "indices have to be int64 [tokens, top_k] beside the gate, dense");
        check.on_gpu(gate);
        std::array<Tensor, 3> out;
        {
            const NoGil no;
            out = gate_balance(gate, indices, mask, (int)top_k);
        }
        return tuple({out[0], out[1], out[2]});
    });
}
PyObject *py_gate_balance_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 4, [&] {
        const Operands check{{"gate_balance_backward"}};
        const Tensor gate = operand(check, a[0], "gate has to be a tensor"), mask = operand(check, a[1], "mask has to be a tensor or None"),
                     share = operand(check, a[2], "share has to be a tensor"), grad = operand(check, a[3], "grad has to be a tensor");
        check.gate(gate, mask);
        check.gate_gradients(gate, share, grad);
        check.on_gpu(gate);
        Tensor out;
        {
            const NoGil no;
            out = gate_balance_backward(gate, mask, share, grad);
        }
        return wrap(out);
    });
}

// (list of tensors) -> bytes that are the same while every one has the same memory, type, sizes and strides
PyObject *py_places(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 1, [&]() -> PyObject * {
        if (!PyList_Check(a[0])) throw std::runtime_error("places: expected a list of tensors");
        std::vector<int64_t> out;
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); i++) {
            const Tensor t = tensor(PyList_GET_ITEM(a[0], i));
            if (!t.defined() || t.layout() != at::kStrided) throw std::runtime_error("places: expected a list of strided tensors");
            out.insert(out.end(), {(int64_t)(uintptr_t)t.data_ptr(), (int64_t)t.scalar_type(), (int64_t)t.device().type(), (int64_t)t.device().index(), t.dim()});
            out.insert(out.end(), t.sizes().begin(), t.sizes().end());
            out.insert(out.end(), t.strides().begin(), t.strides().end());
        }
        return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(out.data()), (Py_ssize_t)(out.size() * sizeof(int64_t)));
    });
}
// (two lists of tensors): whether they are of the same types and sizes, pair by pair, on the same devices, and strided
PyObject *py_alike(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 2, [&]() -> PyObject * {
        if (!PyList_Check(a[0]) || !PyList_Check(a[1]) || PyList_GET_SIZE(a[0]) != PyList_GET_SIZE(a[1])) throw std::runtime_error("alike: expected two lists of one length");
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); i++) {
            const Tensor x = tensor(PyList_GET_ITEM(a[0], i)), y = tensor(PyList_GET_ITEM(a[1], i));
            if (!x.defined() || !y.defined() || x.layout() != at::kStrided || y.layout() != at::kStrided || x.scalar_type() != y.scalar_type() ||
                x.device() != y.device() || x.sizes() != y.sizes())
                Py_RETURN_FALSE;
        }
        Py_RETURN_TRUE;
    });
}

// (params, states, keys, bits): lists of weights, of their states and of the names of the moments in them, scales behind -> a batch,
// or None unless all is as a launch takes it: weights of one type on one GPU, dense and apart, moments and scales that fit them
PyObject *py_adamw_batch(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 4, [&]() -> PyObject * {
        auto b = std::make_unique<Batch>();
        b->params = held(a[0]), b->states = held(a[1]), b->keys = held(a[2]);
        const bool bytes = whole(a[3]) == 8;
        if (b->params.empty() || b->states.size() != b->params.size() || b->keys.size() != (bytes ? 4 : 2))
            throw std::runtime_error("adamw_batch: lists that do not match");
        at::ScalarType *const types = b->types;
        types[0] = bytes ? at::kFloat8_e4m3fn : at::kFloat, types[1] = bytes ? at::kFloat8_e5m2 : at::kFloat, types[2] = types[3] = at::kFloat;
        std::vector<std::pair<uintptr_t, uintptr_t>> lie;
        at::Device device = at::kCPU;
        for (size_t i = 0; i < b->params.size(); i++) {
            const Tensor p = tensor(b->params[i]);
            if (i == 0 && p.defined()) b->type = p.scalar_type(), device = p.device();
            if (!p.defined() || !p.is_cuda() || p.layout() != at::kStrided || !p.is_contiguous() || p.scalar_type() != b->type ||
                p.device() != device || (b->type != at::kFloat && b->type != at::kBFloat16) || !PyDict_Check(b->states[i]))
                Py_RETURN_NONE;
            void *at[4] = {};
            for (size_t k = 0; k < b->keys.size(); k++) {
                PyObject *const o = PyDict_GetItem(b->states[i], b->keys[k]);
                if (o == nullptr || !THPVariable_Check(o)) Py_RETURN_NONE;
                const Tensor m = THPVariable_Unpack(o);
                if (m.scalar_type() != types[k] || m.device() != p.device() || m.layout() != at::kStrided || !m.is_contiguous() ||
                    (k < 2 ? m.sizes() != p.sizes() : m.dim() != 1 || m.numel() != (p.numel() + 255) / 256))
                    Py_RETURN_NONE;
                Py_INCREF(o);
                b->moments.push_back(o);
                at[k] = m.data_ptr();
            }
            vtdge_adamw_tensor x{};
            x.param = p.data_ptr(), x.n = p.numel();
            x.exp_avg = at[0], x.exp_avg_sq = at[1], x.exp_avg_scale = (float *)at[2], x.exp_avg_sq_scale = (float *)at[3];
            b->table.push_back(x);
            if (x.n > 0) lie.emplace_back((uintptr_t)x.param, (uintptr_t)x.param + p.nbytes());
        }
        std::sort(lie.begin(), lie.end());
        for (size_t i = 1; i < lie.size(); i++)
            if (lie[i].first < lie[i - 1].second) Py_RETURN_NONE;
        BatchObject *const out = PyObject_GC_New(BatchObject, batch_type());
        if (out == nullptr) throw python_error();
        out->batch = b.release();
        PyObject_GC_Track(out);
        return reinterpret_cast<PyObject *>(out);
    });
}
// (batch, the group's weights, the optimizer's states, lr, beta1, beta2, eps, decay, step, bits): whether the step was made; if
// not, something is not as it was, or the stream is being captured, and nothing was done
PyObject *py_adamw_step(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(a, n, 10, [&]() -> PyObject * {
        if (Py_TYPE(a[0]) != batch_type()) throw std::runtime_error("adamw_step: expected a batch");
        Batch *const b = reinterpret_cast<BatchObject *>(a[0])->batch;
        double rate[5];
        for (int i = 0; i < 5; i++) rate[i] = real(a[3 + i]);
        const int64_t step = whole(a[8]), bits = whole(a[9]);
        if (!PyDict_Check(a[2]) || !ready(*b, a[1], a[2])) Py_RETURN_FALSE;
        const Tensor &first = THPVariable_Unpack(b->params[0]);
        const c10::DeviceGuard guard(first.device());
        const c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream(first.device().index());
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) {
            (void)hipGetLastError();
            Py_RETURN_FALSE;
        }
        if (status != hipStreamCaptureStatusNone) Py_RETURN_FALSE;
        {
            const NoGil no;
            must(lib.adamw(b->table.data(), (int)b->table.size(), rate[0], rate[1], rate[2], rate[3], rate[4], step, nullptr, code_of(first),
                           (int)bits, stream.stream()),
                 "vtdge_adamw");
        }
        for (PyObject *p : b->params) THPVariable_Unpack(p).unsafeGetTensorImpl()->bump_version();
        Py_RETURN_TRUE;
    });
}

PyMethodDef methods[] = {VT_METHOD(bind), VT_METHOD(linear_cross_entropy), VT_METHOD(cross_entropy), VT_METHOD(cross_entropy_backward),
                         VT_METHOD(balance), VT_METHOD(gate_balance), VT_METHOD(gate_balance_backward), VT_METHOD(places), VT_METHOD(alike), VT_METHOD(adamw_batch),
                         VT_METHOD(adamw_step), VT_METHOD(quantize_blocks), VT_METHOD(dequantize_blocks), VT_METHOD(linear_8bit),
                         VT_METHOD(gelu_8bit), VT_METHOD(layer_norm_8bit), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_training", "The operators of a training step as torch calls them.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__training() { return PyType_Ready(batch_type()) < 0 ? nullptr : PyModule_Create(&module); }
