// The sequence operators for torch tensors: a Python extension module that
// checks tensors, allocates results and workspaces with torch's allocator
// and calls the C entry points on the tensors' device and its current stream.
// Compiled code, because the small calls take less time than a dozen steps of
// the interpreter (one step of one sample: 12 us through ctypes).
//
// snn_b200/sequence.py holds the documented functions; it hands `setup` the
// function that turns a status and a text into the package's exception.
#include "snn_b200.h"

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <Python.h>

namespace {

using at::Tensor;

PyObject *g_raise = nullptr;  // raise(status, text)

// Thrown with the Python exception set.
struct Refused {};

[[noreturn]] void refuse(int status, const char *text) {
    PyObject *r = PyObject_CallFunction(g_raise, "is", status, text);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, text);
    throw Refused();
}
void require(bool ok, const char *text) {
    if (!ok) refuse(SNN_ERR_INVALID_ARGUMENT, text);
}
void check(snn_status_t st, const char *call) {
    if (st != SNN_OK) refuse(st, call);
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return SNN_B200_F32;
        case at::kHalf: return SNN_B200_F16;
        case at::kBFloat16: return SNN_B200_BF16;
        case at::kByte:
        case at::kBool: return SNN_B200_SPIKES;
        default: return -1;
    }
}
int code(const Tensor &t) {
    const int c = code_of(t.scalar_type());
    require(c >= 0, "element type is not one of float32, float16, bfloat16, uint8, bool");
    return c;
}

// ---- autograd ----
// The operators have no autograd formulas: gradients come from calls of their own.
// A result of tensors that require a gradient says so, and going back through it
// is an error; without a history it would only leave their gradients empty.
struct NoFormula : torch::autograd::Node {
    const char *text;
    explicit NoFormula(const char *t) : text(t) {}
    torch::autograd::variable_list apply(torch::autograd::variable_list &&) override {
        TORCH_CHECK_NOT_IMPLEMENTED(false, text);
    }
    std::string name() const override { return "SequenceOperator"; }
};
template <typename... T>
bool wants_gradient(const T &...inputs) {
    return at::GradMode::is_enabled() && ((inputs.defined() && inputs.requires_grad()) || ...);
}
// It leads on to what the inputs come from, but not to the accumulators of leaves: a
// result that lives on would keep one, with the stream of this call, which a backward
// pass of the same leaves captured into a graph could not use.
template <typename... T>
std::shared_ptr<NoFormula> no_formula(const char *text, const T &...inputs) {
    if (!wants_gradient(inputs...)) return nullptr;
    std::shared_ptr<NoFormula> f(new NoFormula(text), torch::autograd::deleteNode);
    const auto lead = [&](const Tensor &t) {
        if (t.defined() && t.grad_fn()) f->add_next_edge(torch::autograd::impl::gradient_edge(t));
    };
    (lead(inputs), ...);
    return f;
}
Tensor &behind(Tensor &result, const std::shared_ptr<NoFormula> &f) {
    if (f && result.defined()) torch::autograd::set_history(result, f);
    return result;
}
// What a call has written to in place is another version of itself.
void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Arguments are borrowed; None is an undefined tensor.
struct Args {
    PyObject *const *v;
    Tensor tensor(int i, bool optional = false) const {
        if (v[i] == Py_None) {
            require(optional, "a tensor expected, not None");
            return Tensor();
        }
        require(THPVariable_Check(v[i]), "a tensor expected");
        const Tensor &t = THPVariable_Unpack(v[i]);
        return t.is_neg() ? t.resolve_neg() : t;  // a sign that is only noted is not in memory
    }
    // One that is written to.
    Tensor place(int i) const {
        require(THPVariable_Check(v[i]), "a tensor expected");
        const Tensor &t = THPVariable_Unpack(v[i]);
        require(!t.is_neg(), "a tensor whose sign is only noted cannot be written to");
        return t;
    }
    bool none(int i) const { return v[i] == Py_None; }
    bool flag(int i) const {
        const int b = PyObject_IsTrue(v[i]);
        if (b < 0) throw Refused();
        return b != 0;
    }
    double number(int i) const {
        const double d = PyFloat_AsDouble(v[i]);
        if (d == -1.0 && PyErr_Occurred()) throw Refused();
        return d;
    }
    int64_t whole(int i) const {
        const int64_t n = PyLong_AsLongLong(v[i]);
        if (n == -1 && PyErr_Occurred()) throw Refused();
        return n;
    }
    // A torch.dtype, or what it is without one.
    at::ScalarType dtype(int i, at::ScalarType otherwise) const {
        if (v[i] == Py_None) return otherwise;
        require(THPDtype_Check(v[i]), "a torch.dtype expected");
        return reinterpret_cast<THPDtype *>(v[i])->scalar_type;
    }
};

// The CUDA device that the tensors are on.
template <typename... T>
int shared_device(const Tensor &first, const T &...others) {
    require(first.is_cuda(), "tensors must be on a CUDA device");
    const int d = first.get_device();
    [[maybe_unused]] const auto same = [&](const Tensor &t) {
        if (t.defined()) require(t.is_cuda() && t.get_device() == d, "tensors must be on one CUDA device");
    };
    (same(others), ...);
    return d;
}
void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

Tensor empty(at::IntArrayRef sizes, at::ScalarType t, const Tensor &like) {
    return at::empty(sizes, like.options().dtype(t).memory_format(c10::nullopt));
}
Tensor scratch(snn_size_t bytes, const Tensor &like) {
    return bytes ? empty({(int64_t)bytes}, at::kByte, like) : Tensor();
}
const void *data(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A float32 tensor of that shape, contiguous.
Tensor state(const Tensor &t, at::IntArrayRef shape, const char *text) {
    if (!t.defined()) return t;
    require(t.scalar_type() == at::kFloat && t.sizes() == shape, text);
    return t.contiguous();
}
// A dimension's stride, or `single` where the dimension is one long and its stride says nothing.
int64_t stride(const Tensor &t, int64_t d, int64_t single) { return t.size(d) > 1 ? t.stride(d) : single; }
// With neighbouring elements along the last dimension.
Tensor rows(const Tensor &t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }

at::ScalarType result_type(const Tensor &x) { return code(x) == SNN_B200_SPIKES ? at::kFloat : x.scalar_type(); }

// ---- packed 4-bit ----
// (x, codes, scales): packs into codes and scales; both None: makes them and returns (codes, scales).
PyObject *quantize(Args a) {
    const Tensor x = a.tensor(0);
    const int dev = shared_device(x), type = code(x);
    require(x.dim() == 2, "mx4_quantize: a 2-D tensor expected");
    snn_size_t nc = 0, ns = 0;
    check(snn_b200_mx4_sizes(x.size(0), x.size(1), &nc, &ns), "snn_b200_mx4_sizes");
    Tensor codes, scales;
    const bool make = a.none(1);
    if (make) {
        codes = empty({(int64_t)nc}, at::kByte, x), scales = empty({(int64_t)ns}, at::kByte, x);
    } else {
        codes = a.place(1), scales = a.place(2);
        shared_device(x, codes, scales);
        require(codes.nbytes() == nc && scales.nbytes() == ns && codes.is_contiguous() && scales.is_contiguous(),
                "mx4_quantize: `out` is of another shape");
    }
    check(snn_b200_mx4_quantize_async(dev, stream_of(dev), data(x), type, x.size(0), x.size(1), x.stride(0),
                                      x.stride(1), out(codes), out(scales)),
          "snn_b200_mx4_quantize_async");
    if (!make) {
        written(codes), written(scales);
        Py_RETURN_NONE;
    }
    PyObject *c = THPVariable_Wrap(std::move(codes)), *s = THPVariable_Wrap(std::move(scales));
    return Py_BuildValue("(NN)", c, s);
}

// The parts of a packed matrix, of which argument i is the first: codes, scales, rows, cols.
struct Packed {
    Tensor codes, scales;
    int64_t rows, cols;
    Packed(const Args &a, int i) : codes(a.tensor(i)), scales(a.tensor(i + 1)), rows(a.whole(i + 2)), cols(a.whole(i + 3)) {
        snn_size_t nc = 0, ns = 0;
        check(snn_b200_mx4_sizes((snn_size_t)rows, (snn_size_t)cols, &nc, &ns), "snn_b200_mx4_sizes");
        require(codes.nbytes() == nc && scales.nbytes() == ns && codes.is_contiguous() && scales.is_contiguous(),
                "a packed matrix whose parts have the sizes of its shape expected");
    }
};

// (codes, scales, rows, cols, dtype)
PyObject *dequantize(Args a) {
    const Packed q(a, 0);
    const int dev = shared_device(q.codes, q.scales);
    Tensor y = empty({q.rows, q.cols}, a.dtype(4, at::kFloat), q.codes);
    check(snn_b200_mx4_dequantize_async(dev, stream_of(dev), data(q.codes), data(q.scales), q.rows, q.cols, out(y),
                                        code(y), q.cols),
          "snn_b200_mx4_dequantize_async");
    return THPVariable_Wrap(std::move(y));
}

const float *bias_of(const Tensor &bias, int64_t n) {
    if (!bias.defined()) return nullptr;
    require(bias.scalar_type() == at::kFloat && bias.dim() == 1 && bias.size(0) == n && bias.is_contiguous(),
            "bias: one contiguous float32 for each row of the weights expected");
    return (const float *)data(bias);
}

// (x packed: 4, w packed: 4, bias, dtype)
PyObject *matmul(Args a) {
    const Packed x(a, 0), w(a, 4);
    const Tensor bias = a.tensor(8, true);
    const int dev = shared_device(x.codes, x.scales, w.codes, w.scales, bias);
    require(x.cols == w.cols, "mx4_matmul: the operands' columns differ");
    Tensor y = empty({x.rows, w.rows}, a.dtype(9, at::kFloat), x.codes);
    check(snn_b200_mx4_matmul_async(dev, stream_of(dev), data(x.codes), data(x.scales), x.rows, data(w.codes),
                                    data(w.scales), w.rows, w.cols, bias_of(bias, w.rows), out(y), code(y), w.rows),
          "snn_b200_mx4_matmul_async");
    behind(y, no_formula("mx4_matmul has no gradient: pass detached tensors", bias));
    return THPVariable_Wrap(std::move(y));
}

// (x, w packed: 4, bias, dtype)
PyObject *linear(Args a) {
    const Tensor x = a.tensor(0), bias = a.tensor(5, true);
    const Packed w(a, 1);
    const int dev = shared_device(x, w.codes, w.scales, bias), type = code(x);
    require(x.dim() > 0 && x.size(-1) == w.cols, "mx4_linear: rows of the weights' number of columns expected");
    int64_t m = 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) m *= x.size(d);
    const Tensor flat = x.dim() == 2 ? x : x.reshape({m, w.cols});
    auto shape = x.sizes().vec();
    shape.back() = w.rows;
    Tensor y = empty(shape, a.dtype(6, result_type(x)), x);
    const snn_size_t need =
        snn_b200_mx4_linear_workspace(data(flat), type, m, w.cols, flat.stride(0), flat.stride(1));
    const Tensor ws = scratch(need, x);
    check(snn_b200_mx4_linear_async(dev, stream_of(dev), data(flat), type, m, w.cols, flat.stride(0), flat.stride(1),
                                    data(w.codes), data(w.scales), w.rows, bias_of(bias, w.rows), out(y), code(y),
                                    w.rows, out(ws), need),
          "snn_b200_mx4_linear_async");
    behind(y, no_formula("mx4_linear has no gradient: pass detached tensors", x, bias));
    return THPVariable_Wrap(std::move(y));
}

// ---- leaky recurrence ----
// An empty [batch, steps, channels] tensor whose steps come first in memory where x's do.
Tensor like(const Tensor &x, at::ScalarType t) {
    const int64_t b = x.size(0), n = x.size(1), c = x.size(2);
    if (b > 1 && n > 1 && x.stride(0) < x.stride(1))
        return at::empty_strided({b, n, c}, {c, b * c, 1}, x.options().dtype(t).memory_format(c10::nullopt));
    return empty({b, n, c}, t, x);
}

struct Sequence {
    Tensor x, gate, lengths;
    snn_b200_leaky_t q = {};
    int dev;
    bool every = false;

    // x, gate, decay, lengths, logit, complement, input_scale from argument i on.
    // A gate expanded over the sequences or the steps is read where it is (one of x's
    // 16-bit type over the steps in 32 bits, as gates without a step stride are); for its gradient
    // (whole) it becomes an array with an element for each of them.
    Sequence(const Args &a, int i, bool whole) : x(a.tensor(i)), gate(a.tensor(i + 1, true)), lengths(a.tensor(i + 3, true)) {
        dev = shared_device(x, gate, lengths);
        require(x.dim() == 3, "leaky: [batch, steps, channels] expected");
        x = rows(x);
        q.batch = x.size(0), q.steps = x.size(1), q.channels = x.size(2);
        q.x_dtype = code(x);
        q.x_batch_stride = stride(x, 0, 0), q.x_step_stride = stride(x, 1, 0);
        q.logit = a.flag(i + 4), q.complement = a.flag(i + 5), q.input_scale = (float)a.number(i + 6);
        require(gate.defined() != !a.none(i + 2), "leaky: either a gate array or a decay is needed");
        if (gate.defined()) {
            int64_t d = gate.dim();
            require(d >= 1 && d <= 3 && gate.size(-1) == x.size(2) && (d < 2 || gate.size(0) == x.size(0)) &&
                        (d < 3 || gate.size(1) == x.size(1)),
                    "leaky: a gate of shape [channels], [batch, channels] or [batch, steps, channels] expected");
            gate = rows(gate);
            const int64_t c = x.size(2) ? x.size(2) : 1;  // of a dimension that is one long: not shared
            if (whole && d > 1 && (stride(gate, 0, c) == 0 || (d > 2 && stride(gate, 1, c) == 0)))
                gate = gate.clone(at::MemoryFormat::Contiguous);
            if (d > 2 && stride(gate, 1, c) == 0 && q.x_dtype != SNN_B200_SPIKES && gate.scalar_type() == x.scalar_type())
                gate = gate.select(1, 0).to(at::kFloat), d = 2;
            q.gate_dtype = code(gate);
            q.gate_batch_stride = d > 1 ? stride(gate, 0, c) : 0, q.gate_step_stride = d > 2 ? stride(gate, 1, c) : 0;
            every = q.gate_step_stride != 0;
        } else {
            q.decay = (float)a.number(i + 2);
        }
        if (lengths.defined())
            require((lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kUInt32) && lengths.dim() == 1 &&
                        lengths.size(0) == x.size(0) && lengths.is_contiguous(),
                    "lengths: one contiguous int32 for each sequence expected");
    }
    const uint32_t *length() const { return (const uint32_t *)data(lengths); }
    int64_t blocks() const { return ((int64_t)q.steps + SNN_B200_LEAKY_BLOCK - 1) / SNN_B200_LEAKY_BLOCK; }
    Tensor workspace(snn_size_t *need, bool backward) const {
        *need = snn_b200_leaky_workspace(&q, backward);
        return scratch(*need, x);
    }
};

// (x, gate, decay, lengths, logit, complement, input_scale, h0, dtype, save)
PyObject *scan(Args a) {
    Sequence s(a, 0, false);
    const int64_t b = s.x.size(0), c = s.x.size(2);
    const Tensor given = a.tensor(7, true);
    if (given.defined()) shared_device(s.x, given);
    const Tensor h0 = state(given, {b, c}, "h0: float32 of shape [batch, channels] expected");
    const bool save = a.flag(9);
    Tensor y = like(s.x, a.dtype(8, result_type(s.x))), h_last = empty({b, c}, at::kFloat, s.x), saved;
    if (save) saved = empty({b, s.blocks(), c}, at::kFloat, s.x);
    s.q.y_dtype = code(y), s.q.y_batch_stride = y.stride(0), s.q.y_step_stride = y.stride(1);
    snn_size_t need;
    const Tensor ws = s.workspace(&need, false);
    check(snn_b200_leaky_scan_async(s.dev, stream_of(s.dev), &s.q, data(s.x), data(s.gate), (const float *)data(h0),
                                    s.length(), out(y), (float *)out(h_last), (float *)out(saved), out(ws), need),
          "snn_b200_leaky_scan_async");
    const auto f = no_formula("leaky_scan has no autograd formula: its gradients come from leaky_scan_backward",
                              a.tensor(0), a.tensor(1, true), given);
    behind(y, f), behind(h_last, f);
    PyObject *py = THPVariable_Wrap(std::move(y)), *ph = THPVariable_Wrap(std::move(h_last));
    if (!save) return Py_BuildValue("(NN)", py, ph);
    return Py_BuildValue("(NNN)", py, ph, THPVariable_Wrap(std::move(saved)));
}

// (x, gate, decay, lengths, logit, complement, input_scale, dy, saved, dh_last)
PyObject *scan_backward(Args a) {
    Sequence s(a, 0, true);
    const int64_t b = s.x.size(0), c = s.x.size(2);
    Tensor dy = a.tensor(7);
    const Tensor saved = a.tensor(8), given = a.tensor(9, true);
    shared_device(s.x, dy, saved, given);
    require(dy.sizes() == s.x.sizes(), "leaky_scan_backward: dy of x's shape expected");
    dy = rows(dy);
    require(saved.dim() == 3 && saved.size(0) == b && saved.size(1) == s.blocks() && saved.size(2) == c &&
                saved.scalar_type() == at::kFloat && saved.is_contiguous(),
            "leaky_scan_backward: `saved` of leaky_scan(..., save=True) expected");
    const Tensor dh_last = state(given, {b, c}, "dh_last: float32 of shape [batch, channels] expected");
    Tensor dx = like(s.x, result_type(s.x)), dh0 = empty({b, c}, at::kFloat, s.x), dgate;
    snn_b200_leaky_t &q = s.q;
    if (s.every) {
        dgate = like(s.gate, s.gate.scalar_type());
        q.dgate_batch_stride = dgate.stride(0), q.dgate_step_stride = dgate.stride(1);
    } else if (s.gate.defined()) {
        dgate = s.gate.dim() > 1 ? empty({b, c}, at::kFloat, s.x) : empty({c}, at::kFloat, s.x);
        q.dgate_batch_stride = q.gate_batch_stride ? c : 0;
    }
    q.y_dtype = code(dy), q.dy_batch_stride = stride(dy, 0, 0), q.dy_step_stride = stride(dy, 1, 0);
    q.dx_batch_stride = dx.stride(0), q.dx_step_stride = dx.stride(1);
    snn_size_t need;
    const Tensor ws = s.workspace(&need, true);
    check(snn_b200_leaky_scan_backward_async(s.dev, stream_of(s.dev), &q, data(s.x), data(s.gate), s.length(),
                                             (const float *)data(saved), data(dy), (const float *)data(dh_last), out(dx),
                                             out(dgate), (float *)out(dh0), out(ws), need),
          "snn_b200_leaky_scan_backward_async");
    // x and the gate ordinarily require a gradient here: this one. Of dy and dh_last it would be a second.
    const auto f = no_formula("leaky_scan_backward has no gradient of its own", a.tensor(7), given);
    behind(dx, f), behind(dgate, f), behind(dh0, f);
    PyObject *pz = dgate.defined() ? THPVariable_Wrap(std::move(dgate)) : Py_NewRef(Py_None);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(dx)), pz, THPVariable_Wrap(std::move(dh0)));
}

// (x, gate, pool, slots, decay, logit, complement, input_scale, dtype)
PyObject *step(Args a) {
    const Tensor x0 = a.tensor(0), gate0 = a.tensor(1, true), pool = a.place(2), slots = a.tensor(3, true);
    const int dev = shared_device(x0, gate0, pool, slots), type = code(x0);
    require(x0.dim() == 2 && pool.dim() == 2 && pool.scalar_type() == at::kFloat && pool.size(1) == x0.size(1) &&
                (pool.stride(1) == 1 || pool.size(1) <= 1),
            "leaky_step: x [batch, channels] and a float32 pool [slot_count, channels] with neighbouring channels expected");
    require(!wants_gradient(pool), "leaky_step: a pool that requires a gradient cannot be updated in place");
    const int64_t b = x0.size(0), c = x0.size(1);
    const Tensor x = rows(x0);
    require(gate0.defined() != !a.none(4), "leaky_step: either a gate array or a decay is needed");
    Tensor gate;
    int64_t gate_stride = 0;
    int gate_type = SNN_B200_F32;
    if (gate0.defined()) {
        const int64_t d = gate0.dim();
        require((d == 1 || (d == 2 && gate0.size(0) == b)) && gate0.size(-1) == c,
                "leaky_step: a gate of shape [channels] or [batch, channels] expected");
        gate = rows(gate0);
        gate_stride = d == 2 ? stride(gate, 0, c ? c : 1) : 0;
        // Expanded over the rows: in 32 bits, as gates without a row stride are.
        if (d == 2 && gate_stride == 0 && type != SNN_B200_SPIKES && gate.scalar_type() == x.scalar_type())
            gate = gate.select(0, 0).to(at::kFloat);
        gate_type = code(gate);
    }
    if (slots.defined())
        require(slots.scalar_type() == at::kInt && slots.dim() == 1 && slots.size(0) == b && slots.is_contiguous(),
                "leaky_step: slots: one contiguous int32 for each row expected");
    Tensor y = empty({b, c}, a.dtype(8, result_type(x)), x);
    check(snn_b200_leaky_step_async(dev, stream_of(dev), b, pool.size(0), c, data(x), type, x.stride(0), data(gate),
                                    gate_type, gate_stride, a.flag(5), a.flag(6),
                                    gate0.defined() ? 0.0f : (float)a.number(4), (float)a.number(7), (float *)out(pool),
                                    pool.stride(0), (const int32_t *)data(slots), out(y), code(y), c),
          "snn_b200_leaky_step_async");
    written(pool);
    behind(y, no_formula("leaky_step has no gradient: pass detached tensors", x0, gate0));
    return THPVariable_Wrap(std::move(y));
}

template <PyObject *(*F)(Args), Py_ssize_t N>
PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (g_raise == nullptr || count != N) {
        PyErr_SetString(PyExc_TypeError, "sequence_ops: wrong number of arguments, or setup was not called");
        return nullptr;
    }
    try {
        return F(Args{args});
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject *setup(PyObject *, PyObject *raise) {
    Py_XSETREF(g_raise, Py_NewRef(raise));
    Py_RETURN_NONE;
}

template <PyObject *(*F)(Args), Py_ssize_t N>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {{"setup", setup, METH_O, nullptr},
                           method<quantize, 3>("quantize"),
                           method<dequantize, 5>("dequantize"),
                           method<matmul, 10>("matmul"),
                           method<linear, 7>("linear"),
                           method<scan, 10>("scan"),
                           method<scan_backward, 10>("scan_backward"),
                           method<step, 9>("step"),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "sequence_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_sequence_ops(void) { return PyModule_Create(&g_module); }
