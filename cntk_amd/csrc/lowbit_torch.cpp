// The low-bit operators on torch tensors: what cntk_amd/lowbit.py calls. A call checks its tensors, makes the results on torch's current
// stream and goes through the C ABI (include/cntk_amd_lowbit.h). Serving and small layers are bound by the host's part of a call: made here it
// takes 4 to 5 us, of which a launch is about two, instead of 9 to 11 through ctypes.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/cntk_amd_lowbit.h"

#include <algorithm>
#include <initializer_list>
#include <utility>
#include <vector>

namespace {

PyObject* g_runtime_error = nullptr; // the package's two exceptions
PyObject* g_logic_error = nullptr;

[[noreturn]] void refuse(const char* text)
{
    PyErr_SetString(g_logic_error, text);
    throw python_error();
}

void check(int rc)
{
    if (rc == CNTKQ_OK)
        return;
    PyErr_SetString(rc == CNTKQ_RUNTIME_ERROR ? g_runtime_error : g_logic_error, cntkq_last_error());
    throw python_error();
}

// One handle per device for the life of the process. A handle is not re-entrant; the interpreter's lock, held throughout every call here,
// keeps calls apart. The calls leave nothing in it but the stream, which is torch's current one.
cntkq_quantizer* handle(int device)
{
    struct Entry
    {
        cntkq_quantizer* h = nullptr;
        hipStream_t stream = nullptr;
        bool known = false;
    };
    static std::vector<Entry>* entries = new std::vector<Entry>();
    if ((size_t) device >= entries->size())
        entries->resize(device + 1);
    Entry& e = (*entries)[device];
    if (e.h == nullptr)
        check(cntkq_create(device, 0, &e.h));
    const hipStream_t stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex) device).stream();
    if (!e.known || e.stream != stream)
    {
        check(cntkq_set_main_stream(e.h, stream));
        e.stream = stream;
        e.known = true;
    }
    return e.h;
}

const at::Tensor& tensor(PyObject* o, const char* what)
{
    if (!THPVariable_Check(o))
    {
        PyErr_Format(g_logic_error, "%s must be a tensor", what);
        throw python_error();
    }
    return THPVariable_Unpack(o);
}

int code_of(at::ScalarType t)
{
    return t == at::kFloat ? CNTKQ_F32 : (t == at::kHalf ? CNTKQ_F16 : (t == at::kBFloat16 ? CNTKQ_BF16 : -1));
}
at::ScalarType type_of(int code)
{
    return code == CNTKQ_F32 ? at::kFloat : (code == CNTKQ_F16 ? at::kHalf : at::kBFloat16);
}
// the element type's code of a tensor of values
int values(const at::Tensor& t, const char* what)
{
    const int code = code_of(t.scalar_type());
    if (code < 0 || !t.is_cuda())
    {
        PyErr_Format(g_logic_error, "%s must be a float32, float16 or bfloat16 device tensor (got %s on %s)", what, c10::toString(t.scalar_type()),
                     t.device().str().c_str());
        throw python_error();
    }
    return code;
}
void same_device(const at::Tensor& a, const at::Tensor& b)
{
    if (a.device() != b.device())
        refuse("all tensors of a call must be on one device");
}
// a packed matrix's buffer
void packed(const at::Tensor& t)
{
    if (t.scalar_type() != at::kByte || !t.is_cuda() || !t.is_contiguous() || t.is_neg())
        refuse("a packed matrix is a contiguous uint8 device tensor");
}

// A tensor as a matrix of its last dimension's rows: in place where its strides allow one (and, if asked for, the values of a row are
// neighbours), a copy otherwise. (A view that stands for its memory's negative is a copy too: data_ptr() does not know of the sign.)
struct Rows
{
    at::Tensor kept; // the copy
    const void* data;
    int64_t rows, cols, row_stride, col_stride;
};
Rows rows_of(const at::Tensor& given, bool contiguous)
{
    Rows r;
    if (given.is_neg())
    {
        at::NoGradGuard no_grad;
        r.kept = given.resolve_neg();
    }
    const at::Tensor t = r.kept.defined() ? r.kept : given;
    if (t.dim() == 2)
    {
        r.rows = t.size(0);
        r.cols = t.size(1);
        r.row_stride = t.stride(0);
        r.col_stride = r.cols > 1 ? t.stride(1) : 1;
        r.data = t.data_ptr();
        if (!contiguous || r.col_stride == 1)
            return r;
    }
    else if (t.dim() == 0)
        refuse("a tensor of at least one dimension is needed");
    at::NoGradGuard no_grad;
    r.cols = t.size(-1);
    r.rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        r.rows *= t.size(i);
    r.kept = t.reshape({r.rows, r.cols});
    if (r.cols > 1 && r.kept.stride(1) != 1)
        r.kept = r.kept.contiguous();
    r.data = r.kept.data_ptr();
    r.row_stride = r.kept.stride(0);
    r.col_stride = 1;
    return r;
}

at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like)
{
    return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
}
at::Tensor bytes(size_t n, const at::Tensor& like)
{
    return make({(int64_t) n}, at::kByte, like);
}
// A tensor of the caller's that is written behind autograd's back: it must not be part of a graph, and what autograd saved of it has to show that it
// changed (`written`, once the call is on its way; `given`: the argument).
void writable(const at::Tensor& t)
{
    if (at::GradMode::is_enabled() && t.requires_grad())
        refuse("out requires grad: the low-bit functions take part in no autograd graph");
    if (t.is_inference() && !c10::InferenceMode::is_enabled())
        refuse("out was made in inference mode and is written outside of it");
}
void written(PyObject* given, const at::Tensor& t)
{
    if (given != Py_None)
        t.unsafeGetTensorImpl()->bump_version();
}
// the caller's result tensor, checked, or a new one
at::Tensor result(PyObject* out, at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like)
{
    if (out == Py_None)
        return make(sizes, type, like);
    const at::Tensor& t = tensor(out, "out");
    if (t.sizes() != sizes || t.scalar_type() != type || t.device() != like.device())
        refuse("out has another shape, type or device than the result");
    if (t.is_neg())
        refuse("out is a view that stands for its memory's negative");
    if (t.dim() == 2 ? t.size(1) > 1 && t.stride(1) != 1 : !t.is_contiguous())
        refuse("out must have contiguous rows");
    writable(t);
    return t;
}
int64_t row_stride(const at::Tensor& t)
{
    return t.dim() == 2 ? t.stride(0) : (t.dim() == 0 ? 1 : t.size(-1));
}

struct Bias
{
    at::Tensor kept;
    const void* data = nullptr;
    int code = CNTKQ_F32;
};

// The bytes of a matrix in memory: `rows` runs of `length`, `pitch` apart and clear of each other.
struct Area
{
    uintptr_t base;
    int64_t rows, pitch, length;

    uintptr_t end() const { return base + (rows - 1) * pitch + length; }
};
// (of values that lie apart in both directions the closer ones count as one run)
Area area(const void* data, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, int64_t size)
{
    if (rows > 1 && cols > 1 && col_stride > row_stride)
    {
        std::swap(rows, cols);
        std::swap(row_stride, col_stride);
    }
    if (rows == 0 || cols == 0)
        return {0, 0, 0, 0};
    Area a = {reinterpret_cast<uintptr_t>(data), rows, row_stride * size, ((cols - 1) * col_stride + 1) * size};
    if (rows == 1 || a.pitch <= a.length)
        a = {a.base, 1, 0, (int64_t) (a.end() - a.base)};
    return a;
}
Area area(const at::Tensor& t) // a result, a packed matrix
{
    return t.dim() == 2 ? area(t.data_ptr(), t.size(0), t.size(1), t.stride(0), t.size(1) > 1 ? t.stride(1) : 1, t.element_size())
                        : area(t.data_ptr(), 1, t.numel(), 0, 1, t.element_size());
}
Area area(const Rows& r, const at::Tensor& like)
{
    return area(r.data, r.rows, r.cols, r.row_stride, r.col_stride, like.element_size());
}
Area area(const Bias& b, int64_t n)
{
    return b.data == nullptr ? Area{0, 0, 0, 0} : area(b.data, 1, n, 0, 1, b.code == CNTKQ_F32 ? 4 : 2);
}
bool overlap(Area a, Area b)
{
    if (a.rows == 0 || b.rows == 0 || a.end() <= b.base || b.end() <= a.base)
        return false;
    // Runs of one that end before the other's next run are left behind until two meet or none are left. Runs at equal distances either meet
    // within the first few or never.
    for (int64_t steps = a.rows > 1 && b.rows > 1 && a.pitch == b.pitch ? 4 : a.rows + b.rows; a.rows > 0 && b.rows > 0 && steps > 0; --steps)
    {
        if (b.base < a.base)
            std::swap(a, b);
        if (b.base < a.base + a.length)
            return true;
        const int64_t behind = a.rows == 1 ? 1 : std::min<int64_t>(a.rows, (b.base - a.base - a.length) / a.pitch + 1);
        a.base += behind * a.pitch;
        a.rows -= behind;
    }
    return false;
}
// The caller's result shares no memory with what the call reads, or with another result of it.
void apart(const at::Tensor& out, std::initializer_list<Area> others)
{
    const Area mine = area(out);
    for (const Area& a : others)
        if (overlap(mine, a))
            refuse("out shares memory with another tensor of the call");
}

int64_t integer(PyObject* o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred())
        throw python_error();
    return v;
}

Bias bias_of(PyObject* o, int64_t n, const at::Tensor& like)
{
    Bias b;
    if (o == Py_None)
        return b;
    const at::Tensor& t = tensor(o, "bias");
    b.code = values(t, "bias");
    if (t.dim() != 1 || t.size(0) != n)
        refuse("bias must have one element per row of the weights");
    same_device(like, t);
    if (t.is_neg() || (n > 1 && t.stride(0) != 1))
    {
        at::NoGradGuard no_grad;
        b.kept = t.resolve_neg().contiguous();
        b.data = b.kept.data_ptr();
    }
    else
        b.data = t.data_ptr();
    return b;
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b)
{
    PyObject* t = PyTuple_New(2);
    if (t == nullptr)
        throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
    return t;
}

void arguments(Py_ssize_t given, Py_ssize_t wanted)
{
    if (given != wanted)
    {
        PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd wanted", given, wanted);
        throw python_error();
    }
}

// quantize(x, buffer or None) -> (buffer, rows, cols)
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 2);
    const at::Tensor& x = tensor(args[0], "x");
    const int code = values(x, "x");
    const Rows r = rows_of(x, false);
    const size_t size = cntkq_mx4_bytes(r.rows, r.cols);
    at::Tensor q;
    if (args[1] == Py_None)
        q = bytes(size, x);
    else
    {
        q = tensor(args[1], "out");
        packed(q);
        same_device(x, q);
        writable(q);
        apart(q, {area(r, x)});
    }
    check(cntkq_mx4_quantize_async(handle(x.get_device()), r.data, code, r.rows, r.cols, r.row_stride, r.col_stride, q.data_ptr(), q.numel(),
                                   nullptr, 0));
    written(args[1], q);
    return Py_BuildValue("(NLL)", THPVariable_Wrap(q), (long long) r.rows, (long long) r.cols);
    END_HANDLE_TH_ERRORS
}

// dequantize(buffer, rows, cols, type code, out or None) -> out
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 5);
    const at::Tensor& q = tensor(args[0], "the packed matrix");
    packed(q);
    const int64_t rows = integer(args[1]), cols = integer(args[2]);
    const int code = (int) integer(args[3]);
    const at::Tensor out = result(args[4], {rows, cols}, type_of(code), q);
    if (args[4] != Py_None)
        apart(out, {area(q)});
    check(cntkq_mx4_dequantize_async(handle(q.get_device()), q.data_ptr(), q.numel(), rows, cols, out.data_ptr(), code, row_stride(out)));
    written(args[4], out);
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// matmul(a's buffer, m, b's buffer, n, k, bias or None, type code, out or None) -> out
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    arguments(nargs, 8);
    const at::Tensor& a = tensor(args[0], "a");
    const at::Tensor& b = tensor(args[2], "b");
    packed(a);
    packed(b);
    same_device(a, b);
    const int64_t m = integer(args[1]), n = integer(args[3]), k = integer(args[4]);
    const Bias bias = bias_of(args[5], n, a);
    const int code = (int) integer(args[6]);
    const at::Tensor out = result(args[7], {m, n}, type_of(code), a);
    if (args[7] != Py_None)
        apart(out, {area(a), area(b), area(bias, n)});
    check(cntkq_mx4_matmul_async(handle(a.get_device()), a.data_ptr(), a.numel(), m, b.data_ptr(), b.numel(), n, k, bias.data, bias.code,
                                 out.data_ptr(), code, row_stride(out)));
    written(args[7], out);
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// linear(x, weights' buffer, n, k, bias or None, save, type code or -1, out or None) -> y, or (y, the 8-bit form's buffer)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    arguments(nargs, 8);
    const at::Tensor& x = tensor(args[0], "x");
    const at::Tensor& w = tensor(args[1], "the weights");
    const int code = values(x, "x");
    packed(w);
    same_device(x, w);
    const int64_t n = integer(args[2]), k = integer(args[3]);
    const bool save = integer(args[5]) != 0;
    int out_code = (int) integer(args[6]);
    out_code = out_code < 0 ? code : out_code;
    const Rows r = rows_of(x, true);
    if (r.cols != k)
    {
        PyErr_Format(g_logic_error, "x has %lld columns, the weights %lld", (long long) r.cols, (long long) k);
        throw python_error();
    }
    const Bias bias = bias_of(args[4], n, x);
    c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = n;
    const at::Tensor y = result(args[7], sizes, type_of(out_code), x);
    if (args[7] != Py_None)
        apart(y, {area(r, x), area(w), area(bias, n)});
    at::Tensor saved, work;
    if (save)
        saved = bytes(cntkq_save8_bytes(r.rows, k), x);
    const size_t need = cntkq_mx4_linear_workspace_bytes(r.rows, n, k, code, save);
    if (need != 0)
        work = bytes(need, x);
    check(cntkq_mx4_linear_async(handle(x.get_device()), r.data, code, r.row_stride, r.rows, w.data_ptr(), w.numel(), n, k, bias.data, bias.code,
                                 y.data_ptr(), out_code, row_stride(y), save ? saved.data_ptr() : nullptr, save ? saved.numel() : 0,
                                 need != 0 ? work.data_ptr() : nullptr, need));
    written(args[7], y);
    return save ? pair(y, saved) : THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// save8(x) -> buffer
PyObject* save8(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 1);
    const at::Tensor& x = tensor(args[0], "x");
    const int code = values(x, "x");
    const Rows r = rows_of(x, true);
    const at::Tensor saved = bytes(cntkq_save8_bytes(r.rows, r.cols), x);
    check(cntkq_save8_async(handle(x.get_device()), r.data, code, r.rows, r.cols, r.row_stride, saved.data_ptr(), saved.numel()));
    return THPVariable_Wrap(saved);
    END_HANDLE_TH_ERRORS
}

// load8(buffer, rows, cols, type code) -> values
PyObject* load8(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 4);
    const at::Tensor& saved = tensor(args[0], "what was kept");
    packed(saved);
    const int64_t rows = integer(args[1]), cols = integer(args[2]);
    const int code = (int) integer(args[3]);
    const at::Tensor out = make({rows, cols}, type_of(code), saved);
    check(cntkq_load8_async(handle(saved.get_device()), saved.data_ptr(), saved.numel(), rows, cols, out.data_ptr(), code, cols));
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// activation_forward(kind, x, gate or None) -> (y, x's buffer, the gate's buffer or None)
PyObject* activation_forward(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 3);
    const int kind = (int) integer(args[0]);
    const at::Tensor& x = tensor(args[1], "x");
    const int code = values(x, "x");
    const Rows r = rows_of(x, true);
    const size_t size = cntkq_save8_bytes(r.rows, r.cols);
    Rows g = {};
    at::Tensor saved_gate;
    if (args[2] != Py_None)
    {
        const at::Tensor& gate = tensor(args[2], "the gate");
        if (gate.sizes() != x.sizes() || gate.scalar_type() != x.scalar_type() || gate.device() != x.device())
            refuse("the gate must be of x's shape and type, on its device");
        g = rows_of(gate, true);
        saved_gate = bytes(size, x);
    }
    const at::Tensor saved = bytes(size, x), y = make(x.sizes(), x.scalar_type(), x);
    check(cntkq_activation_forward_async(handle(x.get_device()), kind, r.data, r.row_stride, g.data, g.row_stride, code, r.rows, r.cols, y.data_ptr(),
                                         r.cols, saved.data_ptr(), saved_gate.defined() ? saved_gate.data_ptr() : nullptr, size));
    if (!saved_gate.defined())
        return Py_BuildValue("(NNO)", THPVariable_Wrap(y), THPVariable_Wrap(saved), Py_None);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(y), THPVariable_Wrap(saved), THPVariable_Wrap(saved_gate));
    END_HANDLE_TH_ERRORS
}

// activation_backward(kind, dy, x's buffer, the gate's buffer or None) -> dx, or (dx, dgate)
PyObject* activation_backward(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 4);
    const int kind = (int) integer(args[0]);
    const at::Tensor& dy = tensor(args[1], "dy");
    const int code = values(dy, "dy");
    const at::Tensor& saved = tensor(args[2], "what was kept");
    packed(saved);
    same_device(dy, saved);
    const bool gated = args[3] != Py_None;
    const Rows r = rows_of(dy, true);
    const at::Tensor dx = make(dy.sizes(), dy.scalar_type(), dy);
    at::Tensor saved_gate, dgate;
    if (gated)
    {
        saved_gate = tensor(args[3], "the kept gate");
        packed(saved_gate);
        same_device(dy, saved_gate);
        if (saved_gate.numel() != saved.numel())
            refuse("what was kept of the gate is of another size");
        dgate = make(dy.sizes(), dy.scalar_type(), dy);
    }
    check(cntkq_activation_backward_async(handle(dy.get_device()), kind, r.data, r.row_stride, code, r.rows, r.cols, saved.data_ptr(),
                                          gated ? saved_gate.data_ptr() : nullptr, saved.numel(), dx.data_ptr(), r.cols,
                                          gated ? dgate.data_ptr() : nullptr, r.cols));
    return gated ? pair(dx, dgate) : THPVariable_Wrap(dx);
    END_HANDLE_TH_ERRORS
}

// weight_gradient(dy, buffer, k, bias, dw or None, db or None, accumulate) -> dw, or (dw, db)
PyObject* weight_gradient(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    arguments(nargs, 7);
    const at::Tensor& dy = tensor(args[0], "dy");
    const int code = values(dy, "dy");
    const at::Tensor& saved = tensor(args[1], "what was kept");
    packed(saved);
    same_device(dy, saved);
    const int64_t k = integer(args[2]);
    const bool bias = integer(args[3]) != 0, accumulate = integer(args[6]) != 0;
    if (accumulate && (args[4] == Py_None || (bias && args[5] == Py_None)))
        refuse("accumulate needs every result's tensor to add to");
    const Rows r = rows_of(dy, true);
    const at::Tensor dw = result(args[4], {r.cols, k}, at::kFloat, dy);
    if (args[4] != Py_None)
        apart(dw, {area(r, dy), area(saved)});
    at::Tensor db, work;
    if (bias)
    {
        db = result(args[5], {r.cols}, at::kFloat, dy);
        if (args[5] != Py_None)
            apart(db, {area(r, dy), area(saved), area(dw)});
    }
    const size_t need = cntkq_weight_gradient_workspace_bytes(r.rows, r.cols, k, code);
    if (need != 0)
        work = bytes(need, dy);
    check(cntkq_weight_gradient_async(handle(dy.get_device()), r.data, code, r.row_stride, r.rows, r.cols, saved.data_ptr(), saved.numel(), k,
                                      static_cast<float*>(dw.data_ptr()), row_stride(dw), bias ? static_cast<float*>(db.data_ptr()) : nullptr,
                                      accumulate, need != 0 ? work.data_ptr() : nullptr, need));
    written(args[4], dw);
    if (bias)
        written(args[5], db);
    return bias ? pair(dw, db) : THPVariable_Wrap(dw);
    END_HANDLE_TH_ERRORS
}

// errors(runtime error class, logic error class)
PyObject* errors(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 2);
    Py_INCREF(args[0]);
    Py_INCREF(args[1]);
    g_runtime_error = args[0];
    g_logic_error = args[1];
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define CNTKQ_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {CNTKQ_METHOD(quantize),           CNTKQ_METHOD(dequantize),          CNTKQ_METHOD(matmul),          CNTKQ_METHOD(linear),
                           CNTKQ_METHOD(save8),              CNTKQ_METHOD(load8),               CNTKQ_METHOD(activation_forward),
                           CNTKQ_METHOD(activation_backward), CNTKQ_METHOD(weight_gradient),    CNTKQ_METHOD(errors),          {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_lowbit", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__lowbit()
{
    return PyModule_Create(&g_module);
}
