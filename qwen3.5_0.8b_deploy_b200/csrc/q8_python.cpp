// Python calls of the 8-bit operators: checks of tensors, outputs and the C ABI's call in one function each.
//
// A product of one token takes the GPU 3.5 us; the same steps in Python, with ctypes for the call, took the host 9 us (quantiser 10, norm block 13, products of
// more rows 14), here 4.8 (6.8, 7.2, 9).  Errors are those of the ctypes binding: its function `fail` raises them.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/b200attn.h"

namespace {

PyObject* g_fail = nullptr;        // fail(status, message) raises

[[noreturn]] void fail(int status, const std::string& message) {
    if (PyObject* r = PyObject_CallFunction(g_fail, "is", status, message.c_str())) Py_DECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, message.c_str());
    throw python_error();
}
[[noreturn]] void refuse(const std::string& message) { fail(B200ATTN_ERR_INVALID, message); }
void check(int status) {
    if (status != 0) fail(status, b200attn_last_error());
}

int code_of(at::ScalarType t) {    // -1: no type of these operators
    return t == at::kBFloat16 ? B200ATTN_DTYPE_BF16 : t == at::kFloat ? B200ATTN_DTYPE_F32 : t == at::kHalf ? B200ATTN_DTYPE_F16 : -1;
}
at::ScalarType type_of(PyObject* dtype, const char* what) {
    if (!THPDtype_Check(dtype)) refuse(std::string(what) + ": a torch.dtype wanted");
    return reinterpret_cast<THPDtype*>(dtype)->scalar_type;
}
int output_code(at::ScalarType t) {
    const int code = code_of(t);
    if (code < 0) refuse(std::string("output type ") + c10::toString(t));
    return code;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + ": a tensor wanted");
    return THPVariable_Unpack(o);
}
bool on_current_device(const at::Tensor& t) { return t.is_cuda() && t.device().index() == c10::cuda::current_device(); }

// A matrix on the current device whose columns lie side by side.  cols, rows: wanted, -1: any number.
struct Matrix {
    at::Tensor t;
    int code = 0;
    int64_t ld = 0, rows = 0, cols = 0;
    void* data() const { return t.data_ptr(); }
};
Matrix matrix(const at::Tensor& t, const char* name, int64_t cols = -1, int64_t rows = -1, bool codes = false) {
    Matrix m;
    m.t = t;
    m.code = codes ? (t.scalar_type() == at::kChar ? 0 : -1) : code_of(t.scalar_type());
    if (m.code < 0) refuse(std::string(name) + ": element type " + c10::toString(t.scalar_type()));
    if (!on_current_device(t)) refuse(std::string(name) + ": not on the current CUDA device");
    if (t.dim() != 2 || (cols >= 0 && t.size(1) != cols) || (rows >= 0 && t.size(0) != rows))
        refuse(std::string(name) + ": wanted [" + (rows >= 0 ? std::to_string(rows) : "rows") + ", " + (cols >= 0 ? std::to_string(cols) : "columns") + "]");
    m.rows = t.size(0);
    m.cols = t.size(1);
    m.ld = m.rows > 1 ? t.stride(0) : std::max(t.stride(0), m.cols);
    if ((m.cols > 1 && t.stride(1) != 1) || m.ld < m.cols)
        refuse(std::string(name) + ": the columns of a row lie side by side and rows do not overlap");
    if (m.rows > INT_MAX || m.cols > INT_MAX) refuse(std::string(name) + ": too large");
    return m;
}
const float* vector(PyObject* o, const char* name, int64_t n) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.numel() != n || !t.is_contiguous() || !on_current_device(t))
        refuse(std::string(name) + ": " + std::to_string(n) + " contiguous fp32 values on the current CUDA device wanted");
    return t.data_ptr<float>();
}

// Autograd does not see what these calls write: a tensor that requires a gradient is refused as PyTorch refuses leaves, and what was written counts as a new version,
// so that a graph that has saved the tensor notices.
void check_writable(const at::Tensor& t, const char* name) {
    if (at::GradMode::is_enabled() && t.requires_grad()) refuse(std::string(name) + ": requires a gradient and would be written to, which is recorded nowhere");
}
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) { return at::Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt)); }
int64_t codes_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
bool truth(PyObject* o) {
    const int r = PyObject_IsTrue(o);
    if (r < 0) throw python_error();
    return r != 0;
}
float number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)v;
}
void arguments(Py_ssize_t given, Py_ssize_t wanted) {
    if (given == wanted) return;
    PyErr_Format(PyExc_TypeError, "%zd arguments wanted, %zd given", wanted, given);
    throw python_error();
}
PyObject* pack(std::initializer_list<at::Tensor> ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    if (!r) throw python_error();
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
    return r;
}

// (x) -> codes, scales
PyObject* quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 1);
    const Matrix x = matrix(tensor(args[0], "quantize_rows"), "quantize_rows");
    const int64_t pitch = codes_pitch(x.cols);
    at::Tensor codes = empty({x.rows, pitch}, at::kChar, x.t), scales = empty({x.rows}, at::kFloat, x.t);
    check(b200attn_q8_quantize(x.data(), x.code, x.ld, (int)x.rows, (int)x.cols, codes.data_ptr<int8_t>(), pitch, scales.data_ptr<float>(), stream()));
    return pack({pitch == x.cols ? codes : codes.narrow(1, 0, x.cols), scales});
    END_HANDLE_TH_ERRORS
}

// What a product writes to: `out`, or a new matrix of `dtype`.
Matrix output(const Matrix& x, int64_t features, at::ScalarType dtype, PyObject* out, bool accumulate) {
    if (out != Py_None) {
        check_writable(tensor(out, "out"), "out");
        return matrix(tensor(out, "out"), "out", features, x.rows);
    }
    if (accumulate) refuse("accumulate wants an output to add to");
    Matrix y;
    y.code = output_code(dtype);
    y.t = empty({x.rows, features}, dtype, x.t);
    y.ld = y.cols = features;
    y.rows = x.rows;
    return y;
}
PyObject* result(PyObject* out, const Matrix& y) {
    if (out == Py_None) return THPVariable_Wrap(y.t);
    written(y.t);
    Py_INCREF(out);
    return out;
}

// (handle, in, out features, x, out_dtype or None, out or None, accumulate) -> y
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 7);
    const auto q = static_cast<b200attn_q8>(PyLong_AsVoidPtr(args[0]));
    const int64_t in = PyLong_AsLongLong(args[1]), features = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) throw python_error();
    const bool accumulate = truth(args[6]);
    const Matrix x = matrix(tensor(args[3], "x"), "x", in);
    const Matrix y = output(x, features, args[4] == Py_None ? x.t.scalar_type() : type_of(args[4], "out_dtype"), args[5], accumulate);
    size_t bytes = 0;
    check(b200attn_q8_workspace(q, (int)x.rows, x.code, &bytes));
    at::Tensor work;                   // of this call: calls on other streams have theirs
    if (bytes) work = empty({(int64_t)bytes}, at::kByte, x.t);
    check(b200attn_q8_forward(q, x.data(), x.code, x.ld, (int)x.rows, y.data(), y.code, y.ld, accumulate, bytes ? work.data_ptr() : nullptr, bytes, stream()));
    return result(args[5], y);
    END_HANDLE_TH_ERRORS
}

// (handle, in, out features, codes, scales, out_dtype, out or None, accumulate) -> y
PyObject* forward_codes(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 8);
    const auto q = static_cast<b200attn_q8>(PyLong_AsVoidPtr(args[0]));
    const int64_t in = PyLong_AsLongLong(args[1]), features = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) throw python_error();
    const bool accumulate = truth(args[7]);
    const Matrix c = matrix(tensor(args[3], "codes"), "codes", in, -1, true);
    if (args[4] == Py_None) refuse("scales: a tensor wanted");
    const float* scales = vector(args[4], "scales", c.rows);
    const Matrix y = output(c, features, type_of(args[5], "out_dtype"), args[6], accumulate);
    const int64_t ld = c.rows > 1 ? c.ld : codes_pitch(c.ld);          // one row may come without the pitch of a matrix
    check(b200attn_q8_forward_codes(q, static_cast<const int8_t*>(c.data()), ld, scales, (int)c.rows, y.data(), y.code, y.ld, accumulate, stream()));
    return result(args[6], y);
    END_HANDLE_TH_ERRORS
}

// (x, y, pre_w, post_w, gate, sigmoid_gate, x_scale, y_scale, eps, out_dtype, in_place) -> x', n or x', codes, scales
PyObject* norm_block(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 11);
    const Matrix x = matrix(tensor(args[0], "x"), "x");
    const bool has_y = args[1] != Py_None, in_codes = args[9] == Py_None, in_place = truth(args[10]);
    if (in_place) check_writable(x.t, "x");
    const at::ScalarType dtype = has_y ? tensor(args[1], "y").scalar_type() : in_codes ? x.t.scalar_type() : type_of(args[9], "out_dtype");
    b200attn_norm_args a{};
    a.dtype = code_of(dtype);
    if (a.dtype < 0 || (!in_codes && type_of(args[9], "out_dtype") != dtype))
        refuse(std::string("norm_block: the output is of the type of y, fp32, fp16 or bf16 (here ") + c10::toString(dtype) + ")");
    a.rows = (int)x.rows;
    a.width = (int)x.cols;
    a.x_dtype = x.code;
    a.d_x = x.data();
    a.ldx = x.ld;
    if (has_y) {
        const Matrix y = matrix(tensor(args[1], "y"), "y", x.cols, x.rows);
        a.d_y = y.data();
        a.ldy = y.ld;
    }
    a.d_pre_w = vector(args[2], "pre_w", x.cols);
    a.d_post_w = vector(args[3], "post_w", x.cols);
    if (args[4] != Py_None) {
        const at::Tensor& g = tensor(args[4], "gate");
        const bool one = g.dim() == 1;
        const Matrix gate = matrix(one ? g.unsqueeze(0) : g, "gate", x.cols, one ? 1 : x.rows);
        if (gate.code != a.dtype) refuse("gate: the type of y wanted");
        a.d_gate = gate.data();
        a.ld_gate = one ? 0 : gate.ld;
        a.gate_kind = truth(args[5]) ? B200ATTN_GATE_SIGMOID : B200ATTN_GATE_AS_IS;
    }
    a.x_scale = number(args[6]);
    a.y_scale = number(args[7]);
    a.eps = number(args[8]);
    const at::Tensor x_out = in_place ? x.t : empty({x.rows, x.cols}, x.t.scalar_type(), x.t);
    a.d_x_out = x_out.data_ptr();
    a.ldx_out = in_place ? x.ld : x.cols;
    if (in_codes) {
        const int64_t pitch = codes_pitch(x.cols);
        at::Tensor codes = empty({x.rows, pitch}, at::kChar, x.t), scales = empty({x.rows}, at::kFloat, x.t);
        a.d_codes = codes.data_ptr<int8_t>();
        a.ld_codes = pitch;
        a.d_scales = scales.data_ptr<float>();
        check(b200attn_norm_block(&a, stream()));
        if (in_place) written(x_out);
        return pack({x_out, pitch == x.cols ? codes : codes.narrow(1, 0, x.cols), scales});
    }
    at::Tensor out = empty({x.rows, x.cols}, dtype, x.t);
    a.d_out = out.data_ptr();
    a.ld_out = x.cols;
    check(b200attn_norm_block(&a, stream()));
    if (in_place) written(x_out);
    return pack({x_out, out});
    END_HANDLE_TH_ERRORS
}

PyObject* set_fail(PyObject*, PyObject* f) {
    Py_INCREF(f);
    Py_XSETREF(g_fail, f);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef g_methods[] = {{"quantize_rows", fast<quantize_rows>(), METH_FASTCALL, nullptr},
                           {"forward", fast<forward>(), METH_FASTCALL, nullptr},
                           {"forward_codes", fast<forward_codes>(), METH_FASTCALL, nullptr},
                           {"norm_block", fast<norm_block>(), METH_FASTCALL, nullptr},
                           {"set_fail", set_fail, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_q8", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__q8() { return PyModule_Create(&g_module); }
