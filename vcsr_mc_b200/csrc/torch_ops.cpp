// The microscaled operators for Python: checks of torch tensors, allocation of results and workspaces from torch's
// allocator on the current stream, and the call into the C ABI, as functions of one CPython module. The same in
// Python around ctypes takes 10 to 12 us per call, several times what the small operators run for. The module does
// no arithmetic; api.py holds the public functions and their documentation.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <string>

#include "vcsrmc.h"

namespace {

PyObject* g_error = nullptr;  // VcsrmcError

struct Fail {
    int status;
    std::string message;
};

[[noreturn]] void invalid(const std::string& what) { throw Fail{VCSRMC_INVALID_ARG, what}; }

void check(int status) {
    if (status == VCSRMC_OK) return;
    char message[1024];
    vcsrmc_last_error(message, sizeof message);
    throw Fail{status, message};
}

// Runs fn and turns what it throws into a Python exception.
template <class Fn>
PyObject* guarded(Fn&& fn) {
    try {
        return fn();
    } catch (const Fail& f) {
        PyObject* args = Py_BuildValue("(is)", f.status, f.message.c_str());
        if (args) PyErr_SetObject(g_error ? g_error : PyExc_RuntimeError, args);
        Py_XDECREF(args);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

struct Owned {  // a reference to give back
    PyObject* p;
    explicit Owned(PyObject* o) : p(o) {}
    ~Owned() { Py_XDECREF(p); }
};

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* none() { return Py_NewRef(Py_None); }

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        invalid("an integer argument is out of range or of another type");
    }
    return v;
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) invalid(std::string(what) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}

int code_of(at::ScalarType t) {
    return t == at::kFloat ? VCSRMC_F32 : t == at::kHalf ? VCSRMC_F16 : t == at::kBFloat16 ? VCSRMC_BF16 : -1;
}

// A dense matrix that an operator takes.
struct Matrix {
    void* p = nullptr;
    int64_t ld = 0, rows = 0, cols = 0;
    int code = 0, device = 0;
};

Matrix dense(const at::Tensor& t, const char* what) {
    Matrix m;
    if (t.layout() != at::kStrided || t.dim() != 2 || (m.code = code_of(t.scalar_type())) < 0)
        invalid(std::string(what) + " must be a 2-D float32, float16 or bfloat16 tensor");
    if (!t.is_cuda()) invalid(std::string(what) + " must be a CUDA tensor");
    m.rows = t.size(0);
    m.cols = t.size(1);
    if (t.stride(1) != 1 && m.cols > 1) invalid("the columns of " + std::string(what) + " must be contiguous");
    m.ld = t.stride(0);
    if (m.rows <= 1) m.ld = std::max<int64_t>(m.cols, 1);  // torch leaves the stride of a single row open
    else if (m.ld < m.cols) invalid("the rows of " + std::string(what) + " must not overlap");
    if (m.cols > INT32_MAX) invalid(std::string(what) + " has too many columns");
    m.p = t.data_ptr();
    m.device = t.get_device();
    return m;
}
Matrix like(PyObject* o, const char* what, const Matrix& x, int code = -1) {
    const Matrix m = dense(tensor(o, what), what);
    if (m.rows != x.rows || m.cols != x.cols || m.device != x.device)
        invalid(std::string(what) + " must have the shape and the device of the tensor it goes with");
    if (code >= 0 && m.code != code) invalid(std::string(what) + " has another type than the tensors it goes with");
    return m;
}
Matrix vector(PyObject* o, const char* what, int device, int64_t n) {
    const at::Tensor& t = tensor(o, what);
    Matrix m;
    m.code = code_of(t.scalar_type());
    if (t.layout() != at::kStrided || t.dim() != 1 || t.size(0) != n || m.code < 0 || !t.is_cuda() || t.get_device() != device ||
        (n > 1 && t.stride(0) != 1))
        invalid(std::string(what) + " must be a contiguous float32, float16 or bfloat16 tensor of " + std::to_string(n) +
                " values on the other tensors' device");
    m.p = t.data_ptr();
    return m;
}

at::Tensor empty(int64_t rows, int64_t cols, at::ScalarType t, int device) {
    return at::detail::empty_cuda({rows, cols}, t, at::Device(at::kCUDA, c10::DeviceIndex(device)), c10::nullopt);
}
at::Tensor empty(int64_t n, at::ScalarType t, int device) {
    return at::detail::empty_cuda({n}, t, at::Device(at::kCUDA, c10::DeviceIndex(device)), c10::nullopt);
}

// An MX matrix: what MXDense holds.
struct Mx {
    at::Tensor data, scale;
    int kind = 0;
    int64_t ldq = 0, lds = 0;
    uint8_t* s() const { return static_cast<uint8_t*>(scale.data_ptr()); }
};

// Rows of elements at multiples of 16 bytes, of scales at multiples of 4.
Mx mx_new(int64_t rows, int64_t cols, int kind, int device) {
    if (kind != VCSRMC_MXF8 && kind != VCSRMC_MXF4) invalid("the microscaled kind must be MXF8 or MXF4");
    Mx m;
    m.kind = kind;
    const int64_t width = kind == VCSRMC_MXF8 ? cols : (cols + 1) / 2, blocks = (cols + 31) / 32;
    m.ldq = (width + 15) / 16 * 16;
    m.lds = (blocks + 3) / 4 * 4;
    m.data = empty(rows, m.ldq, kind == VCSRMC_MXF8 ? at::kFloat8_e4m3fn : at::kByte, device);
    m.scale = empty(rows, m.lds, at::kFloat8_e8m0fnu, device);
    if (m.ldq != width) m.data = m.data.narrow(1, 0, width);
    if (m.lds != blocks) m.scale = m.scale.narrow(1, 0, blocks);
    return m;
}
// Whether a tensor still holds rows x width elements, its rows ld apart.
bool holds(const at::Tensor& t, int64_t rows, int64_t width, int64_t ld) {
    return t.layout() == at::kStrided && t.dim() == 2 && t.element_size() == 1 && t.size(0) == rows && t.size(1) >= width &&
           (rows <= 1 || t.stride(0) == ld) && (t.size(1) <= 1 || t.stride(1) == 1);
}
// From five arguments (data, scale, kind, ldq, lds) that were checked when the matrix was made, and its shape. A tensor may have been
// changed in place since (resize_, set_, t_), and the kernels would follow the old strides out of it: sizes are looked at again.
Mx mx_given(PyObject* const* a, int64_t rows, int64_t cols) {
    Mx m;
    m.data = tensor(a[0], "MX elements");
    m.scale = tensor(a[1], "MX scales");
    m.kind = int(integer(a[2]));
    m.ldq = integer(a[3]);
    m.lds = integer(a[4]);
    if (!m.data.is_cuda() || !m.scale.is_cuda()) invalid("microscaled operators run on CUDA tensors");
    if (!holds(m.data, rows, m.kind == VCSRMC_MXF8 ? cols : (cols + 1) / 2, m.ldq) || !holds(m.scale, rows, (cols + 31) / 32, m.lds) ||
        m.data.get_device() != m.scale.get_device())
        invalid("the tensors of an MX matrix were changed after it was made");
    return m;
}
PyObject* mx_result(const Mx& m) {
    Owned d(wrap(m.data)), s(wrap(m.scale));
    return Py_BuildValue("(OOLL)", d.p, s.p, static_cast<long long>(m.ldq), static_cast<long long>(m.lds));
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream(); }

void count(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) invalid("wrong number of arguments");
}

// (error class): what failures raise
PyObject* set_error(PyObject*, PyObject* cls) {
    Py_XSETREF(g_error, Py_NewRef(cls));
    return none();
}

// (rows, cols, kind, device) -> (data, scale, ldq, lds)
PyObject* mx_empty(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        count(n, 4);
        return mx_result(mx_new(integer(a[0]), integer(a[1]), int(integer(a[2])), int(integer(a[3]))));
    });
}

// (X, kind, out's five or Nones) -> (data, scale, ldq, lds)
PyObject* mx_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        count(n, 7);
        const Matrix x = dense(tensor(a[0], "X"), "X");
        c10::cuda::CUDAGuard guard{c10::DeviceIndex(x.device)};
        const Mx q = a[2] == Py_None ? mx_new(x.rows, x.cols, int(integer(a[1])), x.device) : mx_given(a + 2, x.rows, x.cols);
        check(vcsrmc_mx_quantize(x.p, x.code, x.ld, x.rows, int32_t(x.cols), q.kind, q.data.data_ptr(), q.ldq, q.s(), q.lds,
                                 stream_of(x.device)));
        return mx_result(q);
    });
}

// (Q's five, rows, cols, Y) -> None
PyObject* mx_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        count(n, 8);
        const int64_t rows = integer(a[5]), cols = integer(a[6]);
        const Mx q = mx_given(a, rows, cols);
        const int device = q.data.get_device();
        const Matrix y = dense(tensor(a[7], "out"), "out");
        if (y.rows != rows || y.cols != cols || y.device != device) invalid("out must have Q's shape and device");
        c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
        check(vcsrmc_mx_dequantize(q.data.data_ptr(), q.kind, q.ldq, q.s(), q.lds, rows, int32_t(cols), y.p, y.code, y.ld, stream_of(device)));
        return none();
    });
}

// (handle, device, M, N, B's five, B's rows and columns, O, C, accumulate) -> None
PyObject* spmm_mx(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        count(n, 14);
        auto* d = reinterpret_cast<const vcsrmc_device_format*>(integer(a[0]));
        const int device = int(integer(a[1]));
        const int64_t rows = integer(a[9]), cols = integer(a[10]), O = integer(a[11]);
        const Mx q = mx_given(a + 4, rows, cols);
        const Matrix c = dense(tensor(a[12], "C"), "C");
        if (c.code != VCSRMC_F32) invalid("C must be float32");
        if (c.device != device || q.data.get_device() != device) invalid("A, B and C must be on the same device");
        if (cols < O || c.cols < O || rows < integer(a[3]) || c.rows < integer(a[2]))
            invalid("B and C must hold A's columns and rows, with >= O columns");
        c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
        int64_t bytes = 0;
        check(vcsrmc_spmm_mx_workspace(d, int32_t(std::max<int64_t>(O, 0)), &bytes));
        at::Tensor ws;
        if (bytes > 0) ws = empty(bytes, at::kByte, device);
        check(vcsrmc_spmm_mx(d, q.data.data_ptr(), q.kind, q.ldq, q.s(), q.lds, int32_t(O), static_cast<float*>(c.p), c.ld,
                             int(integer(a[13])), bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(device)));
        return none();
    });
}

// (X, weight, residual, eps, kind, out's five or Nones, residual_out) -> (data, scale, ldq, lds, residual_out, inv_rms)
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 11);
        const Matrix x = dense(tensor(a[0], "X"), "X");
        const Matrix w = vector(a[1], "weight", x.device, x.cols);
        Matrix r, o;
        r.code = x.code;
        if (a[2] != Py_None) r = like(a[2], "residual", x);
        const double eps = PyFloat_AsDouble(a[3]);
        if (eps == -1.0 && PyErr_Occurred()) return nullptr;
        c10::cuda::CUDAGuard guard{c10::DeviceIndex(x.device)};
        at::Tensor h;
        if (a[10] != Py_None) {
            o = like(a[10], "residual_out", x, r.code);
            h = tensor(a[10], "residual_out");
        } else if (a[2] != Py_None) {
            h = empty(x.rows, x.cols, THPVariable_Unpack(a[2]).scalar_type(), x.device);
            o.p = h.data_ptr();
            o.ld = std::max<int64_t>(x.cols, 1);
        }
        const Mx q = a[5] == Py_None ? mx_new(x.rows, x.cols, int(integer(a[4])), x.device) : mx_given(a + 5, x.rows, x.cols);
        const at::Tensor inv = empty(x.rows, at::kFloat, x.device);
        check(vcsrmc_add_rms_norm(x.p, x.code, x.ld, r.p, r.ld, o.p, o.ld, r.code, w.p, w.code, float(eps), x.rows, int32_t(x.cols), q.kind,
                                  q.data.data_ptr(), q.ldq, q.s(), q.lds, static_cast<float*>(inv.data_ptr()), stream_of(x.device)));
        Owned data(wrap(q.data)), scale(wrap(q.scale)), hp(h.defined() ? wrap(h) : Py_NewRef(a[0])), ip(wrap(inv));
        return Py_BuildValue("(OOLLOO)", data.p, scale.p, static_cast<long long>(q.ldq), static_cast<long long>(q.lds), hp.p, ip.p);
    });
}

// (dY, weight, hidden, inv_rms, d_residual, out) -> (dX, dweight)
PyObject* add_rms_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        count(n, 6);
        const Matrix dy = dense(tensor(a[0], "dY"), "dY");
        const Matrix w = vector(a[1], "weight", dy.device, dy.cols);
        const Matrix h = like(a[2], "hidden", dy);
        const Matrix inv = vector(a[3], "inv_rms", dy.device, dy.rows);
        if (inv.code != VCSRMC_F32) invalid("inv_rms must be float32");
        Matrix dr, dx;
        if (a[4] != Py_None) dr = like(a[4], "d_residual", dy, h.code);
        c10::cuda::CUDAGuard guard{c10::DeviceIndex(dy.device)};
        at::Tensor out;
        if (a[5] != Py_None) {
            dx = like(a[5], "out", dy, h.code);
            out = tensor(a[5], "out");
        } else {
            out = empty(dy.rows, dy.cols, THPVariable_Unpack(a[2]).scalar_type(), dy.device);
            dx.p = out.data_ptr();
            dx.ld = std::max<int64_t>(dy.cols, 1);
        }
        const at::Tensor dw = empty(dy.cols, at::kFloat, dy.device);
        int64_t bytes = 0;
        check(vcsrmc_add_rms_norm_backward_workspace(dy.rows, int32_t(dy.cols), &bytes));
        const at::Tensor ws = empty(bytes, at::kByte, dy.device);
        check(vcsrmc_add_rms_norm_backward(dy.p, dy.code, dy.ld, dr.p, dr.ld, h.p, h.ld, h.code, w.p, w.code,
                                           static_cast<const float*>(inv.p), dy.rows, int32_t(dy.cols), dx.p, dx.ld,
                                           static_cast<float*>(dw.data_ptr()), ws.data_ptr(), bytes, stream_of(dy.device)));
        Owned x(wrap(out)), y(wrap(dw));
        return Py_BuildValue("(OO)", x.p, y.p);
    });
}

#define VCSRMC_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"set_error", set_error, METH_O, nullptr},
                         VCSRMC_FAST(mx_empty),
                         VCSRMC_FAST(mx_quantize),
                         VCSRMC_FAST(mx_dequantize),
                         VCSRMC_FAST(spmm_mx),
                         VCSRMC_FAST(add_rms_norm),
                         VCSRMC_FAST(add_rms_norm_backward),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
