// CPython binding of the launch-bound kernels of include/basalt_b200_kernels.h (module basalt_b200._klaunch). A call through ctypes
// converts its arguments in 2.6 us, longer than the launch it makes; a pass of the norm over one row came down from 10.9 to 8.4 us. The
// functions take their C counterparts' arguments in order and return their code. A pointer is an int, None (NULL) or an
// object with a device_ptr() method (a DeviceBuffer); a row stride of None is a row without a gap; a stream of None is the default stream.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdint.h>

#include "../../include/basalt_b200_kernels.h"

namespace {

// Reads arguments one after the other; the first that does not fit its parameter leaves a Python error, and zeros after it.
struct Reader {
    PyObject* const* next;
    bool failed = false;

    uint64_t address() {
        PyObject* o = *next++;
        if (failed || o == Py_None) return 0;
        PyObject* held = nullptr;
        if (!PyLong_Check(o)) {
            if (!(held = PyIndex_Check(o) ? PyNumber_Index(o) : PyObject_CallMethod(o, "device_ptr", nullptr))) return failed = true, 0;
            o = held;
        }
        const uint64_t v = PyLong_AsUnsignedLongLong(o);
        Py_XDECREF(held);
        if (v == (uint64_t)-1 && PyErr_Occurred()) failed = true;
        return v;
    }
    template <class T>
    T* pointer() { return (T*)(uintptr_t)address(); }
    int64_t integer(int64_t none) {
        PyObject* o = *next++;
        if (failed || o == Py_None) return none;
        const int64_t v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) failed = true;
        return v;
    }
    int64_t integer() {
        if (!failed && *next == Py_None) PyErr_SetString(PyExc_TypeError, "an integer is needed"), failed = true;
        return integer(0);
    }
    int small() {   // an int parameter
        const int64_t v = integer();
        if (!failed && (v < INT32_MIN || v > INT32_MAX)) PyErr_SetString(PyExc_OverflowError, "an argument does not fit 32 bits"), failed = true;
        return (int)v;
    }
    float real() {
        PyObject* o = *next++;
        if (failed) return 0.0f;
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) failed = true;
        return (float)v;
    }
};

bool arity(Py_ssize_t got, Py_ssize_t want) {
    if (got == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments are needed, %zd were given", want, got);
    return false;
}

template <class F>
PyObject* launched(const Reader& r, F launch) {
    if (r.failed) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = launch();
    Py_END_ALLOW_THREADS return PyLong_FromLong(rc);
}

PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arity(n, 15)) return nullptr;
    Reader cols_of{args + 13};
    const int64_t cols = cols_of.integer();
    Reader r{args, cols_of.failed};
    const int type = r.small();
    const void* x = r.pointer<void>();
    const int64_t ldx = r.integer(cols);
    const void* residual = r.pointer<void>();
    const int64_t ldr = r.integer(cols);
    void* total = r.pointer<void>();
    const int64_t ldt = r.integer(cols);
    const void* weight = r.pointer<void>();
    const float eps = r.real();
    void* y = r.pointer<void>();
    const int64_t ldy = r.integer(cols);
    float* scales = r.pointer<float>();
    const int64_t rows = r.integer();
    r.next++;
    void* stream = r.pointer<void>();
    return launched(r, [&] { return basalt_k_rms_norm(type, x, ldx, residual, ldr, total, ldt, weight, eps, y, ldy, scales, rows, cols, stream); });
}

PyObject* quantize_e4m3(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arity(n, 9)) return nullptr;
    Reader cols_of{args + 7};
    const int64_t cols = cols_of.integer();
    Reader r{args, cols_of.failed};
    const int type = r.small();
    const void* x = r.pointer<void>();
    const int64_t ldx = r.integer(cols);
    void* q = r.pointer<void>();
    const int64_t ldq = r.integer(cols);
    float* scales = r.pointer<float>();
    const int64_t rows = r.integer();
    r.next++;
    void* stream = r.pointer<void>();
    return launched(r, [&] { return basalt_k_quantize_e4m3(type, x, ldx, q, ldq, scales, rows, cols, stream); });
}

PyObject* matmul_e4m3(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arity(n, 14)) return nullptr;
    Reader sizes{args + 9};
    const int M = sizes.small(), N = sizes.small(), K = sizes.small();
    Reader r{args, sizes.failed};
    const void* a = r.pointer<void>();
    const int64_t lda = r.integer(K);
    const float* a_scales = r.pointer<float>();
    const void* b = r.pointer<void>();
    const int64_t ldb = r.integer(K);
    const float* b_scales = r.pointer<float>();
    const int type = r.small();
    void* c = r.pointer<void>();
    const int64_t ldc = r.integer(N);
    r.next += 3;
    int32_t* status = r.pointer<int32_t>();
    void* stream = r.pointer<void>();
    return launched(r, [&] { return basalt_k_matmul_e4m3(a, lda, a_scales, b, ldb, b_scales, type, c, ldc, M, N, K, status, stream); });
}

PyObject* matmul_w4(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arity(n, 15)) return nullptr;
    Reader sizes{args + 10};
    const int M = sizes.small(), N = sizes.small(), K = sizes.small();
    Reader r{args, sizes.failed};
    const int type = r.small();
    const void* x = r.pointer<void>();
    const int64_t ldx = r.integer(K);
    const void* w = r.pointer<void>();
    const int64_t ldw = r.integer(((int64_t)K + 1) / 2);
    const void* scales = r.pointer<void>();
    const uint8_t* zeros = r.pointer<uint8_t>();
    const int group = r.small();
    void* c = r.pointer<void>();
    const int64_t ldc = r.integer(N);
    r.next += 3;
    int32_t* status = r.pointer<int32_t>();
    void* stream = r.pointer<void>();
    return launched(r, [&] { return basalt_k_matmul_w4(type, x, ldx, w, ldw, scales, zeros, group, c, ldc, M, N, K, status, stream); });
}

#define FAST(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(rms_norm), FAST(quantize_e4m3), FAST(matmul_e4m3), FAST(matmul_w4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_klaunch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__klaunch(void) { return PyModule_Create(&module); }
