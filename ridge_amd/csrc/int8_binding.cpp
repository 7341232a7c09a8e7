// int8_binding.cpp -- the tensors' way to the C ABI in include/ridge_int8.h: the checks of
// arguments, the allocation of results and the current stream behind ridge_amd.int8.
//
// Native because the calls are short: a decoding step's norm runs 3 us on the GPU, and
// checking its six tensors in Python took 6 us on the host (9.3 us a call, 3.2 so).

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <optional>
#include <utility>

#include "ridge_int8.h"

namespace {

PyObject* gError = nullptr;   // ridge_amd.int8.RidgeInt8Error

constexpr int64_t kMostStride = 1 << 23;   // of a product's 8-bit rows

// A refusal: its text becomes gError's.
struct Refusal {
    char text[256];
};

[[noreturn]] void refuse(const char* format, ...) {
    Refusal r;
    va_list args;
    va_start(args, format);
    vsnprintf(r.text, sizeof r.text, format, args);
    va_end(args);
    throw r;
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse("%s must be a tensor", what);
    return THPVariable_Unpack(o);
}

// The tensor, or null for None.
const at::Tensor* optionalTensor(PyObject* o, const char* what) {
    return o == Py_None ? nullptr : &tensor(o, what);
}

int typeCode(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return RIDGE_F16;
        case at::kBFloat16: return RIDGE_BF16;
        case at::kFloat: return RIDGE_F32;
        default: return -1;
    }
}

int typeOf(const at::Tensor& t, const char* what) {
    const int code = typeCode(t.scalar_type());
    if (code < 0) refuse("%s must be float16, bfloat16 or float32, not %s", what, c10::toString(t.scalar_type()));
    return code;
}

void noGradient(const at::Tensor* t) {
    if (t && t->requires_grad() && at::GradMode::is_enabled())
        refuse("the 8-bit operators have no gradient: call them under torch.no_grad()");
    // Level 0 is the only one. Undefined too where forward mode is off; no_grad leaves it on.
    if (t && t->_fw_grad(0).defined())
        refuse("the 8-bit operators have no gradient in forward mode either: take the primal of dual tensors");
}

// A tensor of the caller's that a call has written through its address: a graph that saved it
// notices by its version, as for torch's own writes. (Tensors of inference mode have none.)
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Rows {
    int64_t rows, cols, ld;
};

int64_t to16(int64_t cols) { return (cols + 15) / 16 * 16; }

// A 2-D device tensor whose rows are contiguous.
Rows matrix(const at::Tensor& t, const char* what, const at::Device* device = nullptr) {
    if (!t.is_cuda() || t.dim() != 2 || t.layout() != at::kStrided) refuse("%s must be a 2-D device tensor", what);
    if (device && t.device() != *device)
        refuse("%s is on device %d, not on %d", what, (int)t.device().index(), (int)device->index());
    Rows r = {t.size(0), t.size(1), t.stride(0)};
    if (t.stride(1) != 1 && r.cols > 1) refuse("%s must have contiguous rows", what);
    if (r.rows <= 1) {
        r.ld = r.cols;
    } else if (r.ld < r.cols) {
        refuse("the rows of %s overlap", what);
    }
    return r;
}

void vector(const at::Tensor& t, int64_t n, at::ScalarType type, const at::Device& device, const char* what) {
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || t.device() != device || (n > 1 && t.stride(0) != 1))
        refuse("%s must be %lld contiguous %s on the operands' device", what, (long long)n, c10::toString(type));
}

// 8-bit rows with their scales.
Rows rows8(const at::Tensor& q, const at::Tensor& scale, const char* what, const at::Device* device = nullptr) {
    Rows r = matrix(q, what, device);
    if (q.scalar_type() != at::kChar) refuse("%s must be int8, not %s", what, c10::toString(q.scalar_type()));
    if (r.rows <= 1) r.ld = to16(r.cols);
    if (r.ld % 16 || (uintptr_t)q.data_ptr() % 16)
        refuse("the rows of %s must start at multiples of 16 bytes (as those of empty() do)", what);
    if (r.cols % 16 && r.rows &&
        q.storage_offset() + (r.rows - 1) * r.ld + to16(r.cols) > (int64_t)q.storage().nbytes())
        refuse("the last row of %s ends its memory inside 16 bytes (make it with empty())", what);
    vector(scale, r.rows, at::kFloat, q.device(), "the scales of 8-bit rows");
    return r;
}

// The bytes of a matrix: rows of `bytes`, `stride` apart.
struct Span {
    const char* what;
    int64_t at, rows, bytes, stride;
};

Span span(const at::Tensor& t, const Rows& r, const char* what) {
    const int64_t size = t.element_size();
    return {what, (int64_t)t.data_ptr(), r.rows, r.cols * size, r.ld * size};
}

Span span(const at::Tensor& vector, const char* what) {
    return span(vector, {1, vector.size(0), vector.size(0)}, what);
}

int64_t floorDivide(int64_t n, int64_t d) { return n / d - (n % d < 0); }

// Whether any row of a shares a byte with one of b: column slices of one buffer do not, whose
// rows lie between each other's.
bool meet(Span a, Span b) {
    if (a.rows < 1 || b.rows < 1 || a.bytes < 1 || b.bytes < 1) return false;
    if (a.at >= b.at + (b.rows - 1) * b.stride + b.bytes || b.at >= a.at + (a.rows - 1) * a.stride + a.bytes) return false;
    if (a.rows > b.rows) std::swap(a, b);
    if (b.rows == 1) return true;
    if (a.rows == 1) a.stride = b.stride;
    // The last row of b that begins before the end of a's row i ends behind all others.
    auto row = [&](int64_t i, int64_t least) {
        const int64_t begin = a.at + i * a.stride;
        const int64_t j = std::min(floorDivide(begin + a.bytes - 1 - b.at, b.stride), least + b.rows - 1);
        return j >= least && b.at + j * b.stride + b.bytes > begin;
    };
    // Of equal strides only j - i counts, from 1 - a.rows on.
    if (a.stride == b.stride) {
        b.rows += a.rows - 1;
        return row(0, 1 - a.rows);
    }
    for (int64_t i = 0; i < a.rows; ++i)
        if (row(i, 0)) return true;
    return false;
}

// A call's workgroups read and write in no order: what it writes may be nothing else of it.
void apart(const Span& written, const Span& other) {
    if (meet(written, other)) refuse("%s overlaps %s", written.what, other.what);
}

// An attribute that is a whole number, or a whole number itself.
void* numberOf(PyObject* o, const char* attribute) {
    PyObject* number = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttrString(o, attribute);
    void* value = number ? PyLong_AsVoidPtr(number) : nullptr;
    Py_XDECREF(number);
    if (PyErr_Occurred()) throw python_error();
    return value;
}

// The handle of one of torch's streams, or the handle itself, on the operands' device.
hipStream_t streamOf(PyObject* stream, c10::DeviceIndex device) {
    const hipStream_t handle = (hipStream_t)numberOf(stream, "cuda_stream");
    int64_t on = device;
    hipDevice_t found;
    if (PyObject_HasAttrString(stream, "device_index")) {   // a default stream's handle is null on every device
        on = (int64_t)(intptr_t)numberOf(stream, "device_index");
    } else if (handle && hipStreamGetDevice(handle, &found) == hipSuccess) {
        on = found;
    }
    if (on != device) refuse("the stream is on device %lld, not on the operands' %d", (long long)on, (int)device);
    return handle;
}

// Makes the operands' device current, and the stream: the current one for None, else one
// of torch's streams or a handle. Memory that a call allocates is then that stream's.
class On {
  public:
    On(const at::Device& device, PyObject* stream) : device_(device.index()), before_(c10::hip::current_device()) {
        const hipStream_t p = stream != Py_None ? streamOf(stream, device_) : nullptr;
        if (device_ != before_) c10::hip::set_device(device_);
        if (stream != Py_None) {
            current_ = c10::hip::getCurrentHIPStream(device_);
            c10::hip::setCurrentHIPStream(p ? c10::hip::getStreamFromExternal(p, device_)
                                            : c10::hip::getDefaultHIPStream(device_));
        }
    }
    ~On() {
        if (current_) c10::hip::setCurrentHIPStream(*current_);
        if (device_ != before_) c10::hip::set_device(before_);
    }
    On(const On&) = delete;
    On& operator=(const On&) = delete;
    void* stream() const { return c10::hip::getCurrentHIPStream(device_).stream(); }

  private:
    c10::DeviceIndex device_, before_;
    std::optional<c10::hip::HIPStream> current_;
};

void enqueued(const char* what, int rc) {
    if (rc != 0) refuse("%s returned hipError %d", what, rc);
}

// 8-bit rows to write: the caller's (q, scale), or new ones.
struct RowsOut {
    at::Tensor q, scale;
    int64_t ld = 0;
    RowsOut(PyObject* out, int64_t rows, int64_t cols, const at::Device& device) : given(out) {
        if (out == Py_None) {
            ld = ridge_int8_row_stride(cols);
            q = at::empty({rows, ld}, at::TensorOptions(device).dtype(at::kChar)).narrow(1, 0, cols);
            scale = at::empty({rows}, at::TensorOptions(device).dtype(at::kFloat));
            return;
        }
        if (!PyTuple_Check(out) || PyTuple_GET_SIZE(out) != 2) refuse("out must be (q, scale)");
        q = tensor(PyTuple_GET_ITEM(out, 0), "out's q");
        scale = tensor(PyTuple_GET_ITEM(out, 1), "out's scales");
        const Rows r = rows8(q, scale, "out", &device);
        if (r.rows != rows || r.cols != cols)
            refuse("out holds %lld x %lld, not %lld x %lld", (long long)r.rows, (long long)r.cols, (long long)rows,
                   (long long)cols);
        noGradient(&scale);
        ld = r.ld;
        apart(span(scale, "out's scales"), span8());
    }
    Span span8() const { return span(q, {q.size(0), q.size(1), ld}, "out's q"); }
    // An operand of the call that writes the rows.
    void apartFrom(const Span& other) const {
        if (given == Py_None) return;
        apart(span8(), other);
        apart(span(scale, "out's scales"), other);
    }
    int8_t* at8() const { return (int8_t*)q.data_ptr(); }
    float* atScale() const { return (float*)scale.data_ptr(); }
    void wrote() const {
        if (given == Py_None) return;
        written(q);
        written(scale);
    }
    PyObject* result() const {
        if (given != Py_None) return Py_NewRef(given);
        return Py_BuildValue("(NN)", THPVariable_Wrap(q), THPVariable_Wrap(scale));
    }
    PyObject* given;
};

std::optional<at::ScalarType> optionalType(PyObject* dtype) {
    if (dtype == Py_None) return std::nullopt;
    if (!THPDtype_Check(dtype)) refuse("dtype must be a torch.dtype");
    return ((THPDtype*)dtype)->scalar_type;
}

// A 16- or 32-bit result: the caller's, or a new one of `dtype` (float16 for None).
struct MatrixOut {
    at::Tensor t;
    Rows r;
    int code;
    MatrixOut(PyObject* out, PyObject* dtype, int64_t rows, int64_t cols, const at::Device& device) : given(out) {
        const auto type = optionalType(dtype);
        if (type && typeCode(*type) < 0)
            refuse("the result must be float16, bfloat16 or float32, not %s", c10::toString(*type));
        t = out == Py_None ? at::empty({rows, cols}, at::TensorOptions(device).dtype(type.value_or(at::kHalf)))
                           : tensor(out, "out");
        r = matrix(t, "out", &device);
        code = typeOf(t, "out");
        noGradient(&t);
        if (r.rows != rows || r.cols != cols || (type && t.scalar_type() != *type))
            refuse("out must be %lld x %lld%s%s", (long long)rows, (long long)cols, type ? " of " : "",
                   type ? c10::toString(*type) : "");
    }
    void apartFrom(const Span& other) const {
        if (given != Py_None) apart(span(t, r, "out"), other);
    }
    void wrote() const {
        if (given != Py_None) written(t);
    }
    PyObject* result() const { return given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(t); }
    PyObject* given;
};

PyObject* rowsOf(PyObject* const* args, Py_ssize_t n, bool gated) {
    const char* what = gated ? "gate_up" : "x";
    if (n != 3) refuse("3 arguments are wanted");
    const at::Tensor& x = tensor(args[0], what);
    const Rows r = matrix(x, what);
    const int code = typeOf(x, what);
    noGradient(&x);
    if (r.cols < 1) refuse("%s has no columns", what);
    if (gated && r.cols % 2) refuse("gate_up has %lld columns: two halves are wanted", (long long)r.cols);
    const int64_t cols = gated ? r.cols / 2 : r.cols;
    const On on(x.device(), args[2]);
    const RowsOut out(args[1], r.rows, cols, x.device());
    out.apartFrom(span(x, r, what));
    const auto call = gated ? ridge_int8_silu_mul : ridge_int8_quantize;
    enqueued(gated ? "ridge_int8_silu_mul" : "ridge_int8_quantize",
             call(x.data_ptr(), r.ld, code, out.at8(), out.ld, out.atScale(), r.rows, cols, on.stream()));
    out.wrote();
    return out.result();
}

PyObject* quantizeImpl(PyObject* const* args, Py_ssize_t n) { return rowsOf(args, n, false); }
PyObject* siluMulImpl(PyObject* const* args, Py_ssize_t n) { return rowsOf(args, n, true); }

PyObject* rmsNormImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 7) refuse("7 arguments are wanted");
    const at::Tensor& x = tensor(args[0], "x");
    const Rows r = matrix(x, "x");
    const int code = typeOf(x, "x");
    const at::Device device = x.device();
    const at::Tensor& weight = tensor(args[1], "weight");
    const double eps = PyFloat_AsDouble(args[2]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    const at::Tensor* residual = optionalTensor(args[3], "residual");
    if (!residual && args[4] != Py_None) refuse("residual_out without a residual");
    noGradient(&x);
    noGradient(&weight);
    noGradient(residual);
    if (r.cols < 1) refuse("x has no columns");
    const int weightCode = typeOf(weight, "weight");
    if (weightCode != code && weightCode != RIDGE_F32) refuse("weight must be of x's type or float32");
    vector(weight, r.cols, weight.scalar_type(), device, "weight");
    if (!(eps > 0 && (float)eps > 0 && std::isfinite((float)eps))) refuse("eps must be positive, not %g", eps);
    const On on(device, args[6]);
    Rows in = {0, 0, 0}, to = {0, 0, 0};
    at::Tensor residualOut;
    if (residual) {
        residualOut = args[4] == Py_None ? at::empty({r.rows, r.cols}, x.options()) : tensor(args[4], "residual_out");
        in = matrix(*residual, "residual", &device);
        to = matrix(residualOut, "residual_out", &device);
        if (residual->scalar_type() != x.scalar_type() || in.rows != r.rows || in.cols != r.cols)
            refuse("residual must be like x");
        if (residualOut.scalar_type() != x.scalar_type() || to.rows != r.rows || to.cols != r.cols)
            refuse("residual_out must be like x");
        noGradient(&residualOut);
    }
    const RowsOut out(args[5], r.rows, r.cols, device);
    const Span spanX = span(x, r, "x"), spanWeight = span(weight, "weight");
    out.apartFrom(spanX);
    out.apartFrom(spanWeight);
    if (residual) {
        const Span spanResidual = span(*residual, in, "residual"), spanSum = span(residualOut, to, "residual_out");
        out.apartFrom(spanResidual);
        if (args[4] != Py_None) {
            out.apartFrom(spanSum);
            apart(spanSum, spanWeight);
            // x or residual itself: a thread reads what it then writes.
            for (const Span& from : {spanX, spanResidual})
                if (spanSum.at != from.at || spanSum.stride != from.stride) apart(spanSum, from);
        }
    }
    enqueued("ridge_int8_rms_norm",
             ridge_int8_rms_norm(x.data_ptr(), r.ld, residual ? residual->data_ptr() : nullptr, in.ld, weight.data_ptr(),
                                 weightCode, (float)eps, code, residual ? residualOut.data_ptr() : nullptr, to.ld,
                                 out.at8(), out.ld, out.atScale(), r.rows, r.cols, on.stream()));
    out.wrote();
    if (residual && args[4] != Py_None) written(residualOut);
    PyObject* sum = !residual ? Py_NewRef(Py_None) : args[4] != Py_None ? Py_NewRef(args[4]) : THPVariable_Wrap(residualOut);
    if (args[5] != Py_None)
        return Py_BuildValue("(OON)", PyTuple_GET_ITEM(args[5], 0), PyTuple_GET_ITEM(args[5], 1), sum);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(out.q), THPVariable_Wrap(out.scale), sum);
}

PyObject* dequantizeImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 5) refuse("5 arguments are wanted");
    const at::Tensor &q = tensor(args[0], "q"), &scale = tensor(args[1], "scale");
    const Rows r = rows8(q, scale, "q");
    if (r.cols < 1) refuse("q has no columns");
    noGradient(&scale);
    const On on(q.device(), args[4]);
    const MatrixOut out(args[3], args[2], r.rows, r.cols, q.device());
    out.apartFrom(span(q, r, "q"));
    out.apartFrom(span(scale, "scale"));
    enqueued("ridge_int8_dequantize",
             ridge_int8_dequantize((const int8_t*)q.data_ptr(), r.ld, (const float*)scale.data_ptr(), out.t.data_ptr(),
                                   out.r.ld, out.code, r.rows, r.cols, on.stream()));
    out.wrote();
    return out.result();
}

PyObject* gemmImpl(PyObject* const* args, Py_ssize_t n) {
    if (n != 8) refuse("8 arguments are wanted");
    const at::Tensor &a = tensor(args[0], "a"), &aScale = tensor(args[1], "a_scale");
    const at::Tensor &b = tensor(args[2], "b"), &bScale = tensor(args[3], "b_scale");
    const at::Device device = a.device();
    const Rows ra = rows8(a, aScale, "a"), rb = rows8(b, bScale, "b", &device);
    if (ra.cols != rb.cols) refuse("rows of %lld and of %lld do not chain", (long long)ra.cols, (long long)rb.cols);
    if (ra.cols < 1 || ra.cols > RIDGE_INT8_MAX_K || ra.ld >= kMostStride || rb.ld >= kMostStride)
        refuse("K must be 1 to %d and strides below %lld, not %lld, %lld and %lld", (int)RIDGE_INT8_MAX_K,
               (long long)kMostStride, (long long)ra.cols, (long long)ra.ld, (long long)rb.ld);
    const at::Tensor* bias = optionalTensor(args[4], "bias");
    noGradient(&aScale);
    noGradient(&bScale);
    noGradient(bias);
    const On on(device, args[7]);
    const MatrixOut out(args[6], args[5], ra.rows, rb.rows, device);
    if (bias) vector(*bias, rb.rows, out.t.scalar_type(), device, "bias");
    out.apartFrom(span(a, ra, "a"));
    out.apartFrom(span(b, rb, "b"));
    out.apartFrom(span(aScale, "a_scale"));
    out.apartFrom(span(bScale, "b_scale"));
    if (bias) out.apartFrom(span(*bias, "bias"));
    enqueued("ridge_int8_gemm",
             ridge_int8_gemm((const int8_t*)a.data_ptr(), ra.ld, (const float*)aScale.data_ptr(),
                             (const int8_t*)b.data_ptr(), rb.ld, (const float*)bScale.data_ptr(),
                             bias ? bias->data_ptr() : nullptr, out.t.data_ptr(), out.r.ld, out.code, ra.rows, rb.rows,
                             ra.cols, on.stream()));
    out.wrote();
    return out.result();
}

// One of the calls above as Python sees it: a refusal becomes gError, and an exception of
// torch's (an allocation that fails) the error that torch makes of it.
template <PyObject* (*call)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        return call(args, n);
    } catch (const Refusal& r) {
        PyErr_SetString(gError ? gError : PyExc_RuntimeError, r.text);
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject* setError(PyObject*, PyObject* type) {
    Py_XDECREF(gError);
    gError = Py_NewRef(type);
    Py_RETURN_NONE;
}

PyMethodDef gMethods[] = {
    {"quantize", (PyCFunction)(void (*)(void))entry<quantizeImpl>, METH_FASTCALL, "(x, out, stream)"},
    {"silu_mul", (PyCFunction)(void (*)(void))entry<siluMulImpl>, METH_FASTCALL, "(gate_up, out, stream)"},
    {"rms_norm", (PyCFunction)(void (*)(void))entry<rmsNormImpl>, METH_FASTCALL,
     "(x, weight, eps, residual, residual_out, out, stream)"},
    {"dequantize", (PyCFunction)(void (*)(void))entry<dequantizeImpl>, METH_FASTCALL, "(q, scale, dtype, out, stream)"},
    {"gemm", (PyCFunction)(void (*)(void))entry<gemmImpl>, METH_FASTCALL,
     "(a, a_scale, b, b_scale, bias, dtype, out, stream)"},
    {"set_error", setError, METH_O, "the class that refusals are raised as"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef gModule = {PyModuleDef_HEAD_INIT, "_ridge_int8", "The calls behind ridge_amd.int8.", -1, gMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ridge_int8(void) { return PyModule_Create(&gModule); }
