// binding.hpp -- what the Python extensions share: refusals, tensors as rows of bytes, overlaps,
// streams, and the way from a call's refusal to Python's exception.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <optional>
#include <utility>

// Every extension is one translation unit, and has these for itself.
namespace {

PyObject* gError = nullptr;   // the module's class of errors

// The types' codes in the C headers.
enum { kF16 = 0, kBF16 = 1, kF32 = 2 };

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

[[maybe_unused]] const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse("%s must be a tensor", what);
    return THPVariable_Unpack(o);
}

// The tensor, or null for None.
[[maybe_unused]] const at::Tensor* optionalTensor(PyObject* o, const char* what) {
    return o == Py_None ? nullptr : &tensor(o, what);
}

[[maybe_unused]] int typeCode(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return kF16;
        case at::kBFloat16: return kBF16;
        case at::kFloat: return kF32;
        default: return -1;
    }
}

[[maybe_unused]] int typeOf(const at::Tensor& t, const char* what) {
    const int code = typeCode(t.scalar_type());
    if (code < 0) refuse("%s must be float16, bfloat16 or float32, not %s", what, c10::toString(t.scalar_type()));
    return code;
}

[[maybe_unused]] void noGradient(const at::Tensor* t) {
    if (t && t->requires_grad() && at::GradMode::is_enabled())
        refuse("the 8-bit operators have no gradient: call them under torch.no_grad()");
    // Level 0 is the only one. Undefined too where forward mode is off; no_grad leaves it on.
    if (t && t->_fw_grad(0).defined())
        refuse("the 8-bit operators have no gradient in forward mode either: take the primal of dual tensors");
}

// A tensor of the caller's that a call has written through its address: a graph that saved it
// notices by its version, as for torch's own writes. (Tensors of inference mode have none.)
[[maybe_unused]] void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Rows {
    int64_t rows, cols, ld;
};

// A 2-D device tensor whose rows are contiguous.
[[maybe_unused]] Rows matrix(const at::Tensor& t, const char* what, const at::Device* device = nullptr) {
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

[[maybe_unused]] void vector(const at::Tensor& t, int64_t n, at::ScalarType type, const at::Device& device, const char* what) {
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || t.device() != device || (n > 1 && t.stride(0) != 1))
        refuse("%s must be %lld contiguous %s on the operands' device", what, (long long)n, c10::toString(type));
}

// The bytes of a matrix: rows of `bytes`, `stride` apart.
struct Span {
    const char* what;
    int64_t at, rows, bytes, stride;
};

[[maybe_unused]] Span span(const at::Tensor& t, const Rows& r, const char* what) {
    const int64_t size = t.element_size();
    return {what, (int64_t)t.data_ptr(), r.rows, r.cols * size, r.ld * size};
}

[[maybe_unused]] Span span(const at::Tensor& vector, const char* what) {
    return span(vector, {1, vector.size(0), vector.size(0)}, what);
}

[[maybe_unused]] int64_t floorDivide(int64_t n, int64_t d) { return n / d - (n % d < 0); }

// Whether any row of a shares a byte with one of b: column slices of one buffer do not, whose
// rows lie between each other's.
[[maybe_unused]] bool meet(Span a, Span b) {
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
[[maybe_unused]] void apart(const Span& written, const Span& other) {
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
[[maybe_unused]] hipStream_t streamOf(PyObject* stream, c10::DeviceIndex device) {
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

[[maybe_unused]] void enqueued(const char* what, int rc) {
    if (rc != 0) refuse("%s returned hipError %d", what, rc);
}

// One of an extension's calls as Python sees it: a refusal becomes gError, and an exception of
// torch's (an allocation that fails) the error that torch makes of it.
template <PyObject* (*call)(PyObject* const*, Py_ssize_t)>
[[maybe_unused]] PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        return call(args, n);
    } catch (const Refusal& r) {
        PyErr_SetString(gError ? gError : PyExc_RuntimeError, r.text);
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

[[maybe_unused]] PyObject* setError(PyObject*, PyObject* type) {
    Py_XDECREF(gError);
    gError = Py_NewRef(type);
    Py_RETURN_NONE;
}

}  // namespace
