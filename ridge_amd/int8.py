"""The 8-bit operators over the C ABI in include/ridge_int8.h (libridge_int8.so): rows
held in 8 bits with one scale each, what makes them, and their matrix product.

    empty(rows, cols)          -> (q, scale), buffers laid out for the calls below
    quantize(x)                -> (q, scale) of x's rows
    silu_mul(gate_up)          -> (q, scale) of silu(gate) * up, a row being [gate | up]
    rms_norm(x, weight, eps, residual=r)
                               -> (q, scale, x + r): the norm of x + r, times weight
    gemm(a, a_scale, b, b_scale, bias=None)
                               -> a b^T, scaled by a's rows (tokens) and b's (channels)
    dequantize(q, scale)       -> the values q * scale

q is int8 and scale float32; the 16- and 32-bit tensors are float16, bfloat16 or
float32. Sums, norms and scales are held in 32 bits, and a product's sum is exact: a
row's result is the same, bit for bit, whatever rows are beside it. A weight
[channels, K] goes through quantize() once and is b from then on. Rows may be views: of
any stride and offset in 16 and 32 bits, in 8 bits ones that start at multiples of 16
bytes, which empty() sees to for every number of columns. What a call writes may be nothing
else of the call (rms_norm's residual_out excepted): an output that shares a byte with an
operand is refused, column slices of one buffer are not.

Every call is asynchronous on `stream` (the current one by default) and writes into
`out` where that is given: as everywhere, a tensor that another stream made or will free
is the caller's to order. Outputs that a call allocates itself belong to the stream that
it runs on. Nothing here has a gradient: inputs that need one are refused where gradients
are on, and so are forward mode's dual tensors; a graph that saved a tensor which a call then
writes raises in its backward, as after torch's own in-place operations. There is no
fallback: without the native library every entry point raises.
"""

import ctypes
import importlib.machinery
import importlib.util
import os

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "lib", "libridge_int8.so")
BINDING_PATH = os.path.join(_PKG, "lib", "_ridge_int8.so")

MAX_K = 131071       # of a product: more 8-bit products may not fit a 32-bit sum
MAX_STRIDE = 1 << 23  # of a product's 8-bit rows

_lib = None
_native = None


class RidgeInt8Error(RuntimeError):
    pass


def _built(path):
    if not os.path.exists(path):
        raise RidgeInt8Error("%s is missing: run `python -m ridge_amd.build` (or "
                             "__graft_entry__.build()) first" % path)
    return path


def lib():
    """libridge_int8.so, loaded once: the C ABI itself, for callers that have addresses
    instead of tensors. Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    L = ctypes.CDLL(_built(LIB_PATH))
    p, i, n, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
    for name, args in (
            ("quantize", [p, n, i, p, n, p, n, n, p]),
            ("silu_mul", [p, n, i, p, n, p, n, n, p]),
            ("rms_norm", [p, n, p, n, p, i, f, i, p, n, p, n, p, n, n, p]),
            ("dequantize", [p, n, p, p, n, i, n, n, p]),
            ("gemm", [p, n, p, p, n, p, p, p, n, i, n, n, n, p]),
            ("gemm_form", [n, n, n])):
        function = getattr(L, "ridge_int8_" + name)
        function.restype, function.argtypes = i, args
    L.ridge_int8_row_stride.restype, L.ridge_int8_row_stride.argtypes = n, [n]
    _lib = L
    return L


def _load():
    """The extension that takes tensors (csrc/int8_binding.cpp), loaded once."""
    global _native
    if _native is None:
        import torch  # noqa: F401  its libraries, which the extension is linked to
        loader = importlib.machinery.ExtensionFileLoader("_ridge_int8", _built(BINDING_PATH))
        spec = importlib.util.spec_from_file_location("_ridge_int8", BINDING_PATH, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        module.set_error(RidgeInt8Error)
        _native = module
    return _native


def empty(rows, cols, device=None):
    """(q, scale): uninitialised 8-bit rows and their scales, the rows a multiple of 16
    bytes apart, and of 128 where they are long, which the product reads fastest
    (ridge_int8_row_stride). What is behind `cols` is never looked at."""
    import torch
    device = "cuda" if device is None else device
    q = torch.empty((rows, lib().ridge_int8_row_stride(cols)), dtype=torch.int8, device=device)
    return q[:, :cols], torch.empty(rows, dtype=torch.float32, device=device)


def quantize(x, out=None, stream=None):
    """(q, scale) of the rows of x: scale is a row's largest magnitude over 127, q its
    values over that, rounded to the nearest whole number. A row that holds a NaN or an
    infinity has a scale that is not finite."""
    return (_native or _load()).quantize(x, out, stream)


def silu_mul(gate_up, out=None, stream=None):
    """(q, scale) of silu(gate) * up, where a row of gate_up holds gate and then up:
    [rows, 2 F] -> 8-bit rows of F."""
    return (_native or _load()).silu_mul(gate_up, out, stream)


def rms_norm(x, weight, eps=1e-6, residual=None, residual_out=None, out=None, stream=None):
    """(q, scale, residual_out): s = x + residual, the 8-bit rows of
    s / sqrt(mean(s^2) + eps) * weight, and s rounded to x's type. residual_out may be x
    or residual itself. Without a residual the norm is x's and residual_out is None.
    weight has x's type or is float32."""
    return (_native or _load()).rms_norm(x, weight, eps, residual, residual_out, out, stream)


def dequantize(q, scale, dtype=None, out=None, stream=None):
    """The values q * scale, rounded once to `dtype` (out's, or float16)."""
    return (_native or _load()).dequantize(q, scale, dtype, out, stream)


def gemm(a, a_scale, b, b_scale, bias=None, dtype=None, out=None, stream=None):
    """out[m, n] = (sum over k of a[m, k] b[n, k]) * a_scale[m] * b_scale[n] + bias[n].
    The sum is exact (K at most MAX_K, rows of a and b less than MAX_STRIDE apart), the
    rest is computed in 32 bits and rounded once to `dtype` (out's, or float16), which is
    bias's type too."""
    return (_native or _load()).gemm(a, a_scale, b, b_scale, bias, dtype, out, stream)
