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
float32. Sums, norms and scales are held in 32 bits, and a product's sum is exact. A
weight [channels, K] goes through quantize() once and is b from then on. Rows may be
views: of any stride and offset in 16 and 32 bits, in 8 bits ones that start at multiples
of 16 bytes, which empty() sees to for every number of columns.

Every call is asynchronous on `stream` (the current one by default) and writes into
`out` where that is given: as everywhere, a tensor that another stream made or will free
is the caller's to order. Outputs that a call allocates itself belong to the stream that
it runs on. Nothing here has a gradient: inputs that need one are refused where gradients
are on. There is no fallback: without the native library every entry point raises.
"""

import ctypes
import os

from .gemm import HIP_SUCCESS, _current, _stream_handle

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "lib", "libridge_int8.so")

MAX_K = 131071       # of a product: more 8-bit products may not fit a 32-bit sum
MAX_STRIDE = 1 << 23  # of a product's 8-bit rows

_lib = None
_types = None


class RidgeInt8Error(RuntimeError):
    pass


def lib():
    """Loads libridge_int8.so once. Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RidgeInt8Error("%s is missing: run `python -m ridge_amd.build` (or "
                             "__graft_entry__.build()) first" % LIB_PATH)
    L = ctypes.CDLL(LIB_PATH)
    p, i, n, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
    for name, args in (
            ("quantize", [p, n, i, p, n, p, n, n, p]),
            ("silu_mul", [p, n, i, p, n, p, n, n, p]),
            ("rms_norm", [p, n, p, n, p, i, f, i, p, n, p, n, p, n, n, p]),
            ("dequantize", [p, n, p, p, n, i, n, n, p]),
            ("gemm", [p, n, p, p, n, p, p, p, n, i, n, n, n, p])):
        function = getattr(L, "ridge_int8_" + name)
        function.restype, function.argtypes = i, args
    _lib = L
    return L


def _type_codes():
    """dtype -> the C ABI's number of it."""
    global _types
    if _types is None:
        import torch
        _types = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
    return _types


def _type_of(t, what):
    code = _type_codes().get(t.dtype)
    if code is None:
        raise RidgeInt8Error("%s must be float16, bfloat16 or float32, not %s" % (what, t.dtype))
    return code


def _matrix(t, what, device=None):
    """(rows, cols, stride of the rows) of a 2-D device tensor whose rows are contiguous."""
    if not t.is_cuda or t.dim() != 2:
        raise RidgeInt8Error("%s must be a 2-D device tensor" % what)
    if device is not None and t.device != device:
        raise RidgeInt8Error("%s is on %s, not on %s" % (what, t.device, device))
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise RidgeInt8Error("%s must have contiguous rows" % what)
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise RidgeInt8Error("the rows of %s overlap" % what)
    return rows, cols, ld


def _rows8(q, scale, what, device=None):
    """(rows, cols, stride) of 8-bit rows with their scales."""
    import torch
    rows, cols, ld = _matrix(q, what, device)
    if q.dtype != torch.int8:
        raise RidgeInt8Error("%s must be int8, not %s" % (what, q.dtype))
    if rows <= 1:
        ld = (cols + 15) // 16 * 16
    if ld % 16 or q.data_ptr() % 16:
        raise RidgeInt8Error("the rows of %s must start at multiples of 16 bytes (as those of empty() do)" % what)
    if cols % 16 and rows:
        end = q.storage_offset() + (rows - 1) * ld + (cols + 15) // 16 * 16
        if end > q.untyped_storage().nbytes():
            raise RidgeInt8Error("the last row of %s ends its memory inside 16 bytes (make it with empty())" % what)
    if scale.dtype != torch.float32 or scale.dim() != 1 or scale.shape[0] != rows or scale.device != q.device or \
            (rows > 1 and scale.stride(0) != 1):
        raise RidgeInt8Error("the scales of %s must be %d contiguous float32 on its device" % (what, rows))
    return rows, cols, ld


def _no_gradient(*tensors):
    import torch
    if any(t is not None and t.requires_grad for t in tensors) and torch.is_grad_enabled():
        raise RidgeInt8Error("the 8-bit operators have no gradient: call them under torch.no_grad()")


def _allocate(make, device, stream):
    """make(), with its memory owned by the stream that the call runs on."""
    if stream is None:
        return make()
    import torch
    if isinstance(stream, int):
        if stream == 0:
            stream = torch.cuda.default_stream(device)
        else:
            stream = torch.cuda.ExternalStream(stream, device=device)
    with torch.cuda.stream(stream):
        return make()


def _call(name, device, stream, *args):
    """Calls ridge_int8_<name>(args..., stream) with the operands' device current."""
    if _current()[0]() == device.index:
        rc = getattr(lib(), name)(*args, _stream_handle(stream))
    else:
        import torch
        with torch.cuda.device(device):
            rc = getattr(lib(), name)(*args, _stream_handle(stream))
    if rc != HIP_SUCCESS:
        raise RidgeInt8Error("%s returned hipError %d" % (name, rc))


def empty(rows, cols, device=None):
    """(q, scale): uninitialised 8-bit rows and their scales. The rows lie a multiple of
    16 bytes apart; what is behind `cols` is never looked at."""
    import torch
    device = "cuda" if device is None else device
    q = torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)
    return q[:, :cols], torch.empty(rows, dtype=torch.float32, device=device)


def _rows_out(out, rows, cols, device, stream):
    """(q, scale, stride of q) to write rows x cols to."""
    if out is None:
        out = _allocate(lambda: empty(rows, cols, device), device, stream)
    q, scale = out
    shape = _rows8(q, scale, "out", device)
    if shape[:2] != (rows, cols):
        raise RidgeInt8Error("out holds %d x %d, not %d x %d" % (shape[:2] + (rows, cols)))
    return q, scale, shape[2]


def _some_columns(cols, what):
    if cols < 1:
        raise RidgeInt8Error("%s has no columns" % what)


def quantize(x, out=None, stream=None):
    """(q, scale) of the rows of x: scale is a row's largest magnitude over 127, q its
    values over that, rounded to the nearest whole number. A row that holds a NaN or an
    infinity has a scale that is not finite."""
    rows, cols, ld = _matrix(x, "x")
    code = _type_of(x, "x")
    _no_gradient(x)
    _some_columns(cols, "x")
    q, scale, ldq = _rows_out(out, rows, cols, x.device, stream)
    _call("ridge_int8_quantize", x.device, stream, x.data_ptr(), ld, code, q.data_ptr(), ldq, scale.data_ptr(), rows,
          cols)
    return q, scale


def silu_mul(gate_up, out=None, stream=None):
    """(q, scale) of silu(gate) * up, where a row of gate_up holds gate and then up:
    [rows, 2 F] -> 8-bit rows of F."""
    rows, width, ld = _matrix(gate_up, "gate_up")
    code = _type_of(gate_up, "gate_up")
    _no_gradient(gate_up)
    _some_columns(width, "gate_up")
    if width % 2:
        raise RidgeInt8Error("gate_up has %d columns: two halves are wanted" % width)
    q, scale, ldq = _rows_out(out, rows, width // 2, gate_up.device, stream)
    _call("ridge_int8_silu_mul", gate_up.device, stream, gate_up.data_ptr(), ld, code, q.data_ptr(), ldq,
          scale.data_ptr(), rows, width // 2)
    return q, scale


def rms_norm(x, weight, eps=1e-6, residual=None, residual_out=None, out=None, stream=None):
    """(q, scale, residual_out): s = x + residual, the 8-bit rows of
    s / sqrt(mean(s^2) + eps) * weight, and s rounded to x's type. residual_out may be x
    or residual itself. Without a residual the norm is x's and residual_out is None.
    weight has x's type or is float32."""
    rows, cols, ld = _matrix(x, "x")
    code = _type_of(x, "x")
    _no_gradient(x, weight, residual)
    _some_columns(cols, "x")
    device = x.device
    weight_code = _type_of(weight, "weight")
    if weight_code not in (code, 2) or weight.dim() != 1 or weight.shape[0] != cols or weight.device != device or \
            (cols > 1 and weight.stride(0) != 1):
        raise RidgeInt8Error("weight must be %d contiguous values on x's device, of x's type or float32" % cols)
    if not 0 < eps < float("inf"):
        raise RidgeInt8Error("eps must be positive, not %r" % (eps,))
    r, ldr, o, ldo = None, 0, None, 0
    if residual is not None:
        if residual_out is None:
            import torch
            residual_out = _allocate(lambda: torch.empty((rows, cols), dtype=x.dtype, device=device), device, stream)
        for t, what in ((residual, "residual"), (residual_out, "residual_out")):
            shape = _matrix(t, what, device)
            if t.dtype != x.dtype or shape[:2] != (rows, cols):
                raise RidgeInt8Error("%s must be like x: %d x %d of %s" % (what, rows, cols, x.dtype))
            r, ldr, o, ldo = o, ldo, t.data_ptr(), shape[2]
    elif residual_out is not None:
        raise RidgeInt8Error("residual_out without a residual")
    q, scale, ldq = _rows_out(out, rows, cols, device, stream)
    _call("ridge_int8_rms_norm", device, stream, x.data_ptr(), ld, r, ldr, weight.data_ptr(), weight_code, eps, code,
          o, ldo, q.data_ptr(), ldq, scale.data_ptr(), rows, cols)
    return q, scale, residual_out


def dequantize(q, scale, dtype=None, out=None, stream=None):
    """The values q * scale, rounded once to `dtype` (out's, or float16)."""
    import torch
    rows, cols, ldq = _rows8(q, scale, "q")
    _some_columns(cols, "q")
    if out is None:
        out = _allocate(lambda: torch.empty((rows, cols), dtype=dtype or torch.float16, device=q.device), q.device,
                        stream)
    code = _type_of(out, "out")
    shape = _matrix(out, "out", q.device)
    if shape[:2] != (rows, cols) or (dtype is not None and out.dtype != dtype):
        raise RidgeInt8Error("out must be %d x %d%s" % (rows, cols, "" if dtype is None else " of %s" % dtype))
    _call("ridge_int8_dequantize", q.device, stream, q.data_ptr(), ldq, scale.data_ptr(), out.data_ptr(), shape[2],
          code, rows, cols)
    return out


def gemm(a, a_scale, b, b_scale, bias=None, dtype=None, out=None, stream=None):
    """out[m, n] = (sum over k of a[m, k] b[n, k]) * a_scale[m] * b_scale[n] + bias[n].
    The sum is exact (K at most MAX_K), the rest is computed in 32 bits and rounded once
    to `dtype` (out's, or float16), which is bias's type too."""
    import torch
    M, K, lda = _rows8(a, a_scale, "a")
    N, Kb, ldb = _rows8(b, b_scale, "b", a.device)
    if K != Kb:
        raise RidgeInt8Error("rows of %d and of %d do not chain" % (K, Kb))
    if not 1 <= K <= MAX_K or lda >= MAX_STRIDE or ldb >= MAX_STRIDE:
        raise RidgeInt8Error("K must be 1 to %d and strides below %d, not %d, %d and %d"
                             % (MAX_K, MAX_STRIDE, K, lda, ldb))
    device = a.device
    if out is None:
        out = _allocate(lambda: torch.empty((M, N), dtype=dtype or torch.float16, device=device), device, stream)
    code = _type_of(out, "out")
    shape = _matrix(out, "out", device)
    if shape[:2] != (M, N) or (dtype is not None and out.dtype != dtype):
        raise RidgeInt8Error("out must be %d x %d%s" % (M, N, "" if dtype is None else " of %s" % dtype))
    at = None
    if bias is not None:
        _no_gradient(bias)
        if bias.dtype != out.dtype or bias.dim() != 1 or bias.shape[0] != N or bias.device != device or \
                (N > 1 and bias.stride(0) != 1):
            raise RidgeInt8Error("bias must be %d contiguous values of out's type on its device" % N)
        at = bias.data_ptr()
    _call("ridge_int8_gemm", device, stream, a.data_ptr(), lda, a_scale.data_ptr(), b.data_ptr(), ldb,
          b_scale.data_ptr(), at, out.data_ptr(), shape[2], code, M, N, K)
    return out
