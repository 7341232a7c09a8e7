"""The operators around a cache of keys and values in 8 bits, over the C ABI in
include/ridge_attention.h (libridge_attention.so): what a decoder layer runs between its
projections.

    rope_table(positions, dim)       -> the cosines and sines that norm_rope turns heads by
    norm_rope(q, k, table, positions, q_weight=w, k_weight=w)
                                     -> (q, k), each head normed and turned by its position
    empty_cache(pages, page_size, heads, dim)
                                     -> (k, k_scale, v, v_scale), a cache without values
    write_cache(cache, slots, k, v)  -> cache, with the tokens' rows rounded to 8 bits
    read_cache(cache, slots)         -> (k, v), the values of rows of the cache
    attend(q, cache, pages, lengths) -> the attention of each sequence's newest token

Heads are [tokens, heads, columns] of float16, bfloat16 or float32, of any stride and offset
whose columns are contiguous and which do not overlap (views of a projection's rows among them),
of up to 256 columns. A cache is paged: k and v are int8 [pages, heads, page_size, columns] with a float32
scale for each row, page_size a multiple of 16, rows that start at multiples of 16 bytes. A
slot is a token's place in it, page * page_size + offset. The rows are those of
ridge_amd.int8: a row's largest magnitude over 127 is its scale, and its values over that are
rounded to the nearest whole number.

Sums, norms, softmax statistics and what they are made of are held in 32 bits. A call repeated
with the same operands gives the same bits. Heads that norm_rope turns and rows of the cache do not depend on what is
beside them; attend shares a batch's work evenly, so the last bits of a sequence's result go by
the other sequences' lengths (not by what they hold), unless `pages` has room for 512 tokens
each or fewer. positions, slots, pages and lengths are int32 on the device, so what they say
cannot be refused: a position outside the table, and a page or a length outside the cache, make
NaNs of the rows that ask for them; negative slots are padding.

Calls are asynchronous on `stream` (the current one by default) and write into `out` where
that is given, as those of ridge_amd.int8 do; with all buffers given they can be captured in a
HIP graph (attend allocates its workspace from torch, which a capture keeps in the graph's
own memory). Nothing that a call writes may share a byte with an operand, heads that norm_rope
turns in place excepted. Nothing here has a gradient: inputs that need one are refused where
gradients are on, and dual tensors always. There is no fallback: without the native library
every entry point raises.
"""

import ctypes
import importlib.machinery
import importlib.util
import os

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "lib", "libridge_attention.so")
BINDING_PATH = os.path.join(_PKG, "lib", "_ridge_attention.so")

MAX_DIM = 256    # columns of a head
MAX_AXES = 4     # of a position

_lib = None
_native = None


class RidgeAttentionError(RuntimeError):
    pass


class Heads(ctypes.Structure):
    """ridge_attention_heads_t."""
    _fields_ = [("at", ctypes.c_void_p), ("token", ctypes.c_int64), ("head", ctypes.c_int64), ("heads", ctypes.c_int32)]


class Cache(ctypes.Structure):
    """ridge_attention_cache_t."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "kScale", "vScale")] + \
        [(n, ctypes.c_int64) for n in ("pageStride", "headStride", "tokenStride", "scalePage", "scaleHead", "pages")] + \
        [(n, ctypes.c_int32) for n in ("pageSize", "heads", "dim")]


class Rotation(ctypes.Structure):
    """ridge_attention_rotation_t."""
    _fields_ = [("table", ctypes.c_void_p), ("tableStride", ctypes.c_int64), ("tableRows", ctypes.c_int64),
                ("positions", ctypes.c_void_p), ("positionStride", ctypes.c_int64), ("pairs", ctypes.c_int32),
                ("axes", ctypes.c_int32), ("interleaved", ctypes.c_int32), ("sections", ctypes.c_int32 * MAX_AXES)]


def _built(path):
    if not os.path.exists(path):
        raise RidgeAttentionError("%s is missing: run `python -m ridge_amd.build` (or "
                                  "__graft_entry__.build()) first" % path)
    return path


def lib():
    """libridge_attention.so, loaded once: the C ABI itself, for callers that have addresses
    instead of tensors. Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    L = ctypes.CDLL(_built(LIB_PATH))
    p, i, n, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
    heads, cache, rotation = ctypes.POINTER(Heads), ctypes.POINTER(Cache), ctypes.POINTER(Rotation)
    for name, args in (
            ("norm_rope", [heads, heads, i, p, p, i, f, rotation, heads, heads, n, i, p]),
            ("write", [cache, p, heads, heads, i, n, p]),
            ("read", [cache, p, heads, heads, i, n, p]),
            ("attend", [heads, cache, p, n, n, p, f, n, heads, p, i, n, p, n, p])):
        function = getattr(L, "ridge_attention_" + name)
        function.restype, function.argtypes = i, args
    L.ridge_attention_workspace.restype, L.ridge_attention_workspace.argtypes = n, [n, i, i, i, n, i]
    _lib = L
    return L


def _load():
    """The extension that takes tensors (csrc/attention_binding.cpp), loaded once."""
    global _native
    if _native is None:
        import torch  # noqa: F401  its libraries, which the extension is linked to
        loader = importlib.machinery.ExtensionFileLoader("_ridge_attention", _built(BINDING_PATH))
        spec = importlib.util.spec_from_file_location("_ridge_attention", BINDING_PATH, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        module.set_error(RidgeAttentionError)
        _native = module
    return _native


def rope_table(positions, dim, theta=10000.0, device=None):
    """float32 [positions, dim]: row t has the cosines and then the sines of t * theta^(-2 p / dim)
    for the dim / 2 pairs p, angles and functions in 64 bits. A table of other frequencies (scaled
    ones, or one set for each axis of a position) is laid out the same."""
    import torch
    if dim < 2 or dim % 2:
        raise RidgeAttentionError("a table turns pairs of columns: dim must be even and positive, not %d" % dim)
    device = "cuda" if device is None else device
    rate = float(theta) ** (torch.arange(0, dim, 2, dtype=torch.float64, device=device) / -dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def norm_rope(q, k, table, positions, q_weight=None, k_weight=None, eps=1e-6, sections=None, interleaved=False,
              q_out=None, k_out=None, stream=None):
    """(q_out, k_out): the heads of q [tokens, heads, columns] and of k, each x / sqrt(mean(x^2) +
    eps) * weight where it has a weight ([columns], of q's type or float32), and then turned: with
    pairs = table.shape[1] / 2, columns p and p + pairs (interleaved: 2 p and 2 p + 1) by the
    angle whose cosine is table[t, p] and sine table[t, pairs + p]. Columns from 2 pairs on are
    not turned. t is the token's position, or positions [tokens, axes] with sections saying how
    many pairs, from the first on, each axis turns. One rounding to q's type. q_out may be q and
    k_out k. k may have no heads."""
    return (_native or _load()).norm_rope(q, k, table, positions, q_weight, k_weight, eps, sections, interleaved, q_out,
                                          k_out, stream)


def empty_cache(pages, page_size, heads, dim, device=None):
    """(k, k_scale, v, v_scale): an uninitialised cache of int8 rows [pages, heads, page_size, dim]
    and their float32 scales [pages, heads, page_size]; rows a multiple of 16 bytes apart. Rows
    that no sequence has are never looked at."""
    import torch
    if page_size < 16 or page_size % 16 or not 1 <= dim <= MAX_DIM or heads < 1 or pages < 1:
        raise RidgeAttentionError("page_size must be a multiple of 16 and dim 1 to %d, not %d and %d, of %d pages and %d "
                                  "heads" % (MAX_DIM, page_size, dim, pages, heads))
    device = "cuda" if device is None else device
    parts = []
    for _ in range(2):
        rows = torch.empty((pages, heads, page_size, (dim + 15) // 16 * 16), dtype=torch.int8, device=device)
        parts += [rows[..., :dim], torch.empty((pages, heads, page_size), dtype=torch.float32, device=device)]
    return tuple(parts)


def write_cache(cache, slots, k, v, stream=None):
    """cache, the rows of k and v [tokens, heads, columns] rounded to 8 bits at slots [tokens]. A
    negative slot is padding, and it and one behind the cache are not written. Slots of a call
    must differ: one that comes twice holds the bytes of one token and perhaps the scale of the
    other. A row that holds a NaN or an infinity has a scale that is not finite."""
    return (_native or _load()).write_cache(cache, slots, k, v, stream)


def read_cache(cache, slots, dtype=None, out=None, stream=None):
    """(k, v) [tokens, heads, columns]: the values of the rows at slots [tokens], rounded once to
    `dtype` (out's, or float16). out is (k, v). A negative slot reads as zeros, one behind the
    cache as NaNs."""
    return (_native or _load()).read_cache(cache, slots, dtype, out, stream)


def attend(q, cache, pages, lengths, scale=None, window=None, lse_out=None, out=None, stream=None):
    """out [sequences, heads, columns]: for each head of q, the softmax of scale * (q . k_t) over
    the sequence's tokens t, times v_t. Sequence b has lengths[b] tokens, the new one among them,
    in the pages pages[b]; key head h / (q's heads / the cache's) serves query head h. window:
    only the last that many tokens. scale is 1 / sqrt(columns) by default (2^118 at the most for
    float16). lse_out (float32
    [sequences, heads]) gets the logarithm of the sum of exp(scale * (q . k_t)), by which the
    results over two parts of a sequence are joined. A sequence of no tokens gives zeros, and
    -inf in lse_out. Narrow `pages` to the longest sequence: its columns are what a launch is
    sized by."""
    return (_native or _load()).attend(q, cache, pages, lengths, scale, window, lse_out, out, stream)
