"""The 8-bit operators' library, layout and refusals. No GPU calls: every refusal comes
before one."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

from ridge_amd import int8 as I  # noqa: E402
from test_abi import _declared  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1
P = 1 << 20   # an address that is never followed


def test_every_declared_symbol_is_exported():
    names = _declared(os.path.join(ROOT, "include", "ridge_int8.h"))
    assert len(names) == 7
    L = ctypes.CDLL(I.LIB_PATH)
    assert [n for n in names if not hasattr(L, n)] == []


@pytest.mark.parametrize("cols", [1, 15, 16, 17, 4096])
def test_empty_lays_rows_out_at_multiples_of_16(cols):
    q, scale = I.empty(3, cols, device="cpu")
    assert q.shape == (3, cols) and q.dtype == torch.int8 and q.stride(1) == 1
    assert q.stride(0) % 16 == 0 and q.stride(0) - cols < 16
    assert q.untyped_storage().nbytes() == 3 * q.stride(0)
    assert scale.shape == (3,) and scale.dtype == torch.float32


MAKERS = {
    # name: (arguments, {what: (index, refused value)})
    "quantize": ([P, 64, 0, P, 64, P, 4, 64, None],
                 {"type": (2, 3), "x": (0, None), "x odd": (0, P + 1), "q": (3, P + 8), "ldq": (4, 72),
                  "ldq short": (4, 48), "ldx": (1, 63), "rows": (6, -1), "many rows": (6, 1 << 31), "cols": (7, 0),
                  "scale": (5, None)}),
    "silu_mul": ([P, 128, 1, P, 64, P, 4, 64, None],
                 {"type": (2, -1), "x": (0, None), "q": (3, None), "ldx": (1, 127), "cols": (7, 1 << 30),
                  "rows": (6, -1)}),
    "rms_norm": ([P, 64, P, 64, P, 0, 1e-6, 0, P, 64, P, 64, P, 4, 64, None],
                 {"type": (7, 3), "weight type": (5, 1), "weight": (4, None), "eps": (6, 0.0),
                  "eps nan": (6, float("nan")), "eps inf": (6, float("inf")), "residual alone": (8, None),
                  "residual_out alone": (2, None), "ldx": (1, 63), "ld residual": (3, 63), "ld out": (9, 63),
                  "residual odd": (2, P + 1), "q": (10, P + 1), "ldq": (11, 65), "rows": (13, -1), "cols": (14, 0)}),
    "dequantize": ([P, 64, P, P, 64, 0, 4, 64, None],
                   {"type": (5, 7), "q": (0, None), "q off": (0, P + 4), "ldq": (1, 63), "scale": (2, None),
                    "out": (3, P + 1), "ld": (4, 63), "rows": (6, -5), "cols": (7, 0)}),
    "gemm": ([P, 64, P, P, 64, P, None, P, 32, 0, 16, 32, 64, None],
             {"type": (9, 3), "A": (0, None), "A off": (0, P + 8), "lda": (1, 72), "lda short": (1, 48),
              "lda long": (1, 1 << 23), "scaleA": (2, None), "B": (3, P + 1), "ldb": (4, 8), "scaleB": (5, None),
              "bias odd": (6, P + 1), "C": (7, None), "C odd": (7, P + 1), "ldc": (8, 31), "M": (10, -1),
              "M large": (10, 1 << 31), "N": (11, -1), "K": (12, 0), "K large": (12, I.MAX_K + 1)}),
}


@pytest.mark.parametrize("name,what", [(n, w) for n, (_, bad) in MAKERS.items() for w in bad])
def test_the_library_refuses(name, what):
    args, bad = MAKERS[name]
    args = list(args)
    at, value = bad[what]
    args[at] = value
    if what == "K large":
        args[1] = args[4] = 131072
    assert getattr(I.lib(), "ridge_int8_" + name)(*args) == INVALID


@pytest.mark.parametrize("name,index", [("quantize", 6), ("silu_mul", 6), ("rms_norm", 13), ("dequantize", 6),
                                        ("gemm", 10), ("gemm", 11)])
def test_no_rows_is_a_call_that_does_nothing(name, index):
    args = list(MAKERS[name][0])
    args[index] = 0
    assert getattr(I.lib(), "ridge_int8_" + name)(*args) == 0


def test_host_tensors_are_refused():
    x = torch.zeros((4, 64), dtype=torch.float16)
    q, s = I.empty(4, 64, device="cpu")
    for call in (lambda: I.quantize(x), lambda: I.silu_mul(x), lambda: I.rms_norm(x, x[0]),
                 lambda: I.dequantize(q, s), lambda: I.gemm(q, s, q, s)):
        with pytest.raises(I.RidgeInt8Error, match="device tensor"):
            call()


# What the GPU tests run the forms with, and the products that each is for.
# Form 0 without parts, and with its last round's tiles in quarters and in halves.
FORMS = [(0, 4001, 4093, 2065), (0, 4001, 4103, 2065), (0, 6001, 4100, 1040), (1, 2301, 1805, 2049), (2, 2031, 2031, 1031), (3, 829, 3583, 159), (4, 149, 8887, 4111),
         (5, 49, 8195, 1029), (6, 3, 4001, 1027), (7, 299, 301, 4099), (8, 791, 257, 3469)]


@pytest.mark.parametrize("form,M,N,K", FORMS)
def test_every_form_of_the_product_is_chosen_somewhere(form, M, N, K):
    L = ctypes.CDLL(I.LIB_PATH)
    L.ridge_int8_gemm_form.argtypes = [ctypes.c_int64] * 3
    assert L.ridge_int8_gemm_form(M, N, K) == form


def test_form_of_sizes_without_a_product():
    L = ctypes.CDLL(I.LIB_PATH)
    L.ridge_int8_gemm_form.argtypes = [ctypes.c_int64] * 3
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, I.MAX_K + 1), (1 << 31, 1, 1), (1, -4, 1),
                  (1 << 30, 1 << 30, 16)):
        assert L.ridge_int8_gemm_form(*sizes) == -1
    # Sizes past 16 bits take no form of small tiles, whose arguments hold 16.
    assert 0 <= L.ridge_int8_gemm_form(1, 70000, 64) < 6 and 0 <= L.ridge_int8_gemm_form(70000, 1, 131071) < 6


@pytest.mark.parametrize("cols,stride", [(1, 16), (16, 16), (17, 32), (512, 512), (513, 640), (4096, 4096), (4097, 4224)])
def test_row_stride(cols, stride):
    assert I.lib().ridge_int8_row_stride(cols) == stride
    assert I.empty(2, cols, device="cpu")[0].stride(0) == stride


# A few tokens against wide weights, us in tiles of 16x16 | 64x64 whose workgroups have K alone.
@pytest.mark.parametrize("M,N,K", [
    (2, 8576, 2520),    # 5.6 | 7.3
    (2, 8960, 3412),    # 6.5 | 7.9
    (3, 9728, 3467),    # 7.1 | 8.6
    (3, 11008, 1408),   # 5.1 | 5.6
])
def test_few_tokens_take_the_tiles_that_share_k(M, N, K):
    assert I.lib().ridge_int8_gemm_form(M, N, K) == 6
