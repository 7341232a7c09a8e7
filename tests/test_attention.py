"""The library around the 8-bit cache: layouts, sizes and refusals. No GPU calls: every refusal
comes before one."""
import ctypes
import math
import os

import pytest

torch = pytest.importorskip("torch")

from ridge_amd import attention as A  # noqa: E402
from test_abi import _declared  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1
P = 1 << 20   # an address that is never followed


def test_every_declared_symbol_is_exported():
    names = _declared(os.path.join(ROOT, "include", "ridge_attention.h"))
    assert len(names) == 5
    L = ctypes.CDLL(A.LIB_PATH)
    assert [n for n in names if not hasattr(L, n)] == []


def test_structures_have_the_headers_sizes():
    assert ctypes.sizeof(A.Heads) == 32 and ctypes.sizeof(A.Cache) == 96 and ctypes.sizeof(A.Rotation) == 72


@pytest.mark.parametrize("dim", [2, 64, 80, 128])
def test_rope_table(dim):
    table = A.rope_table(5001, dim, theta=500000.0, device="cpu")
    assert table.shape == (5001, dim) and table.dtype == torch.float32
    for t, p in ((0, 0), (5000, 0), (5000, dim // 2 - 1), (1234, dim // 4)):
        angle = t * 500000.0 ** (-2.0 * p / dim)
        # Rounded once to 32 bits; the angle's 64 carry 5000 * 2^-52.
        assert abs(float(table[t, p]) - math.cos(angle)) <= 2.0 ** -25 + 2.0 ** -38
        assert abs(float(table[t, dim // 2 + p]) - math.sin(angle)) <= 2.0 ** -25 + 2.0 ** -38
    for bad in (0, 7, -2):
        with pytest.raises(A.RidgeAttentionError):
            A.rope_table(4, bad, device="cpu")


@pytest.mark.parametrize("dim", [1, 15, 16, 17, 128, 256])
def test_empty_cache_lays_rows_out_at_multiples_of_16(dim):
    k, k_scale, v, v_scale = A.empty_cache(3, 48, 2, dim, device="cpu")
    for rows, scale in ((k, k_scale), (v, v_scale)):
        assert rows.shape == (3, 2, 48, dim) and rows.dtype == torch.int8 and rows.stride(3) == 1
        assert all(s % 16 == 0 for s in rows.stride()[:3]) and rows.stride(2) - dim < 16
        assert scale.shape == (3, 2, 48) and scale.dtype == torch.float32 and scale.is_contiguous()


@pytest.mark.parametrize("pages,page_size,heads,dim", [(1, 8, 1, 64), (1, 24, 1, 64), (1, 0, 1, 64), (0, 16, 1, 64),
                                                       (1, 16, 0, 64), (1, 16, 1, 0), (1, 16, 1, 257)])
def test_empty_cache_refuses(pages, page_size, heads, dim):
    with pytest.raises(A.RidgeAttentionError):
        A.empty_cache(pages, page_size, heads, dim, device="cpu")


def _heads(heads=4, **changes):
    return A.Heads(**dict(dict(at=P, token=heads * 64, head=64, heads=heads), **changes))


def _cache(**changes):
    return A.Cache(**dict(dict(k=P, v=P, kScale=P, vScale=P, pageStride=2 * 16 * 64, headStride=16 * 64, tokenStride=64,
                               scalePage=32, scaleHead=16, pages=8, pageSize=16, heads=2, dim=64), **changes))


def _rotation(sections=(32, 0, 0, 0), **changes):
    return A.Rotation(**dict(dict(table=P, tableStride=64, tableRows=100, positions=P, positionStride=1, pairs=32, axes=1,
                                  interleaved=0, sections=(ctypes.c_int32 * 4)(*sections)), **changes))


def _norm_rope(q=None, k=None, type=0, q_weight=P, k_weight=P, weight_type=0, eps=1e-6, rotation=None, q_out=None,
               k_out=None, tokens=3, dim=64):
    return A.lib().ridge_attention_norm_rope(q or _heads(), k or _heads(2), type, q_weight, k_weight, weight_type, eps,
                                             rotation or _rotation(), q_out or _heads(), k_out or _heads(2), tokens, dim, None)


@pytest.mark.parametrize("what,changes", [
    ("type", dict(type=3)), ("weight type", dict(weight_type=1)), ("weight off", dict(q_weight=P + 1)),
    ("eps", dict(eps=0.0)), ("eps nan", dict(eps=float("nan"))), ("eps inf", dict(eps=float("inf"))),
    ("tokens", dict(tokens=-1)), ("many tokens", dict(tokens=1 << 31)), ("dim", dict(dim=0)), ("wide", dict(dim=257)),
    ("narrow", dict(dim=63)), ("q", dict(q=_heads(at=None))), ("q off", dict(q=_heads(at=P + 1))),
    ("q's heads", dict(q=_heads(3))), ("k's heads", dict(k_out=_heads(1))), ("stride", dict(k=_heads(2, token=-64))),
    ("head stride", dict(q_out=_heads(head=-1))), ("many heads", dict(q=_heads(65536), q_out=_heads(65536))),
    ("table", dict(rotation=_rotation(table=None))), ("table's stride", dict(rotation=_rotation(tableStride=63))),
    ("no rows", dict(rotation=_rotation(tableRows=0))),
    ("a table of 4 GiB", dict(rotation=_rotation(tableRows=1 << 24))), ("positions", dict(rotation=_rotation(positions=None))),
    ("no pairs", dict(rotation=_rotation((0, 0, 0, 0), pairs=0))), ("axes", dict(rotation=_rotation(axes=0))),
    ("five axes", dict(rotation=_rotation(axes=5))), ("sections", dict(rotation=_rotation((31, 0, 0, 0)))),
    ("sections of two axes", dict(rotation=_rotation((32, 1, 0, 0), axes=2))),
    ("a negative section", dict(rotation=_rotation((33, -1, 0, 0), axes=2))),
])
def test_norm_rope_refuses(what, changes):
    assert _norm_rope(**changes) == INVALID


def test_no_tokens_and_no_heads_are_calls_that_do_nothing():
    assert _norm_rope(tokens=0) == 0
    assert _norm_rope(tokens=0, q=_heads(at=None), rotation=_rotation(positions=None)) == 0
    none = _heads(0, at=None)
    assert _norm_rope(q=none, k=none, q_out=none, k_out=none) == 0
    L = A.lib()
    for call in (L.ridge_attention_write, L.ridge_attention_read):
        assert call(_cache(), None, _heads(2, at=None), _heads(2, at=None), 0, 0, None) == 0
    assert L.ridge_attention_attend(_heads(at=None), _cache(), None, 4, 4, None, 0.125, 0, _heads(at=None), None, 0, 0, None,
                                    0, None) == 0


BAD_CACHES = {
    "k": dict(k=None), "v off": dict(v=P + 8), "kScale": dict(kScale=P + 4), "vScale": dict(vScale=None),
    "page stride": dict(pageStride=2056), "head stride": dict(headStride=-1024), "token stride": dict(tokenStride=72),
    "rows far apart": dict(tokenStride=1 << 27),
    "scale page": dict(scalePage=33), "scale head": dict(scaleHead=-16), "pages": dict(pages=0),
    "many pages": dict(pages=1 << 27), "page size": dict(pageSize=24), "small pages": dict(pageSize=0),
    "heads": dict(heads=0), "many heads": dict(heads=65536), "dim": dict(dim=0), "wide": dict(dim=257),
}


@pytest.mark.parametrize("what", BAD_CACHES)
def test_bad_caches_are_refused(what):
    L, cache = A.lib(), _cache(**BAD_CACHES[what])
    heads = _heads(cache.heads)
    for call in (L.ridge_attention_write, L.ridge_attention_read):
        assert call(cache, P, heads, heads, 0, 3, None) == INVALID
    assert L.ridge_attention_attend(_heads(), cache, P, 4, 4, P, 0.125, 0, _heads(), None, 0, 3, P, 1 << 40, None) == INVALID


@pytest.mark.parametrize("what,changes", [
    ("slots", dict(slots=None)), ("slots off", dict(slots=P + 2)), ("k", dict(k=_heads(2, at=None))),
    ("k's heads", dict(k=_heads(3))), ("v's heads", dict(v=_heads(1))), ("v off", dict(v=_heads(2, at=P + 1))),
    ("stride", dict(v=_heads(2, head=-64))), ("type", dict(type=-1)), ("tokens", dict(tokens=-1)),
    ("many tokens", dict(tokens=1 << 31)),
])
def test_rows_are_refused(what, changes):
    args = dict(dict(slots=P, k=_heads(2), v=_heads(2), type=0, tokens=3), **changes)
    for call in (A.lib().ridge_attention_write, A.lib().ridge_attention_read):
        assert call(_cache(), *args.values(), None) == INVALID


@pytest.mark.parametrize("what,changes", [
    ("q", dict(q=_heads(at=None))), ("heads of q", dict(q=_heads(3), out=_heads(3))), ("out", dict(out=_heads(2))),
    ("pages", dict(pages=None)), ("pages off", dict(pages=P + 1)), ("stride of pages", dict(stride=-4)),
    ("pages each", dict(each=-1)), ("many pages", dict(each=1 << 27)), ("lengths", dict(lengths=None)),
    ("scale", dict(scale=float("inf"))), ("scale nan", dict(scale=float("nan"))), ("window", dict(window=-1)),
    ("lse off", dict(lse=P + 2)), ("type", dict(type=5)), ("batch", dict(batch=-1)), ("many", dict(batch=1 << 30)),
    ("no workspace", dict(each=100, workspace=None)), ("a small workspace", dict(each=100, bytes=1000)),
    ("a workspace off", dict(each=100, workspace=P + 8)),
])
def test_attend_refuses(what, changes):
    args = dict(dict(q=_heads(), cache=_cache(), pages=P, stride=4, each=4, lengths=P, scale=0.125, window=0, out=_heads(),
                     lse=None, type=0, batch=3, workspace=P, bytes=1 << 40), **changes)
    assert A.lib().ridge_attention_attend(*args.values(), None) == INVALID


def test_workspace():
    size = A.lib().ridge_attention_workspace
    assert size(3, 8, 2, 128, 32, 16) == 0       # no sequence is cut
    assert size(128, 8, 2, 128, 64, 16) == 0 < size(127, 8, 2, 128, 64, 16)   # enough heads to fill the card
    assert size(256, 8, 2, 128, 128, 16) == 0 < min(size(255, 8, 2, 128, 128, 16), size(256, 8, 2, 128, 129, 16))
    assert size(128, 34, 2, 128, 64, 16) == size(43, 66, 2, 128, 64, 16) == 0   # tiles of 16 heads count
    assert size(3, 8, 2, 128, 33, 16) == size(1, 4, 1, 128, 1 << 20, 16) > 0
    assert size(3, 8, 2, 128, 33, 16) < size(3, 8, 2, 256, 33, 16) and size(1, 64, 1, 128, 33, 16) == size(1, 16, 1, 128, 33, 16)
    for bad in ((-1, 8, 2, 128, 4, 16), (1 << 31, 8, 2, 128, 4, 16), (3, 9, 2, 128, 4, 16), (3, 8, 0, 128, 4, 16),
                (3, 8, 2, 0, 4, 16), (3, 8, 2, 300, 4, 16), (3, 8, 2, 128, -1, 16), (3, 8, 2, 128, 4, 17),
                (3, 8, 2, 128, 1 << 27, 16)):
        assert size(*bad) < 0


def test_host_tensors_are_refused():
    x = torch.zeros((4, 2, 64), dtype=torch.float16)
    cache = A.empty_cache(2, 16, 2, 64, device="cpu")
    n = torch.zeros(4, dtype=torch.int32)
    table = A.rope_table(8, 64, device="cpu")
    for call in (lambda: A.norm_rope(x, x, table, n), lambda: A.write_cache(cache, n, x, x),
                 lambda: A.read_cache(cache, n), lambda: A.attend(x, cache, n[:, None], n)):
        with pytest.raises(A.RidgeAttentionError, match="device tensor"):
            call()
    for not_a_cache in (None, x, cache[:3], list(cache), (x, x, x, None)):
        with pytest.raises(A.RidgeAttentionError, match="cache"):
            A.read_cache(not_a_cache, n)


def test_without_torch_only_its_extension_is_left_out(monkeypatch, capsys):
    import sys

    from ridge_amd import build
    ran = []
    monkeypatch.setattr(build, "_run", lambda cmd, capture=False: ran.append(cmd) or "")
    monkeypatch.setattr(build.os, "replace", lambda a, b: None)
    monkeypatch.setitem(sys.modules, "torch", None)   # import torch raises ImportError
    assert build.build_attention().endswith("libridge_attention.so")
    assert len(ran) == len(build.ATTENTION_SRCS) + 1 and not any("binding" in word for cmd in ran for word in cmd)
    assert "no torch" in capsys.readouterr().out


def test_attend_refuses_scales_that_float16_has_no_scores_for():
    def attend(type, scale):
        return A.lib().ridge_attention_attend(_heads(), _cache(), P, 4, 4, P, scale, 0, _heads(), None, type, 3, None, 0, None)
    for scale in (2.0 ** 119, -1.01 * 2.0 ** 118):
        assert attend(0, scale) == INVALID
    for type in (0, 1, 2):
        assert attend(type, 2.0 ** 127) == INVALID
