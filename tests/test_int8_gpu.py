"""The 8-bit operators on the GPU against 64-bit references.

Tolerances. u = 2^-24 is half a unit of f32. A scale is a maximum of values that carry
a few roundings each, over 127; a norm's also carries the error of a sum of squares of D
terms, at most as many u as the longest chain of additions is long, halved by the root.
Of q, y / scale is computed with a few u of error (the norm's root cancels), so q lies
within 0.5 + 127 * 16 u of the exact quotient by the *returned* scale's exact value. A
product's sum is exact: each output carries four roundings of f32 in the terms and one to
its type.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from ridge_amd import int8 as I  # noqa: E402
from test_int8 import FORMS  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]
HALF_UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
TINY = 2.0 ** -126


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    I.lib()
    yield
    torch.cuda.synchronize()


def _randn(rows, cols, dtype, seed, wide=0, offset=0):
    """Normal rows with a few wide channels; a view of a wider buffer where asked."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((rows, cols + wide), generator=g, device=DEV)
    x[:, ::17] *= 9
    return x.to(dtype)[:, offset:offset + cols]


def _int8(rows, cols, seed, pad=0, least=-127):
    """8-bit rows whose memory behind `cols` is full of other values."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    ld = (cols + 15) // 16 * 16 + pad
    q = torch.randint(least, 128, (rows, ld), generator=g, device=DEV, dtype=torch.int8)[:, :cols]
    return q, torch.rand(rows, generator=g, device=DEV) * 0.03 + 0.001


def _check_rows(q, scale, y, value_error=8 * U, scale_error=8 * U):
    """q, scale against rows y in 64 bits whose values carry value_error."""
    q, scale, y = q.cpu().double(), scale.cpu().double(), y.cpu().double()
    want = (y.abs().amax(dim=1) / 127).clamp_min(TINY)
    assert torch.all((scale - want).abs() <= want * scale_error), float(((scale - want).abs() / want).max())
    assert float(q.abs().max()) <= 127
    exact = y / want[:, None]
    assert float((q - exact).abs().max()) <= 0.5 + 127 * (8 * U + value_error)


def _sum_error(cols):
    """Of a norm's scale: the longest chain of additions, 32 + 10 + 16 where a row is held
    in registers and cols / 1024 where it is not, halved by the root, and a few more."""
    return (max(58, cols / 1024 + 26) / 2 + 8) * U


# Around every change of form: vectors of 8, rows held by 64, 256 and 1024 threads, rows
# read twice.
WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 511, 512, 513, 1000, 2047, 2048, 2049, 4096, 8192, 8193, 8199, 16384, 16391, 32768,
          32777, 50001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantize(cols, dtype):
    for rows in (1, 5):
        x = _randn(rows, cols, dtype, cols)
        q, scale = I.quantize(x)
        _check_rows(q, scale, x.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_silu_mul(cols, dtype):
    for rows in (1, 5):
        x = _randn(rows, 2 * cols, dtype, cols)
        q, scale = I.silu_mul(x)
        g, u = x.double().chunk(2, dim=1)
        # 1 + exp(-g) carries 3 u (exp's two, its argument's none, one of the sum), the
        # division and the product one each.
        _check_rows(q, scale, g * torch.sigmoid(g) * u)


@pytest.mark.parametrize("weight_f32", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm(cols, dtype, weight_f32):
    eps = 1e-5
    w = (_randn(1, cols, torch.float32, 3)[0] * 0.1 + 1).to(torch.float32 if weight_f32 else dtype)
    for rows in (1, 5):
        x, r = _randn(rows, cols, dtype, cols), _randn(rows, cols, dtype, cols + 1)
        for residual in (None, r):
            s = x.double() if residual is None else x.double() + r.double()
            y = s / (s.square().mean(dim=1, keepdim=True) + eps).sqrt() * w.double()
            q, scale, out = I.rms_norm(x, w, eps, residual=residual)
            # x + residual and the product with the weight are one rounding of f32 each.
            _check_rows(q, scale, y, scale_error=_sum_error(cols))
            if residual is None:
                assert out is None
            else:
                assert out.dtype == dtype
                assert torch.equal(out, (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_wider_buffers_at_odd_offsets(dtype):
    rows, cols = 37, 1003
    x, r = _randn(rows, cols, dtype, 1, 21, 3), _randn(rows, cols, dtype, 2, 5, 1)
    w = _randn(1, cols, dtype, 3, 7, 5)[0]
    buffer = torch.full((rows + 2, 1024 + 32), 99, dtype=torch.int8, device=DEV)
    out = buffer[1:-1, 16:16 + cols], torch.empty(rows, device=DEV)
    for make, plain in ((lambda: I.quantize(x, out=out), lambda: I.quantize(x.contiguous())),
                        (lambda: I.silu_mul(x[:, :1002], out=(out[0][:, :501], out[1])),
                         lambda: I.silu_mul(x[:, :1002].contiguous())),
                        (lambda: I.rms_norm(x, w, residual=r, out=out)[:2],
                         lambda: I.rms_norm(x.contiguous(), w.contiguous(), residual=r.contiguous())[:2])):
        buffer.fill_(99)
        q, scale = make()
        pq, pscale = plain()
        assert torch.equal(q, pq) and torch.equal(scale, pscale)
        inside = torch.zeros_like(buffer, dtype=torch.bool)
        inside[1:-1, 16:16 + q.shape[1]] = True
        assert torch.all(buffer[~inside] == 99), "wrote outside its rows"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [300, 4097, 20000, 40007])
def test_residual_in_place(cols, dtype):
    x, r = _randn(6, cols, dtype, 1), _randn(6, cols, dtype, 2)
    w = torch.ones(cols, dtype=dtype, device=DEV)
    q, scale, out = I.rms_norm(x, w, residual=r)
    for into in (0, 1):
        operands = [x.clone(), r.clone()]
        q2, scale2, out2 = I.rms_norm(operands[0], w, residual=operands[1], residual_out=operands[into])
        assert out2.data_ptr() == operands[into].data_ptr()
        assert torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(out, out2)
        assert torch.equal(operands[1 - into], (x, r)[1 - into])


@pytest.mark.parametrize("cols", [5, 700, 5000, 33000])
def test_rows_without_a_finite_value_do_not_come_back_finite_and_leave_the_others(cols):
    x = _randn(6, cols, torch.bfloat16, 4)
    clean = I.quantize(x)
    bad = x.clone()
    for row, value in ((1, math.nan), (3, math.inf), (4, -math.inf)):
        bad[row, cols // 2] = value
    w = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
    gated = torch.cat([bad, torch.ones_like(bad)], dim=1)
    for q, scale in (I.quantize(bad), I.rms_norm(bad, w)[:2], I.silu_mul(gated)):
        finite = torch.isfinite(scale).tolist()
        # silu(-inf) is 0 * -inf, NaN.
        assert finite == [True, False, True, False, False, True]
        values = I.dequantize(q, scale, torch.float32)
        assert not torch.isfinite(values[[1, 3, 4]]).any()
        assert torch.isfinite(values[[0, 2, 5]]).all()
    q, scale = I.quantize(bad)
    for row in (0, 2, 5):
        assert torch.equal(q[row], clean[0][row]) and scale[row] == clean[1][row]


def test_zero_rows_and_rows_under_the_least_scale():
    x = torch.zeros((4, 100), dtype=torch.float32, device=DEV)
    x[1, 3] = 1e-44                 # under 127 times the smallest normal number: nothing of it is kept
    x[2, 3], x[2, 4] = 127 * TINY, -64.4 * TINY
    x[3, :] = 1.0
    q, scale = I.quantize(x)
    assert torch.isfinite(scale).all() and torch.all(scale >= TINY)
    assert not q[:2].any()
    assert q[2, 3] == 127 and q[2, 4] == -64 and torch.all(q[3] == 127)
    # A norm of zeros is zero: eps keeps the root finite.
    w = torch.ones(100, dtype=torch.float32, device=DEV)
    q, scale, _ = I.rms_norm(torch.zeros_like(x), w, 1e-12)
    assert not q.any() and torch.isfinite(scale).all()


def test_a_sum_of_squares_past_f32_is_not_silently_zero():
    x = torch.full((2, 64), 1.0, dtype=torch.bfloat16, device=DEV)
    x[1] *= 1e25
    _, scale, _ = I.rms_norm(x, torch.ones(64, dtype=torch.bfloat16, device=DEV))
    assert torch.isfinite(scale).tolist() == [True, False]


def test_silu_of_far_values():
    g = torch.tensor([[-1000.0, -100.0, -88.0, 0.0, 50.0, 1000.0]], device=DEV)
    q, scale = I.silu_mul(torch.cat([g, torch.ones_like(g)], dim=1))
    assert torch.equal(q.cpu(), torch.tensor([[0, 0, 0, 0, 6, 127]], dtype=torch.int8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (2, 2049), (7, 4100)])
def test_dequantize(rows, cols, dtype):
    q, scale = _int8(rows, cols, rows, least=-128)
    want = (q.float() * scale[:, None]).to(dtype)
    assert torch.equal(I.dequantize(q, scale, dtype), want)
    buffer = torch.full((rows + 2, cols + 9), 7.0, dtype=dtype, device=DEV)
    I.dequantize(q, scale, out=buffer[1:-1, 4:-5])
    assert torch.equal(buffer[1:-1, 4:-5], want)
    buffer[1:-1, 4:-5] = 7.0
    assert torch.all(buffer == 7.0)


def test_more_elements_than_32_bits_count():
    rows, cols = 70001, 32768
    x = torch.zeros((rows, cols), dtype=torch.float16, device=DEV)
    x[-3:] = _randn(3, cols, torch.float16, 1)
    x[0] = x[-1]
    q, scale = I.quantize(x)
    _check_rows(q[-3:], scale[-3:], x[-3:].double())
    assert torch.equal(q[0], q[-1]) and not q[1:-3].any()
    del x
    v = I.dequantize(q, scale, torch.float16)
    assert torch.equal(v[-3:], (q[-3:].float() * scale[-3:, None]).half())


# ---------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------

def _exact_sums(a, b):
    """Whole-number products in float64, exact: |sum| < 2^31."""
    return a.double() @ b.double().t()


def _check_product(out, a, a_scale, b, b_scale, bias=None):
    term = _exact_sums(a, b) * a_scale.double()[:, None] * b_scale.double()
    add = torch.zeros_like(term) if bias is None else bias.double().expand_as(term)
    want = term + add
    bound = 4 * U * (term.abs() + add.abs()) * 2 + HALF_UNIT[out.dtype] * want.abs() + LEAST[out.dtype]
    off = (out.double() - want).abs()
    assert torch.all(off <= bound * 1.0001), "worst element at %.3f of its bound" % float((off / bound).max())


def _product(M, N, K, dtype, with_bias=False, seed=0, pad=0):
    print("product %d x %d x %d %s" % (M, N, K, dtype), flush=True)
    a, sa = _int8(M, K, seed + 1, pad, -128)
    b, sb = _int8(N, K, seed + 2, pad, -128)
    sb = sb / math.sqrt(K)
    bias = _randn(1, N, dtype, seed + 3)[0] if with_bias else None
    # In a buffer of its own: nothing outside may change.
    buffer = torch.full((M + 2, N + 5), 7.0, dtype=dtype, device=DEV)
    out = buffer[1:-1, 2:-3]
    assert I.gemm(a, sa, b, sb, bias=bias, out=out) is out
    _check_product(out, a, sa, b, sb, bias)
    out.fill_(7.0)
    assert torch.all(buffer == 7.0), "wrote outside C"


@pytest.mark.parametrize("K", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 384, 511, 640, 1000, 4099])
@pytest.mark.parametrize("M", [1, 3, 16, 17, 40, 64, 65, 130, 300])
def test_product_of_every_depth(M, K):
    _product(M, 200, K, torch.float16, seed=M + K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 4096), (2, 17), (5, 1000), (16, 16), (17, 33), (31, 129), (33, 1), (48, 513),
                                 (64, 64), (65, 2047), (100, 300), (128, 128), (129, 257), (255, 1030), (513, 511),
                                 (1100, 1300), (2100, 2070)])
def test_product_of_every_size(M, N, with_bias, dtype):
    _product(M, N, 300, dtype, with_bias, seed=M + N)


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 320), (4100, 4099, 333), (5000, 7000, 640), (300, 16400, 1100),
                                   (16400, 300, 1100), (8200, 8300, 130)])
def test_product_of_large_grids(M, N, K):
    _product(M, N, K, torch.bfloat16, True, seed=K, pad=48)


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_the_longest_sum_fits(M):
    K = I.MAX_K
    a, b = (torch.full((n, K + 1), -128, dtype=torch.int8, device=DEV)[:, :K] for n in (M, 96))
    one = torch.ones(M, device=DEV), torch.ones(96, device=DEV)
    out = I.gemm(a, one[0], b, one[1], dtype=torch.float32)
    assert torch.all(out == float(np.float32(16384 * K)))
    b[0] = 127
    b[1] = 0
    out = I.gemm(a, one[0], b, one[1], dtype=torch.float32)
    assert torch.all(out[:, 0] == float(np.float32(-128 * 127 * K))) and torch.all(out[:, 1] == 0)


@pytest.mark.parametrize("M", [1, 40, 200])
def test_products_with_scales_that_are_not_finite(M):
    a, sa = _int8(M, 100, 1)
    b, sb = _int8(70, 100, 2)
    sa[M // 2], sb[5], sb[6] = math.nan, math.inf, math.nan
    out = I.gemm(a, sa, b, sb)
    finite = torch.isfinite(out)
    assert not finite[M // 2].any() and not finite[:, 5:7].any()
    finite[M // 2], finite[:, 5:7] = True, True
    assert finite.all()


def test_product_with_more_elements_than_32_bits_count():
    M, N, K = 70001, 32768, 40
    a, sa = _int8(M, K, 1)
    b, sb = _int8(N, K, 2)
    out = I.gemm(a, sa, b, sb)
    for rows in (slice(0, 40), slice(65520, 65560), slice(M - 40, M)):
        _check_product(out[rows], a[rows], sa[rows], b, sb)


@pytest.mark.parametrize("M", [1, 30, 300])
def test_product_of_rows_far_apart(M):
    # 8-bit operands of more than 2^32 bytes, rows up to the largest stride apart.
    N, K, ld = 700, 200, (1 << 23) - 16
    memory = torch.empty(N * ld, dtype=torch.int8, device=DEV)
    b = memory.view(N, ld)[:, :K]
    b.copy_(_int8(N, K, 2)[0])
    sb = _int8(N, K, 2)[1]
    a, sa = _int8(M, K, 1)
    _check_product(I.gemm(a, sa, b, sb, dtype=torch.float32), a, sa, b, sb)
    _check_product(I.gemm(b, sb, a, sa, dtype=torch.float32), b, sb, a, sa)


def test_calls_on_a_stream_of_their_own():
    x, w = _randn(300, 1000, torch.float16, 1), _int8(500, 1000, 2)
    weight = torch.ones(1000, dtype=torch.float16, device=DEV)
    q, s, r = I.rms_norm(x, weight, residual=x)
    want = I.gemm(q, s, *w), r, I.dequantize(*I.silu_mul(x)), I.dequantize(*I.quantize(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        q, s, r = I.rms_norm(x, weight, residual=x, stream=stream)
        got = (I.gemm(q, s, *w, stream=stream), r,
               I.dequantize(*I.silu_mul(x, stream=stream), stream=stream),
               I.dequantize(*I.quantize(x, stream=stream), stream=stream))
        side.synchronize()
        for g, t in zip(got, want):
            assert torch.equal(g, t)


def test_calls_are_the_same_every_time_and_in_a_graph():
    x, w = _randn(20, 1500, torch.bfloat16, 1), _int8(2000, 1500, 2)
    weight = torch.ones(1500, dtype=torch.bfloat16, device=DEV)
    rows, r, out = I.empty(20, 1500), torch.empty_like(x), torch.empty((20, 2000), dtype=torch.bfloat16, device=DEV)
    gated = I.empty(20, 1000)

    def step():
        I.rms_norm(x, weight, residual=x, residual_out=r, out=rows)
        I.gemm(*rows, *w, out=out)
        I.silu_mul(out, out=gated)

    def results():
        return [t.clone() for t in (r, rows[0], rows[1], out, gated[0], gated[1])]
    step()
    want = results()
    step()
    assert all(torch.equal(a, b) for a, b in zip(results(), want))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        for t in (r, out, rows[1], gated[1]):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results(), want))
        step()
        torch.cuda.synchronize()


def test_empty_batches():
    x = torch.empty((0, 64), dtype=torch.float16, device=DEV)
    w = _int8(32, 64, 1)
    q, s, r = I.rms_norm(x, torch.ones(64, dtype=torch.float16, device=DEV), residual=x)
    assert q.shape == (0, 64) and s.shape == (0,) and r.shape == (0, 64)
    assert I.gemm(q, s, *w).shape == (0, 32)
    assert I.gemm(*w, q, s).shape == (32, 0)
    assert I.silu_mul(x)[0].shape == (0, 32) and I.quantize(x)[0].shape == (0, 64)
    assert I.dequantize(q, s).shape == (0, 64)


def test_refusals():
    x = _randn(4, 64, torch.float16, 1)
    w = torch.ones(64, dtype=torch.float16, device=DEV)
    q, s = I.quantize(x)
    odd = torch.empty((4, 65), dtype=torch.int8, device=DEV)
    refused = [
        lambda: I.quantize(x[0]), lambda: I.quantize(x.t()), lambda: I.quantize(x.double()),
        lambda: I.quantize(x.expand(4, 64)[:, :0]), lambda: I.quantize(w.expand(4, 64)),
        lambda: I.quantize(x, out=I.empty(4, 63)), lambda: I.quantize(x, out=(odd[:, :64], s)),
        lambda: I.quantize(x, out=(odd[:, 1:], s)), lambda: I.quantize(x, out=(q, s.double())),
        lambda: I.silu_mul(x[:, :63]),
        lambda: I.rms_norm(x, w[:63]), lambda: I.rms_norm(x, w.bfloat16()), lambda: I.rms_norm(x, w, 0.0),
        lambda: I.rms_norm(x, w, residual=x[:2]), lambda: I.rms_norm(x, w, residual=x.bfloat16()),
        lambda: I.rms_norm(x, w, residual_out=x), lambda: I.rms_norm(x, w, float("nan")),
        lambda: I.dequantize(x, s), lambda: I.dequantize(q, s, torch.float64), lambda: I.dequantize(q, s[:2]),
        lambda: I.gemm(q, s, q[:, :32], s), lambda: I.gemm(x, s, q, s), lambda: I.gemm(q, s[:3], q, s),
        lambda: I.gemm(q, s, q, s, bias=w), lambda: I.gemm(q, s, q, s, out=x), lambda: I.gemm(q, s, q, s.cpu()),
        lambda: I.gemm(q, s, q, s, bias=w[:4].float()), lambda: I.gemm(q[:, :0], s, q[:, :0], s),
        # The last row's memory ends inside 16 bytes.
        lambda: I.gemm(torch.empty(4 * 16 - 6, dtype=torch.int8, device=DEV).as_strided((4, 10), (16, 1)), s, q, s),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(I.RidgeInt8Error):
            print("refusal", i, flush=True)
            call()
    y = x.clone().requires_grad_()
    with pytest.raises(I.RidgeInt8Error, match="gradient"):
        I.quantize(y)
    with torch.no_grad():
        assert torch.equal(I.quantize(y)[0], q)


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [1, 7, 65, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_feed_forward_block(tokens, dtype):
    from ridge_amd.int8_mlp import Int8Mlp, plain_block, random_block
    hidden, inner = 1000, 2100
    weights = random_block(hidden, inner, dtype, tokens)
    mlp = Int8Mlp(*weights)
    x, r = _randn(tokens, hidden, dtype, 1) * 0.5, _randn(tokens, hidden, dtype, 2)
    y, s = mlp(x, r)
    space = mlp.workspace(tokens, dtype)
    y2, s2 = mlp(x, r, space)
    assert y2 is space["y"] and s2 is space["residual"]
    assert torch.equal(y, y2) and torch.equal(s, s2)
    want, sums = plain_block(x.double(), r.double(), *(w.double() for w in weights))
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    # Rounding to steps of max / 127 leaves an error of 0.29 steps. Normal rows of 1000 to
    # 2100 reach 3.5 of their standard deviations: 0.8% for each of the four operands, but
    # the norm's rows have channels nine times as wide (27 of a deviation of 2.4: 2.6%)
    # and silu(gate) * up reaches about 15 of its deviations (3.4%). Together 4.6%, of
    # which the gate's share counts about 1.4 times: under 7%.
    assert float((y.double() - want).norm() / want.norm()) < 0.07


def test_feed_forward_block_refuses_weights_of_another_shape():
    from ridge_amd.int8_mlp import Int8Mlp, random_block
    norm_weight, gate_up, down = random_block(64, 96, torch.float16, 1)
    for w in ((norm_weight, gate_up[:-2], down), (norm_weight[:-1], gate_up, down), (norm_weight, gate_up, down.t())):
        with pytest.raises(I.RidgeInt8Error):
            Int8Mlp(*w)


def test_feed_forward_command_in_a_graph():
    from ridge_amd import int8_mlp
    assert int8_mlp.main(["--hidden", "256", "--inner", "512", "--tokens", "1,33", "--steps", "5", "--graph"]) == 0


@pytest.mark.parametrize("M,N,K", [(1, 70000, 33), (70000, 3, 33), (66000, 70, 200)])
def test_products_whose_sizes_do_not_pack(M, N, K):
    _product(M, N, K, torch.float16, True, seed=M)


def test_product_past_the_caches():
    # A C of more than 64 MiB whose rows are whole cache lines, and one a row too narrow.
    for M, N in ((4200, 8192), (4200, 8190), (9000, 4096)):
        a, sa = _int8(M, 200, 1)
        b, sb = _int8(N, 200, 2)
        _check_product(I.gemm(a, sa, b, sb), a, sa, b, sb)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form,M,N,K", FORMS)
def test_every_form_of_the_product(form, M, N, K, dtype):
    _product(M, N, K, dtype, True, seed=K)


@pytest.mark.parametrize("cols", [5003, 16384])
def test_rows_past_the_caches(cols):
    # More than 64 MiB: read and written non-temporally; the same results as a part of it.
    rows = (64 << 20) // (2 * cols) + 5
    x, r = _randn(rows, cols, torch.float16, 1), _randn(rows, cols, torch.float16, 2)
    w = torch.ones(cols, dtype=torch.float16, device=DEV)
    part = slice(rows - 40, rows)
    for make in (lambda t, s: I.quantize(t), lambda t, s: I.silu_mul(t[:, :cols // 2 * 2]),
                 lambda t, s: I.rms_norm(t, w, residual=s)):
        for got, want in zip(make(x, r), make(x[part], r[part])):
            assert torch.equal(got[part], want)
    q, scale = I.quantize(x)
    assert torch.equal(I.dequantize(q, scale)[part], I.dequantize(q[part], scale[part]))


@pytest.mark.parametrize("cols", [600, 2048, 2049, 8192, 11007])
def test_a_row_does_not_depend_on_the_rows_beside_it(cols):
    x, r = _randn(700, cols, torch.bfloat16, 1), _randn(700, cols, torch.bfloat16, 2)
    w, b = torch.ones(cols, dtype=torch.bfloat16, device=DEV), _int8(300, cols, 3)
    for make in (lambda t, s: I.quantize(t), lambda t, s: I.silu_mul(t[:, :cols // 2 * 2]),
                 lambda t, s: I.rms_norm(t, w, residual=s)):
        whole = make(x, r)
        for rows in (slice(0, 1), slice(3, 20), slice(100, 612)):
            for got, want in zip(make(x[rows], r[rows]), whole):
                assert torch.equal(got, want[rows])
    q, scale = I.quantize(x)
    y = I.gemm(q, scale, *b)
    for rows in (slice(0, 1), slice(3, 20), slice(100, 612)):
        assert torch.equal(I.gemm(q[rows], scale[rows], *b), y[rows])


def test_silu_of_values_whose_exponential_comes_near_the_ranges_end():
    g = torch.tensor([[-87.5, -86.0, -85.0, -80.0]], device=DEV)
    u = torch.tensor([[1e36, 1e36, -1e36, 1e34]], device=DEV)
    q, scale = I.silu_mul(torch.cat([g, u], dim=1))
    _check_rows(q, scale, g.double() * torch.sigmoid(g.double()) * u.double())


def test_a_product_of_more_rows_than_the_smallest_tiles_count():
    # 64 x 64 tiles, which few columns ask for, would be more than a launch has.
    M, K = 600_000_000, 16
    a = torch.zeros((M, K), dtype=torch.int8, device=DEV)
    a[-3:] = 5
    sa, b, sb = torch.ones(M, device=DEV), torch.full((1, K), 2, dtype=torch.int8, device=DEV), torch.ones(1, device=DEV)
    out = I.gemm(a, sa, b, sb)
    assert torch.all(out[-3:] == 160) and not out[:-3].any()


def test_no_call_drops_a_gradient():
    x = _randn(4, 64, torch.float16, 1)
    w = torch.ones(64, dtype=torch.float16, device=DEV)
    q, s = I.quantize(x)
    bias = torch.zeros(4, dtype=torch.float16, device=DEV)

    def leaf(t):
        return t.clone().requires_grad_()
    calls = [
        lambda: I.quantize(leaf(x)), lambda: I.silu_mul(leaf(x)), lambda: I.quantize(x, out=(q, leaf(s))),
        lambda: I.rms_norm(leaf(x), w), lambda: I.rms_norm(x, leaf(w)), lambda: I.rms_norm(x, w, residual=leaf(x)),
        lambda: I.rms_norm(x, w, residual=x, residual_out=leaf(x)),
        lambda: I.dequantize(q, leaf(s)), lambda: I.dequantize(q, s, out=leaf(x)),
        lambda: I.gemm(q, leaf(s), q, s), lambda: I.gemm(q, s, q, leaf(s)), lambda: I.gemm(q, s, q, s, bias=leaf(bias)),
        lambda: I.gemm(q, s, q, s, out=leaf(torch.empty((4, 4), dtype=torch.float16, device=DEV))),
    ]
    for call in calls:
        with pytest.raises(I.RidgeInt8Error, match="gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("dtype,exponents", [(torch.float16, (-10, 0, 15)), (torch.bfloat16, (-118, -60, 0, 55)),
                                             (torch.float32, (-118, -60, 0, 55))])
@pytest.mark.parametrize("cols", [3, 700, 20000, 33000])
def test_half_of_a_rows_largest_value_is_a_half_and_goes_to_even(cols, dtype, exponents):
    # 127 (top / 2) / top is 63.5 whatever f32 makes of top / 127.
    bits = {torch.float16: 10, torch.bfloat16: 7, torch.float32: 23}[dtype]
    mantissas = torch.arange(0, 1 << bits, max(1, (1 << bits) // 128 - (bits > 7)), device=DEV)
    for exponent in exponents:
        print("2^%d" % exponent, flush=True)
        top = ((1 + mantissas.double() / 2 ** bits) * 2.0 ** exponent).to(dtype)
        x = torch.zeros((len(top), cols), dtype=dtype, device=DEV)
        x[:, 0], x[:, 1], x[:, -1] = -top, top / 2, -top / 2
        one = torch.ones(cols, dtype=dtype, device=DEV)
        # silu(32) is 32 in f32.
        makers = {"quantize": I.quantize(x), "silu_mul": I.silu_mul(torch.cat([torch.full_like(x, 32), x], dim=1)),
                  "rms_norm": I.rms_norm(x, one)[:2]}
        for name, (q, scale) in makers.items():
            assert torch.all(q[:, 0] == -127) and torch.all(q[:, 1] == 64) and torch.all(q[:, -1] == -64), name
            assert not q[:, 2:-1].any()


# silu(g) u of gates whose e^-g is past f32, where a large u brings the product back. Rows of
# 16 bits as far as their u goes.
FAR = [(torch.float32, [-89.0, -89.5, -90.0, -92.0], 3e38), (torch.float32, [-100.0, -101.0, -102.5, -104.0], 1e35),
       (torch.float32, [-160.0, -165.0, -168.0, -170.0], 3e38), (torch.bfloat16, [-89.0, -90.0, -91.0, -95.0], 1e38),
       (torch.bfloat16, [-120.0, -121.0, -124.0, -130.0], -2e38), (torch.float16, [-88.75, -89.0, -90.0, -92.0], 6e4),
       (torch.float32, [-86.0, -88.0, -88.5, -89.0], 1e30)]


@pytest.mark.parametrize("dtype,gates,up", FAR)
def test_silu_of_gates_whose_exponential_is_past_the_range(dtype, gates, up):
    # e^g to 2 u, the products with g and u one each, the last scaling one: within the 8 u
    # that _check_rows allows.
    for n in (4, 500):
        g = torch.tensor([gates], device=DEV).to(dtype).repeat(3, n // 4)
        u = torch.full_like(g, up)
        q, scale = I.silu_mul(torch.cat([g, u], dim=1))
        _check_rows(q, scale, g.double() * torch.exp(g.double()) / (1 + torch.exp(g.double())) * u.double())


H, B, F = torch.float16, torch.bfloat16, torch.float32
# (form, type, M, N, K) of products whose C goes past the caches: rows of whole cache lines,
# more than 64 MiB. Sizes of up to 65535 rows and more (the two forms of a launch's
# arguments); form 0 with its last round in quarters, halves and whole.
PAST = [(0, H, 4200, 8181, 200), (0, B, 5000, 8180, 100), (0, F, 6100, 8171, 100), (0, H, 174416, 193, 32),
        (0, B, 174416, 193, 32), (0, F, 130662, 129, 33), (1, H, 35553, 1029, 4020), (1, B, 11584, 3443, 4096),
        (1, F, 1542, 13871, 2048), (1, H, 325436, 104, 785), (1, B, 325436, 104, 785), (1, F, 255113, 68, 668),
        (3, H, 56363, 610, 33), (3, B, 56363, 610, 33), (3, F, 1303, 13581, 64), (3, H, 600000, 61, 64),
        (3, B, 600000, 61, 64), (3, F, 261876, 65, 32)]


@pytest.mark.parametrize("form,dtype,M,N,K", PAST)
def test_every_form_past_the_caches_stays_inside_its_rows(form, dtype, M, N, K):
    assert I.lib().ridge_int8_gemm_form(M, N, K) == form
    size = torch.empty((), dtype=dtype).element_size()
    assert M * N * size > 64 << 20
    line = 128 // size
    memory = torch.full((M + 2, (N + line) // line * line), 7.0, dtype=dtype, device=DEV)
    out = memory[1:-1, :N]
    assert out.data_ptr() % 128 == 0 and out.stride(0) * size % 128 == 0 and out.stride(0) > N
    a, sa = _int8(M, K, 1, least=-128)
    b, sb = _int8(N, K, 2, least=-128)
    sb = sb / math.sqrt(K)
    bias = _randn(1, N, dtype, 3)[0]
    I.gemm(a, sa, b, sb, bias=bias, out=out)
    for rows in torch.arange(M, device=DEV).split(1 << 16):
        part = slice(int(rows[0]), int(rows[-1]) + 1)
        _check_product(out[part], a[part], sa[part], b, sb, bias)
    out.fill_(7.0)
    assert torch.all(memory == 7.0), "wrote outside C"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1003, 5002, 16384])
def test_rows_past_the_caches_of_every_type(cols, dtype):
    # Rows of wider buffers: the same bits as a part of them gives, and nothing beside them.
    size = torch.empty((), dtype=dtype).element_size()
    rows = (64 << 20) // (size * cols) + 5
    x, r = _randn(rows, cols, dtype, 1, 5, 3), _randn(rows, cols, dtype, 2, 3, 1)
    w = _randn(1, cols, dtype, 3)[0]
    part = slice(rows - 40, rows)
    ld = I.lib().ridge_int8_row_stride(cols) + 128
    memory = torch.full((rows + 2, ld), 99, dtype=torch.int8, device=DEV)
    total = torch.full((rows + 2, cols + 9), 7.0, dtype=dtype, device=DEV)
    inside = memory[1:-1, 16:16 + cols]
    half = cols // 2
    makers = [lambda t, s, sum_, q, scale: I.quantize(t, out=(q, scale)),
              lambda t, s, sum_, q, scale: I.silu_mul(t[:, :2 * half], out=(q[:, :half], scale)),
              lambda t, s, sum_, q, scale: I.rms_norm(t, w, residual=s, residual_out=sum_, out=(q, scale))]
    for i, make in enumerate(makers):
        width = half if i == 1 else cols
        got = make(x, r, total[1:-1, 4:-5], inside, torch.empty(rows, device=DEV))
        want = make(x[part], r[part], torch.empty((40, cols), dtype=dtype, device=DEV), *I.empty(40, cols))
        for g, t in zip(got, want):
            assert torch.equal(g[part], t)
        inside[:, :width] = 99
        assert torch.all(memory == 99)
        total[1:-1, 4:-5] = 7.0
        assert torch.all(total == 7.0)
    q, scale = I.quantize(x)
    I.dequantize(q, scale, out=total[1:-1, 4:-5])
    assert torch.equal(total[1:-1, 4:-5][part], I.dequantize(q[part], scale[part], dtype))
    total[1:-1, 4:-5] = 7.0
    assert torch.all(total == 7.0)
