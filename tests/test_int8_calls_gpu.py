"""What the 8-bit operators' calls do with the tensors and streams that they are given."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from ridge_amd import int8 as I  # noqa: E402
from test_int8_gpu import DEV, _randn  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    I.lib()
    yield
    torch.cuda.synchronize()


def _operands():
    """(x, weight, q, scale, bias) of 4 rows of 64."""
    x = _randn(4, 64, torch.float16, 1)
    return (x, torch.ones(64, dtype=torch.float16, device=DEV)) + I.quantize(x) + \
        (torch.zeros(4, dtype=torch.float16, device=DEV),)


# Each call with a floating-point buffer of the caller's to write, by what the buffer is.
WRITES = {
    "quantize scale": ((4,), torch.float32, lambda t, x, w, q, s, b: I.quantize(x, out=(q, t))),
    "silu_mul scale": ((4,), torch.float32, lambda t, x, w, q, s, b: I.silu_mul(x, out=(q[:, :32], t))),
    "rms_norm scale": ((4,), torch.float32, lambda t, x, w, q, s, b: I.rms_norm(x, w, out=(q, t))),
    "rms_norm residual_out": ((4, 64), torch.float16, lambda t, x, w, q, s, b: I.rms_norm(x, w, residual=x, residual_out=t)),
    "rms_norm over x": ((4, 64), torch.float16, lambda t, x, w, q, s, b: I.rms_norm(t, w, residual=x, residual_out=t)),
    "rms_norm over residual": ((4, 64), torch.float16, lambda t, x, w, q, s, b: I.rms_norm(x, w, residual=t, residual_out=t)),
    "dequantize out": ((4, 64), torch.float16, lambda t, x, w, q, s, b: I.dequantize(q, s, out=t)),
    "gemm out": ((4, 4), torch.float16, lambda t, x, w, q, s, b: I.gemm(q, s, q, s, out=t)),
}


@pytest.mark.parametrize("what", WRITES)
def test_a_buffer_that_a_graph_saved_is_not_overwritten_in_silence(what):
    shape, dtype, call = WRITES[what]
    operands = _operands()
    buffer = torch.ones(shape, dtype=dtype, device=DEV)
    p = torch.ones(shape, dtype=dtype, device=DEV, requires_grad=True)
    loss = (p * buffer).sum()   # its backward reads the buffer
    with torch.no_grad():
        call(buffer, *operands)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_8_bit_rows_are_versioned_and_read_operands_are_not():
    x, w, q, s, bias = _operands()
    operands = (x, w, q, s, bias)
    before = [t._version for t in operands]
    out = I.empty(4, 64)
    I.quantize(x, out=out), I.rms_norm(x, w, residual=x, out=out), I.gemm(q, s, q, s, bias=bias), I.dequantize(q, s)
    assert [t._version for t in operands] == before
    assert [t._version for t in out] == [2, 2]


def test_buffers_of_inference_mode_are_written_outside_it():
    x, w, q, s, bias = _operands()
    with torch.inference_mode():
        out, rows = torch.empty((4, 4), dtype=torch.float16, device=DEV), I.empty(4, 64)
        I.gemm(q, s, q, s, out=out)
    I.gemm(q, s, q, s, out=out)
    I.quantize(x, out=rows)
    assert torch.equal(out, I.gemm(q, s, q, s)) and torch.equal(rows[0], q)


def test_a_blocks_workspace_is_not_overwritten_under_a_graph_in_silence():
    from ridge_amd.int8_mlp import Int8Mlp, random_block
    mlp = Int8Mlp(*random_block(64, 96, torch.float16, 1))
    x, r = _randn(4, 64, torch.float16, 1), _randn(4, 64, torch.float16, 2)
    space = mlp.workspace(4, torch.float16)
    p = torch.ones(64, dtype=torch.float16, device=DEV, requires_grad=True)
    y, residual = mlp(x, r, space)
    losses = (y * p).sum(), (residual * p).sum()
    mlp(r, x, space)
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_a_tangent_is_refused():
    from torch.autograd import forward_ad
    x, w, q, s, bias = _operands()
    calls = [
        lambda dual: I.quantize(dual(x)), lambda dual: I.silu_mul(dual(x)), lambda dual: I.quantize(x, out=(q, dual(s))),
        lambda dual: I.rms_norm(dual(x), w), lambda dual: I.rms_norm(x, dual(w)),
        lambda dual: I.rms_norm(x, w, residual=dual(x)), lambda dual: I.rms_norm(x, w, residual=x, residual_out=dual(x)),
        lambda dual: I.dequantize(q, dual(s)), lambda dual: I.dequantize(q, s, out=dual(x)),
        lambda dual: I.gemm(q, dual(s), q, s), lambda dual: I.gemm(q, s, q, dual(s)),
        lambda dual: I.gemm(q, s, q, s, bias=dual(bias)),
        lambda dual: I.gemm(q, s, q, s, out=dual(torch.empty((4, 4), dtype=torch.float16, device=DEV))),
    ]

    def dual(t):
        return forward_ad.make_dual(t.clone(), torch.ones_like(t))
    for i, call in enumerate(calls):
        print("call", i, flush=True)
        # Forward mode goes on under no_grad: it is refused there too.
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode, forward_ad.dual_level(), pytest.raises(I.RidgeInt8Error, match="gradient"):
                call(dual)
        with forward_ad.dual_level(), forward_ad._set_fwd_grad_enabled(False):
            call(dual)


def test_functional_transforms_are_refused():
    x, w, q, s, bias = _operands()
    for transform in (lambda: torch.func.jvp(lambda t: I.quantize(t)[1], (x,), (torch.ones_like(x),)),
                      lambda: torch.func.vjp(lambda t: I.quantize(t)[1], x),
                      lambda: torch.func.vmap(lambda t: I.quantize(t)[1])(x.reshape(2, 2, 64))):
        with pytest.raises(RuntimeError):
            transform()


def test_outputs_over_operands_are_refused():
    x, w, q, s, bias = _operands()
    flat = torch.zeros(1024, dtype=torch.float16, device=DEV)
    bytes_ = flat.view(torch.int8)
    f32 = flat.view(torch.float32)
    view = flat[:256].view(4, 64)
    out8 = I.empty(4, 64)
    rows8 = bytes_[:256].view(4, 64)
    C = flat[:16].view(4, 4)
    refused = {
        "shifted by a row": lambda: I.rms_norm(view, w, residual=x, residual_out=flat[64:320].view(4, 64)),
        "shifted by an element": lambda: I.rms_norm(view, w, residual=x, residual_out=flat[1:257].view(4, 64)),
        "another stride": lambda: I.rms_norm(view, w, residual=x, residual_out=flat.as_strided((4, 64), (65, 1))),
        "over the residual": lambda: I.rms_norm(x, w, residual=view, residual_out=flat[64:320].view(4, 64)),
        "x itself, over the residual": lambda: I.rms_norm(view, w, residual=flat[64:320].view(4, 64), residual_out=view),
        "over the weight": lambda: I.rms_norm(x, flat[:64], residual=x, residual_out=view),
        "rows over x": lambda: I.rms_norm(view, w, out=(rows8, s)),
        "rows over the residual": lambda: I.rms_norm(x, w, residual=view, out=(rows8, s)),
        "rows over the sum": lambda: I.rms_norm(x, w, residual=x, residual_out=view, out=(rows8, s)),
        "scales over x": lambda: I.rms_norm(view, w, out=(out8[0], f32[126:130])),
        "scales in the rows": lambda: I.quantize(x, out=(rows8, f32[60:64])),
        "quantize over x": lambda: I.quantize(view, out=(rows8, s)),
        "quantize's scales": lambda: I.quantize(view, out=(out8[0], f32[:4])),
        "silu_mul over its rows": lambda: I.silu_mul(view, out=(rows8[:, :32], s)),
        "dequantize over q": lambda: I.dequantize(rows8, s, out=view),
        "dequantize over its scales": lambda: I.dequantize(q, f32[100:104], out=view),
        "C over a": lambda: I.gemm(rows8, s, q, s, out=C),
        "C over b": lambda: I.gemm(q, s, rows8, s, out=C),
        "C over a_scale": lambda: I.gemm(q, f32[:4], q, s, out=C),
        "C over b_scale": lambda: I.gemm(q, s, q, f32[4:8], out=C),
        "C over the bias": lambda: I.gemm(q, s, q, s, bias=flat[12:16], out=C),
    }
    for name, call in refused.items():
        print(name, flush=True)
        with pytest.raises(I.RidgeInt8Error, match="overlaps"):
            call()


def test_outputs_beside_operands_in_one_buffer():
    x, w, q, s, bias = _operands()
    want = I.quantize(x)
    # x, the residual and the sum as columns of one buffer, the 8-bit rows behind them.
    memory = torch.zeros((4, 64 * 3 + 32), dtype=torch.float16, device=DEV)
    view, residual, total = (memory[:, 64 * i:64 * i + 64] for i in range(3))
    rows8 = memory.view(torch.int8)[:, 384:448]
    view.copy_(x)
    assert torch.equal(I.quantize(view, out=(rows8, s))[0], want[0])
    got = I.rms_norm(view, w, residual=residual, residual_out=total, out=(rows8, s))
    assert torch.equal(got[0], I.rms_norm(x, w)[0]) and torch.equal(total, x)
    # In place, where x and the residual are the same too.
    for into in (view, residual):
        into.copy_(x)
        assert torch.equal(I.rms_norm(into, w, residual=into, residual_out=into)[2], x + x)
    # Halves of one buffer.
    both = torch.zeros((8, 64), dtype=torch.float16, device=DEV)
    both[:4] = x
    assert torch.equal(I.rms_norm(both[:4], w, residual=both[:4], residual_out=both[4:])[2], x + x)


def test_overlap_of_rows_at_any_stride():
    # Random views of one buffer against the bytes that they consist of.
    import random
    rng = random.Random(3)
    memory = torch.zeros(1 << 12, dtype=torch.int8, device=DEV)
    s = torch.ones(9, device=DEV)
    met = 0
    for case in range(600):
        rows, cols = rng.randint(1, 9), rng.randint(1, 40)
        ld8 = 16 * rng.randint((cols + 15) // 16, 8)
        at8 = 16 * rng.randint(0, 40)
        ld16 = ld8 // 2 if rng.random() < 0.5 and ld8 // 2 >= cols else rng.randint(cols, 90)
        at16 = rng.randint(0, 400)
        q = memory.as_strided((rows, cols), (ld8, 1), at8)
        out = memory.view(torch.float16).as_strided((rows, cols), (ld16, 1), at16)
        read = {at8 + i * ld8 + j for i in range(rows) for j in range(cols)}
        written = {2 * (at16 + i * ld16 + j) + e for i in range(rows) for j in range(cols) for e in (0, 1)}
        overlap = bool(read & written)
        met += overlap
        try:
            I.dequantize(q, s[:rows], out=out)
            refused = False
        except I.RidgeInt8Error as e:
            assert "overlaps" in str(e)
            refused = True
        assert refused == overlap, (case, rows, cols, ld8, at8, ld16, at16)
    assert 100 < met < 500


def test_an_earlier_failed_call_is_not_this_ones():
    x, w, q, s, bias = _operands()
    hip = ctypes.CDLL(I.LIB_PATH)   # its runtime, found through it
    calls = [lambda: I.quantize(x), lambda: I.silu_mul(x), lambda: I.rms_norm(x, w), lambda: I.dequantize(q, s),
             lambda: I.gemm(q, s, q, s)]
    for call in calls:
        call()
        assert hip.hipSetDevice(1 << 20) != 0   # a refusal by the runtime, which it also keeps as the last error
        try:
            call()
        finally:
            hip.hipGetLastError()


def test_a_stream_of_another_device_is_refused():
    class Elsewhere:
        cuda_stream, device_index = 0, 1
    x, w, q, s, bias = _operands()
    for call in (lambda t: I.quantize(x, stream=t), lambda t: I.rms_norm(x, w, stream=t),
                 lambda t: I.dequantize(q, s, stream=t), lambda t: I.gemm(q, s, q, s, stream=t)):
        with pytest.raises(I.RidgeInt8Error, match="stream"):
            call(Elsewhere())


def test_streams_by_object_and_by_handle():
    x = _operands()[0]
    want = I.quantize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (None, side, side.cuda_stream, torch.cuda.default_stream(), 0, torch.cuda.ExternalStream(side.cuda_stream)):
        q, scale = I.quantize(x, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(q, want[0]) and torch.equal(scale, want[1])
        assert torch.cuda.current_stream() == torch.cuda.default_stream()
    for stream in ("stream", 1.5, object()):
        with pytest.raises((AttributeError, TypeError)):
            I.quantize(x, stream=stream)


@pytest.mark.parametrize("tokens", [1, 33])
def test_feed_forward_block_without_a_residual(tokens):
    from ridge_amd.int8_mlp import Int8Mlp, plain_block, random_block
    mlp = Int8Mlp(*random_block(256, 512, torch.float16, 1))
    x = _randn(tokens, 256, torch.float16, 2)
    y, residual = mlp(x, None)
    assert residual is x
    space = mlp.workspace(tokens, torch.float16)
    y2, residual = mlp(x, None, space)
    assert y2 is space["y"] and residual is x and torch.equal(y, y2)
    # x + 0 is x: the same block.
    y3, s = mlp(x, torch.zeros_like(x))
    assert torch.equal(y, y3) and torch.equal(s, x)


def test_feed_forward_command_fails_on_results_that_are_not_numbers(monkeypatch):
    from ridge_amd import int8_mlp
    plain = int8_mlp.random_block

    def broken(*args):
        norm_weight, gate_up, down = plain(*args)
        down[0, 0] = math.nan
        return norm_weight, gate_up, down
    args = ["--hidden", "64", "--inner", "64", "--tokens", "1,2", "--steps", "2"]
    assert int8_mlp.main(args) == 0
    monkeypatch.setattr(int8_mlp, "random_block", broken)
    assert int8_mlp.main(args) == 1


def test_ordinary_buffers_are_written_in_inference_mode():
    x, w, q, s, bias = _operands()
    out, rows, total = torch.zeros((4, 4), dtype=torch.float16, device=DEV), I.empty(4, 64), torch.zeros_like(x)
    with torch.inference_mode():
        I.gemm(q, s, q, s, out=out)
        I.rms_norm(x, w, residual=x, residual_out=total, out=rows)
        new = I.gemm(q, s, q, s)
    assert new.is_inference() and torch.equal(out, new) and torch.equal(total, x + x)
