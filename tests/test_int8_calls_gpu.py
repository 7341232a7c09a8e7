"""What the 8-bit operators' calls do with the tensors and streams that they are given."""
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
