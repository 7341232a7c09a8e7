"""attend where values, scales and scores lie far apart, against 64 bits.

Tolerances. u = 2^-24 is half a unit of f32. A score is a sum of D exact products (of 3 D for a query of
f32, whose columns are three parts of bf16), at most as many roundings and 6 of the sum of their
magnitudes; as the exponent of p it carries that as a relative error, with 4 u of its own size and of
the maximum's. p carries 4 u more, its product with a value's scale u, and sums of three parts of n
terms 3 n u. out's numerator and denominator each carry that, relative to the sum of |p v|; a p below
2^-126 of the largest may count nothing, which is within that many times the sum of |v|. (2^-47 where scales
up to 2^-40 alone and past 2^88 meet: no test here has such a p.)
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from ridge_amd import attention as A  # noqa: E402
from test_attention_gpu import DEV, TYPES, U, Batch, _close  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    A.lib()
    yield
    torch.cuda.synchronize()


def _check(b, scale=None):
    """attend of a Batch against 64 bits."""
    lost = 2.0 ** -126
    B, H, D = b.q.shape
    lse = torch.empty((B, H), device=DEV)
    got = A.attend(b.q, b.cache, b.pages, b.lengths, scale=scale, lse_out=lse)
    scale = D ** -0.5 if scale is None else scale
    for i, n in enumerate(b.sizes):
        if n == 0:
            continue
        k, v = b.rows(i)
        q = b.q[i].double().reshape(k.shape[0], -1, D)
        s = q @ k.transpose(1, 2).contiguous() * scale
        most = q.abs() @ k.abs().transpose(1, 2).contiguous() * abs(scale)
        p = torch.softmax(s, dim=2)
        products = 3 * D if b.q.dtype == torch.float32 else D
        off = (products + 6) * U * most + 4 * U * (s.abs() + s.amax(dim=2, keepdim=True).abs()) + (5 + 3 * n) * U
        mass = (p * off).sum(dim=2, keepdim=True) + lost * n
        slack = (p * off) @ v.abs() + mass * (p @ v.abs()) + lost * v.abs().sum(dim=1, keepdim=True)
        _close(got[i], (p @ v).reshape(H, D), slack.reshape(H, D), b.q.dtype)
        want = torch.logsumexp(s, dim=2).reshape(H)
        assert bool(((lse[i].double() - want).abs() <= mass.reshape(H) + 8 * U * want.abs() + 4 * U).all())
    return got


def _tokens(b, i, where):
    """(pages, offsets) of the tokens of sequence i where `where` (of a token's number) is true."""
    t = torch.tensor([t for t in range(b.sizes[i]) if where(t)], device=DEV)
    P = b.cache[0].shape[2]
    return b.pages[i].long()[t // P], t % P


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [10, 20, 24, 31, 34, 38, 42, 60, 100])
def test_a_far_larger_value_of_no_weight_hides_nothing(power, dtype):
    for heads, kv_heads, dim in ((8, 2, 128), (3, 1, 64), (2, 1, 256)):
        b = Batch([700, 300, 40, 3000], heads, kv_heads, dim, 16, dtype)
        b.q[..., 0] = 16
        b.cache[0][..., 0] = 0
        for i, t in ((0, 5), (0, 650), (1, 299), (2, 0), (3, 1500)):
            at = _tokens(b, i, lambda x: x == t)
            b.cache[0][at[0], :, at[1]] = 0
            b.cache[0][at[0], :, at[1], 0] = -127
            b.cache[1][at[0], :, at[1]] = 1.0           # scores of 16 * 127 / 16 and less below the others
            b.cache[3][at[0], :, at[1]] = 0.02 * 2.0 ** power
        _check(b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [30, 36, 40, 70, 90, 110])
def test_rows_of_zeros_keep_their_weight_beside_large_values(power, dtype):
    """Equal scores: the rows of zeros, whose scale is the least there is, count as much as the others,
    be they in a tile before, in another wave's, or in another piece."""
    for first in (32, 128, 256, 2000):
        b = Batch([first + 32, first + 200, 2 * first + 5000], 4, 2, 128, 16, dtype)
        b.q.zero_()
        for i in range(3):
            at = _tokens(b, i, lambda t: t < first)
            b.cache[2][at[0], :, at[1]] = 0
            b.cache[3][at[0], :, at[1]] = 2.0 ** -126
            at = _tokens(b, i, lambda t: t >= first)
            b.cache[3][at[0], :, at[1]] = 2.0 ** power
        _check(b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [-105, -60, -39, -33, 92, 119])
def test_values_that_are_all_tiny_or_huge(power, dtype):
    b = Batch([700, 1, 40, 5000], 8, 2, 128, 16, dtype)
    b.cache[3].mul_(2.0 ** power)
    _check(b)


@pytest.mark.parametrize("dtype,power", [(torch.float16, 10), (torch.float16, 20)] +
                         [(t, p) for t in TYPES[1:] for p in (10, 20, 32, 40, 60, 100)])
def test_a_querys_large_column_hides_no_other(dtype, power):
    """The keys are 0 where the query is large, and its other columns are 2^-power of that."""
    for heads, kv_heads, dim in ((8, 2, 128), (3, 1, 40), (2, 1, 256)):
        b = Batch([700, 300, 40, 3000], heads, kv_heads, dim, 16, dtype)
        b.q.copy_(b.q.double() * 2.0 ** -power)
        b.q[..., 3] = 1.5
        b.cache[0][..., 3] = 0
        for sign in (1, -1):
            _check(b, scale=sign * dim ** -0.5 * 2.0 ** power)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (3, 1, 64), (2, 1, 256), (5, 1, 33)])
def test_queries_of_32_bits_count_with_all_of_them(heads, kv_heads, dim):
    _check(Batch([700, 1, 300, 40, 3000], heads, kv_heads, dim, 16, torch.float32))


FAR_SCALES = [(t, *powers) for t in TYPES[1:] for powers in ((104, 30, -126), (126, 0, -120), (-146, 16, 126), (-130, 0, 126), (-60, -60, 116))]


@pytest.mark.parametrize("dtype,scale,query,key", FAR_SCALES + [(torch.float16, 118, -10, -108), (torch.float16, -140, 10, 126)])
def test_scales_far_from_one(dtype, scale, query, key):
    """Scores of some units, by a scale, query and keys of these powers of two; scores of 0 among them."""
    b = Batch([700, 1, 40, 3000], 4, 2, 128, 16, dtype)
    g = torch.Generator(device=DEV).manual_seed(2)
    b.q.zero_()
    b.q[..., 5] = (1.5 + torch.rand(b.q.shape[:2], generator=g, device=DEV) / 2).to(dtype) * 2.0 ** query
    most = max(1, min(127, int(2.0 ** -(scale + query + key))))
    b.cache[0].copy_(torch.randint(-most, most + 1, b.cache[0].shape, generator=g, device=DEV))
    b.cache[1][b.cache[1].isfinite()] = 2.0 ** key
    for sign in (1, -1):
        _check(b, scale=sign * 1.25 * 2.0 ** scale if scale < 118 else sign * 2.0 ** scale)


def test_scales_without_scores_are_refused():
    b = Batch([5], 4, 2, 64, 16, torch.float16)
    for scale in (2.0 ** 119, -2.0 ** 119, 2.0 ** 127, math.inf):
        with pytest.raises(A.RidgeAttentionError, match="scale"):
            A.attend(b.q, b.cache, b.pages, b.lengths, scale=scale)
    A.attend(b.q.bfloat16(), b.cache, b.pages, b.lengths, scale=2.0 ** 119)
    with pytest.raises(A.RidgeAttentionError, match="scale"):
        A.attend(b.q.bfloat16(), b.cache, b.pages, b.lengths, scale=2.0 ** 127)
