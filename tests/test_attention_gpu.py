"""The operators around the 8-bit cache on the GPU against 64-bit references.

Tolerances. u = 2^-24 is half a unit of f32.
norm_rope: a head's sum of squares adds at most 16 values in a lane and 6 times over lanes, each
addition one rounding; its root halves that, and the mean, eps, the root, the quotient and two
products add one each, a turned value two more: (22 / 2 + 8) u of the magnitudes that are
added, and half a unit of the type.
Rows: the bits of ridge_amd.int8's, which its own tests hold against 64 bits; values read back are
one f32 product, rounded once.
attend: a score is a sum of D products, at most D + 6 roundings of the sum of their magnitudes
(the query's split into 16-bit parts, where it is f32, leaves 2^-22 of it); as the exponent of p
it carries that as a relative error, with 4 u of its own size by the scales, the base's change and the
maximum's subtraction. p carries 4 u more and 2^-21 of its split. Sums over n tokens add at most n
roundings. out's numerator and denominator each carry all that, relative to the sum of |p v|. The
split is of p times the value's scale, relative to the largest p and a power of two within twice
the largest scale S, and lifted by 2^15: its first part of 16 bits is off by 2^-12 of itself or by
2^-25, half of the least step of float16, and the second part by as much of what is left. So a p
however small is off by at most 2^-40 in units of at most 2 S, 2^-39 S |q_t| of the value's whole
numbers q_t (a p that f32 has no number for, below 2^-126, is off by itself, which is less).
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from ridge_amd import attention as A  # noqa: E402
from ridge_amd import int8 as I  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]
HALF_UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    A.lib()
    yield
    torch.cuda.synchronize()


def _randn(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(shape, generator=g, device=DEV)
    x[..., ::17] *= 5
    return x.to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _close(got, want, slack, dtype):
    """got (of dtype) against want in 64 bits, whose f32 value carries `slack`."""
    error = (got.double() - want).abs()
    limit = slack + HALF_UNIT[dtype] * (want.abs() + slack) + LEAST[dtype]
    assert got.dtype == dtype and bool((error <= limit).all()), \
        "%g of the tolerance" % float((error / limit).nan_to_num(nan=math.inf).max())


# ---------------------------------------------------------------------------- norm_rope

def _turned(x, weight, table, positions, sections, interleaved, eps):
    """(norm and rotation in 64 bits, the magnitudes that each value is a sum of)."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(dim=2, keepdim=True) + eps).sqrt() * weight.double()
    pairs = table.shape[1] // 2
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=DEV)
    row = positions.reshape(len(x), -1).long()[:, axis]
    p = torch.arange(pairs, device=DEV)
    c, s = table.double()[row, p][:, None], table.double()[row, pairs + p][:, None]
    one, two = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    z, most = y.clone(), y.abs()
    z[..., one], z[..., two] = y[..., one] * c - y[..., two] * s, y[..., two] * c + y[..., one] * s
    most[..., one], most[..., two] = ((y[..., one] * c).abs() + (y[..., two] * s).abs(),
                                      (y[..., two] * c).abs() + (y[..., one] * s).abs())
    return z, most


def _check_turn(q, k, got, q_weight=None, k_weight=None, table=None, positions=None, sections=None, interleaved=False,
                eps=1e-6):
    for x, y, w in ((q, got[0], q_weight), (k, got[1], k_weight)):
        want, most = _turned(x, w, table, positions, sections or [table.shape[1] // 2], interleaved, eps)
        _close(y, want, 19 * U * most, x.dtype)


# Columns and pairs: whole vectors, the ends of each number of lanes, odd ones.
WIDTHS = [(128, 64), (64, 32), (256, 128), (80, 40), (96, 48), (16, 8), (128, 32), (192, 8), (112, 24), (2, 1), (3, 1),
          (65, 32), (255, 127), (130, 65), (72, 20), (254, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", WIDTHS)
def test_norm_rope(dim, pairs, interleaved, dtype):
    table = A.rope_table(3001, 2 * pairs)
    for tokens, heads, kv_heads in ((1, 5, 2), (37, 32, 8), (3, 1, 0)):
        q, k = _randn((tokens, heads, dim), dtype, dim), _randn((tokens, kv_heads, dim), dtype, dim + 1)
        positions = _ints([(i * 977 + 5) % 3001 for i in range(tokens)])
        for weight in (None, dtype, torch.float32):
            w = {} if weight is None else {"q_weight": _randn((dim,), weight, 3), "k_weight": _randn((dim,), weight, 4)}
            got = A.norm_rope(q, k, table, positions, interleaved=interleaved, **w)
            _check_turn(q, k, got, table=table, positions=positions, interleaved=interleaved, **w)


@pytest.mark.parametrize("sections", [(16, 24, 24), (64, 0, 0), (0, 0, 64), (1, 60, 3), (8, 8, 8, 40), (32, 32)])
def test_axes(sections):
    table = A.rope_table(500, 128)
    q, k = _randn((19, 4, 128), torch.float16, 1), _randn((19, 2, 128), torch.float16, 2)
    positions = _ints([[(i * 31 + a * 7) % 500 for a in range(len(sections))] for i in range(19)])
    for interleaved in (False, True):
        got = A.norm_rope(q, k, table, positions, sections=sections, interleaved=interleaved)
        _check_turn(q, k, got, table=table, positions=positions, sections=sections, interleaved=interleaved)


def test_norm_of_one_of_them():
    table, positions = A.rope_table(50, 64), _ints([3, 4, 5])
    q, k, w = _randn((3, 4, 64), torch.float16, 1), _randn((3, 2, 64), torch.float16, 2), _randn((64,), torch.float16, 3)
    for weights in ({"q_weight": w}, {"k_weight": w}):
        _check_turn(q, k, A.norm_rope(q, k, table, positions, **weights), table=table, positions=positions, **weights)


@pytest.mark.parametrize("dim,pairs", [(128, 64), (128, 16), (65, 20)])
def test_norm_rope_of_views_in_place_and_beside(dim, pairs):
    table, positions = A.rope_table(99, 2 * pairs), _ints([7, 0, 98, 13])
    w = _randn((dim,), torch.bfloat16, 5)
    qkv = _randn((4, 3, 8 * dim + 7), torch.bfloat16, 1)[:, 1, 3:3 + 8 * dim].view(4, 8, dim)   # odd offsets and strides
    q, k = qkv[:, :5], qkv[:, 5:7]
    want = A.norm_rope(q.contiguous(), k.contiguous(), table, positions, q_weight=w, k_weight=w)
    # Heads before tokens, into columns of one buffer.
    out = torch.zeros((7, 4, 2 * dim), dtype=torch.bfloat16, device=DEV)
    to = out[:5, :, :dim].transpose(0, 1), out[5:, :, dim:].transpose(0, 1)
    got = A.norm_rope(q, k, table, positions, q_weight=w, k_weight=w, q_out=to[0], k_out=to[1])
    assert got[0] is to[0] and got[1] is to[1]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert float(out[:5, :, dim:].abs().max()) == 0 and float(out[5:, :, :dim].abs().max()) == 0
    v = qkv[:, 7:].clone()
    got = A.norm_rope(q, k, table, positions, q_weight=w, k_weight=w, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 7:], v)


def test_a_token_does_not_depend_on_the_others():
    table = A.rope_table(4000, 128)
    w = _randn((128,), torch.float16, 5)
    q, k = _randn((9000, 6, 128), torch.float16, 1), _randn((9000, 2, 128), torch.float16, 2)
    positions = (torch.arange(9000, device=DEV) % 4000).int()
    many = A.norm_rope(q, k, table, positions, q_weight=w, k_weight=w)
    for t in (0, 4500, 8999):
        one = A.norm_rope(q[t:t + 1], k[t:t + 1], table, positions[t:t + 1], q_weight=w, k_weight=w)
        assert torch.equal(one[0][0], many[0][t]) and torch.equal(one[1][0], many[1][t])


def test_positions_outside_the_table_make_nans_of_what_they_turn():
    table = A.rope_table(10, 64)
    q = _randn((4, 3, 96), torch.float16, 1)
    got, _ = A.norm_rope(q, q[:, :0], table, _ints([9, 10, -1, 2 ** 31 - 1]))
    assert bool(got[0].isfinite().all())
    assert bool(got[1:, :, :64].isnan().all()) and torch.equal(got[:, :, 64:], q[:, :, 64:])
    got, _ = A.norm_rope(q, q[:, :0], table, _ints([[9, 10]] * 4), sections=(20, 12))
    assert bool(got[:, :, :20].isfinite().all()) and bool(got[:, :, 20:32].isnan().all())


def test_values_that_are_not_numbers_stay_in_their_head_or_pair():
    table = A.rope_table(10, 64)
    w = torch.ones(96, device=DEV)
    for dim in (96, 95):
        x = _randn((1, 4, dim), torch.float32, 1)
        x[0, 1, 5], x[0, 2, 90], x[0, 3, 70] = math.nan, math.inf, 3e30
        none = x[:, :0]
        plain = A.norm_rope(x, none, table, _ints([3]))[0].isfinite()
        assert bool(plain[0, 0].all()) and bool(plain[0, 3].all())
        assert (~plain[0, 1]).nonzero().flatten().tolist() == [5, 37] and (~plain[0, 2]).nonzero().flatten().tolist() == [90]
        normed = A.norm_rope(x, none, table, _ints([3]), q_weight=w[:dim])[0]
        # A sum of squares past the range of f32 is not silent either.
        assert bool(normed[0, 0].isfinite().all()) and bool(normed[0, 1:].isnan().all())


def test_heads_of_zeros():
    table = A.rope_table(10, 64)
    x = torch.zeros((2, 2, 64), dtype=torch.float16, device=DEV)
    got = A.norm_rope(x, x, table, _ints([1, 2]), q_weight=torch.ones(64, device=DEV), k_weight=torch.ones(64, device=DEV))
    assert float(got[0].abs().max()) == 0 and float(got[1].abs().max()) == 0


# ---------------------------------------------------------------------------- the cache

def _filled(pages, page_size, heads, dim, value=77):
    cache = A.empty_cache(pages, page_size, heads, dim)
    for t in cache:
        t.fill_(value)
    return cache


def _at(cache, slots):
    """The cache's rows and scales at slots: (k, k_scale, v, v_scale) with tokens in front."""
    P = cache[0].shape[2]
    slots = slots.long()
    return tuple(t[slots // P, :, slots % P] for t in cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 8, 9, 16, 64, 65, 72, 127, 128, 129, 200, 256])
@pytest.mark.parametrize("page_size", [16, 48])
def test_write_and_read(page_size, dim, dtype):
    for tokens, heads in ((1, 1), (5, 3), (130, 8)):
        cache = _filled(tokens // page_size + 2, page_size, heads, dim)
        before = [t.clone() for t in cache]
        slots = torch.randperm(cache[0].shape[0] * page_size, device=DEV)[:tokens].int()
        k, v = _randn((tokens, heads, dim), dtype, dim), _randn((tokens, heads, dim), dtype, dim + 1)
        assert A.write_cache(cache, slots, k, v) is cache
        got = _at(cache, slots)
        for x, q, scale in ((k, *got[:2]), (v, *got[2:])):
            want = I.quantize(x.reshape(-1, dim).contiguous())
            assert torch.equal(q.reshape(-1, dim), want[0]) and torch.equal(scale.reshape(-1), want[1])
        for out in (torch.float16, torch.bfloat16, torch.float32):
            for x, q, scale in zip(A.read_cache(cache, slots, dtype=out), got[::2], got[1::2]):
                assert x.dtype == out and torch.equal(x, (q.float() * scale[..., None]).to(out))
        # Nothing else was written.
        here = torch.zeros(cache[0].shape[0] * page_size, dtype=torch.bool, device=DEV)
        here[slots.long()] = True
        here = here.view(-1, 1, page_size)
        for now, then in zip(cache, before):
            mask = here.expand(-1, heads, -1)
            assert torch.equal(now[~mask], then[~mask])


def test_padding_and_slots_outside():
    cache = _filled(2, 16, 2, 64)
    k = _randn((5, 2, 64), torch.float16, 1)
    slots = _ints([-1, 31, 32, -2 ** 31, 2 ** 31 - 1])
    A.write_cache(cache, slots, k, k)
    assert torch.equal(cache[0][1, :, 15], I.quantize(k[1])[0])
    for t in cache:
        t = t.clone()
        t[1, :, 15] = 77
        assert bool((t == 77).all())
    x, _ = A.read_cache(cache, slots)
    assert float(x[0].abs().max()) == 0 and float(x[3].abs().max()) == 0
    assert bool(x[2].isnan().all()) and bool(x[4].isnan().all()) and bool(x[1].isfinite().all())
    out = torch.full((5, 2, 64), 3.0, dtype=torch.float16, device=DEV), torch.zeros((5, 2, 64), dtype=torch.float16, device=DEV)
    assert A.read_cache(cache, slots, out=out)[0] is out[0]


def test_rows_of_zeros_tiny_values_and_none_numbers():
    cache = _filled(1, 16, 1, 128)
    x = torch.zeros((4, 1, 128), device=DEV)
    x[1, 0, :3] = torch.tensor([1e-42, -2e-42, 3e-42], device=DEV)
    x[2, 0, 5], x[3, 0, 5] = math.nan, -math.inf
    A.write_cache(cache, _ints([0, 1, 2, 3]), x, x)
    want = I.quantize(x[:, 0])
    assert torch.equal(cache[0][0, 0, :2], want[0][:2]) and torch.equal(cache[1][0, 0, :2], want[1][:2])
    assert not bool(cache[1][0, 0, 2:4].isfinite().any())
    assert not bool(A.read_cache(cache, _ints([2, 3]), dtype=torch.float32)[0].isfinite().any())


def test_rows_of_every_magnitude_have_quantizes_bits():
    g = torch.Generator(device=DEV).manual_seed(3)
    power = torch.arange(-149, 128, device=DEV).repeat_interleave(8)
    x = (torch.rand((len(power), 2, 64), generator=g, device=DEV) * 2 - 1) * torch.ldexp(torch.ones((), device=DEV), power // 2)[:, None, None]
    x = x * torch.ldexp(torch.ones((), device=DEV), power - power // 2)[:, None, None]
    x[::2, :, 0] *= 2   # and a largest value that may be any
    x[::5, :, 1] = x[::5, :, 0] / 2
    x = torch.where(x.isfinite(), x, torch.ones_like(x))
    cache = A.empty_cache(len(power) // 16 + 1, 16, 2, 64)
    slots = torch.arange(len(power), device=DEV).int()
    A.write_cache(cache, slots, x, x.flip(2))
    got = _at(cache, slots)
    for rows, q, scale in ((x, *got[:2]), (x.flip(2), *got[2:])):
        want = I.quantize(rows.reshape(-1, 64))
        assert torch.equal(q.reshape(-1, 64), want[0]) and torch.equal(scale.reshape(-1), want[1])


def _strided_caches(pages, page_size, heads, dim):
    """The same cache laid out in other orders: heads behind tokens, k and v between each other, pages apart."""
    wide = (dim + 15) // 16 * 16
    a = torch.zeros((pages, page_size, 2, heads, wide + 16), dtype=torch.int8, device=DEV)
    s = torch.zeros((2, heads, pages + 1, 2 * page_size), device=DEV)
    yield (a[:, :, 0, :, :dim].transpose(1, 2), s[0, :, 1:, :page_size].transpose(0, 1),
           a[:, :, 1, :, :dim].transpose(1, 2), s[1, :, 1:, :page_size].transpose(0, 1))
    b = torch.zeros((heads, 2, pages, page_size, wide), dtype=torch.int8, device=DEV)
    t = torch.zeros((pages, 2, heads, page_size), device=DEV)
    yield (b[:, 0, ..., :dim].transpose(0, 1), t[:, 0], b[:, 1, ..., :dim].transpose(0, 1), t[:, 1])


@pytest.mark.parametrize("dim", [64, 72, 128])
def test_caches_in_other_orders(dim):
    k, v = _randn((70, 3, dim), torch.float16, 1), _randn((70, 3, dim), torch.float16, 2)
    slots = torch.randperm(6 * 16, device=DEV)[:70].int()
    q = _randn((2, 6, dim), torch.float16, 3)
    pages, lengths = _ints([[5, 0, 2], [1, 3, 4]]), _ints([33, 48])
    plain = _filled(6, 16, 3, dim, 0)
    A.write_cache(plain, slots, k, v)
    want = A.read_cache(plain, slots), A.attend(q, plain, pages, lengths)
    for cache in _strided_caches(6, 16, 3, dim):
        A.write_cache(cache, slots, k, v)
        for a, b in zip(A.read_cache(cache, slots), want[0]):
            assert torch.equal(a, b)
        assert torch.equal(A.attend(q, cache, pages, lengths), want[1])


# ---------------------------------------------------------------------------- attend

class Batch:
    """Sequences of the given lengths in a cache whose other rows are full of what must not be read."""

    def __init__(self, lengths, heads, kv_heads, dim, page_size, dtype, seed=1, spare=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        held = [-(-n // page_size) for n in lengths]
        total = sum(held) + spare
        self.cache = A.empty_cache(total, page_size, kv_heads, dim)
        order = torch.randperm(total, generator=g, device=DEV).int()
        self.pages = torch.full((len(lengths), max(held + [1])), -7, dtype=torch.int32, device=DEV)
        self.lengths, self.sizes = _ints(lengths), lengths
        at = 0
        used = torch.zeros((total, page_size), dtype=torch.bool, device=DEV)
        for b, n in enumerate(held):
            self.pages[b, :n] = order[at:at + n]
            used[order[at:at + n].long()] = True
            if lengths[b] % page_size:
                used[order[at + n - 1].long(), lengths[b] % page_size:] = False
            at += n
        for rows, scale in (self.cache[:2], self.cache[2:]):
            rows.copy_(torch.randn(rows.shape, generator=g, device=DEV).mul_(40).round_().clamp_(-127, 127))
            scale.copy_(torch.rand(scale.shape, generator=g, device=DEV) * 0.02 + 0.01)
            scale.masked_fill_(~used[:, None], math.nan)
        self.q = (torch.randn((len(lengths), heads, dim), generator=g, device=DEV) * 1.5).to(dtype)

    def rows(self, b, window=None):
        """(k, v) [heads, tokens, dim] of the sequence, in 64 bits."""
        n, P = self.sizes[b], self.cache[0].shape[2]
        t = torch.arange(max(0, n - (window or n)), n, device=DEV)
        page, at = self.pages[b].long()[t // P], t % P
        scale = self.cache[3][page, :, at].double()[..., None]
        self.least = scale.amax(dim=0, keepdim=True).transpose(0, 1) * 2.0 ** -39 if len(t) else None
        self.whole = self.cache[2][page, :, at].double().abs().transpose(0, 1)
        return [(r[page, :, at].double() * s[page, :, at].double()[..., None]).transpose(0, 1)
                for r, s in (self.cache[:2], self.cache[2:])]

    def exact(self, scale=None, window=None):
        """(out, lse, what out's f32 value may be off by, and lse's)."""
        B, H, D = self.q.shape
        scale = D ** -0.5 if scale is None else scale
        out, lse = torch.zeros((B, H, D), dtype=torch.float64, device=DEV), torch.full((B, H), -math.inf, dtype=torch.float64, device=DEV)
        slack, lse_slack = torch.zeros_like(out), torch.zeros((B, H), dtype=torch.float64, device=DEV)
        for b in range(B):
            k, v = self.rows(b, window)
            n = k.shape[1]
            if n == 0:
                continue
            KV = k.shape[0]
            q = self.q[b].double().reshape(KV, H // KV, D)
            s = q @ k.transpose(1, 2).contiguous() * scale
            most = q.abs() @ k.abs().transpose(1, 2).contiguous() * abs(scale)
            p = torch.softmax(s, dim=2)
            off = (D + 6) * U * most + (2.0 ** -22 * most if self.q.dtype == torch.float32 else 0)
            off = off + 4 * U * (s.abs() + s.amax(dim=2, keepdim=True).abs()) + 4 * U + 2.0 ** -21 + n * U
            out[b] = (p @ v).reshape(H, D)
            # Each p with its own relative error; the denominator's is their mean.
            slack[b] = ((p * off) @ v.abs() + (p * off).sum(dim=2, keepdim=True) * (p @ v.abs())
                        + self.least * self.whole.sum(dim=1, keepdim=True)).reshape(H, D)
            lse[b] = torch.logsumexp(s, dim=2).reshape(H)
            lse_slack[b] = ((p * off).sum(dim=2) + 4 * U * torch.logsumexp(s, dim=2).abs() + 4 * U).reshape(H)
        return out, lse, slack, lse_slack

    def check(self, scale=None, window=None):
        lse = torch.empty(self.q.shape[:2], device=DEV)
        got = A.attend(self.q, self.cache, self.pages, self.lengths, scale=scale, window=window, lse_out=lse)
        out, want, slack, lse_slack = self.exact(scale, window)
        _close(got, out, slack, self.q.dtype)
        empty = want == -math.inf
        assert torch.equal(lse == -math.inf, empty) and float(got[empty].abs().sum()) == 0
        assert bool(((lse.double() - want).abs()[~empty] <= lse_slack[~empty]).all())
        assert torch.equal(A.attend(self.q, self.cache, self.pages, self.lengths, scale=scale, window=window), got)
        return got, lse


LENGTHS = [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 511, 512, 513, 777, 1024,
           1025, 1600]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (16, 1, 256), (7, 1, 80), (3, 3, 72), (34, 2, 96),
                                                (5, 1, 1), (6, 2, 200), (71, 1, 64), (1, 1, 128), (32, 2, 33)])
def test_attend(heads, kv_heads, dim, dtype):
    Batch(LENGTHS, heads, kv_heads, dim, 16, dtype).check()


@pytest.mark.parametrize("page_size", [16, 32, 48, 80, 256, 1024])
def test_pages_of_any_size(page_size):
    Batch(LENGTHS, 8, 2, 64, page_size, torch.float16).check()


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 33, 100, 256, 500, 1599, 1600, 1601, 2 ** 40])
def test_windows(window):
    b = Batch(LENGTHS, 8, 2, 64, 16, torch.bfloat16)
    # What lies before the window must not be read either.
    held = b.pages.tolist()
    for i, n in enumerate(b.sizes):
        for t in range(max(0, n - window)):
            page, at = held[i][t // 16], t % 16
            if t % 16 == 0 and t + 16 <= n - window:
                b.pages[i, t // 16] = 2 ** 31 - 1
            b.cache[1][page, :, at] = b.cache[3][page, :, at] = math.nan
    b.check(window=window)


@pytest.mark.parametrize("length", [1700, 4095, 4096, 4097, 8192, 10000, 20011, 32768, 32769, 70001])
def test_long_sequences(length):
    Batch([length, 1, length // 3], 8, 2, 128, 64, torch.float16).check()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 3.0])
def test_scales(scale):
    Batch(LENGTHS, 8, 2, 64, 16, torch.float32).check(scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_scale_of_zero_weighs_all_tokens_alike(dtype):
    """Whatever the keys: times a scale of 0 in place of f32's smallest, they would count by some hundredths."""
    b = Batch([300, 1, 700, 0], 8, 2, 128, 16, dtype)
    b.cache[1].mul_(1e38)
    b.check(scale=0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_and_values_of_any_size(dtype):
    """Softmaxes of one token, scores far from zero, values of all magnitudes in one sequence."""
    b = Batch([700, 300, 40], 8, 2, 128, 16, dtype)
    b.q.mul_(30)
    b.check()
    b.cache[1].mul_(1e-3), b.cache[3].mul_(100)
    b.check()
    # One value row of zeros has the least scale there is; another is a thousand times the others.
    b = Batch([700, 300, 40], 8, 2, 128, 16, dtype)
    for i, t in ((0, 5), (0, 650), (1, 299), (2, 0)):
        page = int(b.pages[i, t // 16])
        b.cache[2][page, :, t % 16] = 0
        b.cache[3][page, :, t % 16] = 2.0 ** -126
    page = int(b.pages[0, 20])
    b.cache[3][page, :, 7] *= 1000
    b.check()
    # Queries whose largest column hides the others' size.
    b.q.mul_(1e-4)
    b.q[:, ::2, 3] = 100
    b.check()


def test_a_far_sum_of_small_probabilities_counts():
    # One token in front of many whose probabilities are each below 2^-24 of its own.
    n = 60000
    b = Batch([n], 1, 1, 64, 16, torch.float32)
    b.q.zero_()
    b.q[0, 0, 0] = 1
    rows, scale = b.cache[0], b.cache[1]
    rows.zero_()
    scale[scale.isfinite()] = 1.0
    b.cache[3][b.cache[3].isfinite()] = 1.0
    b.cache[2].fill_(1)
    page = int(b.pages[0, 0])
    rows[page, 0, 0, 0] = 17
    b.cache[2][page, 0, 0] = 0
    out, _ = b.check(scale=1.0)
    want = (n - 1) / (n - 1 + math.exp(17))
    assert abs(float(out[0, 0, 0]) - want) < 1e-4 * want


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_in_the_cache_counts_twice_or_never(dtype):
    """Values that tell each token: uniform probabilities over v_t = 1 at t % dim, whole numbers of tokens."""
    n, dim = 5 * 128 + 77, 128
    b = Batch([n], 4, 1, dim, 16, dtype)
    b.q.zero_()
    b.cache[2].zero_()
    b.cache[3][b.cache[3].isfinite()] = 1.0
    for t in range(n):
        b.cache[2][int(b.pages[0, t // 16]), 0, t % 16, t % dim] = 1
    out = A.attend(b.q, b.cache, b.pages, b.lengths)
    want = torch.tensor([6.0 if d < 77 else 5.0 for d in range(dim)], device=DEV, dtype=torch.float64) / n
    assert bool(((out.double() - want).abs() <= want * (HALF_UNIT[dtype] + 2.0 ** -20)).all())


def _near(got, want):
    """Two results of float16 whose f32 values differ by their cut: one rounding apart at the most."""
    return bool(((got.double() - want.double()).abs() <= want.double().abs() * 2.0 ** -10 + 1e-4 * float(want.abs().max())).all())


def test_lengths_and_pages_outside_the_cache_make_nans_of_their_sequence():
    # The others keep their values, but for what another cut of the batch makes of the last bits.
    b = Batch([100, 600, 40, 64, 90], 8, 2, 64, 16, torch.float16)
    want = A.attend(b.q, b.cache, b.pages, b.lengths)
    lse = torch.empty((5, 8), device=DEV)
    lengths = b.lengths.clone()
    lengths[0], lengths[2] = -1, b.pages.shape[1] * 16 + 1
    got = A.attend(b.q, b.cache, b.pages, lengths, lse_out=lse)
    for i in range(5):
        if i in (0, 2):
            assert bool(got[i].isnan().all()) and bool(lse[i].isnan().all())
        else:
            assert _near(got[i], want[i]) and bool(lse[i].isfinite().all())
    for bad in (-1, b.cache[0].shape[0], 2 ** 31 - 1, -2 ** 31):
        for at in (0, 17, 37):
            pages = b.pages.clone()
            pages[1, at] = bad
            got = A.attend(b.q, b.cache, pages, b.lengths, lse_out=lse)
            assert bool(got[1].isnan().all()) and bool(lse[1].isnan().all())
            for i in (0, 2, 3, 4):
                assert _near(got[i], want[i])
    # Pages behind the length and before the window are not looked at.
    pages = b.pages.clone()
    pages[1, :20] = -1
    assert bool(A.attend(b.q, b.cache, pages, b.lengths, window=100)[1].isfinite().all())


def test_rows_that_are_not_numbers_come_out():
    b = Batch([300, 300], 8, 2, 64, 16, torch.float16)
    want = A.attend(b.q, b.cache, b.pages, b.lengths)
    for part in (1, 3):
        for bad in (math.nan, math.inf):
            cache = tuple(t.clone() for t in b.cache)
            cache[part][int(b.pages[1, 10]), 1, 3] = bad
            got = A.attend(b.q, cache, b.pages, b.lengths)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1, :4], want[1, :4])
            # A key's infinite scale may give a token all of the softmax or nothing of it.
            if part == 3 or math.isnan(bad):
                assert not bool(got[1, 4:].isfinite().all(dim=1).any())
    q = b.q.clone()
    q[1, 2, 5] = math.nan
    got = A.attend(q, b.cache, b.pages, b.lengths)
    assert bool(got[1, 2].isnan().all())
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (20, 1, 64), (6, 6, 80)])
def test_calls_repeat_their_bits_and_short_sequences_keep_theirs(heads, kv_heads, dim):
    b = Batch([3000, 17, 900, 0, 513, 9000] + [256] * 40, heads, kv_heads, dim, 16, torch.float16)
    lse = torch.empty((46, heads), device=DEV)
    many = A.attend(b.q, b.cache, b.pages, b.lengths, lse_out=lse)
    again = torch.empty_like(lse)
    assert torch.equal(A.attend(b.q, b.cache, b.pages, b.lengths, lse_out=again), many) and torch.equal(again, lse)
    # Sequences of up to 512 tokens, in pages for no more: one workgroup each, whatever is beside them.
    few = b.lengths[6:], b.pages[6:, :32]
    some = A.attend(b.q[6:], b.cache, few[1], few[0])
    for i in (0, 39):
        assert torch.equal(A.attend(b.q[6 + i:7 + i], b.cache, few[1][i:i + 1], few[0][i:i + 1])[0], some[i])


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 64), (40, 2, 128), (2, 2, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_batches_of_all_sorts(heads, kv_heads, dim, dtype):
    """Shares of rounds that begin and end anywhere: in the first and the last sequence, between sequences
    of none, several heads a workgroup and several workgroups a head, more sequences than a wave has lanes."""
    for lengths in ([0] * 70 + [700], [5000] + [0] * 3, [600], [129] * 63, [129] * 64, [129] * 65 + [3000],
                    [(i * 389) % 1500 for i in range(150)], [(i * 389) % 2500 for i in range(300)], [1] * 300, [20000, 1, 1, 20000]):
        b = Batch(lengths, heads, kv_heads, dim, 16, dtype)
        if b.pages.shape[1] <= 32:
            b.pages = torch.cat([b.pages, torch.full((len(lengths), 33), -1, dtype=torch.int32, device=DEV)], dim=1)
        b.check()


@pytest.mark.parametrize("width", [1, 130])
def test_more_sequences_than_one_launch_takes(width):
    # All of them on one page; in 130 pages each they share their rounds, in one each has its own.
    n, cache = 66001, _filled(2, 16, 1, 16, 1)
    g = torch.Generator(device=DEV).manual_seed(1)
    cache[0].copy_(torch.randint(-127, 128, cache[0].shape, generator=g, device=DEV))
    cache[2].copy_(torch.randint(-127, 128, cache[2].shape, generator=g, device=DEV))
    cache[1].fill_(0.01), cache[3].fill_(0.02)
    q = torch.randn((n, 2, 16), generator=g, device=DEV).half()
    lengths = torch.randint(0, 17, (n,), generator=g, device=DEV, dtype=torch.int32)
    pages = torch.ones((n, 1), dtype=torch.int32, device=DEV).expand(n, width).contiguous()
    lse = torch.empty((n, 2), device=DEV)
    got = A.attend(q, cache, pages, lengths, lse_out=lse)
    k, v = cache[0][1, 0].double() * cache[1][1, 0].double()[:, None], cache[2][1, 0].double() * cache[3][1, 0].double()[:, None]
    s = q.double() @ k.t() / 4
    s = torch.where(torch.arange(16, device=DEV) < lengths[:, None, None], s, -math.inf)
    want = torch.softmax(s, dim=2).nan_to_num(nan=0.0) @ v
    # 16 products and 16 tokens: 2^-16 of the magnitudes is far more than f32 loses.
    _close(got, want, 2.0 ** -16 * 127 * 0.02, torch.float16)
    exact = torch.logsumexp(s, dim=2)
    assert torch.equal(lse == -math.inf, exact == -math.inf)
    assert float((lse.double() - exact)[lse.isfinite()].abs().max()) < 1e-4


@pytest.mark.parametrize("dim", [64, 80, 33, 256])
def test_queries_and_results_of_any_stride(dim):
    b = Batch([700, 33, 0, 5], 6, 2, dim, 16, torch.bfloat16)
    want = A.attend(b.q, b.cache, b.pages, b.lengths)
    memory = torch.zeros((6, 4, 2 * dim + 3), dtype=torch.bfloat16, device=DEV)
    q, out = memory[..., 1:1 + dim].transpose(0, 1), memory[..., dim + 2:2 * dim + 2].transpose(0, 1)
    q.copy_(b.q)
    pages = torch.full((4, 2 * b.pages.shape[1] + 5), -1, dtype=torch.int32, device=DEV)[:, 3:3 + b.pages.shape[1]]
    pages.copy_(b.pages)
    assert A.attend(q, b.cache, pages, b.lengths, out=out) is out
    assert torch.equal(out, want) and torch.equal(q, b.q)
    assert float(memory[..., 0].abs().max()) == 0 and float(memory[..., dim + 1].abs().max()) == 0


def test_sequences_that_share_their_pages():
    b = Batch([640], 4, 2, 64, 16, torch.float16)
    pages, lengths = b.pages.expand(3, -1), _ints([640, 100, 639])
    q = _randn((3, 4, 64), torch.float16, 8)
    got = A.attend(q, b.cache, pages, lengths)
    for i, n in enumerate((640, 100, 639)):
        assert _near(got[i], A.attend(q[i:i + 1], b.cache, b.pages, _ints([n]))[0])


def test_no_sequences_and_no_pages():
    b = Batch([5, 0], 4, 2, 64, 16, torch.float16)
    assert A.attend(b.q[:0], b.cache, b.pages[:0], b.lengths[:0]).shape == (0, 4, 64)
    lse = torch.empty((2, 4), device=DEV)
    out = A.attend(b.q, b.cache, b.pages[:, :0], _ints([0, 1]), lse_out=lse)
    assert float(out[0].abs().max()) == 0 and bool((lse[0] == -math.inf).all())
    assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all())


def test_offsets_past_32_bits():
    # 5.2 GB of rows each; the sequence lies in the last pages.
    pages, page_size, heads, dim = 40000, 64, 8, 256
    cache = A.empty_cache(pages, page_size, heads, dim)
    assert cache[0].numel() > 2 ** 32
    n = 300
    slots = torch.arange(n, device=DEV).int() + (pages - 5) * page_size
    k, v = _randn((n, heads, dim), torch.float16, 1), _randn((n, heads, dim), torch.float16, 2)
    A.write_cache(cache, slots, k, v)
    got = A.read_cache(cache, slots)
    small = A.empty_cache(5, page_size, heads, dim)
    A.write_cache(small, torch.arange(n, device=DEV).int(), k, v)
    for a, b in zip(got, A.read_cache(small, torch.arange(n, device=DEV).int())):
        assert torch.equal(a, b)
    q = _randn((1, 16, dim), torch.float16, 3)
    lengths = _ints([n])
    far = A.attend(q, cache, _ints([list(range(pages - 5, pages))]), lengths)
    assert torch.equal(far, A.attend(q, small, _ints([[0, 1, 2, 3, 4]]), lengths))
    # Heads far apart: 2^32 bytes and more between a view's tokens.
    wide = torch.empty((3, 1 << 31), dtype=torch.float16, device=DEV)[:, :4 * 64].view(3, 4, 64)
    wide.copy_(_randn((3, 4, 64), torch.float16, 4))
    table, positions = A.rope_table(20, 64), _ints([1, 2, 3])
    near = A.norm_rope(wide.contiguous(), wide[:, :0], table, positions)[0]
    assert torch.equal(A.norm_rope(wide, wide[:, :0], table, positions, q_out=wide)[0], near)
