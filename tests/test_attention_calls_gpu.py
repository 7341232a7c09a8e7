"""What the calls around the 8-bit cache do with the tensors and streams that they are given, and a
run of them together."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from ridge_amd import attention as A  # noqa: E402
from ridge_amd import int8 as I  # noqa: E402
from test_attention_gpu import DEV, Batch, _filled, _ints, _randn  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    A.lib()
    yield
    torch.cuda.synchronize()


def _operands(dtype=torch.float16):
    """What every call takes: 4 tokens of 4 query and 2 key heads of 64."""
    o = {"q": _randn((4, 4, 64), dtype, 1), "k": _randn((4, 2, 64), dtype, 2), "v": _randn((4, 2, 64), dtype, 3),
         "w": _randn((64,), dtype, 4), "table": A.rope_table(50, 64), "positions": _ints([3, 1, 4, 1]),
         "cache": _filled(3, 16, 2, 64, 1), "slots": _ints([0, 17, 33, 34]), "pages": _ints([[0, 1], [2, 0], [1, 1], [2, 1]]),
         "lengths": _ints([20, 32, 1, 16])}
    return o


def _norm_rope(o, **changes):
    o = dict(o, **changes)
    return A.norm_rope(o["q"], o["k"], o["table"], o["positions"], q_weight=o["w"], k_weight=o["w"],
                       q_out=o.get("q_out"), k_out=o.get("k_out"), stream=o.get("stream"))


def _write(o, **changes):
    o = dict(o, **changes)
    return A.write_cache(o["cache"], o["slots"], o["k"], o["v"], stream=o.get("stream"))


def _read(o, **changes):
    o = dict(o, **changes)
    return A.read_cache(o["cache"], o["slots"], out=o.get("out"), dtype=o.get("dtype"), stream=o.get("stream"))


def _attend(o, **changes):
    o = dict(o, **changes)
    return A.attend(o["q"], o["cache"], o["pages"], o["lengths"], lse_out=o.get("lse"), out=o.get("out"),
                    window=o.get("window"), scale=o.get("scale"), stream=o.get("stream"))


def _with(cache, index, tensor):
    return cache[:index] + (tensor,) + cache[index + 1:]


def test_wrong_arguments_are_refused():
    o = _operands()
    cache, q, k = o["cache"], o["q"], o["k"]
    f64, ints = q.double(), o["positions"]
    wide = torch.zeros((4, 1, 320), dtype=torch.float16, device=DEV)
    refused = {
        "q of 64 bits": lambda: _norm_rope(o, q=f64), "k of another type": lambda: _norm_rope(o, k=k.float()),
        "k of other tokens": lambda: _norm_rope(o, k=k[:3]), "k of another width": lambda: _norm_rope(o, k=k[..., :32]),
        "q in two dimensions": lambda: _norm_rope(o, q=q[0]), "columns apart": lambda: _norm_rope(o, q=q[..., ::2], k=k[..., ::2]),
        "320 columns": lambda: _norm_rope(o, q=wide, k=wide), "overlapping heads": lambda: _norm_rope(o, q=q[:1].expand(4, 4, 64)),
        "a table of 16 bits": lambda: _norm_rope(o, table=o["table"].half()), "odd columns of a table": lambda: _norm_rope(o, table=o["table"][:, :33]),
        "a wide table": lambda: _norm_rope(o, table=A.rope_table(50, 66)), "no rows": lambda: _norm_rope(o, table=o["table"][:0]),
        "table on the host": lambda: _norm_rope(o, table=o["table"].cpu()),
        "positions of 64 bits": lambda: _norm_rope(o, positions=ints.long()), "few positions": lambda: _norm_rope(o, positions=ints[:3]),
        "five axes": lambda: _norm_rope(o, positions=ints[:, None].expand(4, 5).contiguous()),
        "no sections": lambda: _norm_rope(o, positions=ints[:, None].expand(4, 2).contiguous()),
        "sections of 31": lambda: A.norm_rope(q, k, o["table"], ints, sections=[31]),
        "sections of 33": lambda: A.norm_rope(q, k, o["table"], ints, sections=[33]),
        "negative sections": lambda: A.norm_rope(q, k, o["table"], ints[:, None].expand(4, 2).contiguous(), sections=[33, -1]),
        "two sections of one axis": lambda: A.norm_rope(q, k, o["table"], ints, sections=[16, 16]),
        "a short weight": lambda: _norm_rope(o, w=o["w"][:63]), "a weight of another type": lambda: _norm_rope(o, w=o["w"].bfloat16()),
        "two types of weights": lambda: A.norm_rope(q, k, o["table"], ints, q_weight=o["w"], k_weight=o["w"].float()),
        "eps of 0": lambda: A.norm_rope(q, k, o["table"], ints, eps=0.0), "eps of nan": lambda: A.norm_rope(q, k, o["table"], ints, eps=math.nan),
        "another q_out": lambda: _norm_rope(o, q_out=k.clone()), "k_out of another type": lambda: _norm_rope(o, k_out=k.float()),
        "a cache of three": lambda: _write(o, cache=cache[:3]), "a list": lambda: _write(o, cache=list(cache)),
        "16-bit rows": lambda: _write(o, cache=_with(cache, 0, cache[0].half())),
        "other pages of v": lambda: _write(o, cache=_with(cache, 2, cache[2][:2])),
        "v of other strides": lambda: _write(o, cache=_with(cache, 2, torch.zeros((3, 2, 16, 80), dtype=torch.int8, device=DEV)[..., :64])),
        "k for v": lambda: _write(o, cache=_with(cache, 2, cache[0])),
        "one scale for both": lambda: _write(o, cache=_with(cache, 3, cache[1])),
        "short scales": lambda: _write(o, cache=_with(cache, 1, cache[1][..., :8])), "scales of 64 bits": lambda: _write(o, cache=_with(cache, 3, cache[3].double())),
        "pages of 8": lambda: _write(o, cache=tuple(t[:, :, :8] for t in cache)),
        "no pages": lambda: _write(o, cache=tuple(t[:0] for t in cache)),
        "rows at 8": lambda: _read(o, cache=tuple(t[..., 8:40] if t.dim() == 4 else t for t in cache)),
        "rows 72 apart": lambda: _read(o, cache=tuple(torch.zeros((3, 2, 16, 72), dtype=torch.int8, device=DEV)[..., :64] if t.dim() == 4 else t for t in cache)),
        "pages over each other": lambda: _read(o, cache=tuple(t[:1].expand(3, *t.shape[1:]) for t in cache)),
        "k of other heads": lambda: _write(o, k=q), "v of other tokens": lambda: _write(o, v=k[:2]), "v of another type": lambda: _write(o, v=o["v"].float()),
        "slots of 64 bits": lambda: _write(o, slots=o["slots"].long()), "few slots": lambda: _write(o, slots=o["slots"][:3]),
        "slots apart": lambda: _read(o, slots=torch.zeros(8, dtype=torch.int32, device=DEV)[::2]),
        "reading into integers": lambda: _read(o, dtype=torch.int8), "out of another type": lambda: _read(o, out=(k, o["v"]), dtype=torch.float32),
        "out alone": lambda: _read(o, out=(k,)), "out of q's heads": lambda: _read(o, out=(q, q)),
        "three heads on two": lambda: _attend(o, q=q[:, :3]), "another width": lambda: _attend(o, q=q[..., :32]),
        "q of 8 bits": lambda: _attend(o, q=q.to(torch.int8)), "pages of 64 bits": lambda: _attend(o, pages=o["pages"].long()),
        "pages of three": lambda: _attend(o, pages=o["pages"][:3]), "pages apart": lambda: _attend(o, pages=torch.zeros((4, 4), dtype=torch.int32, device=DEV)[:, ::2]),
        "lengths of three": lambda: _attend(o, lengths=o["lengths"][:3]), "lengths of 64 bits": lambda: _attend(o, lengths=o["lengths"].long()),
        "a window of 0": lambda: _attend(o, window=0), "a negative window": lambda: _attend(o, window=-5),
        "an infinite scale": lambda: _attend(o, scale=math.inf), "a scale of nan": lambda: _attend(o, scale=math.nan),
        "lse of q's type": lambda: _attend(o, lse=torch.zeros((4, 4), dtype=torch.float16, device=DEV)),
        "lse of other heads": lambda: _attend(o, lse=torch.zeros((4, 2), device=DEV)), "lse on the host": lambda: _attend(o, lse=torch.zeros((4, 4))),
        "out of another shape": lambda: _attend(o, out=k.clone()), "lengths on the host": lambda: _attend(o, lengths=o["lengths"].cpu()),
    }
    for name, call in refused.items():
        print(name, flush=True)
        with pytest.raises(A.RidgeAttentionError):
            call()
    with pytest.raises(TypeError):
        A.norm_rope(q, k, o["table"], ints, sections=["a"])


def test_outputs_over_operands_are_refused():
    o = _operands()
    flat = torch.zeros(8192, dtype=torch.float16, device=DEV)
    f32, bytes_, i32 = flat.view(torch.float32), flat.view(torch.int8), flat.view(torch.int32)
    q, k = flat[:1024].view(4, 4, 64), flat[:512].view(4, 2, 64)
    cache = A.empty_cache(1, 16, 2, 64)
    over = (bytes_[:2048].view(1, 2, 16, 64), cache[1], cache[2], cache[3])
    slots, pages = _ints([0, 1, 2, 3]), _ints([[0]] * 4)
    lse = f32[:16].view(4, 4)
    refused = {
        "q_out a row on": lambda: _norm_rope(o, q=q, q_out=flat[256:1280].view(4, 4, 64)),
        "q_out an element on": lambda: _norm_rope(o, q=q, q_out=flat[1:1025].view(4, 4, 64)),
        "q_out in another order": lambda: _norm_rope(o, q=q, q_out=flat[:1024].view(4, 4, 64).transpose(0, 1)),
        "q_out over k": lambda: _norm_rope(o, k=k, q_out=q), "k_out over q": lambda: _norm_rope(o, q=q, k_out=k),
        "both into one": lambda: _norm_rope(o, q_out=q, k_out=k),
        "q_out over the weight": lambda: _norm_rope(o, w=flat[64:128], q_out=q),
        "q_out over the table": lambda: _norm_rope(o, table=f32[:3200].view(50, 64), q_out=q),
        "k_out over the positions": lambda: _norm_rope(o, positions=i32[100:104].zero_(), k_out=k),
        "writing over k": lambda: _write(o, cache=over, slots=slots, k=k), "writing over v": lambda: _write(o, cache=over, slots=slots, v=k),
        "writing over the slots": lambda: _write(o, cache=over, slots=i32[5:9]),
        "reading over the rows": lambda: _read(o, cache=over, slots=slots, out=(k, o["v"])),
        "reading over the slots": lambda: _read(o, slots=i32[:4].zero_(), out=(o["k"], k)),
        "both values into one": lambda: _read(o, out=(k, k)),
        "out over q": lambda: _attend(o, q=q, out=q), "out over the cache": lambda: _attend(o, cache=over, pages=pages, out=q),
        "out over the pages": lambda: _attend(o, pages=i32[:8].zero_().view(4, 2), out=q),
        "out over the lengths": lambda: _attend(o, lengths=i32[8:12].zero_(), out=q),
        "lse over out": lambda: _attend(o, lse=lse, out=q), "lse over q": lambda: _attend(o, lse=lse, q=q),
        "lse over the scales": lambda: _attend(o, cache=_with(cache, 3, f32[:32].view(1, 2, 16)), pages=pages, lse=lse),
        "lse over the lengths": lambda: _attend(o, lengths=i32[8:12].zero_(), lse=lse),
    }
    for name, call in refused.items():
        print(name, flush=True)
        with pytest.raises(A.RidgeAttentionError, match="overlap"):
            call()


def test_gradients_and_tangents_are_refused():
    from torch.autograd import forward_ad
    o = _operands()
    cache, out, lse = o["cache"], torch.zeros_like(o["q"]), torch.zeros((4, 4), device=DEV)
    calls = [
        lambda f: _norm_rope(o, q=f(o["q"])), lambda f: _norm_rope(o, k=f(o["k"])), lambda f: _norm_rope(o, w=f(o["w"])),
        lambda f: _norm_rope(o, table=f(o["table"])), lambda f: _norm_rope(o, q_out=f(out)),
        lambda f: _write(o, k=f(o["k"])), lambda f: _write(o, v=f(o["v"])), lambda f: _write(o, cache=_with(cache, 1, f(cache[1]))),
        lambda f: _read(o, cache=_with(cache, 3, f(cache[3]))), lambda f: _read(o, out=(f(o["k"]), o["v"].clone())),
        lambda f: _attend(o, q=f(o["q"])), lambda f: _attend(o, cache=_with(cache, 1, f(cache[1]))),
        lambda f: _attend(o, out=f(out)), lambda f: _attend(o, lse=f(lse)),
    ]

    def leaf(t):
        return t.clone().requires_grad_()

    def dual(t):
        return forward_ad.make_dual(t.clone(), torch.ones_like(t))
    for i, call in enumerate(calls):
        print("call", i, flush=True)
        with pytest.raises(A.RidgeAttentionError, match="gradient"):
            call(leaf)
        with torch.no_grad():
            call(leaf)
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode, forward_ad.dual_level(), pytest.raises(A.RidgeAttentionError, match="gradient"):
                call(dual)


def test_buffers_that_a_graph_saved_are_not_overwritten_in_silence():
    o = _operands()
    writes = {
        "q_out": ((4, 4, 64), torch.float16, lambda t: _norm_rope(o, q_out=t)),
        "in place": ((4, 2, 64), torch.float16, lambda t: _norm_rope(o, k=t, k_out=t)),
        "scales": ((3, 2, 16), torch.float32, lambda t: _write(o, cache=_with(o["cache"], 3, t))),
        "values": ((4, 2, 64), torch.float16, lambda t: _read(o, out=(t, torch.zeros_like(t)))),
        "out": ((4, 4, 64), torch.float16, lambda t: _attend(o, out=t)),
        "lse": ((4, 4), torch.float32, lambda t: _attend(o, lse=t)),
    }
    for name, (shape, dtype, call) in writes.items():
        print(name, flush=True)
        buffer = torch.ones(shape, dtype=dtype, device=DEV)
        p = torch.ones(shape, dtype=dtype, device=DEV, requires_grad=True)
        loss = (p * buffer).sum()
        with torch.no_grad():
            call(buffer)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    read = {name: t for name, t in o.items() if name != "cache"}
    before = {name: t._version for name, t in read.items()}
    _norm_rope(o), _write(o), _read(o), _attend(o)
    assert {name: t._version for name, t in read.items()} == before
    with torch.inference_mode():
        made = torch.empty_like(o["q"]), A.empty_cache(3, 16, 2, 64)
    _attend(o, out=made[0]), _write(o, cache=made[1])


def test_streams():
    o = _operands()
    _write(o)
    torch.cuda.synchronize()
    want = _norm_rope(o), _read(o), _attend(o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        got = _norm_rope(o, stream=stream), _read(o, stream=stream), _attend(o, stream=stream)
        assert _write(o, stream=stream) is o["cache"]
        side.synchronize()
        for a, b in zip(got[0] + got[1] + (got[2],), want[0] + want[1] + (want[2],)):
            assert torch.equal(a, b)
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    # What a call allocates belongs to its stream: memory that the side stream still writes is not
    # handed to the current one.
    for call in (_norm_rope, _read, _attend):
        with pytest.raises((A.RidgeAttentionError, TypeError, AttributeError)):
            call(o, stream="stream")


def test_two_calls_at_once_do_not_share_anything():
    batches = [Batch([3000, 100, 9000, 0], 8, 2, 64, 16, torch.float16, seed=s) for s in (1, 2)]
    want = [A.attend(b.q, b.cache, b.pages, b.lengths) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                got.append(A.attend(b.q, b.cache, b.pages, b.lengths))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_a_failed_call_of_the_program_is_not_taken_for_this_ones():
    o = _operands()
    hip = ctypes.CDLL("libamdhip64.so")
    try:
        assert hip.hipSetDevice(999) != 0
        _norm_rope(o), _write(o), _read(o), _attend(o)
    finally:
        hip.hipGetLastError()   # cleared: torch's calls would report it


def test_graphs_replay_with_new_values():
    b = Batch([700, 100, 1500, 0, 33], 8, 2, 64, 16, torch.float16, spare=4)
    n, table = len(b.sizes), A.rope_table(2000, 64)
    q, k, v = _randn((n, 8, 64), torch.float16, 1), _randn((n, 2, 64), torch.float16, 2), _randn((n, 2, 64), torch.float16, 3)
    # The last pages are nobody's: new tokens go there, and count nowhere.
    free = sorted(set(range(b.cache[0].shape[0])) - set(int(p) for p in b.pages.flatten()))[0]
    slots = _ints([free * 16 + i for i in range(n)])
    lse = torch.empty((n, 8), device=DEV)

    def run():
        turned = A.norm_rope(q, k, table, b.lengths)
        A.write_cache(b.cache, slots, turned[1], v)
        return turned + A.read_cache(b.cache, slots) + (A.attend(turned[0], b.cache, b.pages, b.lengths, lse_out=lse), lse)
    run()
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run()[:-1])
        graphs.append(graph)
    for i in range(6):
        q.copy_(_randn(q.shape, torch.float16, 10 + i)), v.copy_(_randn(v.shape, torch.float16, 20 + i))
        lengths = _ints([(m * (i + 1)) % (m + 1) for m in b.sizes])
        b.lengths.copy_(lengths)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got, got_lse = [t.clone() for t in results[i % 2]], lse.clone()
        want = run()
        for a, c in zip(got + [got_lse], want):
            assert torch.equal(a, c)


def test_a_prompt_and_then_tokens_one_by_one():
    """Sequences of different prompts, written at once with padding, then grown by a token at a time;
    each step against the keys and values of all tokens in 64 bits, rounded as the cache rounds them."""
    heads, kv_heads, dim, page_size, dtype = 6, 2, 80, 16, torch.float16
    prompts, steps = [5, 33, 16, 1], 20
    g = torch.Generator(device=DEV).manual_seed(5)
    table = A.rope_table(100, 64)
    w = _randn((dim,), dtype, 6)
    n, each = len(prompts), 4
    cache = _filled(n * each, page_size, kv_heads, dim)
    pages = torch.randperm(n * each, generator=g, device=DEV).int().view(n, each)

    def slots_of(b, t):
        return int(pages[b, t // page_size]) * page_size + t % page_size

    def new(tokens):
        return [torch.randn((tokens, h, dim), generator=g, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads)]
    longest = max(prompts)
    held = [[] for _ in prompts]
    q, k, v = new(n * longest)
    positions = _ints([t for _ in prompts for t in range(longest)])
    slots = _ints([slots_of(b, t) if t < prompts[b] else -1 for b in range(n) for t in range(longest)])
    q, k = A.norm_rope(q, k, table, positions, q_weight=w, k_weight=w)
    A.write_cache(cache, slots, k, v)
    for b, m in enumerate(prompts):
        held[b] = [t[b * longest:b * longest + m] for t in (k, v)]
    lengths = list(prompts)
    for _ in range(steps):
        q, k, v = new(n)
        q, k = A.norm_rope(q, k, table, _ints(lengths), q_weight=w, k_weight=w)
        A.write_cache(cache, _ints([slots_of(b, lengths[b]) for b in range(n)]), k, v)
        lengths = [m + 1 for m in lengths]
        got = A.attend(q, cache, pages, _ints(lengths))
        for b in range(n):
            held[b] = [torch.cat([t, x[b:b + 1]]) for t, x in zip(held[b], (k, v))]
            keys, values = ((r.double() * s.double()[:, None]).view(-1, kv_heads, dim).transpose(0, 1)
                            for r, s in (I.quantize(t.reshape(-1, dim)) for t in held[b]))
            p = torch.softmax(q[b].double().view(kv_heads, -1, dim) @ keys.transpose(1, 2).contiguous() * dim ** -0.5, dim=2)
            want = (p @ values).view(heads, dim)
            # f32 sums of 80 products and up to 53 tokens, whose relative error is below 2^-14 of what they add,
            # and the rounding to float16.
            most = (p @ values.abs()).view(heads, dim)
            assert bool(((got[b].double() - want).abs() <= 2.0 ** -14 * most + 2.0 ** -11 * want.abs() + 2.0 ** -24).all())
    # The same prefix read back.
    slots = _ints([slots_of(1, t) for t in range(lengths[1])])
    for x, t in zip(A.read_cache(cache, slots, dtype=torch.float32), held[1]):
        r, s = I.quantize(t.reshape(-1, dim))
        assert torch.equal(x.view(-1, dim), r.float() * s[:, None])


def test_two_parts_of_a_sequence_are_joined_by_their_lse():
    b = Batch([900], 8, 2, 128, 16, torch.float32)
    lse = torch.empty((1, 8), device=DEV)
    whole = A.attend(b.q, b.cache, b.pages, b.lengths, lse_out=lse)
    parts = []
    for first, length in ((0, 320), (20, 580)):
        part = torch.empty((1, 8), device=DEV)
        parts.append((A.attend(b.q, b.cache, b.pages[:, first:], _ints([length]), lse_out=part), part))
    weight = torch.softmax(torch.stack([p[1] for p in parts]), dim=0)
    joined = sum(w[..., None] * p[0] for w, p in zip(weight, parts))
    assert float((joined - whole).abs().max()) < 1e-5 * float(whole.abs().max())
    assert float((torch.logsumexp(torch.stack([p[1] for p in parts]), dim=0) - lse).abs().max()) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_block(dtype):
    from ridge_amd import int8_attention as B
    hidden, heads, kv_heads, dim, sequences, length = 256, 8, 2, 64, 5, 70
    norm_weight, qkv, out, q_weight, k_weight = B.random_block(hidden, heads, kv_heads, dim, dtype, 1)
    table = A.rope_table(length, dim)
    block = B.Int8Attention(norm_weight, qkv, out, heads, kv_heads, table, q_weight, k_weight)
    cache, pages, slots, lengths, every = B.random_cache(sequences, length, kv_heads, dim, 16, dtype, 2)
    x, r = _randn((sequences, hidden), dtype, 3), _randn((sequences, hidden), dtype, 4)
    space = block.workspace(sequences, dtype)
    y, total = block(x, r, cache, lengths - 1, slots, pages, lengths, space)
    assert y.data_ptr() == space["y"].data_ptr() and torch.equal(total, x + r)
    cached = [A.read_cache(cache, every[b, :-1], dtype=torch.float32) for b in range(sequences)]
    want, _, k, v = B.plain_block(x.float(), r.float(), norm_weight.float(), qkv.float(), out.float(), heads, kv_heads, table,
                                  cached, lengths - 1, q_weight.float(), k_weight.float())
    # Rows of 8 bits are off by 0.4% of their largest value: four of them in a row, and the weights.
    assert float((y.float() - want).norm() / want.norm()) < 0.05
    for new, at in ((k, 0), (v, 1)):
        got = A.read_cache(cache, slots, dtype=torch.float32)[at]
        assert float((got - new).norm() / new.norm()) < 0.05
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block(x, r, cache, lengths - 1, slots, pages, lengths, space)
    for i in range(3):
        x.copy_(_randn(x.shape, dtype, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = space["y"].clone()
        assert torch.equal(block(x, r, cache, lengths - 1, slots, pages, lengths)[0], got)
    # The sum is x itself without a residual.
    assert block(x, None, cache, lengths - 1, slots, pages, lengths)[1] is x
    with pytest.raises(A.RidgeAttentionError):
        B.Int8Attention(norm_weight, qkv, out, 7, kv_heads, table)


def test_the_command():
    from ridge_amd import int8_attention as B
    args = ["--hidden", "512", "--heads", "8", "--kv-heads", "2", "--dim", "64", "--sequences", "1,3", "--length", "600",
            "--steps", "3"]
    assert B.main(args) == 0
    assert B.main(args + ["--graph", "--dtype", "bfloat16", "--page-size", "16"]) == 0


@pytest.mark.parametrize("handle", [False, True])
def test_a_call_on_a_stream_has_its_memory_from_there(handle):
    """The workspace and the result: the current stream, which runs ahead, is given none of it."""
    b = Batch([3000, 100, 9000, 0], 8, 2, 64, 16, torch.float16)
    bytes_ = A.lib().ridge_attention_workspace(4, 8, 2, 64, b.pages.shape[1], 16)
    want = A.attend(b.q, b.cache, b.pages, b.lengths)
    busy = torch.zeros((4096, 4096), device=DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()

    def held():
        return sum(s["total_size"] for s in torch.cuda.memory_snapshot() if s["stream"] == side.cuda_stream)
    before = held()
    for _ in range(3):
        with torch.cuda.stream(side):
            for _ in range(8):
                busy.add_(1)
        got = A.attend(b.q, b.cache, b.pages, b.lengths, stream=side.cuda_stream if handle else side)
        others = [torch.full((bytes_,), 255, dtype=torch.uint8, device=DEV) for _ in range(4)]
        others += [torch.full_like(got, math.nan) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del others
    assert bytes_ > 0 and held() - before >= bytes_
    assert torch.cuda.current_stream() == torch.cuda.default_stream()


def test_functional_transforms_and_tensors_without_memory_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    o = _operands()
    two = {n: torch.stack([t, t]) for n, t in o.items() if n != "cache"}
    for name, call in (("q", _norm_rope), ("positions", _norm_rope), ("k", _write), ("slots", _write), ("slots", _read), ("q", _attend),
                       ("lengths", _attend), ("pages", _attend)):
        print(name, flush=True)
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda t: call(o, **{name: t}))(two[name])
    for call in (lambda t: _norm_rope(o, q=t)[0], lambda t: _attend(o, q=t)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (o["q"],), (torch.ones_like(o["q"]),))
        with pytest.raises(RuntimeError):
            torch.func.vjp(call, o["q"])
    with FakeTensorMode() as mode:
        fake = {n: mode.from_tensor(t) for n, t in o.items() if n != "cache"}
        fake["cache"] = tuple(mode.from_tensor(t) for t in o["cache"])
        for call in (_norm_rope, _write, _read, _attend):
            with pytest.raises(A.RidgeAttentionError):
                call(fake)
