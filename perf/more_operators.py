"""The 8-bit cache's workloads: keys and values held in 8 bits in pages, what makes them,
and the attention of new tokens over them.

A served decoder layer with an 8-bit cache runs, between its projections: the norms of
the query's and key's heads with the position rotation, the writing of the new keys and
values, and the attention of each sequence's newest token over its pages. A prompt's
continuation reads rows of the cache back. A case is one such call on buffers that the
caller owns.

    own                  False: the plain form, elementary torch operations in 32 bits;
                         True: the calls of ridge_amd.attention
    listed()             the standing cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call
    run(state)           one pass, and its outputs
    work(case)           the bytes and operations a pass cannot do without
    exact(case, seed)    the outputs in 64 bits, without this package's code

A cache is (k, k_scale, v, v_scale): 8-bit rows [pages, heads, page_size, dim] and their
scales [pages, heads, page_size]. A slot is a token's place in it, page * page_size +
offset; a negative one is padding, neither written nor read. Writing returns the values
that the rows stand for, so its pass includes the call that reads them back.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
THETA = 10000.0

# No case costs more than the largest listed ones.
MOST_ROW_VALUES = 16384 * 40 * 128       # heads' values of a pass over rows
MOST_ATTEND_BYTES = int(1.6e9)
MOST_POSITIONS = 32768                   # rows of a table of rotations

_attention = None


def _ops():
    """ridge_amd.attention, imported where the framework's own calls run."""
    global _attention
    if _attention is None:
        from ridge_amd import attention
        _attention = attention
    return _attention


def _named(name, case):
    return dict(case, name=name) if name else case


def _rope(name, tokens, heads, kv_heads, dim, dtype, turned=None, norm=True, axes=1, interleaved=False):
    """`turned` of a head's dim columns are rotated, by positions on `axes` axes."""
    return _named(name, {"kind": "norm_rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                         "dtype": dtype, "turned": turned or dim, "norm": norm, "axes": axes,
                         "interleaved": interleaved})


def _rows(name, kind, tokens, kv_heads, dim, page_size, dtype, spread, padding=False):
    """`spread`: each token of a sequence of its own, at a slot anywhere; else prompts, page
    after page. `padding`: every eleventh token is none."""
    return _named(name, {"kind": kind, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page_size": page_size,
                         "dtype": dtype, "spread": spread, "padding": padding})


def _attend(name, batch, longest, shortest, heads, kv_heads, dim, page_size, dtype, window=0, empty=False, lse=False):
    """Sequences of `shortest` to `longest` tokens; `empty`: every fifth of none."""
    return _named(name, {"kind": "attend", "batch": batch, "longest": longest, "shortest": shortest, "heads": heads,
                         "kv_heads": kv_heads, "dim": dim, "page_size": page_size, "dtype": dtype, "window": window,
                         "empty": empty, "lse": lse})


def listed():
    return [
        # One decoding token: launch and host latency.
        _rope("norm_rope_1x32+8x128", 1, 32, 8, 128, "f16"),
        # The prompts of a prefill: memory traffic alone.
        _rope("norm_rope_16384x32+8x128", 16384, 32, 8, 128, "bf16"),
        # Patches of images among text: heads of 80, three axes, neighbours as pairs.
        _rope("norm_rope_axes_2311x14+2x80", 2311, 14, 2, 80, "f16", axes=3, interleaved=True),
        # One decoding token's key and value into the cache.
        _rows("write_1x8x128", "write", 1, 8, 128, 16, "f16", True),
        # A prefill's keys and values.
        _rows("write_16384x8x128", "write", 16384, 8, 128, 64, "bf16", False),
        # A padded batch of a small model: an odd head, pages that are no power of two.
        _rows("read_777x3x72", "read", 777, 3, 72, 48, "f16", True, True),
        # A long shared prefix that a prompt's continuation attends to in 16 bits.
        _rows("read_32768x8x128", "read", 32768, 8, 128, 64, "bf16", False),
        # One sequence with a short prompt: latency.
        _attend("attend_1x300_32/8x128", 1, 300, 300, 32, 8, 128, 16, "f16"),
        # One sequence with a very long one: the whole card on its length.
        _attend("attend_1x131072_32/8x128", 1, 131072, 131072, 32, 8, 128, 64, "bf16"),
        # A decoding batch of chats.
        _attend("attend_32x4096_32/8x128", 32, 4096, 512, 32, 8, 128, 16, "bf16"),
        # One shared head of keys, 71 query heads of 64, a window, sequences of no tokens,
        # and the sums that a caller joins with another part's.
        _attend("attend_odd_13x5003_71/1x64", 13, 5003, 1, 71, 1, 64, 48, "f16", window=1777, empty=True, lse=True),
        # The largest: long documents, the cache's bytes alone.
        _attend("attend_64x16384_32/8x128", 64, 16384, 8192, 32, 8, 128, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng):
    """A head's columns: the common ones, or any even number."""
    return rng.choice([64, 80, 96, 128, 128, 128, 192, 256, 2 * rng.randint(8, 128)])


def draw(rng):
    kind = rng.choice(["norm_rope", "write", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    while True:
        dim, kv_heads = _dim(rng), rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
        page_size = 16 * rng.choice([1, 1, 2, 3, 4, 4, 8, 16])
        if kind == "norm_rope":
            turned = rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)])
            case = _rope("", _log_int(rng, 1, 16384), heads, kv_heads, dim, dtype, turned, rng.random() < 0.7,
                         rng.choice([1, 1, 2, 3]), rng.random() < 0.3)
            if case["tokens"] * (heads + kv_heads) * dim <= MOST_ROW_VALUES:
                return case
        elif kind != "attend":
            case = _rows("", kind, _log_int(rng, 1, 32768), kv_heads, dim, page_size, dtype, rng.random() < 0.4,
                         rng.random() < 0.3)
            if case["tokens"] * kv_heads * dim * 2 <= MOST_ROW_VALUES:
                return case
        else:
            longest = _log_int(rng, 1, 131072)
            window = rng.choice([0, 0, 0, _log_int(rng, 1, longest)])
            case = _attend("", _log_int(rng, 1, 256), longest, rng.randint(max(1, longest // 8), longest), heads,
                           kv_heads, dim, page_size, dtype, window, rng.random() < 0.2, rng.random() < 0.3)
            # The whole cache lies on the card, whatever the window lets a pass read.
            if work(dict(case, window=0))["bytes"] <= MOST_ATTEND_BYTES and heads <= 128:
                return case


def _sections(case):
    """How many of the rotated pairs each axis turns: about equal parts, the first the largest."""
    pairs, axes = case["turned"] // 2, case["axes"]
    each = pairs // axes
    return [pairs - each * (axes - 1)] + [each] * (axes - 1)


def _lengths(case):
    """Each sequence's tokens, spread over the case's range."""
    lo, span = case["shortest"], case["longest"] - case["shortest"]
    lengths = [lo + int(round(span * ((1 + b * 0.618034) % 1 if b else 1))) for b in range(case["batch"])]
    return [0 if case["empty"] and b % 5 == 4 else n for b, n in enumerate(lengths)]


def _kept(case):
    """Each sequence's tokens that its window lets through."""
    return [min(n, case["window"] or n) for n in _lengths(case)]


def _heads(g, tokens, heads, dim, dtype):
    """Heads out of a projection: normal, with one column in 32 six times as wide."""
    x = torch.randn((tokens, heads, dim), generator=g, device=DEVICE)
    x *= torch.where(torch.rand((heads, dim), generator=g, device=DEVICE) < 1 / 32, 6.0, 1.0)
    return x.to(dtype)


def _cache(g, pages, heads, page_size, dim):
    """A cache of rows of normal values; rows 16 bytes apart at the least, as the framework lays them out."""
    shape, cache = (pages, heads, page_size), []
    for _ in range(2):
        rows = torch.empty(shape + ((dim + 15) // 16 * 16,), dtype=torch.int8, device=DEVICE)
        for part in rows.split(max(1, (1 << 26) // (heads * page_size * rows.shape[3]))):
            part.copy_(torch.randn(part.shape, generator=g, device=DEVICE).mul_(40).round_().clamp_(-127, 127))
        scale = torch.rand(shape, generator=g, device=DEVICE).mul_(0.01).add_(0.02)
        cache += [rows[..., :dim], scale]
    return tuple(cache)


def _slots(g, case):
    T, P = case["tokens"], case["page_size"]
    pages = T // P + 8
    if case["spread"]:
        slots = torch.randperm(pages * P, generator=g, device=DEVICE)[:T]
    else:
        at = torch.arange(T, device=DEVICE)
        slots = torch.randperm(pages, generator=g, device=DEVICE)[at // P] * P + at % P
    if case["padding"]:
        slots[10::11] = -1
    return pages, slots.to(torch.int32)


def _table(rows, pairs):
    """Cosines and then sines of each position's angles, for a base of 10000."""
    rate = THETA ** (-torch.arange(pairs, dtype=torch.float64, device=DEVICE) / pairs)
    angle = torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dtype, dim = case["kind"], TYPES[case["dtype"]], case["dim"]
    state = dict(case, dtype=dtype)
    if kind == "norm_rope":
        T, H, KV = case["tokens"], case["heads"], case["kv_heads"]
        qkv = _heads(g, T, H + 2 * KV, dim, dtype)     # the projection's rows: q, k and v beside each other
        state["q"], state["k"] = qkv[:, :H], qkv[:, H:H + KV]
        state["q_out"] = torch.empty((T, H, dim), dtype=dtype, device=DEVICE)
        state["k_out"] = torch.empty((T, KV, dim), dtype=dtype, device=DEVICE)
        state["sections"] = _sections(case)
        state["table"] = _table(MOST_POSITIONS, case["turned"] // 2)
        # Of text one token behind the other, from anywhere on; of patches each axis its own.
        state["positions"] = torch.randint(MOST_POSITIONS, (T if case["axes"] > 1 else 1, case["axes"]), generator=g,
                                           device=DEVICE, dtype=torch.int32)
        if case["axes"] == 1:
            state["positions"] = (state["positions"] + torch.arange(T, device=DEVICE)[:, None]).remainder(MOST_POSITIONS).int()
        for name in ("q_weight", "k_weight"):
            state[name] = torch.randn(dim, generator=g, device=DEVICE).mul_(0.1).add_(1).to(dtype) if case["norm"] else None
    elif kind == "attend":
        B, P, lengths = case["batch"], case["page_size"], _lengths(case)
        held = [-(-n // P) for n in lengths]
        state["cache"] = _cache(g, sum(held) + 1, case["kv_heads"], P, dim)
        order = torch.randperm(sum(held) + 1, generator=g, device=DEVICE).to(torch.int32)
        state["pages"] = torch.zeros((B, max(max(held), 1)), dtype=torch.int32, device=DEVICE)
        for b, part in enumerate(order[:sum(held)].split(held)):
            state["pages"][b, :held[b]] = part
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        q = torch.randn((B, case["heads"], dim), generator=g, device=DEVICE)
        q *= torch.where(torch.rand((B, case["heads"], 1), generator=g, device=DEVICE) < 0.25, 3.0, 1.0)   # some heads look at few tokens
        state["q"], state["out"] = q.to(dtype), torch.empty_like(q, dtype=dtype)
        state["lse_out"] = torch.empty((B, case["heads"]), device=DEVICE) if case["lse"] else None
        state["kept"] = list(zip(lengths, _kept(case)))
    else:
        pages, state["slots"] = _slots(g, case)
        state["cache"] = _cache(g, pages, case["kv_heads"], case["page_size"], dim)
        shape = case["tokens"], case["kv_heads"], dim
        if kind == "write":
            state["k"], state["v"] = _heads(g, *shape, dtype), _heads(g, *shape, dtype)
        state["values"] = torch.empty(shape, dtype=dtype, device=DEVICE), torch.empty(shape, dtype=dtype, device=DEVICE)
    return state


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


def _run_own(state):
    ops, kind = _ops(), state["kind"]
    if kind == "norm_rope":
        q, k = ops.norm_rope(state["q"], state["k"], state["table"], state["positions"], q_weight=state["q_weight"],
                             k_weight=state["k_weight"], eps=EPS, sections=state["sections"],
                             interleaved=state["interleaved"], q_out=state["q_out"], k_out=state["k_out"])
        return {"q": q, "k": k}
    if kind == "attend":
        out = ops.attend(state["q"], state["cache"], state["pages"], state["lengths"], window=state["window"] or None,
                         lse_out=state["lse_out"], out=state["out"])
        return {"out": out, "lse": state["lse_out"]}
    if kind == "write":
        ops.write_cache(state["cache"], state["slots"], state["k"], state["v"])
    k, v = ops.read_cache(state["cache"], state["slots"], out=state["values"])
    return {"k": k, "v": v}


def _plain_turn(x, weight, state):
    y, half, pairs = x.float(), state["turned"] // 2, torch.arange(state["turned"] // 2, device=DEVICE)
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(dim=2, keepdim=True) + EPS) * weight.float()
    axis = torch.repeat_interleave(torch.tensor(state["sections"], device=DEVICE), output_size=half)
    row = state["positions"][:, axis].long()                       # [tokens, pairs]
    cos, sin = state["table"][row, pairs][:, None], state["table"][row, half + pairs][:, None]
    if state["interleaved"]:
        first, second = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
    else:
        first, second = y[..., :half], y[..., half:2 * half]
    turned = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack(turned, dim=3).flatten(2) if state["interleaved"] else torch.cat(turned, dim=2)
    return torch.cat([turned, y[..., 2 * half:]], dim=2).to(state["dtype"])


def _plain_norm_rope(state):
    return {"q": _plain_turn(state["q"], state["q_weight"], state), "k": _plain_turn(state["k"], state["k_weight"], state)}


def _plain_write(state):
    values = []
    for x in (state["k"].double(), state["v"].double()):   # 32 bits lose the halves between two whole numbers
        top = x.abs().amax(dim=2, keepdim=True)
        y = torch.round(127 * x / top.clamp_min(127 * torch.finfo(torch.float32).tiny)) * (top / 127)
        values.append(torch.where(state["slots"][:, None, None] >= 0, y, torch.zeros_like(y)).to(state["dtype"]))
    return dict(zip("kv", values))


def _plain_read(state):
    k, k_scale, v, v_scale = state["cache"]
    page, at = state["slots"].long() // state["page_size"], state["slots"].long() % state["page_size"]
    page = page.clamp_min(0)
    values = []
    for rows, scale in ((k, k_scale), (v, v_scale)):
        y = rows[page, :, at].float() * scale[page, :, at][..., None]
        values.append(torch.where(state["slots"][:, None, None] >= 0, y, torch.zeros_like(y)).to(state["dtype"]))
    return dict(zip("kv", values))


def _plain_attend(state):
    (k, k_scale, v, v_scale), q, P = state["cache"], state["q"].float(), state["page_size"]
    B, H, D = q.shape
    KV = k.shape[1]
    out, lse = torch.zeros_like(q), torch.full((B, H), -math.inf, device=DEVICE)
    for b, (n, kept) in enumerate(state["kept"]):
        if kept == 0:
            continue
        pages = state["pages"][b, (n - kept) // P:(n - 1) // P + 1].long()
        start = (n - kept) % P

        def rows(values, scale):
            y = values[pages].float() * scale[pages][..., None]
            return y.transpose(0, 1).reshape(KV, -1, D)[:, start:start + kept]
        s = q[b].reshape(KV, H // KV, D) @ rows(k, k_scale).transpose(1, 2).contiguous() * D ** -0.5
        top = s.amax(dim=2, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(dim=2, keepdim=True)
        out[b] = (p @ rows(v, v_scale) / total).reshape(H, D)
        lse[b] = (top + total.log()).reshape(H)
    return {"out": out.to(state["dtype"]), "lse": lse if state["lse"] else None}


_PLAIN = {"norm_rope": _plain_norm_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}


def work(case):
    E, D, KV = 4 if case["dtype"] == "f32" else 2, case["dim"], case["kv_heads"]
    if case["kind"] == "norm_rope":
        T, values = case["tokens"], case["tokens"] * (case["heads"] + KV) * D
        # A position's rotations are read once for all heads.
        table = min(T * case["axes"], MOST_POSITIONS) * 4 * case["turned"] // case["axes"]
        return {"bytes": 2 * E * values + table + 4 * T * case["axes"] + (2 * E * D if case["norm"] else 0),
                "flops": 7 * values}
    if case["kind"] == "attend":
        kept = _kept(case)
        pages = sum(-(-n // case["page_size"]) for n in kept)
        rows = case["batch"] * case["heads"]
        return {"bytes": 2 * sum(kept) * KV * (D + 4) + 2 * E * rows * D + 4 * pages + 4 * len(kept)
                + (4 * rows if case["lse"] else 0), "flops": 4 * sum(kept) * case["heads"] * D}
    values = case["tokens"] * KV * D * 2
    if case["kind"] == "write":     # the values in, what the rows stand for out
        return {"bytes": 2 * E * values + 4 * case["tokens"], "flops": 4 * values}
    return {"bytes": (1 + E) * values + 8 * case["tokens"] * KV + 4 * case["tokens"], "flops": values}


def _turn64(x, weight, state):
    y, half, T = x.double(), state["turned"] // 2, x.shape[0]
    if weight is not None:
        power = torch.linalg.vector_norm(y, dim=-1, keepdim=True).square() / y.shape[-1] + EPS
        y = y / power.sqrt() * weight.double()
    table = state["table"].double()
    cos, sin = torch.empty((2, T, 1, half), dtype=torch.float64, device=DEVICE)
    begin = 0
    for a, n in enumerate(state["sections"]):
        rows = table[state["positions"][:, a].long()]
        cos[:, 0, begin:begin + n] = rows[:, begin:begin + n]
        sin[:, 0, begin:begin + n] = rows[:, half + begin:half + begin + n]
        begin += n
    z = y.clone()
    pair = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if state["interleaved"] else (slice(0, half), slice(half, 2 * half))
    z[..., pair[0]] = y[..., pair[0]] * cos - y[..., pair[1]] * sin
    z[..., pair[1]] = y[..., pair[0]] * sin + y[..., pair[1]] * cos
    return z


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "norm_rope":
        return {"q": _turn64(state["q"], state["q_weight"], state), "k": _turn64(state["k"], state["k_weight"], state)}
    if kind == "attend":
        (k, k_scale, v, v_scale), q, P = state["cache"], state["q"].double(), case["page_size"]
        B, H, D = q.shape
        group = H // case["kv_heads"]
        out, lse = torch.zeros_like(q), torch.full((B, H), -math.inf, dtype=torch.float64, device=DEVICE)
        for b, (n, kept) in enumerate(state["kept"]):
            at = torch.arange(n - kept, n, device=DEVICE)
            if kept == 0:
                continue
            page, offset = state["pages"][b].long()[at // P], at % P
            for h in range(case["kv_heads"]):
                keys = k[page, h, offset].double() * k_scale[page, h, offset].double().unsqueeze(1)
                own_heads = slice(h * group, (h + 1) * group)
                s = (keys @ q[b, own_heads].t()).t() / math.sqrt(D)
                values = v[page, h, offset].double() * v_scale[page, h, offset].double().unsqueeze(1)
                out[b, own_heads] = torch.softmax(s, dim=1) @ values
                lse[b, own_heads] = torch.logsumexp(s, dim=1)
        return {"out": out, "lse": lse if case["lse"] else None}
    here = state["slots"].ge(0).double()[:, None, None]
    if kind == "write":
        values = []
        for x in (state["k"].double(), state["v"].double()):
            top = torch.linalg.vector_norm(x, ord=math.inf, dim=-1).unsqueeze(-1)
            top = torch.where(top > 0, top, torch.ones_like(top))
            values.append((x * 127).div(top).round_().mul_(top).div_(127) * here)
        return {"k": values[0], "v": values[1]}
    k, k_scale, v, v_scale = state["cache"]
    slots = state["slots"].long().clamp_min(0)
    page, at = torch.div(slots, case["page_size"], rounding_mode="floor"), slots.remainder(case["page_size"])
    return {"k": k[page, :, at].double() * k_scale[page, :, at].double().unsqueeze(-1) * here,
            "v": v[page, :, at].double() * v_scale[page, :, at].double().unsqueeze(-1) * here}
