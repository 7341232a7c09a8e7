"""The 8-bit operators' workloads: rows held in 8 bits with a scale each, and the
matrix product of such rows.

A served model with 8-bit weights runs, for every matrix product, one operator that
makes 8-bit rows out of activations (a norm with the residual's addition, a gated
activation, or the rows as they are) and the product of those rows with the weight's,
one scale for each token and one for each channel. A case is one such call, or the
two together, on buffers that the caller owns.

    own                  False: the plain form, elementary torch operations in 32 bits;
                         True: the calls of ridge_amd.int8
    listed()             the standing cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call
    run(state)           one pass, and its outputs
    work(case)           the bytes and operations a pass cannot do without
    exact(case, seed)    the outputs in 64 bits, without this package's code

Operators whose result is 8-bit rows return the values these stand for (q times the
row's scale) in the input's type, so their pass includes the call that makes those.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6

# No case costs more than the largest listed ones.
MOST_ELEMENTS = 16384 * 8192
MOST_MNK = 8192 * 8192 * 8192
MOST_GEMM_BYTES = 4 * 8192 * 8192

_int8 = None


def _ops():
    """ridge_amd.int8, imported where the framework's own calls run."""
    global _int8
    if _int8 is None:
        from ridge_amd import int8
        _int8 = int8
    return _int8


def _rows(name, kind, rows, cols, dtype, wide=0):
    case = {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "wide": wide}
    return dict(case, name=name) if name else case


def _gemm(name, kind, M, N, K, dtype, bias):
    case = {"kind": kind, "M": M, "N": N, "K": K, "dtype": dtype, "bias": bias}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token's norm in a decoding step: launch and host latency.
        _rows("rms_norm_1x4096", "rms_norm", 1, 4096, "f16"),
        # The norm over a long prompt batch: memory traffic alone.
        _rows("rms_norm_16384x8192", "rms_norm", 16384, 8192, "bf16"),
        # The gated activation of a few decoding sequences, an odd width.
        _rows("silu_mul_13x11007", "silu_mul", 13, 11007, "f16"),
        # The gated activation of a prompt.
        _rows("silu_mul_4096x16384", "silu_mul", 4096, 16384, "bf16"),
        # Attention's output before its projection, rows cut out of a wider buffer.
        _rows("quantize_333x5000_of_5064", "quantize", 333, 5000, "bf16", 64),
        # A whole weight matrix when a model is loaded.
        _rows("quantize_16384x8192", "quantize", 16384, 8192, "f16"),
        # One token: the weight's bytes are all there is to move.
        _gemm("gemm_1x4096x4096", "gemm", 1, 4096, 4096, "f16", False),
        # A decoding batch on a wide layer with a bias.
        _gemm("gemm_48x8192x4096", "gemm", 48, 8192, 4096, "bf16", True),
        # Ragged in every direction: a batch of prompts without padding, an odd
        # number of channels, and a K that ends inside a 16-byte chunk.
        _gemm("gemm_1531x5003x2050", "gemm", 1531, 5003, 2050, "f16", True),
        # The headline benchmark's square.
        _gemm("gemm_4096cube", "gemm", 4096, 4096, 4096, "f16", False),
        # The largest: the matrix pipes alone.
        _gemm("gemm_8192cube", "gemm", 8192, 8192, 8192, "bf16", False),
        # The start of a feed-forward block for a few tokens: norm, then product.
        _gemm("norm_gemm_8x12288x4096", "norm_gemm", 8, 12288, 4096, "f16", False),
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Half of the widths are whole 128s, the others whatever comes, odd ones among them."""
    n = _log_int(rng, lo, hi)
    return max(128, n // 128 * 128) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["rms_norm", "silu_mul", "quantize", "gemm", "gemm", "gemm", "norm_gemm"])
    dtype = rng.choice(["f16", "bf16"])
    while True:
        if kind in ("gemm", "norm_gemm"):
            M = _log_int(rng, 1, 8192 if kind == "gemm" else 2048)
            N, K = _width(rng, 32, 16384), _width(rng, 32, 16384)
            case = _gemm("", kind, M, N, K, rng.choice([dtype, dtype, "f32"]) if kind == "gemm" else dtype,
                         rng.random() < 0.3)
            if M * N * K <= MOST_MNK and work(case)["bytes"] <= MOST_GEMM_BYTES:
                return case
        else:
            rows, cols = _log_int(rng, 1, 16384), _width(rng, 32, 16384)
            if rows * cols * (2 if kind == "silu_mul" else 1) <= MOST_ELEMENTS:
                return _rows("", kind, rows, cols, dtype, rng.choice([0, 0, 0, 8, 56, 1]))


def _activations(g, rows, cols, dtype, wide=0):
    """A residual stream's values: normal, with one channel in 256 twelve times as wide.
    With `wide`, the rows of a buffer that many columns wider."""
    x = torch.randn((rows, cols + wide), generator=g, device=DEVICE)
    x *= torch.where(torch.rand(cols + wide, generator=g, device=DEVICE) < 1 / 256, 12.0, 1.0)
    return x.to(dtype)[:, :cols]


def _int8_buffer(rows, cols):
    """8-bit rows as the framework lays them out: rows a multiple of 16 bytes apart."""
    return torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=DEVICE)[:, :cols]


def _int8_rows(g, rows, cols):
    """8-bit rows of normal values, and scales of like rows."""
    q = _int8_buffer(rows, cols)
    q.copy_(torch.randn((rows, cols), generator=g, device=DEVICE).mul_(32).round_().clamp_(-127, 127))
    return q, torch.rand(rows, generator=g, device=DEVICE).mul_(0.03).add_(0.01)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["dtype"]]
    state = {"kind": kind, "dtype": dtype}
    if kind in ("gemm", "norm_gemm"):
        M, N, K = case["M"], case["N"], case["K"]
        if kind == "gemm":
            state["a"], state["a_scale"] = _int8_rows(g, M, K)
        state["b"], state["b_scale"] = _int8_rows(g, N, K)
        state["b_scale"] *= 0.02
        state["bias"] = torch.randn(N, generator=g, device=DEVICE).to(dtype) if case["bias"] else None
        state["out"] = torch.empty((M, N), dtype=dtype, device=DEVICE)
        rows, cols = M, K
    else:
        rows, cols = case["rows"], case["cols"]
        width = 2 * cols if kind == "silu_mul" else cols
        state["x"] = _activations(g, rows, width, dtype, case["wide"])
        state["values"] = torch.empty((rows, cols), dtype=dtype, device=DEVICE)
    if kind in ("rms_norm", "norm_gemm"):
        if kind == "norm_gemm":
            state["x"] = _activations(g, rows, cols, dtype)
        state["residual"] = _activations(g, rows, cols, dtype)
        state["weight"] = torch.randn(cols, generator=g, device=DEVICE).mul_(0.1).add_(1).to(dtype)
        state["residual_out"] = torch.empty((rows, cols), dtype=dtype, device=DEVICE)
    if kind != "gemm":
        state["rows8"] = _int8_buffer(rows, cols), torch.empty(rows, dtype=torch.float32, device=DEVICE)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    ops, kind, dtype = _ops(), state["kind"], state["dtype"]
    if kind == "gemm":
        return ops.gemm(state["a"], state["a_scale"], state["b"], state["b_scale"], bias=state["bias"],
                        out=state["out"])
    if kind == "norm_gemm":
        q, scale, residual = ops.rms_norm(state["x"], state["weight"], EPS, residual=state["residual"],
                                          residual_out=state["residual_out"], out=state["rows8"])
        y = ops.gemm(q, scale, state["b"], state["b_scale"], bias=state["bias"], out=state["out"])
        return {"y": y, "residual": residual}
    if kind == "rms_norm":
        q, scale, residual = ops.rms_norm(state["x"], state["weight"], EPS, residual=state["residual"],
                                          residual_out=state["residual_out"], out=state["rows8"])
        return {"values": ops.dequantize(q, scale, out=state["values"]), "residual": residual}
    make = ops.silu_mul if kind == "silu_mul" else ops.quantize
    q, scale = make(state["x"], out=state["rows8"])
    return {"values": ops.dequantize(q, scale, out=state["values"])}


def _plain_rows(y):
    """(q, scale) of 32-bit rows: whole numbers up to 127, and the step of each row."""
    scale = (y.abs().amax(dim=1, keepdim=True) / 127).clamp_min(torch.finfo(torch.float32).tiny)
    return torch.round(y / scale), scale


def _plain_norm(state):
    s = state["x"].float() + state["residual"].float()
    y = s * torch.rsqrt((s * s).mean(dim=1, keepdim=True) + EPS) * state["weight"].float()
    return y, s.to(state["dtype"])


def _plain_product(q, scale, state):
    y = (q @ state["b"].float().t()) * scale * state["b_scale"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["dtype"])


def _run_plain(state):
    kind, dtype = state["kind"], state["dtype"]
    if kind == "gemm":
        return _plain_product(state["a"].float(), state["a_scale"][:, None], state)
    if kind in ("rms_norm", "norm_gemm"):
        y, residual = _plain_norm(state)
        q, scale = _plain_rows(y)
        if kind == "norm_gemm":
            return {"y": _plain_product(q, scale, state), "residual": residual}
        return {"values": (q * scale).to(dtype), "residual": residual}
    y = state["x"].float()
    if kind == "silu_mul":
        gate, up = y.chunk(2, dim=1)
        y = gate / (1 + torch.exp(-gate)) * up
    q, scale = _plain_rows(y)
    return {"values": (q * scale).to(dtype)}


def work(case):
    E = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("gemm", "norm_gemm"):
        M, N, K = case["M"], case["N"], case["K"]
        a = M * K + 4 * M if case["kind"] == "gemm" else 3 * E * M * K + E * K
        return {"bytes": a + N * K + 4 * N + E * M * N + (E * N if case["bias"] else 0), "flops": 2 * M * N * K}
    rows, cols = case["rows"], case["cols"]
    if case["kind"] == "rms_norm":  # x and the residual in, the residual and the values out
        return {"bytes": 4 * E * rows * cols + E * cols, "flops": 8 * rows * cols}
    return {"bytes": (3 if case["kind"] == "silu_mul" else 2) * E * rows * cols, "flops": 6 * rows * cols}


def _nearest_steps(y):
    """Each row's values moved to the nearest multiple of its largest magnitude's 127th."""
    top = torch.linalg.vector_norm(y, ord=math.inf, dim=-1).unsqueeze(-1)
    step = torch.where(top > 0, top, torch.ones_like(top)) / 127
    return y.div(step).round_().mul_(step)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind in ("rms_norm", "norm_gemm"):
        r = state["x"].double() + state["residual"].double()
        power = torch.linalg.vector_norm(r, dim=-1).square_().div_(r.shape[1]).add_(EPS)
        held = _nearest_steps(r * state["weight"].double() / power.sqrt_().unsqueeze(-1))
        if kind == "rms_norm":
            return {"values": held, "residual": r}
    elif kind == "gemm":
        held = state["a"].double().mul_(state["a_scale"].double().unsqueeze(-1))
    else:
        x = state["x"].double()
        if kind == "silu_mul":
            x = x[:, :case["cols"]] * torch.sigmoid(x[:, :case["cols"]]) * x[:, case["cols"]:]
        return {"values": _nearest_steps(x)}
    y = held @ (state["b"].double() * state["b_scale"].double().unsqueeze(-1)).t()
    if state["bias"] is not None:
        y += state["bias"].double()
    return y if kind == "gemm" else {"y": y, "residual": r}
