"""A gated feed-forward block in 8 bits, as a decoder layer runs it:

    h = norm(x + residual) * norm_weight            rms_norm, 8-bit rows
    [gate | up] = h gate_up^T                       gemm, 16-bit
    a = silu(gate) * up                             silu_mul, 8-bit rows
    y = a down^T                                    gemm, 16-bit

    python -m ridge_amd.int8_mlp [--hidden 4096] [--inner 8192] [--tokens 1,16,256,4096]
                                 [--dtype float16] [--steps 200] [--graph]

prints, for each number of tokens, the block's time and how far y is from the same block
in 32 bits with the weights as they were. --graph replays the four launches as a HIP
graph. Weights and inputs are random; sizes default to the framework's own.
"""

import argparse

from . import int8


class Int8Mlp:
    """The block with its weights in 8 bits, quantised once: gate_up [2 inner, hidden]
    (gate's rows, then up's) and down [hidden, inner], one scale for each row."""

    def __init__(self, norm_weight, gate_up, down, eps=1e-6):
        if gate_up.shape[0] != 2 * down.shape[1] or gate_up.shape[1] != down.shape[0] or \
                norm_weight.shape != (down.shape[0],):
            raise int8.RidgeInt8Error("gate_up %s, down %s and norm_weight %s are not one block's"
                                      % (tuple(gate_up.shape), tuple(down.shape), tuple(norm_weight.shape)))
        self.hidden, self.inner, self.eps = down.shape[0], down.shape[1], eps
        self.norm_weight = norm_weight
        self.gate_up = int8.quantize(gate_up)
        self.down = int8.quantize(down)

    def workspace(self, tokens, dtype):
        """The buffers of a pass over `tokens` rows, for callers that keep them."""
        import torch
        device = self.norm_weight.device
        return {"h": int8.empty(tokens, self.hidden, device),
                "gate_up": torch.empty((tokens, 2 * self.inner), dtype=dtype, device=device),
                "a": int8.empty(tokens, self.inner, device),
                "y": torch.empty((tokens, self.hidden), dtype=dtype, device=device),
                "residual": torch.empty((tokens, self.hidden), dtype=dtype, device=device)}

    def __call__(self, x, residual=None, workspace=None):
        """(y, x + residual), on the current stream; both in the workspace where one is given.
        Without a residual, as before a model's first block, the sum is x itself."""
        w = workspace or self.workspace(x.shape[0], x.dtype)
        h, h_scale, total = int8.rms_norm(x, self.norm_weight, self.eps, residual=residual,
                                          residual_out=None if residual is None else w["residual"], out=w["h"])
        gate_up = int8.gemm(h, h_scale, *self.gate_up, out=w["gate_up"])
        a, a_scale = int8.silu_mul(gate_up, out=w["a"])
        return int8.gemm(a, a_scale, *self.down, out=w["y"]), x if residual is None else total


def plain_block(x, residual, norm_weight, gate_up, down, eps=1e-6):
    """The block in the inputs' own precision, of elementary operations: (y, x + residual)."""
    s = x + residual
    h = s / (s.square().mean(dim=1, keepdim=True) + eps).sqrt() * norm_weight
    gate, up = (h @ gate_up.t()).chunk(2, dim=1)
    return (gate / (1 + (-gate).exp()) * up) @ down.t(), s


def random_block(hidden, inner, dtype, seed, device="cuda"):
    """(norm_weight, gate_up, down) of a random block whose values stay of order one."""
    import torch
    g = torch.Generator(device=device).manual_seed(seed)
    norm_weight = torch.randn(hidden, generator=g, device=device).mul_(0.1).add_(1).to(dtype)
    gate_up = torch.randn((2 * inner, hidden), generator=g, device=device).mul_(hidden ** -0.5).to(dtype)
    down = torch.randn((hidden, inner), generator=g, device=device).mul_(inner ** -0.5).to(dtype)
    return norm_weight, gate_up, down


def _time(step, steps):
    """Microseconds a step, the middle of five windows."""
    import torch
    for _ in range(20):
        step()
    got = []
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(steps):
            step()
        end.record()
        end.synchronize()
        got.append(start.elapsed_time(end) / steps * 1e3)
    return sorted(got)[2]


def main(argv=None):
    import torch
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--inner", type=int, default=8192)
    ap.add_argument("--tokens", default="1,16,256,4096", help="numbers of tokens, separated by commas")
    ap.add_argument("--dtype", default="float16", choices=["float16", "bfloat16"])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--graph", action="store_true", help="replay the pass as a HIP graph")
    args = ap.parse_args(argv)
    dtype = getattr(torch, args.dtype)
    weights = random_block(args.hidden, args.inner, dtype, 1)
    mlp = Int8Mlp(*weights)
    worst = 0.0
    for tokens in (int(t) for t in args.tokens.split(",")):
        x = torch.randn((tokens, args.hidden), device="cuda").to(dtype)
        residual = torch.randn((tokens, args.hidden), device="cuda").to(dtype)
        space = mlp.workspace(tokens, dtype)

        def step():
            mlp(x, residual, space)
        step()
        if args.graph:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            step = graph.replay
        us = _time(step, args.steps)
        want = plain_block(x.float(), residual.float(), *(w.float() for w in weights))[0]
        off = float((space["y"].float() - want).norm() / want.norm())
        worst = max(worst, off if off == off else float("inf"))   # a NaN is no error within any bound
        print("%6d tokens  %9.2f us  %8.1f TOP/s  error %.2f%%"
              % (tokens, us, 6.0 * tokens * args.hidden * args.inner / us / 1e6, 100 * off), flush=True)
    return 0 if worst < 0.1 else 1


if __name__ == "__main__":
    raise SystemExit(main())
