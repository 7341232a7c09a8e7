"""The attention half of a decoder layer over a cache in 8 bits, for one new token of each
sequence:

    h = norm(x + residual) * norm_weight            int8.rms_norm, 8-bit rows
    [q | k | v] = h qkv^T                           int8.gemm, 16-bit
    q, k = norm and rotation of their heads         attention.norm_rope, in place
    cache[slots] = k, v                             attention.write_cache, 8-bit rows
    o = softmax(q K^T) V over each sequence         attention.attend
    y = o out^T                                     int8.quantize and int8.gemm

    python -m ridge_amd.int8_attention [--hidden 4096] [--heads 32] [--kv-heads 8] [--dim 128]
                                       [--sequences 1,16,64] [--length 4096] [--page-size 64]
                                       [--dtype float16] [--steps 200] [--graph]

prints, for each number of sequences, the block's time and how far y is from the same block
in 32 bits with the weights as they were and the cache's values. --graph replays the block's
launches as a HIP graph. Weights, inputs and what the cache holds are random.
"""

import argparse

from . import attention, int8
from .int8_mlp import _time


class Int8Attention:
    """The block with its weights in 8 bits, quantised once: qkv [(heads + 2 kv_heads) dim, hidden]
    (the query heads' rows, then the keys', then the values') and out [hidden, heads dim], one
    scale for each row. q_weight and k_weight [dim] norm the heads, or are None. table has the
    rotations (attention.rope_table)."""

    def __init__(self, norm_weight, qkv, out, heads, kv_heads, table, q_weight=None, k_weight=None, eps=1e-6):
        hidden = out.shape[0]
        if norm_weight.shape != (hidden,) or qkv.shape[1] != hidden or heads < 1 or kv_heads < 1 or heads % kv_heads or \
                out.shape[1] % heads or qkv.shape[0] * heads != out.shape[1] * (heads + 2 * kv_heads):
            raise attention.RidgeAttentionError("qkv %s, out %s and norm_weight %s are not one block's of %d heads on %d"
                                                % (tuple(qkv.shape), tuple(out.shape), tuple(norm_weight.shape), heads,
                                                   kv_heads))
        self.hidden, self.heads, self.kv_heads, self.dim = hidden, heads, kv_heads, out.shape[1] // heads
        self.norm_weight, self.q_weight, self.k_weight, self.table, self.eps = norm_weight, q_weight, k_weight, table, eps
        self.qkv, self.out = int8.quantize(qkv), int8.quantize(out)

    def workspace(self, tokens, dtype):
        """The buffers of a pass over one token of each of `tokens` sequences, for callers that keep them."""
        import torch
        device, width = self.norm_weight.device, self.heads * self.dim
        return {"h": int8.empty(tokens, self.hidden, device),
                "qkv": torch.empty((tokens, width + 2 * self.kv_heads * self.dim), dtype=dtype, device=device),
                "o": torch.empty((tokens, self.heads, self.dim), dtype=dtype, device=device),
                "o8": int8.empty(tokens, width, device),
                "y": torch.empty((tokens, self.hidden), dtype=dtype, device=device),
                "residual": torch.empty((tokens, self.hidden), dtype=dtype, device=device)}

    def __call__(self, x, residual, cache, positions, slots, pages, lengths, workspace=None):
        """(y, x + residual), on the current stream; both in the workspace where one is given. Row b of
        x is sequence b's new token, which goes to slots[b] and is the last of lengths[b]. Without a
        residual, as before a model's first block, the sum is x itself."""
        w = workspace or self.workspace(x.shape[0], x.dtype)
        h, h_scale, total = int8.rms_norm(x, self.norm_weight, self.eps, residual=residual,
                                          residual_out=None if residual is None else w["residual"], out=w["h"])
        heads = int8.gemm(h, h_scale, *self.qkv, out=w["qkv"]).view(x.shape[0], -1, self.dim)
        q, k, v = heads.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        attention.norm_rope(q, k, self.table, positions, q_weight=self.q_weight, k_weight=self.k_weight, eps=self.eps,
                            q_out=q, k_out=k)
        attention.write_cache(cache, slots, k, v)
        o = attention.attend(q, cache, pages, lengths, out=w["o"])
        o8, o_scale = int8.quantize(o.view(x.shape[0], -1), out=w["o8"])
        return int8.gemm(o8, o_scale, *self.out, out=w["y"]), x if residual is None else total


def plain_block(x, residual, norm_weight, qkv, out, heads, kv_heads, table, cached, positions, q_weight=None,
                k_weight=None, eps=1e-6):
    """The block in the inputs' own precision, of elementary operations: (y, x + residual, k, v), the
    last two being the new token's. cached: each sequence's keys and values [tokens, kv_heads, dim]
    before the new token."""
    import torch
    s = x + residual
    h = s / (s.square().mean(dim=1, keepdim=True) + eps).sqrt() * norm_weight
    q, k, v = (h @ qkv.t()).view(len(x), heads + 2 * kv_heads, -1).split([heads, kv_heads, kv_heads], dim=1)

    def turned(t, weight):
        if weight is not None:
            t = t / (t.square().mean(dim=2, keepdim=True) + eps).sqrt() * weight
        half = table.shape[1] // 2
        c, s = table[positions.long(), None].split(half, dim=2)
        a, b, rest = t[..., :half], t[..., half:2 * half], t[..., 2 * half:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], dim=2)
    q, k = turned(q, q_weight), turned(k, k_weight)
    rows = []
    for i, (keys, values) in enumerate(cached):
        keys, values = (torch.cat(t).transpose(0, 1).contiguous() for t in ((keys, k[i:i + 1]), (values, v[i:i + 1])))
        p = q[i].view(kv_heads, heads // kv_heads, -1) @ keys.transpose(1, 2).contiguous() * keys.shape[2] ** -0.5
        p = (p - p.amax(dim=2, keepdim=True)).exp()
        rows.append((p / p.sum(dim=2, keepdim=True) @ values).reshape(-1))
    return torch.stack(rows) @ out.t(), s, k, v


def random_block(hidden, heads, kv_heads, dim, dtype, seed, device="cuda"):
    """(norm_weight, qkv, out, q_weight, k_weight) of a random block whose values stay of order one."""
    import torch
    g = torch.Generator(device=device).manual_seed(seed)

    def near_one(n):
        return torch.randn(n, generator=g, device=device).mul_(0.1).add_(1).to(dtype)
    width = heads * dim
    qkv = torch.randn((width + 2 * kv_heads * dim, hidden), generator=g, device=device).mul_(hidden ** -0.5).to(dtype)
    out = torch.randn((hidden, width), generator=g, device=device).mul_(width ** -0.5).to(dtype)
    return near_one(hidden), qkv, out, near_one(dim), near_one(dim)


def random_cache(sequences, length, kv_heads, dim, page_size, dtype, seed, device="cuda"):
    """(cache, pages, slots, lengths, every) of sequences of `length` tokens: all but the last one in the
    cache, on pages in a random order, the slots that the last ones go to, and all tokens' slots."""
    import torch
    g = torch.Generator(device=device).manual_seed(seed)
    each = -(-length // page_size)
    cache = attention.empty_cache(sequences * each, page_size, kv_heads, dim, device)
    pages = torch.randperm(sequences * each, generator=g, device=device).to(torch.int32).view(sequences, each)
    at = torch.arange(length, device=device)
    slots = pages[:, at // page_size] * page_size + (at % page_size).to(torch.int32)
    for b in range(sequences):
        k, v = (torch.randn((length - 1, kv_heads, dim), generator=g, device=device).to(dtype) for _ in range(2))
        attention.write_cache(cache, slots[b, :-1], k, v)
    lengths = torch.full((sequences,), length, dtype=torch.int32, device=device)
    return cache, pages, slots[:, -1].contiguous(), lengths, slots


def main(argv=None):
    import torch
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--dim", type=int, default=128)
    ap.add_argument("--sequences", default="1,16,64", help="numbers of sequences, separated by commas")
    ap.add_argument("--length", type=int, default=4096, help="tokens of a sequence, the new one among them")
    ap.add_argument("--page-size", type=int, default=64)
    ap.add_argument("--dtype", default="float16", choices=["float16", "bfloat16"])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--graph", action="store_true", help="replay the pass as a HIP graph")
    args = ap.parse_args(argv)
    dtype = getattr(torch, args.dtype)
    norm_weight, qkv, out, q_weight, k_weight = random_block(args.hidden, args.heads, args.kv_heads, args.dim, dtype, 1)
    table = attention.rope_table(args.length, args.dim)
    block = Int8Attention(norm_weight, qkv, out, args.heads, args.kv_heads, table, q_weight, k_weight)
    worst = 0.0
    for sequences in (int(t) for t in args.sequences.split(",")):
        cache, pages, slots, lengths, every = random_cache(sequences, args.length, args.kv_heads, args.dim, args.page_size,
                                                           dtype, 2)
        x, residual = (torch.randn((sequences, args.hidden), device="cuda").to(dtype) for _ in range(2))
        positions = lengths - 1
        space = block.workspace(sequences, dtype)

        def step():
            block(x, residual, cache, positions, slots, pages, lengths, space)
        step()
        if args.graph:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            step = graph.replay
        us = _time(step, args.steps)
        cached = [attention.read_cache(cache, every[b, :-1], dtype=torch.float32) for b in range(sequences)]
        want = plain_block(x.float(), residual.float(), norm_weight.float(), qkv.float(), out.float(), args.heads,
                           args.kv_heads, table, cached, positions, q_weight.float(), k_weight.float())[0]
        off = float((space["y"].float() - want).norm() / want.norm())
        worst = max(worst, off if off == off else float("inf"))   # a NaN is no error within any bound
        held = 2.0 * sequences * args.length * args.kv_heads * (args.dim + 4)
        print("%6d sequences of %d  %9.2f us  cache %7.1f GB/s  error %.2f%%"
              % (sequences, args.length, us, held / us / 1e3, 100 * off), flush=True)
    return 0 if worst < 0.1 else 1


if __name__ == "__main__":
    raise SystemExit(main())
