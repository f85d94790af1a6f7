"""A decoder layer served from 8-bit weights and an 8-bit paged key/value cache.

Prompts of different lengths go through the layer in one call, then every sequence decodes token by token:

    RMSNorm + q/k/v projection -> kv_append (rotation, cache) -> kv_attention -> output projection
    RMSNorm -> moe (router, top-k experts)

``python examples/decode_layer.py`` runs it at the sizes given on the command line with random weights, then prints the
time of a decode step, captured in a CUDA graph as a server would, and the bytes that the cache holds.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import popcorn_b200 as pc  # noqa: E402


class DecoderLayer:
    """Weights, quantized once, and the cache of ``pages`` pages."""

    eps = 1e-5

    def __init__(self, hidden, heads, kv_heads, dim, experts, inter, top_k, pages, page_size=16, positions=4096,
                 seed=0, device="cuda"):
        gen = torch.Generator(device).manual_seed(seed)

        def weights(*shape):  # int8 codes and a scale per output channel
            q, s = pc.quantize(torch.randn(shape, generator=gen, device=device).flatten(0, -2) * shape[-1] ** -0.5)
            return q.view(shape), s.view(shape[:-1])

        self.heads, self.kv_heads, self.dim, self.top_k = heads, kv_heads, dim, top_k
        self.norm1 = torch.rand(hidden, generator=gen, device=device) + 0.5
        self.norm2 = torch.rand(hidden, generator=gen, device=device) + 0.5
        self.qkv = weights((heads + 2 * kv_heads) * dim, hidden)
        self.o = weights(hidden, heads * dim)
        self.router = torch.randn((experts, hidden), generator=gen, device=device) * hidden ** -0.5
        self.gate, self.up, self.down = (weights(experts, inter, hidden), weights(experts, inter, hidden),
                                         weights(experts, hidden, inter))
        angle = torch.arange(positions, device=device)[:, None] * 1e4 ** (-torch.arange(0, dim, 2, device=device) / dim)
        self.cos, self.sin = angle.cos(), angle.sin()
        self.cache = pc.KvCache.empty(pages, kv_heads, dim, page_size, device)

    def __call__(self, x, table, start, length, first=None, max_tokens=None, routing=False):
        """x f32 [tokens, hidden], the sequences' new tokens one after the other (``first`` as in kv_append);
        ``start`` and ``length`` int32 [seqs]: cached tokens before and after this call."""
        qkv = pc.rmsnorm_dequantize_matmul(x, self.norm1, self.eps, *self.qkv).view(len(x), -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = pc.kv_append(self.cache, k, v, table, start, first=first, q=q, cos=self.cos, sin=self.sin)
        a = pc.kv_attention(self.cache, q, table, length, first=first, max_tokens=max_tokens)
        x = x + pc.dequantize_matmul(a.view(len(x), -1), *self.o)
        z = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * self.norm2
        y = pc.moe(z, self.router, *self.gate, *self.up, *self.down, self.top_k, routing=routing)
        return (x + y[0], *y[1:]) if routing else x + y


def block_table(longest, seqs, page_size, device="cuda"):
    """Pages for ``seqs`` sequences of up to ``longest`` tokens each: (int32 [seqs, pages], number of pages)."""
    each = -(-longest // page_size)
    return torch.randperm(seqs * each, device=device).to(torch.int32).view(seqs, each), seqs * each


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("hidden", 2048), ("heads", 32), ("kv-heads", 8), ("dim", 64), ("experts", 16),
                        ("inter", 1024), ("top-k", 4), ("seqs", 4), ("prompt", 500), ("steps", 32)):
        p.add_argument("--" + name, type=int, default=value)
    o = p.parse_args()
    table, pages = block_table(o.prompt + o.steps + 8, o.seqs, 16)
    layer = DecoderLayer(o.hidden, o.heads, o.kv_heads, o.dim, o.experts, o.inter, o.top_k, pages,
                         positions=o.prompt + o.steps + 8)
    new = torch.tensor([max(1, o.prompt * (b + 1) // o.seqs) for b in range(o.seqs)], dtype=torch.int32)
    first = torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0).to(torch.int32)]).cuda()
    length = new.cuda()
    x = torch.randn((int(new.sum()), o.hidden), device="cuda")
    y = layer(x, table, torch.zeros_like(length), length, first=first, max_tokens=int(new.max()))

    # Decode: the lengths advance on the device, so one graph serves every step.
    x = y[first[1:].long() - 1].contiguous()
    after = length + 1

    def step():
        x.copy_(layer(x, table, length, after))
        length.add_(1), after.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(o.steps):
        graph.replay()
    t1.record()
    torch.cuda.synchronize()
    bits = pc.device_errors()
    if bits:
        raise SystemExit(f"device error bits {bits:#x}")
    held = 2 * int(length.sum()) * o.kv_heads * o.dim
    print(f"prompts of {new.tolist()} tokens, then {o.steps} steps of {o.seqs} sequences: "
          f"{t0.elapsed_time(t1) * 1e3 / o.steps:.1f} us a step, {held / 1e6:.2f} MB of codes cached")


if __name__ == "__main__":
    main()
