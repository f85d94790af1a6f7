"""GPU: the cache, the attention and the experts together, as examples/decode_layer.py runs them.

The layer is compared with the same layer in 64 bits over the values that the cache holds. Its projections are within
1e-5 normwise of that (popcorn's tolerance for the f32 path), attention and experts within 1e-5 of their inputs'; the
sums of a few such errors, grown by the softmax's slope (scores of a few units), stay under 2e-4 of a row's norm.
Experts are those that the layer picked: a near tie may go either way.
"""
import importlib.util
import os

import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_layer.py")
    spec = importlib.util.spec_from_file_location("decode_layer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _plain(layer, x, table, lengths, new, experts, weights):
    """The layer in 64 bits, reading keys and values from the cache."""
    import torch

    f64 = torch.float64
    full = lambda w: w[0].to(f64) * w[1].to(f64)[..., None]  # noqa: E731
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + layer.eps) * w.to(f64)  # noqa: E731
    x = x.to(f64)
    qkv = (norm(x, layer.norm1) @ full(layer.qkv).T).view(len(x), -1, layer.dim)
    group, half = layer.heads // layer.kv_heads, layer.dim // 2
    out, at = torch.zeros((len(x), layer.heads, layer.dim), dtype=f64, device=x.device), 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        k, v = (t.to(f64).transpose(1, 2).reshape(-1, layer.kv_heads, layer.dim)[:n].repeat_interleave(group, 1)
                for t in pc.kv_read(layer.cache, table[b].contiguous()))
        q = qkv[at: at + m, :layer.heads]
        cos, sin = (t[n - m: n, None].to(f64) for t in (layer.cos, layer.sin))
        q = torch.cat([q[..., :half] * cos - q[..., half:] * sin, q[..., half:] * cos + q[..., :half] * sin], -1)
        s = torch.einsum("ihd,jhd->hij", q, k) * layer.dim ** -0.5
        pos = torch.arange(n, device=x.device)
        s = s.masked_fill(pos[None, None] > pos[n - m:, None], float("-inf"))
        out[at: at + m] = torch.einsum("hij,jhd->ihd", s.softmax(-1), v)
        at += m
    x = x + out.flatten(1) @ full(layer.o).T
    z = norm(x, layer.norm2)
    g, u, d = (full(w) for w in (layer.gate, layer.up, layer.down))
    y = torch.zeros_like(x)
    for t in range(len(x)):
        for e, p in zip(experts[t].tolist(), weights[t].tolist()):
            y[t] += p * (d[e] @ (torch.nn.functional.silu(g[e] @ z[t]) * (u[e] @ z[t])))
    return x + y


@pytest.mark.parametrize("hidden, heads, kv_heads, dim, page", [(256, 8, 2, 64, 16), (320, 4, 4, 128, 32), (512, 6, 2, 80, 64)])
def test_layer_over_prompts_and_steps(cuda, hidden, heads, kv_heads, dim, page):
    import torch

    ex = _example()
    new = [37, 1, 16]
    table, pages = ex.block_table(64, len(new), page, cuda)
    layer = ex.DecoderLayer(hidden, heads, kv_heads, dim, 8, 192, 2, pages, page, positions=64, seed=hidden, device=cuda)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    lengths = list(new)
    x = torch.randn((sum(new), hidden), generator=torch.Generator(cuda).manual_seed(1), device=cuda)
    y, experts, weights = layer(x, table, ints([0] * 3), ints(lengths), first=ints([0, 37, 38, 54]), max_tokens=37,
                                routing=True)
    for step in range(4):
        want = _plain(layer, x, table, lengths, new, experts, weights)
        assert ((y - want).norm(dim=1) <= 2e-4 * want.norm(dim=1)).all()
        last = torch.tensor(new, device=cuda).cumsum(0) - 1
        x, new = y[last].contiguous(), [1, 1, 1]
        y, experts, weights = layer(x, table, ints(lengths), ints([n + 1 for n in lengths]), routing=True)
        lengths = [n + 1 for n in lengths]
    assert pc.device_errors() == 0


def test_example_runs(cuda, monkeypatch, capsys):
    import sys

    ex = _example()
    monkeypatch.setattr(sys, "argv", ["decode_layer.py", "--hidden", "512", "--heads", "8", "--kv-heads", "2", "--experts",
                                      "8", "--inter", "256", "--prompt", "90", "--steps", "3"])
    ex.main()
    assert "us a step" in capsys.readouterr().out
