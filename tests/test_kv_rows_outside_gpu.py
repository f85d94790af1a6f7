"""GPU: an append leaves rows that belong to no sequence alone: those before the first sequence's run as those behind the
last one's. Their keys, values and queries are not looked at, and no error is reported."""
import numpy as np
import pytest

import popcorn_b200 as pc
from test_kv_gpu import Cache, _cast, _f32, _put, _rng, _tables, _turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("old, first, tokens", [([0, 5], [2, 5, 9], 12), ([30, 0], [7, 8, 8], 8), ([3, 20], [60, 150, 200], 230)])
def test_rows_of_no_sequence(cuda, kind, rotate, old, first, tokens):
    import torch

    rng = _rng("outside rows", tokens)
    heads, q_heads, dim, page = 2, 4, 64, 16
    table = np.int32(rng.permutation(24)[:22].reshape(2, 11))
    c = Cache(rng, 24, heads, page, dim, cuda)
    k, v = (_cast(rng.standard_normal((tokens, heads, dim)), kind) for _ in range(2))
    q = _cast(rng.standard_normal((tokens, q_heads, dim)), kind)
    lo, hi, new = first[0], first[-1], np.diff(first).tolist()
    pos = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)]).astype(int)
    cos, sin = _tables(256, dim) if rotate else (None, None)
    turned = lambda x: _turn(_f32(x[lo:hi]), pos, cos, sin, False) if rotate else _f32(x[lo:hi])  # noqa: E731
    _put(c.k, c.ks, turned(k), table, old, new, page)
    _put(c.v, c.vs, _f32(v[lo:hi]), table, old, new, page)
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    out = torch.full((tokens, q_heads, dim), 7.0, dtype=q.dtype, device=cuda)
    k[:lo], k[hi:], v[:lo], v[hi:] = (float("nan"),) * 4
    pc.kv_append(c.dev, k.to(cuda), v.to(cuda), up(table), up(np.int32(old)), first=up(np.int32(first)), q=q.to(cuda),
                 q_out=out, cos=up(cos), sin=up(sin))
    c.same()
    assert pc.device_errors() == 0
    assert torch.equal(out[lo:hi].cpu(), _cast(turned(q), kind))
    assert (out[:lo] == 7).all() and (out[hi:] == 7).all()
