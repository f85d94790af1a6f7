"""GPU: windows as wide as an int64 is hide nothing, whatever the positions: the answer is the one without a window, bit
for bit."""
import numpy as np
import pytest

import popcorn_b200 as pc
from test_kv_gpu import Cache, _cast, _first, _pages, _rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("length, new", [([2, 70], [9, 3]), ([30, 200], [90, 60])])  # more queries than tokens among them
def test_windows_wider_than_every_position(cuda, kind, causal, wide, length, new):
    import torch

    rng = _rng("window", len(kind) + causal)
    heads, group, dim, page = 2, 2, 64, 16
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    if wide:  # not a small call
        table = np.concatenate([table, np.full((len(length), (1 << 19) // page), -9, np.int32)], 1)
    q = _cast(rng.standard_normal((sum(new), heads * group, dim)), kind).to(cuda)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    call = lambda window: pc.kv_attention(c.dev, q, up(table), up(np.int32(length)), first=up(_first(new)),  # noqa: E731
                                          max_tokens=max(new), causal=causal, window=window)
    want = call(0)
    assert want[-1].any()
    for window in ((1 << 31) - 1, 1 << 31, 1 << 32, (1 << 63) - 1):
        assert torch.equal(call(window), want), window
    assert pc.device_errors() == 0
