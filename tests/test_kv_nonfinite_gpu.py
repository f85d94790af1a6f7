"""GPU: a query row that sees a block with a non-finite scale gives NaN, whatever the block's codes and the sign of the
score: a key scale of infinity makes scores of -inf out of negative products, a value scale of infinity makes infinities
out of codes. Rows that do not see the block keep their bits."""
import numpy as np
import pytest

import popcorn_b200 as pc
from test_kv_gpu import Cache, _cast, _first, _pages, _rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("scale", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim", [64, 80, 128, 192])
def test_blocks_with_non_finite_scales(cuda, kind, scale, wide, dim):
    import torch

    rng = _rng("nonfinite", dim)
    heads, group, page, length, new = 2, 2, 16, [100, 1, 64], [60, 1, 64]
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    if wide:  # 16-bit types at dim 64 and 128: the kernel for prompts
        table = np.concatenate([table, np.full((len(length), (1 << 19) // page), -9, np.int32)], 1)
    c = Cache(rng, pages, heads, page, dim, cuda)
    c.dev.k.abs_().clamp_(1, 127)  # with the sign of a row's query: all scores of one sign
    c.dev.v.abs_().clamp_(1, 127)
    q = torch.from_numpy(np.abs(rng.standard_normal((sum(new), heads * group, dim))) + 0.1)
    q[::2] *= -1
    q = _cast(q.numpy(), kind).to(cuda)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    call = lambda: pc.kv_attention(c.dev, q, up(table), up(np.int32(length)), first=up(_first(new)), max_tokens=max(new))  # noqa: E731
    want = call()
    assert torch.isfinite(want).all()
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(length, new)])
    seq = np.repeat(np.arange(3), new)
    for scales in (c.dev.k_scale, c.dev.v_scale):
        for b, block in ((0, 5), (1, 0), (2, 2)):  # tokens 80 to 95, the only token, tokens 32 to 47
            at = int(table[b, block])
            kept = scales[at, 1].item()
            scales[at, 1] = scale
            got = call()
            sees = torch.zeros(want.shape[:2], dtype=torch.bool, device=cuda)
            sees[up((seq == b) & (pos >= block * page)), group:] = True
            assert torch.isnan(got[sees]).all()
            assert torch.equal(got[~sees], want[~sees])
            scales[at, 1] = kept
    assert pc.device_errors() == 0
