"""GPU: what attention adds to the rounding of its f16 and f32 outputs.

Rounding the exact result to f16 has a certain root mean square error. The kernels' other errors (scores in f32 from exact
products, probabilities of 22 bits, f32 sums) are of the order of 2^-18 of the result, a fiftieth of it; together they may
make the error at most 5 % larger, which leaves them a third of the rounding's. One f16 for a probability is an error of
the same size as the rounding and makes it 35 % larger. The same holds in calls for few rows and for prompts."""
import numpy as np
import pytest

import popcorn_b200 as pc
from test_kv_gpu import Cache, _attend, _cast, _f32, _first, _pages, _rng, lse_v

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("length, new", [([700, 300], [1, 1]), ([700, 300], [9, 4]), ([600, 333], [150, 70]), ([64, 64], [64, 64])])
def test_f16_results_are_nearly_the_rounded_exact_ones(cuda, dim, wide, length, new):
    import torch

    rng = _rng("prompt error", dim, *new)
    heads, group, page = 2, 2, 16
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    if wide:  # not a small call
        table = np.concatenate([table, np.full((len(length), (1 << 19) // page), -9, np.int32)], 1)
    q = _cast(rng.standard_normal((sum(new), heads * group, dim)), "float16")
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    got = pc.kv_attention(c.dev, q.to(cuda), up(table), up(np.int32(length)), first=up(_first(new)), max_tokens=max(new))
    lse_v.clear()
    want = _attend(c, _f32(q).astype(np.float64), table, length, new, group, True, 0, dim ** -0.5)[0]
    rounding = np.linalg.norm(want.astype(np.float16).astype(np.float64) - want)
    assert np.linalg.norm(_f32(got).astype(np.float64) - want) <= 1.05 * rounding
