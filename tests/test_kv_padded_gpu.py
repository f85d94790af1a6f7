"""GPU: attention over batches that are padded. The buffer of query rows is longer than the sequences' runs of them, as a
server's buffer of a fixed size is whose `first` changes from step to step. Every row of a sequence is answered, however
the sizes that the host knows (tokens, max_tokens, seqs) relate to the lengths that only the device knows, and rows of no
sequence keep what they hold. Tolerances are those of test_kv_gpu.py."""
import numpy as np
import pytest

import popcorn_b200 as pc
from test_kv_gpu import Cache, _cast, _check, _f32, _pages, _rng

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


def _up(a, cuda):
    return _torch().from_numpy(np.ascontiguousarray(a)).to(cuda)


def _wide(table, page):
    """A block table that could hold long sequences: the call is not a small one."""
    return np.concatenate([table, np.full((len(table), (1 << 19) // page), -9, np.int32)], 1)


PADDED = [
    # heads, group, dim, page, tokens, max_tokens, lengths, queries
    (2, 1, 64, 16, 256, 256, [300], [10]),            # one sequence in a buffer of 256 rows
    (2, 1, 128, 16, 256, None, [300], [10]),          # the same, max_tokens left to its default
    (1, 4, 128, 32, 128, 64, [200, 77], [3, 64]),     # tokens is seqs max_tokens, one sequence short
    (2, 2, 64, 16, 192, 64, [100, 40, 500], [1, 0, 2]),
    (1, 8, 128, 64, 100, 50, [60, 1000], [5, 50]),
    (1, 3, 64, 16, 80, 40, [7, 90], [12, 33]),        # more queries than tokens
    (2, 1, 128, 16, 96, 48, [200, 300], [48, 47]),
]


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", range(len(PADDED)))
def test_rows_behind_the_last_sequence(cuda, kind, wide, case):
    torch = _torch()
    heads, group, dim, page, tokens, most, length, new = PADDED[case]
    rng = _rng("padded", case)
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    table = _wide(table, page) if wide else table
    used = sum(new)
    q = _cast(rng.standard_normal((tokens, heads * group, dim)) * 1.5, kind)
    first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    out = torch.full((tokens, heads * group, dim), 7.0, dtype=q.dtype, device=cuda)
    lse = torch.full((tokens, heads * group), 7.0, device=cuda)
    got = pc.kv_attention(c.dev, q.to(cuda), _up(table, cuda), _up(np.int32(length), cuda), first=_up(first, cuda),
                          max_tokens=most, out=out, lse=lse)
    assert pc.device_errors() == 0
    assert (got[used:] == 7).all() and (lse[used:] == 7).all()
    _check(c, _f32(q[:used]).astype(np.float64), _f32(got[:used]).astype(np.float64),
           lse[:used].cpu().numpy().astype(np.float64), table, length, new, group, True, 0, dim ** -0.5, kind)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_graph_whose_sequence_boundaries_change(cuda, kind):
    torch = _torch()
    rng = _rng("padded graph", 1)
    heads, group, dim, page, length, most = 2, 2, 64, 16, [400, 333], 64
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    table = _wide(table, page)
    q = _cast(rng.standard_normal((2 * most, heads * group, dim)) * 1.5, kind)
    dq, dtable, dlength = q.to(cuda), _up(table, cuda), _up(np.int32(length), cuda)
    first = _up(np.int32([0, most, 2 * most]), cuda)
    out, lse = torch.zeros_like(dq), torch.zeros((2 * most, heads * group), device=cuda)
    call = lambda: pc.kv_attention(c.dev, dq, dtable, dlength, first=first, max_tokens=most, out=out, lse=lse)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new in ([64, 64], [5, 15], [1, 64], [0, 30], [64, 0]):
        first.copy_(_up(np.int32([0, new[0], sum(new)]), cuda))
        out.fill_(7), lse.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        used = sum(new)
        assert (out[used:] == 7).all() and (lse[used:] == 7).all()
        _check(c, _f32(q[:used]).astype(np.float64), _f32(out[:used]).astype(np.float64),
               lse[:used].cpu().numpy().astype(np.float64), table, length, new, group, True, 0, dim ** -0.5, kind)
    assert pc.device_errors() == 0
