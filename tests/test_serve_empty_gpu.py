"""GPU: the serving operators' Python functions take batches without tokens or without sequences: they give empty results,
or the caller's outputs as they are, like the C entry points' calls without work."""
import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_batches_without_work(cuda, kind):
    import torch

    dtype = getattr(torch, kind)
    cache = pc.KvCache.empty(4, 2, 64, 16, device=cuda)
    cache.k.fill_(3), cache.v.fill_(4), cache.k_scale.fill_(0.5), cache.v_scale.fill_(0.25)
    z = lambda *shape, dtype=dtype: torch.zeros(shape, dtype=dtype, device=cuda)  # noqa: E731
    i32 = lambda *shape: z(*shape, dtype=torch.int32)  # noqa: E731
    cos = z(8, 32, dtype=torch.float32)
    for seqs, width in ((0, 0), (0, 3), (2, 3), (1, 0)):
        table, start, first = i32(seqs, width), i32(seqs), i32(seqs + 1)
        out = pc.kv_append(cache, z(0, 2, 64), z(0, 2, 64), table, start, first=first, q=z(0, 4, 64), cos=cos, sin=cos)
        assert out.shape == (0, 4, 64) and out.dtype == dtype
        assert pc.kv_append(cache, z(0, 2, 64), z(0, 2, 64), table, start, first=first) is None
        lse = z(0, 4, dtype=torch.float32)
        for most in (None, 1, 5):
            out = pc.kv_attention(cache, z(0, 4, 64), table, start, first=first, max_tokens=most, lse=lse)
            assert out.shape == (0, 4, 64) and out.dtype == dtype
        if seqs == 0:  # one token a sequence, of none
            assert pc.kv_append(cache, z(0, 2, 64), z(0, 2, 64), table, start) is None
            assert pc.kv_attention(cache, z(0, 4, 64), table, start).shape == (0, 4, 64)
    # tokens of no sequence
    out = torch.full((3, 4, 64), 7.0, dtype=dtype, device=cuda)
    none = dict(first=i32(1))
    assert (pc.kv_attention(cache, z(3, 4, 64), i32(0, 2), i32(0), out=out, **none) == 7).all()
    assert (pc.kv_append(cache, z(3, 2, 64), z(3, 2, 64), i32(0, 2), i32(0), q=z(3, 4, 64), q_out=out, **none) == 7).all()
    torch.cuda.synchronize()
    assert (cache.k == 3).all() and (cache.v == 4).all() and (cache.k_scale == 0.5).all() and (cache.v_scale == 0.25).all()
    assert pc.device_errors() == 0


def test_checks_come_before_empty_batches(cuda):
    import torch

    cache = pc.KvCache.empty(4, 2, 64, 16, device=cuda)
    z = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=cuda)  # noqa: E731
    i32 = lambda *shape: z(*shape, dtype=torch.int32)  # noqa: E731
    for k in (z(0, 3, 64), z(0, 2, 32), z(0, 2, 64, dtype=torch.float64)):
        with pytest.raises(ValueError, match="kv_append"):
            pc.kv_append(cache, k, k, i32(0, 3), i32(0))
    for q in (z(0, 3, 64), z(0, 2, 32), z(0, 2, 64, dtype=torch.float64)):
        with pytest.raises(ValueError, match="kv_attention"):
            pc.kv_attention(cache, q, i32(0, 3), i32(0))


def test_experts_without_tokens(cuda):
    import torch

    E, F, K = 4, 32, 64
    z = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=cuda)  # noqa: E731
    codes = lambda *shape: z(*shape, dtype=torch.int8)  # noqa: E731
    layer = [z(E, K), codes(E, F, K), z(E, F), codes(E, F, K), z(E, F), codes(E, K, F), z(E, K)]
    assert pc.moe(z(0, K), *layer, top_k=2).shape == (0, K)
    out, experts, weights = pc.moe(z(0, K), *layer, top_k=2, routing=True)
    assert out.shape == (0, K) and experts.shape == weights.shape == (0, 2) and experts.dtype is torch.int32
    with pytest.raises(ValueError, match="moe"):
        pc.moe(z(0, K + 1), *layer, top_k=2)
