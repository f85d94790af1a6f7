"""GPU: the experts' router may be the output of the call before on the same stream, also of one that lets the next
kernel start before it has written: the library's decode products, appends and read-backs do."""
import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu

E, F, K = 4, 64, 4096


def _producers(kind, gen, cuda):
    """Calls that write an f32 router [E, K], each another one, and the router's memory."""
    import torch

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    if kind == "product":  # one row of activations, E K output channels
        inner = 2048
        w = torch.randint(-127, 128, (E * K, inner), generator=gen, dtype=torch.int8, device=cuda)
        scale = torch.full((E * K,), 3e-4 / inner ** 0.5, device=cuda)
        out = torch.zeros((1, E * K), device=cuda)
        xs = [torch.randn((1, inner), generator=gen, device=cuda) for _ in range(8)]
        return [lambda x=x: pc.dequantize_matmul(x, w, scale, out=out) for x in xs], out.view(E, K)
    cache = pc.KvCache.empty(16, 4, 128, 16, device=cuda)
    if kind == "append":  # the rotated queries of E sequences, 32 heads of 128
        out = torch.zeros((E, 32, 128), device=cuda)
        k = torch.randn((E, 4, 128), generator=gen, device=cuda)
        table, start = i32(*range(E)).view(E, 1), i32(*range(E))
        qs = [torch.randn((E, 32, 128), generator=gen, device=cuda) / 40 for _ in range(8)]
        return [lambda q=q: pc.kv_append(cache, k, k, table, start, q=q, q_out=out) for q in qs], out.view(E, K)
    out, v = torch.zeros((2, 4, 16, 128), device=cuda), torch.zeros((2, 4, 16, 128), device=cuda)  # two pages' values
    cache.k.copy_(torch.randint(-127, 128, cache.k.shape, generator=gen, dtype=torch.int8, device=cuda))
    cache.k_scale.fill_(3e-4)
    pages = [i32(2 * a, 2 * a + 1) for a in range(8)]
    return [lambda p=p: pc.kv_read(cache, p, k_out=out, v_out=v) for p in pages], out.view(E, K)


@pytest.mark.parametrize("kind", ["product", "append", "read"])
def test_router_written_by_the_call_before(cuda, kind):
    import torch

    gen = torch.Generator(cuda).manual_seed(len(kind))
    codes = lambda *s: torch.randint(-127, 128, s, generator=gen, dtype=torch.int8, device=cuda)  # noqa: E731
    layer = [codes(E, F, K), torch.rand((E, F), generator=gen, device=cuda) / 5000, codes(E, F, K),
             torch.rand((E, F), generator=gen, device=cuda) / 5000, codes(E, K, F), torch.rand((E, K), generator=gen, device=cuda) / 500]
    x = torch.randn((3, K), generator=gen, device=cuda)
    calls, router = _producers(kind, gen, cuda)
    wants = []
    for call in calls:
        call()
        torch.cuda.synchronize()
        wants.append([t.clone() for t in pc.moe(x, router, *layer, top_k=2, routing=True)])
        torch.cuda.synchronize()
    assert not any(torch.equal(wants[0][2], w[2]) for w in wants[1:])
    for _ in range(20):
        gots = []
        for call in calls:
            call()
            gots.append(pc.moe(x, router, *layer, top_k=2, routing=True))
        for got, want in zip(gots, wants):
            for g, t in zip(got, want):
                assert torch.equal(g, t)
