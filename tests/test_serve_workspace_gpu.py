"""GPU: the serving operators' workspaces (include/popcorn_serve.h): the library's pool, a caller's buffer whatever is in
it, and the refusal of one that is too small or unaligned give the same bits, or leave the output alone."""
import ctypes

import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu

BAD, OK = pc.POPCORN_ERROR_INVALID_VALUE, pc.POPCORN_SUCCESS


def _run(call, need, align, out):
    """call(workspace pointer or None, bytes) -> status, results in out."""
    import torch

    assert need > 0
    torch.cuda.synchronize()
    assert call(None, 0) == OK
    torch.cuda.synchronize()
    want = out.clone()
    for fill in (0, 255):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=out.device)
        assert ws.data_ptr() % align == 0
        out.fill_(7)
        torch.cuda.synchronize()
        assert call(ws.data_ptr(), need) == OK
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    ws = torch.zeros(need + 2 * align, dtype=torch.uint8, device=out.device)
    out.fill_(7)
    torch.cuda.synchronize()
    assert call(ws.data_ptr(), need - 1) == BAD
    assert call(ws.data_ptr() + align // 2, need + align) == BAD
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert pc.device_errors() == 0


@pytest.mark.parametrize("kind, code", [("float32", pc.TYPE_F32), ("float16", pc.TYPE_F16), ("bfloat16", pc.TYPE_BF16)])
@pytest.mark.parametrize("new, width", [([1, 1, 1], 40), ([5, 1, 3], 40), ([200, 90, 1], 40), ([200, 90, 1], 20000)])
def test_attention_workspace(cuda, kind, code, new, width):
    import torch

    lib = pc.load_library()
    gen = torch.Generator(cuda).manual_seed(5)
    pages, heads, group, page, dim = 130, 2, 2, 16, 64
    codes = [torch.randint(-127, 128, (pages, heads, page, dim), generator=gen, dtype=torch.int8, device=cuda) for _ in "kv"]
    scales = [torch.rand((pages, heads), generator=gen, device=cuda) / 60 for _ in "kv"]
    cache = pc.KvCache(*codes, *scales)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.zeros((3, width), dtype=torch.int32, device=cuda)
    table[:, :40] = ints(list(range(120))).view(3, 40)
    first, length = ints([0, new[0], new[0] + new[1], sum(new)]), ints([600, 333, 40])
    q = torch.randn((sum(new), heads * group, dim), generator=gen, device=cuda).to(getattr(torch, kind))
    out = torch.empty_like(q)
    struct = ctypes.byref(cache._struct)
    need = lib.popcornKvAttentionWorkspace(struct, code, 3, sum(new), max(new), heads * group)

    def call(ws, size):
        return lib.popcornKvAttention(out.data_ptr(), None, q.data_ptr(), heads * group * dim, dim, code, struct,
                                      table.data_ptr(), width, first.data_ptr(), length.data_ptr(), 3, sum(new), max(new),
                                      heads * group, 1, 0, dim ** -0.5, ws, size, None)

    _run(call, need, 16, out)


@pytest.mark.parametrize("M, K, F, E, top", [(1, 256, 128, 8, 2), (9, 2560, 64, 4, 2), (70, 128, 48, 6, 3), (5, 100, 52, 4, 2)])
def test_moe_workspace(cuda, M, K, F, E, top):
    import torch

    lib = pc.load_library()
    gen = torch.Generator(cuda).manual_seed(6)
    codes = lambda *s: torch.randint(-127, 128, s, generator=gen, dtype=torch.int8, device=cuda)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=gen, device=cuda) / 1000  # noqa: E731
    x, router = torch.randn((M, K), generator=gen, device=cuda), torch.randn((E, K), generator=gen, device=cuda)
    w = [codes(E, F, K), rand(E, F), codes(E, F, K), rand(E, F), codes(E, K, F), rand(E, K)]
    out = torch.empty_like(x)

    def call(ws, size):
        return lib.popcornMoe_i8f32(out.data_ptr(), None, None, x.data_ptr(), router.data_ptr(), *(t.data_ptr() for t in w),
                                    M, K, F, E, top, 1, ws, size, None)

    _run(call, lib.popcornMoeWorkspace(M, K, F, E, top), 256, out)
