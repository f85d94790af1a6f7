"""GPU: the serving operators on a stream given with the call while another one is current. Workspaces and outputs belong
to the given stream: earlier work of the current stream does not write into them, later tensors of the current stream do
not take a workspace's memory while the kernels run, and an output that the current stream still reads is not handed out
again."""
import threading

import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu

DELAY = 20_000_000  # clock cycles, about 10 ms: long against a call, on either stream


def _ints(cuda, *v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device=cuda)


def _attention(kind, new):
    """Split tasks: partial results and join entries go through the workspace."""
    def make(cuda):
        import torch

        gen = torch.Generator(cuda).manual_seed(7)
        heads, group, dim, page, pages = 2, 4, 128, 16, 512
        codes = [torch.randint(-127, 128, (pages, heads, page, dim), generator=gen, dtype=torch.int8, device=cuda) for _ in "kv"]
        scales = [torch.rand((pages, heads), generator=gen, device=cuda) / 60 for _ in "kv"]
        cache = pc.KvCache(*codes, *scales)
        width = (1 << 19) // page if new > 1 else pages // 2
        table = torch.zeros((2, width), dtype=torch.int32, device=cuda)
        table[:, : pages // 2] = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).view(2, -1).to(cuda, torch.int32)
        first, length = _ints(cuda, 0, new, 2 * new), _ints(cuda, 4000, 3333)
        q = torch.randn((2 * new, heads * group, dim), generator=gen, device=cuda).to(getattr(torch, kind))
        q2 = (q * 2 + 1).contiguous()

        def call(other=False, **kw):
            return [pc.kv_attention(cache, q2 if other else q, table, length, first=first, max_tokens=new, **kw)]

        return call

    return make


def _moe(tokens, routing):
    def make(cuda):
        import torch

        gen = torch.Generator(cuda).manual_seed(8)
        E, F, K = 16, 256, 1024
        codes = lambda *s: torch.randint(-127, 128, s, generator=gen, dtype=torch.int8, device=cuda)  # noqa: E731
        rand = lambda *s: torch.rand(s, generator=gen, device=cuda) / 2000  # noqa: E731
        layer = [torch.randn((E, K), generator=gen, device=cuda) / 16, codes(E, F, K), rand(E, F), codes(E, F, K), rand(E, F),
                 codes(E, K, F), rand(E, K)]
        x = torch.randn((tokens, K), generator=gen, device=cuda)
        x2 = x.flip(0).contiguous() + 0.5

        def call(other=False, **kw):
            got = pc.moe(x2 if other else x, *layer, top_k=3, routing=routing, **kw)
            return list(got) if routing else [got]

        return call

    return make


def _append(cuda):
    import torch

    gen = torch.Generator(cuda).manual_seed(9)
    cache = pc.KvCache.empty(64, 2, 64, 16, device=cuda)
    k, q = torch.randn((300, 2, 64), generator=gen, device=cuda), torch.randn((300, 8, 64), generator=gen, device=cuda)
    q2, table = q + 1, torch.arange(40, dtype=torch.int32, device=cuda).view(2, 20)
    first, start = _ints(cuda, 0, 200, 300), _ints(cuda, 0, 0)
    cos, sin = torch.rand((300, 32), generator=gen, device=cuda), torch.rand((300, 32), generator=gen, device=cuda)
    return lambda other=False, **kw: [pc.kv_append(cache, k, k, table, start, first=first, q=q2 if other else q, cos=cos,
                                                   sin=sin, **kw)]


def _read(cuda):
    import torch

    gen = torch.Generator(cuda).manual_seed(10)
    cache = pc.KvCache.empty(64, 2, 64, 16, device=cuda)
    cache.k.copy_(torch.randint(-127, 128, cache.k.shape, generator=gen, dtype=torch.int8, device=cuda))
    cache.v.copy_(cache.k.flip(0)), cache.k_scale.fill_(0.5), cache.v_scale.fill_(0.25)
    lists = torch.arange(64, dtype=torch.int32, device=cuda), torch.arange(63, -1, -1, dtype=torch.int32, device=cuda)
    return lambda other=False, **kw: list(pc.kv_read(cache, lists[other], **kw))


OPERATORS = {"rows f32": _attention("float32", 1), "rows bf16": _attention("bfloat16", 1), "prompt f16": _attention("float16", 70),
             "moe 1": _moe(1, False), "moe 9": _moe(9, True), "moe 70": _moe(70, False), "append": _append, "read": _read}


def _sizes(call):
    """Bytes of the outputs and of what else a call allocates."""
    import torch

    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    most = torch.cuda.max_memory_allocated() - before
    held = [t.untyped_storage().nbytes() for t in out]
    return held + ([most - sum(held)] if most > sum(held) else [])


@pytest.mark.parametrize("name", OPERATORS)
def test_given_stream_and_tensors_of_the_current_one(cuda, name):
    import torch

    call = OPERATORS[name](cuda)
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    sizes = _sizes(call)
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()

    def block(n, fill):
        return torch.full((n,), fill, dtype=torch.uint8, device=cuda)

    for fill in (0xFF, 0x00, 0x3C):
        # Blocks that the current stream has still to write to are free again when the call allocates.
        torch.cuda.empty_cache()
        torch.cuda._sleep(DELAY)
        for n in sizes:
            block(n, fill)
        got = call(stream=side)
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        # The call's kernels begin late, after the current stream has taken and written blocks of the same sizes.
        del got
        with torch.cuda.stream(side):
            torch.cuda._sleep(DELAY)
        got = call(stream=side)
        kept = [block(n, fill) for n in sizes * 3]
        current.synchronize()
        side.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert all((t == fill).all() for t in kept)  # nor did the kernels write into those
        del got, kept
    assert pc.device_errors() == 0


@pytest.mark.parametrize("name", OPERATORS)
def test_output_that_the_current_stream_still_reads(cuda, name):
    import torch

    call = OPERATORS[name](cuda)
    want, others = [t.clone() for t in call()], [t.clone() for t in call(True)]
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    for _ in range(3):
        got = call(stream=side)
        current.wait_stream(side)
        torch.cuda._sleep(DELAY)
        copies = [t.clone() for t in got]  # after the delay
        del got
        again = call(True, stream=side)  # at once
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(copies, want))
        assert all(torch.equal(g, w) for g, w in zip(again, others))


@pytest.mark.parametrize("name", OPERATORS)
def test_handles_of_the_default_streams_and_graphs(cuda, name):
    import torch

    call = OPERATORS[name](cuda)
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for handle in (0, 1, 2, torch.cuda.default_stream(), side, side.cuda_stream):  # 1, 2: legacy, per thread
            got = call(stream=handle)
            torch.cuda.synchronize()
            assert all(torch.equal(g, w) for g, w in zip(got, want)), handle
            assert torch.cuda.current_stream() == side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fork = torch.cuda.Stream()
        fork.wait_stream(torch.cuda.current_stream())
        got = call(stream=fork)
        torch.cuda.current_stream().wait_stream(fork)
    for _ in range(2):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_threads_on_their_own_streams(cuda):
    import torch

    calls = [make(cuda) for make in OPERATORS.values()]
    wants = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        try:
            for _ in range(10):
                for call, want in zip(calls[i:] + calls[:i], wants[i:] + wants[:i]):
                    got = call(stream=stream)
                    stream.synchronize()
                    if not all(torch.equal(g, w) for g, w in zip(got, want)):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    assert pc.device_errors() == 0
