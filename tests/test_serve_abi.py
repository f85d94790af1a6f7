"""CPU: the serving operators' C entry points (include/popcorn_serve.h) are declared, exported and keep the library's
argument conventions for calls that launch nothing: a null buffer that is not optional is refused before any size is
looked at, a call without work succeeds, sizes the kernels do not take are refused."""
import ctypes
import os
import re
import subprocess

import pytest

import popcorn_b200 as pc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x1000  # never dereferenced
BAD, OK = pc.POPCORN_ERROR_INVALID_VALUE, pc.POPCORN_SUCCESS


def test_header_python_list_library_and_archive_agree(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "popcorn_serve.h")).read(), flags=re.S)
    names = re.findall(r"^\s*(?:popcornStatus_t|int64_t)\s+(popcorn\w+)\s*\(", text, flags=re.M)
    assert sorted(names) == sorted(pc.SERVE_SYMBOLS)
    out = subprocess.run(["nm", "-g", "--defined-only", os.path.join(ROOT, "lib", "libpopcorn.a")], capture_output=True,
                         text=True, check=True).stdout
    defined = set(re.findall(r" [TW] (\w+)$", out, flags=re.M))
    for name in names:
        assert hasattr(lib, name) and name in defined, name


def test_cache_struct_layout_matches_the_header():
    assert ctypes.sizeof(pc.KvCacheStruct) == 64
    assert [getattr(pc.KvCacheStruct, f).offset for f, _ in pc.KvCacheStruct._fields_] == list(range(0, 64, 8))


def _cache(**change):
    c = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, pages=4, heads=2, page_size=16, dim=64)
    c.update(change)
    return pc.KvCacheStruct(*(c[f] for f, _ in pc.KvCacheStruct._fields_))


def _append(lib, cache=None, **change):
    a = dict(k=FAKE, kt=128, kh=64, v=FAKE, vt=128, vh=64, type=0, table=FAKE, width=3, first=FAKE, start=FAKE, seqs=2,
             tokens=5, q_out=None, q=None, qt=256, qh=64, q_heads=4, cos=None, sin=None, positions=10, rot=64, inter=0,
             stream=None)
    assert set(change) <= set(a)
    a.update(change)
    c = cache or _cache()
    return lib.popcornKvAppend(ctypes.byref(c), *a.values())


def _attend(lib, struct=None, **change):
    a = dict(out=FAKE, lse=None, q=FAKE, qt=256, qh=64, type=0, cache=None, table=FAKE, width=3, first=FAKE, length=FAKE,
             seqs=2, tokens=5, most=4, q_heads=4, causal=1, window=0, scale=0.1, ws=None, bytes=0, stream=None)
    assert set(change) <= set(a)
    c = struct or _cache()
    a["cache"] = ctypes.byref(c)
    a.update(change)
    return lib.popcornKvAttention(*a.values())


CACHES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0)]
WRONG_CACHES = [dict(k=FAKE + 8), dict(pages=0), dict(heads=0), dict(page_size=8), dict(page_size=24),
                dict(page_size=512), dict(dim=8), dict(dim=72), dict(dim=272)]


def test_append_refusals(lib):
    for c in CACHES + WRONG_CACHES:
        assert _append(lib, _cache(**c)) == BAD, c
    for c in CACHES:  # null before sizes
        assert _append(lib, _cache(**c), tokens=0) == BAD, c
    for name in ("k", "v", "table", "start"):
        assert _append(lib, **{name: None}) == BAD and _append(lib, tokens=0, **{name: None}) == BAD, name
    for change in (dict(q=FAKE), dict(q_out=FAKE), dict(cos=FAKE), dict(sin=FAKE), dict(type=3), dict(type=-1),
                   dict(width=0), dict(first=None), dict(q=FAKE, q_out=FAKE + 16, q_heads=0),
                   dict(q=FAKE, q_out=FAKE, qh=128), dict(cos=FAKE, sin=FAKE, rot=12), dict(cos=FAKE, sin=FAKE, rot=72),
                   dict(cos=FAKE, sin=FAKE, rot=0), dict(cos=FAKE, sin=FAKE, positions=0)):
        assert _append(lib, **change) == BAD, change
    for change in (dict(tokens=0), dict(seqs=0), dict(tokens=-1), dict(seqs=-3)):
        assert _append(lib, **change) == OK, change


def test_read_refusals(lib):
    read = lambda cache, k=FAKE, v=FAKE, kind=0, pages=FAKE, n=2: lib.popcornKvRead(  # noqa: E731
        k, v, kind, ctypes.byref(cache), pages, n, None)
    for c in CACHES + WRONG_CACHES:
        assert read(_cache(**c)) == BAD, c
    for change in (dict(k=0), dict(v=0), dict(pages=0), dict(kind=7), dict(k=FAKE + 4), dict(v=FAKE + 8),
                   dict(n=1 << 31)):
        assert read(_cache(), **change) == BAD, change
    assert lib.popcornKvRead(FAKE, FAKE, 0, None, FAKE, 2, None) == BAD
    for n in (0, -1):
        assert read(_cache(), n=n) == OK


def test_attention_refusals(lib):
    for c in CACHES + WRONG_CACHES:
        assert _attend(lib, _cache(**c)) == BAD, c
    for name in ("out", "q", "table", "length", "cache"):
        assert _attend(lib, **{name: None}) == BAD and _attend(lib, tokens=0, **{name: None}) == BAD, name
    for change in (dict(type=5), dict(width=0), dict(width=1 << 28), dict(first=None), dict(most=0), dict(q_heads=3),
                   dict(q_heads=0), dict(q_heads=65538), dict(out=FAKE + 4), dict(tokens=1 << 30)):
        assert _attend(lib, **change) == BAD, change
    for change in (dict(tokens=0), dict(seqs=0), dict(tokens=-1)):
        assert _attend(lib, **change) == OK, change
    c = _cache()
    for sizes in ((9, 2, 5, 4, 4), (0, 0, 5, 4, 4), (0, 2, 5, 4, 3), (0, 2, 0, 4, 4)):
        assert lib.popcornKvAttentionWorkspace(ctypes.byref(c), *sizes) == 0, sizes
    assert lib.popcornKvAttentionWorkspace(None, 0, 2, 5, 4, 4) == 0


def test_moe_refusals(lib):
    def call(*null, experts=None, weights=None, M=2, K=64, F=32, E=4, top=2, ws=None, n=0):
        names = ["out", "x", "router", "qg", "sg", "qu", "su", "qd", "sd"]
        p = {name: 0 if name in null else FAKE for name in names}
        return lib.popcornMoe_i8f32(p["out"], experts, weights, *(p[n] for n in names[1:]), M, K, F, E, top, 1, ws, n,
                                    None)

    for name in ("out", "x", "router", "qg", "sg", "qu", "su", "qd", "sd"):
        assert call(name) == BAD and call(name, M=0) == BAD, name
    for change in (dict(experts=FAKE), dict(weights=FAKE), dict(top=0), dict(top=5), dict(top=-1), dict(E=257, top=1),
                   dict(E=64, top=17), dict(K=65552), dict(F=65552), dict(ws=FAKE, n=16), dict(ws=FAKE + 16, n=1 << 30)):
        assert call(**change) == BAD, change
    for change in (dict(M=0), dict(K=0), dict(F=0), dict(E=0), dict(M=-4)):
        assert call(**change) == OK, change
    assert lib.popcornMoeWorkspace(2, 64, 32, 4, 5) == 0 and lib.popcornMoeWorkspace(0, 64, 32, 4, 2) == 0
    need = [lib.popcornMoeWorkspace(m, 64, 32, 4, 2) for m in (1, 8, 64, 1000)]
    assert 0 < need[0] < need[1] < need[2] == need[3]  # 64 tokens are one pass


def test_binding_refuses_tensors_that_are_not_on_a_gpu():
    torch = pytest.importorskip("torch")
    x = torch.zeros((2, 64))
    with pytest.raises(ValueError, match="x: a CUDA tensor"):
        pc.moe(x, x, x, x, x, x, x, x, top_k=1)
    q, s = torch.zeros((2, 1, 16, 64), dtype=torch.int8), torch.zeros((2, 1))
    for args in ((q, q, s, s), (x, x, s, s), (q, q[:1], s, s), (q, q, s[0], s), (q.float(), q, s, s)):
        with pytest.raises(ValueError, match="KvCache"):
            pc.KvCache(*args)
