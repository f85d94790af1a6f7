"""GPU: the paged 8-bit key/value cache (include/popcorn_serve.h): append with rotation, read-back, attention.

Append and read-back are IEEE f32 operation by operation, so they are compared bit for bit with a numpy restatement.
Attention is compared with softmax attention in 64 bits over the cached values. Its tolerance follows from its
arithmetic, per element and relative to the largest visible |value| V:

* a score is exact but for the query's fixed point (half a unit of qmax / 32512 for 16-bit types, of qmax / 2^21 for
  f32) and a few f32 roundings of the score: ds = scale * sum|k| * unit / 2 + 8 * 2^-24 * |s|max
* a probability changes by a factor of at most exp(2 ds) relative to the others: 2 ds V
* probabilities are rounded to f16 (2^-11) for 16-bit types, the f32 path keeps 22 bits and sums in f32 over at most
  a few hundred tiles: 2^-11 V or 2^-19 V
* the result is rounded to its type: 2^-11, 2^-8 or 2^-24 of |out| <= V, and f16 has no values between 0 and 2^-24
"""
import zlib

import numpy as np
import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _torch():
    import torch

    return torch


def _rng(*key):
    return np.random.default_rng([zlib.crc32(k.encode()) if isinstance(k, str) else k for k in key])


def _pages(rng, need, spare=3):
    """Block table for sequences of `need` pages each, in random order; unused entries are nonsense."""
    total = sum(need) + spare
    order = rng.permutation(total)
    table = np.full((len(need), max(max(need), 1) + 1), -7, np.int32)
    table[:, -1] = 1 << 30
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    return table, total


def _first(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def _cast(a, kind):
    return _torch().from_numpy(np.ascontiguousarray(a, np.float32)).to(getattr(_torch(), kind))


def _f32(t):
    return t.float().cpu().numpy()


# ------------------------------------------------------------------ append
def _turn(x, pos, cos, sin, inter):
    """f32, one rounding per product and sum."""
    r = cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    out = x.copy()
    a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if inter else (x[..., :r], x[..., r:2 * r])
    lo, hi = a * c - b * s, b * c + a * s
    if inter:
        out[..., 0:2 * r:2], out[..., 1:2 * r:2] = lo, hi
    else:
        out[..., :r], out[..., r:2 * r] = lo, hi
    return out


def _put(codes, scale, x, table, old, new, page):
    f32 = np.float32
    first = _first(new)
    for b, (o, n) in enumerate(zip(old, new)):
        for p in range(o // page, (o + n - 1) // page + 1 if n else 0):
            lo, hi = max(o, p * page), min(o + n, (p + 1) * page)
            at, row = table[b, p], lo - p * page
            v = x[first[b] + lo - o: first[b] + hi - o]
            for h in range(codes.shape[1]):
                before = scale[at, h] if row else f32(0)
                with np.errstate(invalid="ignore"):
                    now = np.fmax.reduce(np.abs(v[:, h]), axis=None, initial=f32(0)) / f32(127)
                if now < 2.0 ** -80:
                    now = f32(0)
                s = max(before, now)
                if row and s != before:
                    codes[at, h, :row] = np.rint(codes[at, h, :row].astype(f32) * (before / s)).astype(np.int8)
                if s > 0:
                    with np.errstate(invalid="ignore"):
                        q = np.rint(v[:, h] / s)
                    q = np.clip(np.where(np.isnan(q), 0, q), -128, 127)
                else:
                    q = np.zeros_like(v[:, h])
                codes[at, h, row: row + hi - lo] = q.astype(np.int8)
                scale[at, h] = s


class Cache:
    """A cache on the device and its copy on the host."""

    def __init__(self, rng, pages, heads, page, dim, cuda):
        torch = _torch()
        self.k, self.v = (np.clip(np.rint(rng.standard_normal((pages, heads, page, dim)) * 40), -128, 127)
                          .astype(np.int8) for _ in range(2))
        self.ks, self.vs = ((rng.random((pages, heads)) * 0.03 + 0.005).astype(np.float32) for _ in range(2))
        self.dev = pc.KvCache(*(torch.from_numpy(a.copy()).to(cuda) for a in (self.k, self.v, self.ks, self.vs)))

    def same(self):
        for name in ("k", "v", "k_scale", "v_scale"):
            host = getattr(self, name.replace("_scale", "s"))
            np.testing.assert_array_equal(getattr(self.dev, name).cpu().numpy(), host, err_msg=name)


def _tables(positions, rot):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


APPENDS = [
    # heads, q_heads, dim, page, rot, interleaved, old, new
    (1, 1, 16, 16, 16, False, [0], [1]),
    (3, 6, 64, 16, 32, True, [15, 16, 17, 0], [1, 1, 1, 1]),
    (2, 4, 128, 16, 128, False, [5, 0, 31, 100], [40, 1, 2, 17]),
    (4, 4, 80, 32, 80, False, [7, 63], [70, 1]),
    (8, 32, 128, 64, 64, True, [64, 1], [129, 200]),
    (1, 8, 256, 16, 256, False, [3] * 40, [1] * 40),
    (2, 2, 48, 256, 8, True, [250], [300]),
    (5, 5, 64, 16, 0, False, [0, 0, 9], [16, 0, 33]),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_matches_its_definition_bit_for_bit(cuda, kind, case):
    torch = _torch()
    heads, q_heads, dim, page, rot, inter, old, new = APPENDS[case]
    rng = _rng("append", case)
    table, pages = _pages(rng, [(o + n + page - 1) // page for o, n in zip(old, new)])
    c = Cache(rng, pages, heads, page, dim, cuda)
    total = sum(new)
    k, v = (_cast(rng.standard_normal((total, heads, dim)) * 3 ** rng.standard_normal((total, 1, 1)), kind)
            for _ in range(2))
    q = _cast(rng.standard_normal((total, q_heads, dim)), kind)
    pos = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)]).astype(int)
    cos, sin = _tables(int(pos.max()) + 1, rot) if rot else (None, None)
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    one = all(n == 1 for n in new)
    args = dict(first=None if one and case % 2 else up(_first(new)), q=q.to(cuda), cos=up(cos), sin=up(sin),
                interleaved=inter)
    kr, qr = (_turn(_f32(x), pos, cos, sin, inter) if rot else _f32(x) for x in (k, q))
    _put(c.k, c.ks, kr, table, old, new, page)
    _put(c.v, c.vs, _f32(v), table, old, new, page)
    for _ in range(2):  # the second call finds everything in place
        got = pc.kv_append(c.dev, k.to(cuda), v.to(cuda), up(table), up(np.int32(old)), **args)
        c.same()
        assert torch.equal(got.cpu(), _cast(qr, kind))
    assert pc.device_errors() == 0


@pytest.mark.parametrize("kind", TYPES)
def test_append_strides_alignment_and_in_place_queries(cuda, kind):
    torch = _torch()
    rng = _rng("strides", 1)
    heads, dim, page, old, new = 3, 64, 16, [11, 2], [9, 30]
    total = sum(new)
    table, pages = _pages(rng, [(o + n + page - 1) // page for o, n in zip(old, new)])
    cos, sin = _tables(64, dim)
    pos = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)])
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    for shift, layout in ((0, "token"), (1, "token"), (0, "head"), (3, "head")):
        c = Cache(rng, pages, heads, page, dim, cuda)
        # one buffer with q, k and v interleaved, off alignment by `shift` elements
        fused = _cast(rng.standard_normal((total, 3 * heads, dim)), kind)
        buf = torch.zeros(fused.numel() + 8, dtype=fused.dtype, device=cuda)
        if layout == "token":
            view = buf[shift: shift + fused.numel()].view(total, 3 * heads, dim)
        else:
            view = buf[shift: shift + fused.numel()].view(3 * heads, total, dim).transpose(0, 1)
        view.copy_(fused)
        q, k, v = view[:, :heads], view[:, heads: 2 * heads], view[:, 2 * heads:]
        want = _f32(fused)
        _put(c.k, c.ks, _turn(want[:, heads: 2 * heads], pos, cos, sin, False), table, old, new, page)
        _put(c.v, c.vs, want[:, 2 * heads:], table, old, new, page)
        turned = _cast(_turn(want[:, :heads], pos, cos, sin, False), kind)
        got = pc.kv_append(c.dev, k, v, up(table), up(np.int32(old)), first=up(_first(new)), q=q, cos=up(cos),
                           sin=up(sin))
        c.same()
        assert torch.equal(got.cpu(), turned)
        own = q.contiguous()
        again = pc.kv_append(c.dev, k, v, up(table), up(np.int32(old)), first=up(_first(new)), q=own, q_out=own,
                             cos=up(cos), sin=up(sin))
        assert again.data_ptr() == own.data_ptr() and torch.equal(own.cpu(), turned)


def test_append_zeros_tiny_values_nan_and_infinity(cuda):
    torch = _torch()
    rng = _rng("edge", 1)
    c = Cache(rng, 4, 5, 16, 32, cuda)
    k = rng.standard_normal((3, 5, 32)).astype(np.float32)
    k[:, 0] = 0.0                     # a block of zeros: scale 0, codes 0
    k[:, 1] = 1e-30                   # below the smallest scale: the same
    k[1, 2, 3] = np.nan               # skipped by the maximum, code 0
    k[1, 3, 5] = np.inf               # infinite scale
    k[:, 4] *= 1e-20                  # small but kept
    v = k[::-1].copy()
    table, old, new = np.int32([[2]]), [0], [3]
    _put(c.k, c.ks, k, table, old, new, 16)
    _put(c.v, c.vs, v, table, old, new, 16)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    pc.kv_append(c.dev, up(k), up(v), up(table), up(np.int32(old)), first=up(_first(new)))
    c.same()
    assert c.ks[2, 0] == 0 and c.ks[2, 1] == 0 and np.isinf(c.ks[2, 3]) and c.ks[2, 4] > 0
    # a later token after zeros sets the scale afresh
    k2 = rng.standard_normal((1, 5, 32)).astype(np.float32)
    k2[:, 3] = 0
    _put(c.k, c.ks, k2, table, [3], [1], 16)
    _put(c.v, c.vs, k2, table, [3], [1], 16)
    pc.kv_append(c.dev, up(k2), up(k2), up(table), up(np.int32([3])))
    c.same()


def test_append_skips_and_reports_what_lies_outside(cuda):
    torch = _torch()
    rng = _rng("outside", 1)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    c = Cache(rng, 4, 2, 16, 64, cuda)
    x = up(rng.standard_normal((5, 2, 64)).astype(np.float32))
    # page index past the pool, negative page, position past the table, negative position; the last one is fine
    table, start = np.int32([[4], [-1], [0], [1], [3]]), np.int32([0, 3, 16, -1, 2])
    pc.kv_append(c.dev, x, x, up(table), up(start))
    torch.cuda.synchronize()
    assert pc.device_errors() == 0x2000 << 16 and pc.device_errors() == 0
    _put(c.k, c.ks, _f32(x)[4:], table[4:], [2], [1], 16)
    _put(c.v, c.vs, _f32(x)[4:], table[4:], [2], [1], 16)
    c.same()
    # a position past the rotation tables
    cos, sin = _tables(2, 64)
    pc.kv_append(c.dev, x[4:], x[4:], up(table[4:]), up(start[4:]), cos=up(cos), sin=up(sin))
    assert pc.device_errors() == 0x2000 << 16
    c.same()
    # runs of tokens that do not ascend: whatever is written stays inside, and the call ends
    for first in ([0, 5, 0, 5, 0, 5], [5, 4, 3, 2, 1, 0], [-3, 9, 9, 9, 9, 9]):
        pc.kv_append(c.dev, x, x, up(np.int32([[0], [1], [2], [3], [0]])), up(np.int32([0] * 5)), first=up(np.int32(first)))
    torch.cuda.synchronize()
    pc.device_errors()


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", [(2, 1, 16, 16), (5, 3, 32, 80), (9, 8, 64, 128), (3, 2, 256, 256)])
def test_read_gives_code_times_scale(cuda, kind, shape):
    torch = _torch()
    rng = _rng("read", *shape)
    c = Cache(rng, *shape, cuda)
    pages = rng.permutation(shape[0])[: max(1, shape[0] - 1)].astype(np.int32)
    k, v = pc.kv_read(c.dev, torch.from_numpy(pages).to(cuda), dtype=getattr(torch, kind))
    for got, codes, scale in ((k, c.k, c.ks), (v, c.v, c.vs)):
        want = codes[pages].astype(np.float32) * scale[pages][..., None, None]
        assert torch.equal(got.cpu(), _cast(want, kind))
    assert pc.device_errors() == 0
    k, v = pc.kv_read(c.dev, torch.tensor([shape[0], -1], dtype=torch.int32, device=cuda))
    assert not k.any() and not v.any()
    assert pc.device_errors() == 0x2000 << 16


# --------------------------------------------------------------- attention
def _attend(c, q, table, length, new, group, causal, window, scale):
    """64-bit softmax attention over the cached values; also the log denominators and the tolerance's parts."""
    first = _first(new)
    page = c.k.shape[2]
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    ds_parts, top = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for b, n in enumerate(new):
        at = table[b, : (length[b] + page - 1) // page]
        if not n or not len(at):
            continue
        for h in range(c.k.shape[1]):
            k = (c.k[at, h].astype(np.float64) * c.ks[at, h].astype(np.float64)[:, None, None]).reshape(-1, c.k.shape[3])
            v = (c.v[at, h].astype(np.float64) * c.vs[at, h].astype(np.float64)[:, None, None]).reshape(-1, c.k.shape[3])
            for i in range(n):
                pos = length[b] - n + i
                lo = max(0, pos + 1 - window) if window > 0 else 0
                hi = pos + 1 if causal else length[b]
                if hi <= lo:
                    continue
                t = first[b] + i
                for j in range(h * group, (h + 1) * group):
                    s = k[lo:hi] @ q[t, j] * scale
                    m = s.max()
                    p = np.exp(s - m)
                    out[t, j] = p @ v[lo:hi] / p.sum()
                    lse[t, j] = m + np.log(p.sum())
                    unit = np.abs(q[t, j]).max()
                    ds_parts[t, j] = np.abs(k[lo:hi]).sum(1).max() * unit * abs(scale) / 2
                    top[t, j] = np.abs(s).max()
                    out_v = np.abs(v[lo:hi]).max()
                    lse_v[t, j] = out_v if (t, j) in lse_v else out_v
    return out, lse, ds_parts, top


lse_v = {}


def _check(c, q, got, lse, table, length, new, group, causal, window, scale, kind):
    lse_v.clear()
    want, want_lse, ds, top = _attend(c, q, table, length, new, group, causal, window, scale)
    ds = ds / (2 ** 21 if kind == "float32" else 32512) + 8 * 2.0 ** -24 * top
    rounding = {"float32": 2.0 ** -19 + 2.0 ** -24, "float16": 2 * 2.0 ** -11, "bfloat16": 2.0 ** -11 + 2.0 ** -8}[kind]
    big = np.zeros(q.shape[:2])
    for (t, j), x in lse_v.items():
        big[t, j] = x
    tol = (2 * np.expm1(ds) + rounding) * big + (2.0 ** -25 if kind == "float16" else 0.0)
    err = np.abs(got - want)
    assert (err <= tol[..., None]).all(), (err.max(), tol.min(), np.argwhere(err > tol[..., None])[:4])
    seen = np.isfinite(want_lse)
    assert (np.isneginf(lse) == ~seen).all()
    assert (got[~seen] == 0).all()
    assert (np.abs(lse[seen] - want_lse[seen]) <= ds[seen] + 2.0 ** -20 * (1 + np.abs(want_lse[seen]))).all()


ATTENDS = [
    # heads, group, dim, page, lengths, queries, causal, window
    (1, 1, 16, 16, [1], [1], True, 0),
    (2, 1, 64, 16, [1, 15, 16, 17, 0, 33], [1] * 6, True, 0),
    (2, 4, 128, 32, [700, 1, 64], [1] * 3, True, 0),
    (1, 8, 128, 16, [2000], [1], True, 0),
    (2, 3, 80, 64, [100, 257], [3, 1], True, 0),
    (3, 5, 96, 16, [31, 200, 0, 2], [4, 9, 2, 3], True, 0),     # more queries than tokens: rows that see nothing
    (1, 12, 256, 16, [300, 40], [2, 1], True, 0),
    (2, 2, 192, 128, [129, 500], [1, 1], True, 0),
    (4, 1, 128, 16, [90, 400], [40, 33], True, 0),
    (2, 4, 64, 16, [333, 1000], [5, 1], True, 64),
    (2, 2, 128, 32, [200, 65], [7, 65], True, 1),
    (1, 3, 64, 16, [77, 130], [20, 3], False, 0),
    (1, 2, 128, 64, [150], [50], False, 30),
    (1, 32, 128, 16, [513], [1], True, 0),
    (2, 4, 128, 16, [40] * 150, [1] * 150, True, 0),            # more sequences than threads of a block
    (2, 2, 64, 16, [600, 3], [290, 3], True, 0),
    (1, 1, 128, 256, [5000], [1], True, 0),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_against_64_bits(cuda, kind, case):
    torch = _torch()
    heads, group, dim, page, length, new, causal, window = ATTENDS[case]
    rng = _rng("attend", case)
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    total = sum(new)
    q = _cast(rng.standard_normal((total, heads * group, dim)) * 1.5, kind)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    one = all(n == 1 for n in new)
    lse = torch.zeros((total, heads * group), device=cuda)
    got = pc.kv_attention(c.dev, q.to(cuda), up(table), up(np.int32(length)), lse=lse,
                          first=None if one and case % 2 else up(_first(new)),
                          max_tokens=max(new) if case % 3 else None, causal=causal, window=window)
    again = pc.kv_attention(c.dev, q.to(cuda), up(table), up(np.int32(length)), first=up(_first(new)),
                            max_tokens=max(new) if case % 3 else None, causal=causal, window=window)
    assert pc.device_errors() == 0
    assert torch.equal(got, again)  # no order of blocks changes a result
    _check(c, _f32(q).astype(np.float64), _f32(got).astype(np.float64), lse.cpu().numpy().astype(np.float64), table, length, new,
           group, causal, window, dim ** -0.5, kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_scales_strides_and_unlike_blocks(cuda, kind, scale):
    """Block scales that differ by 10^20, zero scales, a peaked softmax, strided unaligned queries."""
    torch = _torch()
    rng = _rng("scales", int(scale * 10) + 9)
    heads, group, dim, page, length, new = 2, 2, 64, 16, [200, 90], [2, 1]
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    for codes, s in ((c.k, c.ks), (c.v, c.vs)):
        s *= (10.0 ** rng.integers(-20, 1, s.shape)).astype(np.float32)
        zero = rng.random(s.shape) < 0.1
        s[zero] = 0
        codes[zero] = 0
    c.dev = pc.KvCache(*(torch.from_numpy(a.copy()).to(cuda) for a in (c.k, c.v, c.ks, c.vs)))
    q = _cast(rng.standard_normal((3, heads * group, dim)), kind)
    buf = torch.zeros(2 * q.numel() + 3, dtype=q.dtype, device=cuda)
    view = buf[3:].view(3, heads * group, 2 * dim)[..., dim:]
    view.copy_(q)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    lse = torch.zeros((3, heads * group), device=cuda)
    got = pc.kv_attention(c.dev, view, up(table), up(np.int32(length)), first=up(_first(new)), max_tokens=2, lse=lse,
                          scale=scale)
    _check(c, _f32(q).astype(np.float64), _f32(got).astype(np.float64), lse.cpu().numpy().astype(np.float64), table, length, new,
           group, True, 0, scale, kind)


@pytest.mark.parametrize("kind", TYPES)
def test_attention_unseen_blocks_and_rows_do_not_matter(cuda, kind):
    """NaN scales in pages that no query sees and codes past the end change nothing; those that a row sees, and
    non-finite queries, give NaN there and nowhere else."""
    torch = _torch()
    rng = _rng("unseen", 1)
    heads, group, dim, page, length, new = 2, 2, 128, 16, [40, 100], [3, 1]
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    q = _cast(rng.standard_normal((4, heads * group, dim)), kind).to(cuda)
    call = lambda window=0: pc.kv_attention(c.dev, q, up(table), up(np.int32(length)), first=up(_first(new)),  # noqa: E731
                                            max_tokens=3, window=window)
    want, want20 = call(), call(20)
    used = set(table[0, :3]) | set(table[1, :7])
    for p in set(range(pages)) - used:
        for s in (c.dev.k_scale, c.dev.v_scale):
            s[p] = float("nan")
    c.dev.k[int(table[0, 2]), :, 8:] = 77   # past length 40
    c.dev.v[int(table[0, 2]), :, 8:] = -77
    assert torch.equal(call(), want)
    # pages behind the window
    for s in (c.dev.k_scale, c.dev.v_scale):
        s[int(table[1, 0])] = float("nan")
        s[int(table[1, 1]), 0] = float("inf")
    assert torch.equal(call(20), want20)
    got = call()
    assert torch.isnan(got[3]).all() and torch.equal(got[:3], want[:3])
    # the last block of sequence 0: rows 0, 1, 2 stand at positions 37, 38, 39 and all see it; a query with an
    # infinity spoils its own row
    q[1, 1, 5] = float("inf")
    got = call(20)
    assert torch.isnan(got[1, 1]).all()
    keep = torch.ones((4, heads * group), dtype=torch.bool)
    keep[1, 1] = False
    assert torch.equal(got[keep], want20[keep])


def test_attention_reports_pages_and_lengths_outside(cuda):
    torch = _torch()
    rng = _rng("report", 1)
    c = Cache(rng, 4, 2, 16, 64, cuda)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    q = up(rng.standard_normal((3, 4, 64)).astype(np.float32))
    # sequence 0: middle page outside the pool; sequence 1: longer than its table; sequence 2: negative length
    got = pc.kv_attention(c.dev, q, up(np.int32([[0, 9, 1], [1, 2, 3], [-1, -1, -1]])), up(np.int32([48, 1000, -5])))
    assert pc.device_errors() == 0x4000 << 16
    assert torch.isfinite(got).all() and not got[2].any()
    short = pc.kv_attention(c.dev, q, up(np.int32([[0, 1], [1, 2], [0, 0]])), up(np.int32([32, 32, 0])))
    lse = torch.zeros((3, 4), device=cuda)
    full = pc.kv_attention(c.dev, q, up(np.int32([[0, 1, 0], [1, 2, 3], [0, 0, 0]])), up(np.int32([32, 48, 0])), lse=lse)
    assert torch.allclose(got[0], short[0], rtol=0, atol=1e-5)  # the bad page counts as unseen
    assert torch.allclose(got[1], full[1], rtol=0, atol=1e-5)  # (another batch is cut into other runs)
    assert pc.device_errors() == 0
    for first in ([0, 3, 0, 3], [3, 2, 1, 0], [-2, 5, 7, 9]):
        pc.kv_attention(c.dev, q, up(np.int32([[0], [1], [2]])), up(np.int32([16, 16, 16])), first=up(np.int32(first)))
    torch.cuda.synchronize()
    pc.device_errors()


def test_long_cache_offsets_pass_32_bits(cuda):
    """A pool of more than 2^31 codes a half: pages at its end, appended, read and attended."""
    torch = _torch()
    heads, page, dim = 8, 64, 128
    pages = (1 << 31) // (heads * page * dim) + 64
    cache = pc.KvCache.empty(pages, heads, dim, page, device=cuda)
    rng = _rng("long", 1)
    table = np.int32([[pages - 1, 3, pages - 2]])
    new = [150]
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    k, v = (rng.standard_normal((150, heads, dim)).astype(np.float32) for _ in range(2))
    pc.kv_append(cache, up(k), up(v), up(table), up(np.int32([0])), first=up(_first(new)))
    small = Cache(rng, 3, heads, page, dim, cuda)
    for codes, scale, x in ((small.k, small.ks, k), (small.v, small.vs, v)):
        codes[:] = 0
        scale[:] = 0
        _put(codes, scale, x, np.int32([[0, 1, 2]]), [0], new, page)
    kk, vv = pc.kv_read(cache, up(table[0]))
    assert np.array_equal(_f32(kk), small.k.astype(np.float32) * small.ks[..., None, None])
    assert np.array_equal(_f32(vv), small.v.astype(np.float32) * small.vs[..., None, None])
    small.dev = pc.KvCache(*(up(a) for a in (small.k, small.v, small.ks, small.vs)))
    q = up(rng.standard_normal((1, 16, dim)).astype(np.float32))
    got = pc.kv_attention(cache, q, up(table), up(np.int32([150])))
    want = pc.kv_attention(small.dev, q, up(np.int32([[0, 1, 2]])), up(np.int32([150])))
    assert torch.equal(got, want)


def test_side_streams_and_graphs(cuda):
    """Append and attention on a side stream, and replayed from a graph."""
    torch = _torch()
    rng = _rng("stream", 1)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    heads, dim, page = 2, 128, 16
    cache = pc.KvCache.empty(40, heads, dim, page, device=cuda)
    table = up(np.arange(40, dtype=np.int32).reshape(2, 20))
    k = up(rng.standard_normal((600, heads, dim)).astype(np.float32))
    first = up(np.int32([0, 300, 600]))
    start, length = up(np.int32([0, 0])), up(np.int32([300, 300]))
    q = up(rng.standard_normal((600, 4, dim)).astype(np.float32))
    pc.kv_append(cache, k, k * 2, table, start, first=first)
    want = pc.kv_attention(cache, q, table, length, first=first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache2 = pc.KvCache.empty(40, heads, dim, page, device=cuda)
    k2 = k * 2
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        pc.kv_append(cache2, k, k2, table, start, first=first)
        got = pc.kv_attention(cache2, q, table, length, first=first)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pc.kv_append(cache2, k, k2, table, start, first=first)
        pc.kv_attention(cache2, q, table, length, first=first, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_python_refusals(cuda):
    torch = _torch()
    z = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=cuda)  # noqa: E731
    cache = pc.KvCache.empty(4, 2, 64, 16, device=cuda)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    k, q, table, start, first = z(3, 2, 64), z(3, 4, 64), torch.zeros((2, 2), dtype=torch.int32, device=cuda), i32(0, 0), i32(0, 1, 3)
    cos = z(32, 32)
    good = dict(k=k, v=k, table=table, start=start, first=first, q=q, cos=cos, sin=cos)
    assert pc.kv_append(cache, **good).shape == q.shape
    for name, bad in (("k", k.half()), ("k", k[:, :1]), ("k", k[0]), ("k", k.cpu()), ("k", k.double()), ("v", k[:2]),
                      ("v", k.transpose(1, 2).contiguous().transpose(1, 2)), ("table", table.long()), ("table", table[0]),
                      ("table", table.t()[:1]), ("start", start[:1]), ("start", start.cpu()), ("first", first[:2]),
                      ("first", None), ("q", q[..., :32]), ("q", q.bfloat16()), ("cos", cos[0]), ("cos", cos.half()),
                      ("sin", None), ("sin", cos[:5]), ("cos", cos[:, ::2]), ("q_out", q[:, :2]), ("q_out", q.half())):
        with pytest.raises(ValueError, match="kv_append"):
            pc.kv_append(cache, **{**good, name: bad})
    with pytest.raises(pc.PopcornError):
        pc.kv_append(cache, **{**good, "cos": z(32, 30), "sin": z(32, 30)})  # rot_dim 60
    length = i32(1, 2)
    good = dict(q=q, table=table, length=length, first=first)
    assert pc.kv_attention(cache, **good).shape == q.shape
    for name, bad in (("q", q[:, :3]), ("q", q[..., :32]), ("q", q.double()), ("q", q.cpu()), ("q", q[0]),
                      ("table", table.long()), ("length", length[:1]), ("length", length.float()), ("first", None),
                      ("out", q.half()), ("out", q[:, ::2]), ("lse", z(3, 5)), ("lse", z(4, 3).t())):
        with pytest.raises(ValueError, match="kv_attention"):
            pc.kv_attention(cache, **{**good, name: bad})
    with pytest.raises(pc.PopcornError):
        pc.kv_attention(cache, **good, max_tokens=0)
    pages = i32(0, 1)
    for kw in (dict(pages=pages.long()), dict(pages=pages.cpu()), dict(pages=pages[None]), dict(pages=pages, dtype=torch.int8),
               dict(pages=pages, k_out=z(2, 2, 16, 32)), dict(pages=pages, v_out=z(2, 2, 16, 64, dtype=torch.float16))):
        with pytest.raises(ValueError, match="kv_read"):
            pc.kv_read(cache, **kw)
    assert pc.kv_read(cache, pages[:0])[0].shape == (0, 2, 16, 64)


PROMPTS = [
    # heads, group, dim, page, lengths, queries, causal, window
    (1, 1, 64, 16, [300], [257], True, 0),
    (2, 1, 128, 32, [130, 48, 5], [47, 48, 5], True, 0),            # rows on both sides of the kernels' border
    (2, 4, 128, 16, [700, 90, 12, 0], [100, 12, 1, 0], True, 0),
    (1, 8, 128, 64, [2000], [70], True, 0),
    (3, 5, 64, 16, [31, 200, 0, 2], [40, 9, 20, 3], True, 0),       # more queries than tokens: rows that see nothing
    (2, 4, 64, 16, [333, 1000], [50, 130], True, 64),
    (2, 3, 128, 128, [200, 650], [70, 65], True, 1),
    (1, 2, 128, 16, [150, 129], [50, 129], False, 30),
    (1, 3, 64, 32, [777, 130], [20, 300], False, 0),
    (4, 2, 128, 256, [1025, 511], [256, 1], True, 0),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompts_against_64_bits(cuda, kind, wide, case):
    """Small calls, and the same ones with a block table that could hold long sequences."""
    torch = _torch()
    heads, group, dim, page, length, new, causal, window = PROMPTS[case]
    rng = _rng("prompts", case)
    table, pages = _pages(rng, [(n + page - 1) // page for n in length])
    c = Cache(rng, pages, heads, page, dim, cuda)
    if wide:
        table = np.concatenate([table, np.full((len(length), (1 << 19) // page), -9, np.int32)], 1)
    q = _cast(rng.standard_normal((sum(new), heads * group, dim)) * 1.5, kind)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    lse = torch.zeros((sum(new), heads * group), device=cuda)
    call = lambda most, lse=None: pc.kv_attention(c.dev, q.to(cuda), up(table), up(np.int32(length)),  # noqa: E731
                                                  first=up(_first(new)), max_tokens=most, causal=causal,
                                                  window=window, lse=lse)
    got = call(max(new), lse)
    assert torch.equal(got, call(max(new)))
    assert pc.device_errors() == 0
    _check(c, _f32(q).astype(np.float64), _f32(got).astype(np.float64), lse.cpu().numpy().astype(np.float64), table, length, new,
           group, causal, window, dim ** -0.5, kind)


@pytest.mark.parametrize("tokens", [3, 40])
def test_append_rounds_values_next_to_halves(cuda, tokens):
    """Codes at k + 1/2 and a few ulps beside it, for scales from 1e-22 to the largest, and blocks of zeros, NaN and
    infinities: decode and prompt forms of the kernel give the definition's codes."""
    torch = _torch()
    rng = _rng("halves", tokens)
    top = np.float32([1.0, 127.0, 3e-20, 7e20, 3.4e38, 0.0, 1e-30, 1.0, 1.0])
    heads, dim, page = len(top), 64, 64
    c = Cache(rng, 3, heads, page, dim, cuda)
    half = rng.integers(-127, 127, (tokens, heads, dim)) + 0.5
    with np.errstate(over="ignore"):
        k = (half * (top / np.float32(127))[None, :, None].astype(np.float64)).astype(np.float32)
    k = (k.view(np.int32) + rng.integers(-3, 4, k.shape)).astype(np.int32).view(np.float32)
    k[0, :, 0] = top
    k[:, 5] = 0.0
    k[1, 7, 9] = np.nan
    k[2, 8, 60] = -np.inf
    v = np.ascontiguousarray(k[:, ::-1])
    table, old, new = np.int32([[1]]), [0], [tokens]
    _put(c.k, c.ks, k, table, old, new, page)
    _put(c.v, c.vs, v, table, old, new, page)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    pc.kv_append(c.dev, up(k), up(v), up(table), up(np.int32(old)), first=up(_first(new)))
    c.same()
    assert pc.device_errors() == 0
