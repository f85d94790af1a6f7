"""Measured cases of the operators around the quantized linear layers of a decoder: the paged 8-bit key/value
cache (append with the position rotation, read-back, attention) and the mixture-of-experts layer on int8 experts.

``listed()`` are the cases that stand for real use, ``draw(rng)`` gives others of the same ranges, ``prepare`` makes
what a program has in hand before a call, ``run`` is one pass. With ``own`` false ``run`` is the plain form in
elementary torch operations (32-bit arithmetic, one rounding at the end); with ``own`` true it calls the library.
``exact`` restates each operator from its definition in 64 bits.

The cache: codes int8 [pages, heads, page, dim] and one f32 scale for each (page, head), keys and values apart; a value
is code * scale. Sequence b's token at position p lies in page table[b, p // page], row p % page. Appending sets the
block's scale to max(old scale, max|new| / 127) (no old scale for a page that the append begins), re-encodes the
block's earlier codes as rint(code * (old / new)) and writes rint(value / scale) for the new tokens.
"""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SMALLEST_SCALE = 2.0 ** -80  # a block scale below it counts as zero


def listed():
    return [
        # One user's chat: the next token of one sequence, 32 heads of 128 (the 7B linear stack's qkv width).
        dict(name="append 1 token f32", op="append", type="float32", seqs=1, tokens=1, ragged=False, context=777,
             heads=32, q_heads=32, dim=128, page=16, rot=128, interleaved=False),
        # A serving batch's next tokens, grouped heads, ragged lengths.
        dict(name="append batch bf16", op="append", type="bfloat16", seqs=64, tokens=1, ragged=True, context=4096,
             heads=8, q_heads=32, dim=128, page=32, rot=128, interleaved=False),
        # Drafted tokens on small heads, partial interleaved rotation, odd counts.
        dict(name="append drafts f16", op="append", type="float16", seqs=9, tokens=37, ragged=True, context=1111,
             heads=5, q_heads=15, dim=64, page=16, rot=32, interleaved=True),
        # Prompts entering the cache, some behind a cached prefix that ends inside a page.
        dict(name="append prompts f32", op="append", type="float32", seqs=4, tokens=2048, ragged=True, context=500,
             heads=8, q_heads=32, dim=128, page=64, rot=128, interleaved=False),
        # The smallest attention: one sequence's next token, a kilo-token context.
        dict(name="attend 1x1000 f32", op="attend", type="float32", seqs=1, tokens=1, ragged=False, context=1000,
             heads=32, q_heads=32, dim=128, page=16, window=0),
        # A batch of the 7B shape (one key/value head for each query head) at 4096 tokens.
        dict(name="attend 16x4096 f32", op="attend", type="float32", seqs=16, tokens=1, ragged=False, context=4096,
             heads=32, q_heads=32, dim=128, page=16, window=0),
        # A serving batch with grouped heads and ragged lengths.
        dict(name="attend ragged bf16", op="attend", type="bfloat16", seqs=64, tokens=1, ragged=True, context=8192,
             heads=8, q_heads=32, dim=128, page=32, window=0),
        # One long document.
        dict(name="attend 1x131075 f16", op="attend", type="float16", seqs=1, tokens=1, ragged=False, context=131075,
             heads=8, q_heads=32, dim=128, page=64, window=0),
        # Checking drafted tokens against the cache, small heads, a sliding window.
        dict(name="attend drafts bf16", op="attend", type="bfloat16", seqs=12, tokens=5, ragged=True, context=3001,
             heads=4, q_heads=12, dim=64, page=16, window=1024),
        # A chunk of two prompts over what is cached of them.
        dict(name="attend prompt bf16", op="attend", type="bfloat16", seqs=2, tokens=1024, ragged=False, context=4000,
             heads=8, q_heads=32, dim=128, page=64, window=0),
        # One token through two of sixteen experts of the 7B MLP's size.
        dict(name="moe 1 of 16x11008 f32", op="moe", tokens=1, experts=16, top=2, hidden=4096, inter=11008,
             renorm=True),
        # A small batch over many small experts.
        dict(name="moe 16 of 64x1424 f32", op="moe", tokens=16, experts=64, top=6, hidden=2048, inter=1424,
             renorm=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "moe"])
    if op == "moe":
        c = dict(op=op, tokens=_log(rng, 1, 32), experts=rng.choice([4, 8, 16, 24, 48, 64]), top=rng.choice([1, 2, 3, 4, 6, 8]),
                 hidden=rng.choice([512, 1024, 1280, 2048, 2560, 4096]), inter=16 * _log(rng, 24, 688),
                 renorm=rng.random() < 0.5)
        c["top"] = min(c["top"], c["experts"])
        while c["experts"] * c["inter"] * c["hidden"] > 16 * 11008 * 4096 or c["inter"] == 3072:
            c["inter"] = 16 * _log(rng, 24, 400)
        return c
    heads = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    c = dict(op=op, type=rng.choice(sorted(TYPES)), seqs=_log(rng, 1, 64), ragged=rng.random() < 0.7, heads=heads,
             q_heads=heads * rng.choice([1, 2, 3, 4, 4, 8]), dim=rng.choice([64, 128, 128, 128]),
             page=rng.choice([16, 32, 64]))
    kind = rng.choice(["one", "one", "drafts", "prompt"])
    c["tokens"] = 1 if kind == "one" else rng.randint(2, 8) if kind == "drafts" else _log(rng, 33, 1024)
    if kind == "prompt":
        c["seqs"] = min(c["seqs"], 3)
        while c["q_heads"] > 64:
            c["q_heads"] -= heads
    if op == "append":
        c["context"] = _log(rng, 1, 4095)
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2])
        c["interleaved"] = rng.random() < 0.3
    else:
        most = 1 << 17 if kind == "one" else 4000
        most = max(17, min(most, (1 << 28) // (c["seqs"] * heads * c["dim"])))
        if kind == "prompt":
            most = max(17, min(most, (1 << 28) // (c["seqs"] * c["q_heads"] * c["tokens"])))
        c["context"] = _log(rng, 16, most)
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4000)])
    if c["context"] == 3072:
        c["context"] += 1
    return c


def _lengths(case):
    """(tokens already cached, new tokens) of each sequence: the same ones for every seed."""
    r = random.Random("%d %d %d %d" % (case["seqs"], case["tokens"], case["context"], case["heads"]))
    if not case["ragged"]:
        return [case["context"]] * case["seqs"], [case["tokens"]] * case["seqs"]
    old = [r.randint(0, case["context"]) for _ in range(case["seqs"])]
    new = [r.randint(1, case["tokens"]) for _ in range(case["seqs"])]
    old[r.randrange(case["seqs"])] = case["context"]
    new[r.randrange(case["seqs"])] = case["tokens"]
    return old, new


def _touched(case):
    """(sequence, page of the sequence) of the pages that an append writes to."""
    old, new = _lengths(case)
    return [(b, p) for b in range(case["seqs"])
            for p in range(old[b] // case["page"], (old[b] + new[b] - 1) // case["page"] + 1)]


def _seen(case):
    """For each sequence: (key tokens that some query sees, query-key pairs)."""
    old, new = _lengths(case)
    w = case["window"]
    out = []
    for o, n in zip(old, new):
        first = max(0, o - w + 1) if w else 0
        out.append((o + n - first, sum(min(o + i + 1, w) if w else o + i + 1 for i in range(n))))
    return out


def work(case):
    if case["op"] == "moe":
        m, e, k, f, t = case["tokens"], case["experts"], case["hidden"], case["inter"], case["top"]
        used = e * (1 - (1 - t / e) ** m)  # experts that some token picks, on average
        flops = 2.0 * m * e * k + 6.0 * m * t * k * f
        return {"bytes": used * (3.0 * k * f + 8 * f + 4 * k) + 4.0 * e * k + 8.0 * m * k + 8 * m * t, "flops": flops}
    size = TYPES[case["type"]].itemsize
    old, new = _lengths(case)
    total, h, d = sum(new), case["heads"], case["dim"]
    table = 4 * sum((o + n + case["page"] - 1) // case["page"] for o, n in zip(old, new))
    if case["op"] == "append":
        blocks = len(_touched(case)) * h
        moved = total * size * (2 * h + 2 * case["q_heads"]) * d + total * 4 * case["rot"]
        # the touched blocks' codes and scales read and written, and their values read back
        return {"bytes": moved + blocks * 2 * (2 * case["page"] * d + 8 + 4 * case["page"] * d) + table,
                "flops": total * (h + case["q_heads"]) * case["rot"] * 3.0 + blocks * case["page"] * d * 8.0}
    seen = _seen(case)
    keys, pairs = sum(s for s, _ in seen), sum(p for _, p in seen)
    return {"bytes": keys * h * (2 * d + 8 / case["page"]) + 2 * total * case["q_heads"] * d * size + table,
            "flops": 4.0 * pairs * case["q_heads"] * d}


def _cache(case, pages, gen, dev):
    shape = (pages, case["heads"], case["page"], case["dim"])
    make = lambda: torch.randn(shape, generator=gen, device=dev).mul_(36).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    scale = lambda by: (torch.rand(shape[:2], generator=gen, device=dev) + 0.5).mul_(by)  # noqa: E731
    return make(), make(), scale(1 / 36), scale(1 / 50)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "moe":
        m, e, k, f = case["tokens"], case["experts"], case["hidden"], case["inter"]

        def matrix(n, kk):
            q = torch.randint(-127, 128, (e, n, kk), generator=gen, device=dev, dtype=torch.int8)
            return q, (torch.rand((e, n), generator=gen, device=dev) + 0.5) / (73 * math.sqrt(kk))

        s = dict(case=case, x=torch.randn((m, k), generator=gen, device=dev),
                 router=torch.randn((e, k), generator=gen, device=dev) * (1.5 / math.sqrt(k)))
        s["gate"], s["up"], s["down"] = matrix(f, k), matrix(f, k), matrix(k, f)
        return s
    old, new = _lengths(case)
    page = case["page"]
    need = [(o + n + page - 1) // page for o, n in zip(old, new)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: sum(need)].tolist()
    table, at = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at: at + n], dtype=torch.int32)
        at += n
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    kind = TYPES[case["type"]]
    kc, vc, ks, vs = _cache(case, pages, gen, dev)
    total, h, d = sum(new), case["heads"], case["dim"]
    s = dict(case=case, kc=kc, vc=vc, ks=ks, vs=vs, table=table.to(dev), first=whole(first), start=whole(old),
             length=whole([o + n for o, n in zip(old, new)]), most=max(new),
             q=torch.randn((total, case["q_heads"], d), generator=gen, device=dev).to(kind))
    if case["op"] == "append":
        # keys and values as two slices of one projection's output, as a fused qkv product leaves them
        kv = torch.randn((total, 2, h, d), generator=gen, device=dev)
        s["k"], s["v"] = kv.to(kind)[:, 0], (kv * 0.7).to(kind)[:, 1]
        angle = torch.arange(max(o + n for o, n in zip(old, new)), dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        s["cos"], s["sin"] = angle.cos().float().to(dev), angle.sin().float().to(dev)
        s["touched"] = whole([int(table[b, p]) for b, p in _touched(case)])
    if own:
        import popcorn_b200 as pc

        s["cache"] = pc.KvCache(kc, vc, ks, vs)  # the handle that a program keeps
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "moe": _own_moe}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "moe": _plain_moe}[op](state)


def _own_append(s):
    import popcorn_b200 as pc

    q = pc.kv_append(s["cache"], s["k"], s["v"], s["table"], s["start"], first=s["first"], q=s["q"], cos=s["cos"],
                     sin=s["sin"], interleaved=s["case"]["interleaved"])
    k, v = pc.kv_read(s["cache"], s["touched"])
    return {"q": q, "k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}


def _own_attend(s):
    import popcorn_b200 as pc

    return pc.kv_attention(s["cache"], s["q"], s["table"], s["length"], first=s["first"], max_tokens=s["most"],
                           window=s["case"]["window"])


def _own_moe(s):
    import popcorn_b200 as pc

    out, experts, weights = pc.moe(s["x"], s["router"], *s["gate"], *s["up"], *s["down"], top_k=s["case"]["top"],
                                   renormalize=s["case"]["renorm"], routing=True)
    return {"out": out, "experts": experts, "weights": weights}


def _places(s):
    """Sequence and position of each new token."""
    total = s["q"].shape[0]
    at = torch.arange(total, device=s["q"].device, dtype=torch.int32)
    b = torch.searchsorted(s["first"][1:], at, right=True)
    return b, s["start"][b] + at - s["first"][b]


def _rotated(x, cos, sin, interleaved):
    x, r = x.float(), cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * r:]], -1)


def _plain_put(codes, scale, values, page, row, old, at):
    """Appends values [tokens, heads, dim] at (page, row) to the keys or the values of the cache: `at` lists the pages
    that get new rows, old[page] counts the rows that earlier appends filled."""
    most = torch.zeros_like(scale).index_reduce_(0, page, values.abs().amax(-1), "amax")
    now = most / torch.full_like(most, 127)  # a division by a tensor is IEEE's, one by a number is not
    now = torch.where(now < SMALLEST_SCALE, torch.zeros_like(now), now)
    before = torch.where(old[:, None] == 0, torch.zeros_like(scale), scale)  # none for a page that begins now
    fresh = torch.maximum(before, now)
    ratio = torch.where(fresh > 0, before / fresh, torch.ones_like(fresh))[at][..., None, None]
    earlier = (torch.arange(codes.shape[2], device=codes.device) < old[at][:, None])[:, None, :, None]
    kept = codes[at]
    codes[at] = torch.where(earlier, torch.round(kept.float() * ratio).to(torch.int8), kept)
    by = fresh[page][..., None]
    codes[page, :, row] = torch.where(by > 0, torch.round(values / by), torch.zeros_like(values)).clamp(-128, 127).to(torch.int8)
    scale[at] = fresh[at]


def _plain_append(s):
    c = s["case"]
    b, pos = _places(s)
    page = s["table"][b, pos // c["page"]].long()
    row = (pos % c["page"]).long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    k, v = _rotated(s["k"], cos, sin, c["interleaved"]), s["v"].float()
    old = torch.full((s["kc"].shape[0],), c["page"], device=row.device).index_reduce_(0, page, row, "amin")
    at = s["touched"].long()
    _plain_put(s["kc"], s["ks"], k, page, row, old, at)
    _plain_put(s["vc"], s["vs"], v, page, row, old, at)
    return {"q": _rotated(s["q"], cos, sin, c["interleaved"]).to(s["q"].dtype),
            "k": s["kc"][at].float() * s["ks"][at][..., None, None],
            "v": s["vc"][at].float() * s["vs"][at][..., None, None], "k_scale": s["ks"], "v_scale": s["vs"]}


def _plain_attend(s):
    c = s["case"]
    n, h, g, d, most = c["seqs"], c["heads"], c["q_heads"] // c["heads"], c["dim"], s["most"]
    b, pos = _places(s)
    i = pos - s["start"][b]
    q = torch.zeros((n, most, h, g, d), device=pos.device)
    q[b, i] = s["q"].float().view(-1, h, g, d)
    at = s["table"].clamp(min=0).long()
    k = (s["kc"][at].float() * s["ks"][at][..., None, None]).transpose(1, 2).reshape(n, h, -1, d)
    v = (s["vc"][at].float() * s["vs"][at][..., None, None]).transpose(1, 2).reshape(n, h, -1, d)
    scores = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(n, h, most * g, d), k.transpose(2, 3)) / math.sqrt(d)
    key = torch.arange(k.shape[2], device=pos.device)
    query = s["start"][:, None] + torch.arange(most, device=pos.device)
    sees = key <= query[..., None]
    if c["window"]:
        sees &= key > query[..., None] - c["window"]
    scores = scores.view(n, h, most, g, -1).masked_fill_(~sees[:, None, :, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p.view(n, h, most * g, -1), v) / p.sum(-1).view(n, h, most * g, 1)
    return out.view(n, h, most, g, d)[b, :, i].reshape(-1, h * g, d).to(s["q"].dtype)


def _plain_moe(s):
    c, x = s["case"], s["x"]
    m, t = c["tokens"], c["top"]
    p = torch.softmax(torch.matmul(x, s["router"].t()), -1)
    # a stable descending sort: of equal probabilities the lowest index comes first
    weights, experts = torch.sort(p, dim=-1, descending=True, stable=True)
    weights, experts = weights[:, :t], experts[:, :t]
    if c["renorm"]:
        weights = weights / weights.sum(-1, keepdim=True)
    silu = lambda v: v / (1 + torch.exp(-v))  # noqa: E731
    if m * t <= c["experts"]:  # the chosen experts' weights, token by token
        w = lambda j: s[j][0][experts].float() * s[j][1][experts][..., None]  # noqa: E731
        hid = silu(torch.matmul(w("gate"), x[:, None, :, None])) * torch.matmul(w("up"), x[:, None, :, None])
        y = torch.matmul(w("down"), hid)[..., 0]
    else:  # every expert on every token
        w = lambda j: s[j][0].float().mul_(s[j][1][..., None]).transpose(1, 2)  # noqa: E731
        hid = silu(torch.matmul(x, w("gate"))) * torch.matmul(x, w("up"))
        y = torch.matmul(hid, w("down")).transpose(0, 1)[torch.arange(m, device=x.device)[:, None], experts]
    return {"out": (y * weights[..., None]).sum(1), "experts": experts.to(torch.int32), "weights": weights}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "moe": _exact_moe}[case["op"]](s)


def _exact_turn(x, pos, c):
    """Rotation by complex numbers: the pair (a, b) is a + ib, turned by the table's cos + i sin."""
    table = torch.complex(c[0].double(), c[1].double())[pos][:, None]
    x, r = x.double(), table.shape[-1]
    pair = x[..., :2 * r].unflatten(-1, (r, 2) if c[2] else (2, r))
    pair = pair if c[2] else pair.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * table)
    return torch.cat([(z if c[2] else z.transpose(-1, -2)).flatten(-2), x[..., 2 * r:]], -1)


def _exact_append(s):
    case = s["case"]
    old, new = _lengths(case)
    page, turn = case["page"], (s["cos"], s["sin"], case["interleaved"])
    pos = torch.tensor([o + i for o, n in zip(old, new) for i in range(n)], device="cuda")
    k, v = _exact_turn(s["k"], pos, turn), s["v"].double()
    out = {"q": _exact_turn(s["q"], pos, turn), "k": [], "v": []}
    scales = {"k": s["ks"].double(), "v": s["vs"].double()}
    first = 0
    for b, (o, n) in enumerate(zip(old, new)):
        for p in range(o // page, (o + n - 1) // page + 1):
            lo, hi = max(o, p * page), min(o + n, (p + 1) * page)
            at = int(s["table"][b, p])
            for name, codes, values in (("k", s["kc"], k), ("v", s["vc"], v)):
                x = values[first + lo - o: first + hi - o].transpose(0, 1)
                before = scales[name][at] * (1.0 if lo > p * page else 0.0)
                now = torch.maximum(before, x.abs().amax((1, 2)) / 127)
                block = codes[at].double()
                block[:, :lo - p * page] = torch.round(block[:, :lo - p * page] * (before / now)[:, None, None])
                block[:, lo - p * page: hi - p * page] = torch.round(x / now[:, None, None])
                out[name].append(block * now[:, None, None])
                scales[name][at] = now
        first += n
    return {"q": out["q"], "k": torch.stack(out["k"]), "v": torch.stack(out["v"]), "k_scale": scales["k"],
            "v_scale": scales["v"]}


def _exact_attend(s):
    case = s["case"]
    old, new = _lengths(case)
    h, g, page = case["heads"], case["q_heads"] // case["heads"], case["page"]
    if sum(p for _, p in _seen(case)) * case["q_heads"] * case["dim"] > 2e11:
        return None  # 64-bit products of this size take too long
    out, first = [], 0
    for b, (o, n) in enumerate(zip(old, new)):
        at = s["table"][b, : (o + n + page - 1) // page].long()
        flat = lambda c, x: (c[at].double() * x[at].double()[..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, : o + n]  # noqa: E731
        k, v = flat(s["kc"], s["ks"]), flat(s["vc"], s["vs"])
        q = s["q"][first: first + n].double().unflatten(1, (h, g))
        z = torch.einsum("nhgd,hkd->hgnk", q, k) * case["dim"] ** -0.5
        ahead = torch.arange(o + n, device="cuda") - torch.arange(o, o + n, device="cuda")[:, None]
        hidden = ahead > 0
        if case["window"]:
            hidden |= ahead <= -case["window"]
        p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
        out.append(torch.einsum("hgnk,hkd->nhgd", p, v).flatten(1, 2))
        first += n
    return torch.cat(out)


def _exact_moe(s):
    case = s["case"]
    x, t = s["x"].double(), case["top"]
    z = torch.einsum("mk,ek->me", x, s["router"].double())
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    experts = torch.argsort(p, dim=1, descending=True, stable=True)[:, :t]
    weights = torch.gather(p, 1, experts)
    if case["renorm"]:
        weights = weights / weights.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        picked = experts == e
        who = picked.any(1).nonzero()[:, 0]
        if not len(who):
            continue
        w = lambda j: s[j][0][e].double() * s[j][1][e].double()[:, None]  # noqa: E731
        a = torch.einsum("mk,fk->mf", x[who], w("gate"))
        y = torch.einsum("mf,kf->mk", a * torch.sigmoid(a) * torch.einsum("mk,fk->mf", x[who], w("up")), w("down"))
        out[who] += y * (weights * picked).sum(1)[who, None]
    return {"out": out, "experts": None, "weights": weights}
