"""GPU: the mixture-of-experts layer on int8 experts (include/popcorn_serve.h) against a restatement in 64 bits.

Tolerance, per output: each product sum is exact or joined by at most 16 + max(K, F) / 32 f32 roundings, so with
eps = (16 + max(K, F) / 32) 2^-24 a dot product is off by at most eps times the sum of its terms' magnitudes; a hidden
value inherits gate and up errors (|silu'| < 1.1), a weight the logits' (a relative 2 dz).
"""
import numpy as np
import pytest

import popcorn_b200 as pc

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


def _layer(M, K, F, E, seed, ties=False):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)).astype(np.float32)
    router = (rng.standard_normal((E, K)) * 2 / np.sqrt(K)).astype(np.float32)
    if ties:
        router[:] = router[rng.integers(0, max(1, E // 3), E)]

    def matrix(n, k):
        return (rng.integers(-128, 128, (E, n, k)).astype(np.int8),
                ((rng.random((E, n)) + 0.5) / (73 * np.sqrt(k))).astype(np.float32))

    return x, router, matrix(F, K), matrix(F, K), matrix(K, F)


def _call(layer, top, renorm, cuda, routing=True, shift=0):
    torch = _torch()

    def up(a):  # `shift` bytes or elements off the allocation's alignment
        a = torch.from_numpy(np.ascontiguousarray(a))
        buf = torch.empty(a.numel() + 16, dtype=a.dtype, device=cuda)
        view = buf[shift: shift + a.numel()].view(a.shape)
        view.copy_(a)
        return view

    x, router, gate, upm, down = layer
    got = pc.moe(up(x), up(router), *map(up, gate), *map(up, upm), *map(up, down), top_k=top, renormalize=renorm,
                 routing=routing)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in got] if routing else got.cpu().numpy()


def _reference(layer, top, renorm):
    x, router, (qg, sg), (qu, su), (qd, sd) = layer
    (M, K), F = x.shape, qg.shape[1]
    x, router = x.astype(np.float64), router.astype(np.float64)
    eps = (16 + max(K, F) / 32) * 2.0 ** -24
    z = x @ router.T
    dz = eps * np.abs(x) @ np.abs(router).T + 2.0 ** -22
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    experts = np.argsort(-z, axis=1, kind="stable")[:, :top]
    weights = np.take_along_axis(p, experts, 1)
    if renorm:
        weights = weights / weights.sum(1, keepdims=True)
    out, tol = np.zeros((M, K)), np.zeros((M, K))
    for m in range(M):
        dw = 4 * dz[m].max() + 8 * eps
        for e, w in zip(experts[m], weights[m]):
            g, u = ((q[e].astype(np.float64) * s[e].astype(np.float64)[:, None]) for q, s in ((qg, sg), (qu, su)))
            d = qd[e].astype(np.float64) * sd[e].astype(np.float64)[:, None]
            gv, uv = g @ x[m], u @ x[m]
            ga, ua = np.abs(g) @ np.abs(x[m]), np.abs(u) @ np.abs(x[m])
            silu = gv / (1 + np.exp(-gv))
            h = silu * uv
            dh = eps * (1.1 * ga * np.abs(uv) + np.abs(silu) * ua + np.abs(h)) + 2.0 ** -29 * np.abs(h).max()
            out[m] += w * (d @ h)
            tol[m] += w * (np.abs(d) @ (dh + (eps + dw) * np.abs(h)))
    return out, tol, experts, weights, dz


CASES = [
    # M, K, F, E, top, renormalize
    (1, 64, 64, 4, 2, True),
    (1, 512, 1424, 16, 2, True),
    (2, 1024, 96, 8, 8, False),
    (3, 208, 80, 5, 3, True),          # multiples of 16 that are not of 64
    (4, 256, 256, 64, 6, False),
    (7, 4096, 176, 3, 1, True),
    (16, 512, 272, 64, 4, True),
    (33, 320, 144, 4, 4, False),       # every expert sees every token
    (64, 128, 64, 256, 16, True),
    (70, 128, 112, 6, 2, True),        # more than one pass
    (1, 16, 16, 1, 1, False),
    (3, 100, 52, 4, 2, True),          # sizes of the plain kernels
    (1, 7, 3, 2, 2, False),
    (65, 33, 20, 9, 3, True),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_moe_against_64_bits(cuda, case):
    M, K, F, E, top, renorm = CASES[case]
    layer = _layer(M, K, F, E, 100 + case)
    want, tol, experts, weights, dz = _reference(layer, top, renorm)
    out, got_experts, got_weights = _call(layer, top, renorm, cuda)
    np.testing.assert_array_equal(got_experts, experts)
    assert (np.abs(got_weights - weights) <= (4 * dz.max(1, keepdims=True) + 2.0 ** -20) * weights).all()
    assert (np.abs(out - want) <= tol).all(), (np.abs(out - want) / tol).max()
    np.testing.assert_array_equal(_call(layer, top, renorm, cuda, routing=False), out)  # and the same bits again


@pytest.mark.parametrize("shift", [1, 4, 8])
def test_moe_unaligned_buffers(cuda, shift):
    layer = _layer(5, 256, 128, 6, 7)
    want, tol, experts, _, _ = _reference(layer, 2, True)
    out, got_experts, _ = _call(layer, 2, True, cuda, shift=shift)
    np.testing.assert_array_equal(got_experts, experts)
    assert (np.abs(out - want) <= tol).all()


def test_moe_ties_go_to_the_lowest_index(cuda):
    for M, E, top in ((3, 12, 5), (20, 48, 8)):
        layer = _layer(M, 256, 64, E, 11, ties=True)
        want, tol, experts, _, _ = _reference(layer, top, True)
        x, router = layer[0].astype(np.float64), layer[1].astype(np.float64)
        # equal rows of the router: equal logits in 64 bits only if numpy sums them alike, so rank by row content
        _, kind = np.unique(router, axis=0, return_inverse=True)
        z = np.stack([(x * router[np.flatnonzero(kind == k)[0]]).sum(1) for k in range(kind.max() + 1)], 1)[:, kind.ravel()]
        order = np.argsort(-z, axis=1, kind="stable")[:, :top]
        out, got, _ = _call(layer, top, True, cuda)
        np.testing.assert_array_equal(got, order)
        assert np.isfinite(out).all()


def test_moe_extreme_magnitudes_and_zero_tokens(cuda):
    layer = _layer(6, 256, 128, 8, 21)
    x = layer[0]
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e12
    x[3, 5:] = 0
    x[4] *= (10.0 ** np.random.default_rng(1).integers(-12, 3, 256)).astype(np.float32)
    layer[1][:] *= np.float32(1e-3)
    with np.errstate(over="ignore"):
        want, tol, experts, _, _ = _reference(layer, 3, True)
    out, got, _ = _call(layer, 3, True, cuda)
    rows = [1, 3, 4, 5]  # (logits of 1e9 make one expert certain: row 2's order is checked, its weights may underflow)
    assert not out[0].any()
    np.testing.assert_array_equal(got[[2, *rows], :1], experts[[2, *rows], :1])
    assert (np.abs(out[rows] - want[rows]) <= tol[rows] + 1e-44).all()
    assert np.isfinite(out[2]).all()


@pytest.mark.parametrize("sizes", [(256, 128), (100, 52)])
def test_moe_nan_stays_with_its_token(cuda, sizes):
    layer = _layer(5, *sizes, 4, 31)
    clean = _call(layer, 2, True, cuda, routing=False)
    for bad in (np.nan, np.inf):
        layer[0][3, 17] = bad
        out, experts, _ = _call(layer, 2, True, cuda)
        assert np.isnan(out[3]).all()
        np.testing.assert_array_equal(out[[0, 1, 2, 4]], clean[[0, 1, 2, 4]])
        assert ((experts >= 0) & (experts < 4)).all()


def test_moe_expert_offsets_pass_32_bits(cuda):
    """Codes of one matrix beyond 2^31 bytes: the last expert lies past them."""
    torch = _torch()
    E, F, K = 18, 11008, 11008
    small = _layer(1, K, F, 1, 41)
    gate = torch.zeros((E, F, K), dtype=torch.int8, device=cuda)
    gate[-1] = torch.from_numpy(small[2][0][0]).to(cuda)
    scale = torch.zeros((E, F), device=cuda)
    scale[-1] = torch.from_numpy(small[2][1][0]).to(cuda)
    x = torch.from_numpy(small[0]).to(cuda)
    router = torch.zeros((E, K), device=cuda)
    router[-1] = x[0] / 100
    out = pc.moe(x, router, gate, scale, gate, scale, gate, scale, top_k=1)
    one = [t[-1:].contiguous() for t in (gate, scale)]
    want = pc.moe(x, router[-1:].contiguous(), *one, *one, *one, top_k=1)
    assert out.abs().max() > 0
    assert torch.allclose(out, want, rtol=1e-5, atol=0)


def test_moe_refusals(cuda):
    torch = _torch()
    x, router, gate, up, down = ([torch.from_numpy(a).to(cuda) for a in (t if isinstance(t, tuple) else (t,))]
                                 for t in _layer(2, 64, 32, 4, 51))
    args = [*x, *router, *gate, *up, *down]
    assert pc.moe(*args, top_k=2).shape == (2, 64)
    for i in range(len(args)):
        for change in (lambda t: t.double(), lambda t: t[..., :-1], lambda t: t.cpu()):
            bad = list(args)
            bad[i] = change(bad[i])
            with pytest.raises((ValueError, pc.PopcornError)):
                pc.moe(*bad, top_k=2)
    for top in (0, 5, -1):
        with pytest.raises((pc.PopcornError, RuntimeError)):
            pc.moe(*args, top_k=top)
    with pytest.raises(ValueError):
        pc.moe(*args, top_k=2, out=torch.zeros((2, 63), device=cuda))


@pytest.mark.parametrize("M, K, F, E, top", [
    # wide hidden sizes: more than 16 output channels to an SM, by tokens of a pass and tokens of an expert
    (3, 2560, 272, 4, 2), (8, 2560, 48, 16, 2), (12, 2560, 80, 3, 2), (33, 2560, 64, 4, 2), (57, 2544, 32, 30, 1),
    (2, 4096, 80, 4, 2), (3, 4096, 320, 4, 2), (9, 4096, 64, 8, 1), (20, 4096, 64, 4, 3), (41, 4096, 48, 2, 1),
    (60, 4096, 48, 8, 4), (5, 5120, 48, 4, 2), (64, 5120, 32, 64, 2), (6, 9488, 32, 2, 1),
])
def test_moe_wide_hidden_sizes(cuda, M, K, F, E, top):
    layer = _layer(M, K, F, E, 900 + M)
    want, tol, experts, weights, dz = _reference(layer, top, True)
    out, got_experts, got_weights = _call(layer, top, True, cuda)
    np.testing.assert_array_equal(got_experts, experts)
    assert (np.abs(got_weights - weights) <= (4 * dz.max(1, keepdims=True) + 2.0 ** -20) * weights).all()
    assert (np.abs(out - want) <= tol).all(), (np.abs(out - want) / tol).max()
    np.testing.assert_array_equal(_call(layer, top, True, cuda, routing=False), out)
