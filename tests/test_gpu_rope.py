"""Rotary positions against long double on the CPU."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _h():
    import h3mi
    return h3mi


def _ref(x, positions, freqs, interleaved, inverse, amplitude):
    """(result, bound) of float64 [n, rows, heads, dim]; rows at a position below 0 as they are."""
    rot, x = 2 * len(freqs), x.astype(np.longdouble)
    a = positions.astype(np.longdouble)[..., None] * freqs.astype(np.longdouble)
    c, s = (amplitude * f(a)[:, :, None] for f in (np.cos, np.sin))
    s = -s if inverse else s
    first = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    out, off = x.copy(), np.zeros(x.shape)
    u, v = x[..., first], x[..., second]
    out[..., first], out[..., second] = u * c - v * s, u * s + v * c
    # The angle: two roundings in 64 bits and the factor's (3 2^-53 of it), then one to 32 bits of at most half a turn (pi 2^-25).
    # Sine and cosine: two steps of 1 at most (2^-22), the amplitude's product and the two products and the sum (4 2^-24).
    off[..., first] = off[..., second] = (np.abs(u) + np.abs(v)) * abs(amplitude) * (
        np.abs(a)[:, :, None] * 3 * 2.0 ** -53 + math.pi * 2.0 ** -25 + 2.0 ** -22 + 4 * 2.0 ** -24)
    # and the result's own rounding, of what is within that of the exact one
    half = torch.finfo(torch.bfloat16).eps / 2
    off[..., :rot] += half * (np.abs(out[..., :rot]) + off[..., :rot]) + 2.0 ** -134
    gone = positions < 0
    out[gone], off[gone] = x[gone], 0
    return out.astype(np.float64), off.astype(np.float64)


def _bf(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16)


def _check(got, x, positions, freqs, interleaved, inverse, amplitude):
    want, off = _ref(x.double().numpy(), positions.numpy(), freqs.numpy(), interleaved, inverse, amplitude)
    d = np.abs(got.double().cpu().numpy() - want)
    assert got.shape == x.shape and (d <= off).all(), (d - off).max()


@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (128, 32), (128, 96), (64, 64), (64, 16), (256, 256), (80, 80), (80, 48), (72, 16), (128, 126),
                                     (128, 2), (64, 24), (40, 40), (8, 8), (8, 2), (512, 512), (512, 510), (104, 40), (128, 124), (64, 4), (72, 60)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,rows,hq,hk", [(1, 1, 3, 3), (3, 37, 5, 1), (2, 300, 2, 4)])
def test_rope(dim, rot, interleaved, n, rows, hq, hk):
    """Views of a projection's output, in place and into new tensors, forth and back; rows behind a sequence's own."""
    h = _h()
    rng = np.random.default_rng(dim * rot + rows)
    qkv = _bf(rng, n, rows, hq + 2 * hk, dim)
    positions = torch.from_numpy(rng.integers(0, 200000, (n, 1)) + np.arange(rows)).to(torch.int32)
    positions[:, rows - rows // 3:] = -1
    positions[-1, 0] = 0
    freqs, amplitude = h.rotary_frequencies(rot, scaling="yarn", factor=4.0, device="cpu")
    for inverse in (False, True):
        d = qkv.to(DEV)
        q, k = d[:, :, :hq], d[:, :, hq:hq + hk]
        args = (positions.to(DEV), freqs.to(DEV))
        new = h.rotary(q, k, *args, interleaved=interleaved, inverse=inverse, amplitude=amplitude)
        assert torch.equal(d.cpu(), qkv) and all(t.is_contiguous() for t in new)
        got = h.rotary_(q, k, *args, interleaved=interleaved, inverse=inverse, amplitude=amplitude)
        assert got[0] is q and got[1] is k
        for y, z, x in ((q, new[0], qkv[:, :, :hq]), (k, new[1], qkv[:, :, hq:hq + hk])):
            _check(y, x, positions, freqs, interleaved, inverse, amplitude)
            assert torch.equal(y, z)
        assert torch.equal(d[:, :, hq + hk:].cpu(), qkv[:, :, hq + hk:])  # the values between
        assert torch.equal(h.rotary(qkv[:, :, :hq].to(DEV), None, *args, interleaved, inverse, amplitude)[0], new[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(interleaved):
    """The angle of a position of 31 bits is as good as that of a near one."""
    h = _h()
    rng = np.random.default_rng(4)
    positions = torch.tensor([[0, 1, 2, 4095, 131071, 1 << 20, (1 << 24) + 1, (1 << 30) + 1, 2 ** 31 - 1, -1, -2 ** 31]], dtype=torch.int32)
    freqs = torch.from_numpy(np.concatenate([np.linspace(0, math.pi, 60), [1.0, 100.0, 1e-9, -0.5]]))
    x = _bf(rng, 1, 11, 4, 128)
    _check(h.rotary(x.to(DEV), None, positions.to(DEV), freqs.to(DEV), interleaved=interleaved)[0], x, positions, freqs, interleaved, False, 1.0)


@pytest.mark.parametrize("n,rows,hq,hk,dim,rot", [(1, 3001, 56, 56, 128, 128), (4, 701, 40, 8, 128, 64), (300, 1, 40, 8, 128, 128), (1, 9001, 1, 1, 64, 64),
                                                  (1, 1, 600, 300, 256, 256), (2, 1500, 24, 24, 64, 32), (1, 5, 56, 56, 128, 126),
                                                  (2, 1500, 24, 24, 64, 12)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_every_split_of_the_rows(n, rows, hq, hk, dim, rot, interleaved):
    """Many rows to a workgroup, many workgroups to a row."""
    h = _h()
    rng = np.random.default_rng(rows)
    q, k = _bf(rng, n, rows, hq, dim), _bf(rng, n, rows, hk, dim)
    positions = torch.from_numpy(rng.integers(-1, 5000, (n, rows))).to(torch.int32)
    freqs, _ = h.rotary_frequencies(rot, device="cpu")
    got = h.rotary(q.to(DEV), k.to(DEV), positions.to(DEV), freqs.to(DEV), interleaved=interleaved)
    for y, x in zip(got, (q, k)):
        some = rng.choice(rows, min(rows, 60), replace=False)
        _check(y[:, some], x[:, some], positions[:, some], freqs, interleaved, False, 1.0)
    # all of it against the products in torch, to a step of bf16
    a = positions.to(DEV).double()[..., None] * freqs.to(DEV)
    c, s = (f(a).float()[:, :, None] for f in (torch.cos, torch.sin))
    for y, x in zip(got, (q, k)):
        x = x.to(DEV)
        u, v = (x[..., 0:rot:2].float(), x[..., 1:rot:2].float()) if interleaved else (x[..., :rot // 2].float(), x[..., rot // 2:rot].float())
        pair = (u * c - v * s, u * s + v * c)
        want = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
        want = torch.where((positions.to(DEV) >= 0)[..., None, None], want, x[..., :rot].float())
        assert ((y[..., :rot].float() - want).abs() <= 2.0 ** -8 * want.abs() * 1.01 + 1e-5).all()
        assert torch.equal(y[..., rot:], x[..., rot:])


def test_sequences_between_each_other():
    """Strides that run over sequences first, and one row of many sequences."""
    h = _h()
    rng = np.random.default_rng(6)
    freqs, _ = h.rotary_frequencies(128, device="cpu")
    for n, rows in ((5, 7), (5, 1), (1, 7)):
        x = _bf(rng, rows, n, 6, 128)
        positions = torch.from_numpy(rng.integers(0, 99, (n, rows))).to(torch.int32)
        d = x.to(DEV)
        t = d.transpose(0, 1)
        h.rotary_(t[:, :, :4], t[:, :, 4:], positions.to(DEV), freqs.to(DEV))
        _check(t, x.transpose(0, 1), positions, freqs, False, False, 1.0)


@pytest.mark.parametrize("hq,hk", [(4, 4), (5, 2)])
def test_q_and_k_of_one_buffer(hq, hk):
    """All of a sequence's q rows before its k rows, all of a token's: in place, with heads of their own."""
    h = _h()
    rng = np.random.default_rng(16)
    n, rows, dim = 3, 37, 128
    freqs, _ = h.rotary_frequencies(dim, device="cpu")
    positions = torch.from_numpy(rng.integers(-1, 9999, (n, rows))).to(torch.int32)
    for tokens_first in (False, True):
        a, b = (rows, n) if tokens_first else (n, rows)
        x = _bf(rng, a, b * (hq + hk) * dim)
        d = x.to(DEV)

        def sides(t):
            two = t[:, :b * hq * dim].unflatten(1, (b, hq, dim)), t[:, b * hq * dim:].unflatten(1, (b, hk, dim))
            return [s.transpose(0, 1) for s in two] if tokens_first else two

        h.rotary_(*sides(d), positions.to(DEV), freqs.to(DEV))
        for got, was in zip(sides(d), sides(x)):
            _check(got, was, positions, freqs, False, False, 1.0)


def test_inverse_is_the_gradient():
    """<g, R x> = <R' g, x>, and differences of R along a direction; to the roundings of both sides."""
    h = _h()
    rng = np.random.default_rng(7)
    freqs, amplitude = h.rotary_frequencies(64, scaling="yarn", factor=16.0)
    positions = torch.from_numpy(rng.integers(0, 99999, (2, 50))).to(torch.int32).to(DEV)
    x, g = (_bf(rng, 2, 50, 3, 128).to(DEV) for _ in range(2))
    for interleaved in (False, True):
        y = h.rotary(x, None, positions, freqs, interleaved, False, amplitude)[0].double()
        b = h.rotary(g, None, positions, freqs, interleaved, True, amplitude)[0].double()
        left, right = (g.double() * y).sum(), (b * x.double()).sum()
        half = 2.0 ** -8
        most = half * ((g.double() * y).abs().sum() + (b * x.double()).abs().sum()) * 1.01
        assert abs(left - right) <= most
        # R is linear: R (x + g) - R x = R g
        both = (x.float() + g.float()).to(torch.bfloat16)
        step = (both.double() - x.double())
        d = h.rotary(both, None, positions, freqs, interleaved, False, amplitude)[0].double() - y
        want = h.rotary(step.to(torch.bfloat16), None, positions, freqs, interleaved, False, amplitude)[0].double()
        slack = half * (d.abs() + 2 * y.abs() + want.abs() * 2) * 1.01 + half * amplitude * 2 * step.abs().amax(-1, keepdim=True) + 1e-5
        assert ((d - want).abs() <= slack).all()


@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 60), (256, 126)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_transpose_pair_by_pair(dim, rot, interleaved):
    """<g, R x> = <R' g, x> over every pair of elements, within the roundings of its four results; a rotation the wrong way round,
    or none, passes it in few pairs."""
    h = _h()
    rng = np.random.default_rng(dim + rot)
    freqs, amplitude = h.rotary_frequencies(rot, scaling="yarn", factor=16.0)
    positions = torch.from_numpy(rng.integers(1, 99999, (2, 50))).to(torch.int32).to(DEV)
    x, g = (_bf(rng, 2, 50, 3, dim).to(DEV) for _ in range(2))

    def pairs(t):
        t = t[..., :rot].double()
        return t.unflatten(-1, (-1, 2)) if interleaved else t.unflatten(-1, (2, -1)).transpose(-1, -2)

    y = pairs(h.rotary(x, None, positions, freqs, interleaved, False, amplitude)[0])
    u, w = pairs(x), pairs(g)

    def within(b):
        b = pairs(b)
        # each result is off by half a step at most, 2^-8 of it, and by what 32 bits add, less than a hundredth of that beside
        # the larger of the pair's elements
        most = 2.0 ** -8 * ((w * y).abs() + (b * u).abs()).sum(-1) + 2.0 ** -15 * amplitude * w.abs().sum(-1) * u.abs().sum(-1)
        return ((w * y).sum(-1) - (b * u).sum(-1)).abs() <= most

    turned = h.rotary(g, None, positions, freqs, interleaved, True, amplitude)[0]
    assert within(turned).all()
    # the slow pairs of a short turn hardly move: the first half of them
    for wrong in (h.rotary(g, None, positions, freqs, interleaved, False, amplitude)[0], h.rotary(g, None, torch.zeros_like(positions), freqs, interleaved, True, amplitude)[0]):
        assert within(wrong)[..., :rot // 4].double().mean() < 0.1
    if rot < dim:
        assert torch.equal(turned[..., rot:], g[..., rot:])


def test_special_values_stay_in_their_pairs():
    h = _h()
    rng = np.random.default_rng(8)
    freqs, _ = h.rotary_frequencies(128)
    positions = torch.tensor([[5, -1, 7]], dtype=torch.int32, device=DEV)
    x = _bf(rng, 1, 3, 2, 128).to(DEV)
    for interleaved in (False, True):
        want = h.rotary(x, None, positions, freqs, interleaved)[0]
        bad = x.clone()
        bad[0, 0, 1, 10], bad[0, 1, 0, 3] = float("nan"), float("inf")
        got = h.rotary(bad, None, positions, freqs, interleaved)[0]
        other = 11 if interleaved else 74
        hit = torch.zeros_like(x, dtype=torch.bool)
        hit[0, 0, 1, 10] = hit[0, 0, 1, other] = True
        assert got[hit].isnan().all() and got[0, 1, 0, 3] == float("inf")
        hit[0, 1, 0, 3] = True
        assert torch.equal(got[~hit], want[~hit])


def test_frequencies():
    h = _h()
    i = np.arange(32)
    f, amp = h.rotary_frequencies(64, base=500.0, device="cpu")
    assert f.dtype == torch.float64 and np.allclose(f, 500.0 ** (-i / 32), rtol=1e-14) and amp == 1.0
    assert np.allclose(h.rotary_frequencies(64, scaling="linear", factor=8.0)[0].cpu(), 10000.0 ** (-i / 32) / 8, rtol=1e-14)
    f = h.rotary_frequencies(64, scaling="ntk", factor=8.0)[0].cpu().numpy()
    assert f[0] == 1.0 and np.isclose(f[31], 10000.0 ** (-31 / 32) / 8, rtol=1e-12)
    f, amp = h.rotary_frequencies(64, scaling="yarn", factor=8.0, window=4096)
    plain, f = 10000.0 ** (-i / 32), f.cpu().numpy()
    turns = 4096 * plain / (2 * math.pi)
    assert np.allclose(f[turns >= 34], plain[turns >= 34]) and np.allclose(f[turns <= 0.7], plain[turns <= 0.7] / 8) and np.isclose(amp, 1 + 0.1 * math.log(8))
    # quotients of up to 8, each off by at most 8 roundings of 2^-53 (4 of either number): equal ones differ by 2 * 8 * 8 of them
    assert (np.diff(plain / f) >= -128 * 2.0 ** -53).all()
    for kw in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.5), dict(rot_dim=8, scaling="other"), dict(rot_dim=8, window=0)):
        with pytest.raises(ValueError):
            h.rotary_frequencies(**kw)


def test_captured_and_streams():
    h = _h()
    rng = np.random.default_rng(9)
    freqs, _ = h.rotary_frequencies(128)
    q, k = _bf(rng, 2, 33, 4, 128).to(DEV), _bf(rng, 2, 33, 1, 128).to(DEV)
    positions = torch.zeros(2, 33, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    h.rotary(q, k, positions, freqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = h.rotary(q, k, positions, freqs)
    for r in range(4):
        positions.random_(-1, 9999)
        q.normal_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = h.rotary(q, k, positions, freqs)
        want = h.rotary(q, k, positions, freqs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(out, want, beside)), r


def test_rows_past_32_bits():
    """Of tensors of more than 2^32 bytes the last rows are turned as they are alone, in place and into new ones."""
    h = _h()
    rows, heads, some = 300_000, 56, 50
    x = torch.empty((1, rows, heads, 128), device=DEV, dtype=torch.bfloat16).normal_()
    assert x.numel() * 2 > 2 ** 32
    freqs, _ = h.rotary_frequencies(128)
    positions = torch.arange(rows, dtype=torch.int32, device=DEV)[None]
    want = h.rotary(x[:, -some:], None, positions[:, -some:].contiguous(), freqs)[0]
    assert torch.equal(h.rotary(x, None, positions, freqs)[0][:, -some:], want)
    h.rotary_(x, None, positions, freqs)
    assert torch.equal(x[:, -some:], want)


def test_refusals():
    h = _h()
    freqs, _ = h.rotary_frequencies(64)
    positions = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device=DEV)
    k = q.clone()
    for args, msg in (((q.float(), k, positions, freqs), "q must be bfloat16"), ((q, k[:, :2], positions, freqs), "k must be"),
                      ((q, k[..., :32], positions, freqs), "k must be"), ((q, k, positions.long(), freqs), "positions"), ((q, k, positions[0], freqs), "positions"),
                      ((q, k, positions, freqs.float()), "freqs"), ((q, k.cpu(), positions, freqs), "k is on"), ((q.transpose(2, 3), None, positions, freqs), "contiguous"),
                      ((q[..., :32].expand(2, 3, 4, 32), None, positions, freqs[:8]), "contiguous")):
        with pytest.raises(ValueError, match=msg):
            h.rotary(*args)
    for call, msg in ((lambda: h.rotary_(q, q, positions, freqs), "overlap"), (lambda: h.rotary_(q, q[:, :, 1:], positions, freqs), "overlap"),
                      (lambda: h.rotary_(q[:1].expand(2, 3, 4, 64), None, positions, freqs), "shorter"),
                      (lambda: h.rotary(q, k, positions, torch.ones(33, dtype=torch.float64, device=DEV)), "rot=66"),
                      (lambda: h.rotary(q, k, positions, freqs, amplitude=float("inf")), "amplitude"),
                      (lambda: h.rotary_(q.view(-1)[4:4 + 2 * 3 * 3 * 64].view(2, 3, 3, 64), None, positions, freqs), "aligned"),
                      (lambda: h.rotary_(q.as_strided((2, 3, 2, 64), (256, 128, 64, 1)), None, positions, freqs), "overlap")):
        with pytest.raises(h._lib.H3miError, match=msg):
            call()
    with pytest.raises(RuntimeError, match="no gradient"):
        h.rotary(q.requires_grad_(), None, positions, freqs)
    with torch.no_grad():
        h.rotary(q, None, positions, freqs)


def test_nothing_to_do():
    h = _h()
    freqs, _ = h.rotary_frequencies(64)
    for n, rows in ((0, 3), (2, 0)):
        x = torch.zeros(n, rows, 4, 64, dtype=torch.bfloat16, device=DEV)
        y, z = h.rotary(x, None, torch.zeros(n, rows, dtype=torch.int32, device=DEV), freqs)
        assert y.shape == x.shape and z is None
