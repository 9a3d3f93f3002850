"""A step of many requests as a program runs it: projection, pages, rotary positions, the 4-bit cache and attention over it, on
the GPU alone; each part against its plain form, eager and captured, with sequences that come, grow, wait for pages and go."""
import numpy as np
import pytest
import torch

import kv4_ref as R4
import kv_ref as R
from pages_ref import Pool
from test_gpu_rope import _ref as rope_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Model:
    """One layer's projection and what a program keeps beside it."""

    def __init__(self, n, rows, heads, kv, dim, blocks, pages, rot, interleaved, seed):
        import h3mi
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.n, self.rows, self.heads, self.kv, self.dim = n, rows, heads, kv, dim
        width, out = 256, (heads + 2 * kv) * dim
        self.w = torch.randint(-127, 128, (out, width), generator=g, device=DEV, dtype=torch.int8)
        self.ws = torch.rand(out, generator=g, device=DEV) * 1e-3 + 1e-4
        self.x = torch.zeros(n * rows, width, device=DEV, dtype=torch.bfloat16)
        self.counts, self.keep = (torch.zeros(n, dtype=torch.int32, device=DEV) for _ in range(2))
        self.freqs, self.amplitude = h3mi.rotary_frequencies(rot, scaling="yarn", factor=4.0, window=512)
        self.interleaved = interleaved
        self.fresh(blocks, pages)

    def fresh(self, blocks, pages):
        import h3mi
        self.pool, self.cache = h3mi.kv_pool(pages), h3mi.kv_cache(pages, self.kv, self.dim, bits=4)
        self.tables = torch.full((self.n, blocks), -1, dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(self.n, dtype=torch.int32, device=DEV)

    def step(self):
        import h3mi
        h3mi.kv_release_(self.pool, self.tables, self.lens, self.keep)
        granted, positions, slots = h3mi.kv_extend_(self.pool, self.tables, self.lens, self.rows, counts=self.counts)
        qkv = h3mi.w8a8_linear(self.x, self.w, self.ws).view(self.n, self.rows, -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv, self.kv], 2)
        before = qkv.clone()
        h3mi.rotary_(q, k, positions, self.freqs, interleaved=self.interleaved, amplitude=self.amplitude)
        h3mi.kv_write_(self.cache, k, v, self.tables, self.lens, counts=granted)
        out = h3mi.kv_attention(q, self.cache, self.tables, self.lens, causal=True, counts=granted)
        return out, granted, positions, slots, before, qkv


def _change(m, rng, r):
    """Some sequences lose all, or some, of their tokens; the others get up to `rows` more."""
    lens = m.lens.cpu().numpy()
    keep = np.where(rng.random(m.n) < 0.3, 0, np.where(rng.random(m.n) < 0.2, lens // 2, 2 ** 31 - 1))
    m.keep.copy_(torch.from_numpy(keep.astype(np.int32)))
    m.counts.copy_(torch.from_numpy(rng.integers(0, m.rows + 1, m.n).astype(np.int32)))
    m.x.normal_()
    return keep


SHAPES = [(4, 90, 6, 2, 128, 8, 14, 64, True), (3, 1, 10, 2, 128, 3, 4, 128, False), (2, 150, 2, 2, 256, 6, 9, 256, False), (5, 40, 4, 4, 64, 4, 9, 64, True)]


@pytest.mark.parametrize("shape", SHAPES)
def test_step(shape):
    m, rng = Model(*shape, seed=1), np.random.default_rng(shape[1])
    ref = Pool(m.pool.free.cpu().numpy(), int(m.pool.count), m.tables.cpu().numpy(), m.lens.cpu().numpy())
    plain = R4.Cache4(shape[6], m.kv, m.dim)
    short = 0
    for r in range(400):
        keep = _change(m, rng, r)
        if r >= 8:  # and then all grow, until some wait for pages
            if short:
                break
            keep = np.full(m.n, 2 ** 31 - 1)
            m.keep.fill_(2 ** 31 - 1), m.counts.fill_(m.rows)
        ref.release(keep)
        want = ref.extend(m.rows, m.counts.cpu().numpy())
        out, granted, positions, slots, before, qkv = m.step()
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip((granted, positions, slots), want)) and ref.same(m.pool, m.tables, m.lens) == []
        short += int((want[0] < m.counts.cpu().numpy()).sum())
        turned, kept = m.heads + m.kv, before[:, :, m.heads + m.kv:]
        exact, off = rope_ref(before[:, :, :turned].double().cpu().numpy(), want[1], m.freqs.cpu().numpy(), m.interleaved, False, m.amplitude)
        assert (np.abs(qkv[:, :, :turned].double().cpu().numpy() - exact) <= off).all() and torch.equal(qkv[:, :, turned:], kept)
        q, k, v = (t.double().cpu().numpy() for t in qkv.split([m.heads, m.kv, m.kv], 2))
        R4.write(plain, k, v, ref.tables, ref.lens, want[0])
        assert plain.same(m.cache) == []
        exact, mag, top = R.attention(plain.plain(), q, ref.tables, ref.lens, want[0], True)
        d = np.abs(out.double().cpu().numpy() - exact)
        assert (d <= R.bound(exact, mag, top, m.dim)).all() and (d[mag == 0] == 0).all()
        # a slot is where the token went
        at = torch.from_numpy(want[2]).reshape(-1)
        rows = at[at >= 0]
        if len(rows):
            got = m.cache.v.cpu()[rows // 64, :, rows % 64]
            assert torch.equal(got, torch.from_numpy(R4.quantize(v.reshape(-1, m.kv, m.dim)[(at >= 0).numpy()])[0]))
    assert short > 0


@pytest.mark.parametrize("shape", SHAPES)
def test_captured_step(shape):
    """One captured step, replayed as the sequences change, beside an eager program of its own pool and cache; another stream
    is at work between."""
    m, eager = Model(*shape, seed=2), Model(*shape, seed=2)
    m.step()
    m.fresh(shape[5], shape[6])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step()
    side = torch.cuda.Stream()
    rng = np.random.default_rng(4)
    for r in range(6):
        _change(eager, rng, r)
        for name in ("keep", "counts", "x"):
            getattr(m, name).copy_(getattr(eager, name))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            torch.randn(1 << 20, device=DEV).sum()
        want = eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r
        assert all(torch.equal(a, b) for a, b in zip((*m.pool, *m.cache, m.tables, m.lens), (*eager.pool, *eager.cache, eager.tables, eager.lens))), r
