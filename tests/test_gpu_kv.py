"""The 8-bit key/value cache against plain forms on the CPU: written bytes are pinned, reading is exact, selections are
equal, attention is within the bounds that kv_ref.bound derives."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _h():
    import h3mi
    return h3mi


def _bf(a):
    """float32 array of bf16 values -> bf16 GPU tensor"""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16).to(DEV)


def _np(t):
    return t.detach().float().cpu().numpy()


def _round(a):
    return torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16).float().numpy()


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _tables(rng, n, blocks, spare=2):
    return rng.permutation(n * blocks + spare)[:n * blocks].reshape(n, blocks).astype(np.int32)


# ------------------------------------------------------------------ writing and reading


@pytest.mark.parametrize("heads,dim", [(3, 64), (2, 128), (5, 256)])
@pytest.mark.parametrize("steps", [
    [(100, 100)], [(64, 64), (1, 65), (1, 66), (70, 136)], [(1, 1), (62, 63), (1, 64), (1, 65)], [(130, 130), (3, 100), (200, 256)],
])
def test_write_is_pinned(heads, dim, steps):
    """A chain of writes (rows, length after it), every row in use; the tokens grow so that scales do."""
    h = _h()
    rng = np.random.default_rng(len(steps) * dim)
    blocks = 4
    ref = R.Cache(2 * blocks + 2, heads, dim, seed=1)
    cache, tables = ref.to(), _tables(rng, 2, blocks)
    for x, (rows, end) in enumerate(steps):
        k = _round(rng.standard_normal((2, rows, heads, dim)) * 3.0 ** x)
        v = _round(rng.standard_normal((2, rows, heads, dim)) * 1.5 ** x)
        lens = np.array([end, max(end - 5, 0)])
        counts = np.array([rows, max(rows - 5, 0)])
        R.write(ref, k, v, tables, lens, counts)
        assert h.kv_write_(cache, _bf(k), _bf(v), _i32(tables), _i32(lens), counts=_i32(counts)) is cache
        assert ref.same(cache) == []


def test_write_of_views_and_without_counts():
    h = _h()
    rng = np.random.default_rng(5)
    heads, dim, rows = 3, 128, 77
    qkv = _round(rng.standard_normal((2, rows, 3, heads, dim)))
    ref = R.Cache(6, heads, dim, seed=2)
    cache, tables, lens = ref.to(), _tables(rng, 2, 2), np.array([77, 100])
    t = _bf(qkv)
    h.kv_write_(cache, t[:, :, 1], t[:, :, 2], _i32(tables), _i32(lens))
    R.write(ref, qkv[:, :, 1], qkv[:, :, 2], tables, lens, [rows, rows])
    assert ref.same(cache) == []


@pytest.mark.parametrize("first,second", [
    (1.0, 1.0), (1.0, 0.25), (1.0, 2.0), (1.0, 2.0078125), (1.0, 255.0), (1.0, 256.0), (1.0, 258.0), (1.0, 1e30), (0.0, 3.0),
    (3.0, 0.0), (1e-38, 1e-38), (1e-38, 3e-38), (9.2e-41, 1.0), (1e-40, 3e-40), (3e38, 3e38), (1e-3, 3e38),
    (1.0, np.inf), (np.inf, 1.0), (np.nan, 1.0), (1.0, np.nan), (1.0, -np.inf),
])
def test_scale_growth(first, second):
    """The second write of a block against its first, at the edges of every rule."""
    h = _h()
    rng = np.random.default_rng(9)
    heads, dim = 2, 64
    ref = R.Cache(2, heads, dim, seed=3)
    cache, tables = ref.to(), np.array([[1]], np.int32)
    for end, rows, top in ((20, 20, first), (21, 1, second), (40, 19, 1.0 if np.isfinite(first) else first)):
        x = rng.uniform(-1, 1, (2, 1, rows, heads, dim))
        x[:, :, 0, :, 3] = 1.0  # the largest is `top` itself
        with np.errstate(invalid="ignore"):
            x = _round(x * top)
        R.write(ref, x[0], x[1], tables, [end], [rows])
        h.kv_write_(cache, _bf(x[0]), _bf(x[1]), _i32(tables), _i32([end]))
        assert ref.same(cache) == [], (end, first, second)


def test_write_drops_what_has_no_place():
    """Lengths past the table, rows before token 0, negative counts and lengths, pages outside the pool, no rows."""
    h = _h()
    rng = np.random.default_rng(11)
    heads, dim, rows = 2, 64, 90
    ref = R.Cache(9, heads, dim, seed=4)
    cache = ref.to()
    tables = np.array([[0, 1], [2, 9], [3, 4], [-1, 5], [6, 7], [8, 2147483647]], np.int32)
    lens, counts = np.array([140, 128, 30, 128, -5, 100]), np.array([90, 90, 90, 200, 20, -3])
    k, v = (_round(rng.standard_normal((6, rows, heads, dim))) for _ in range(2))
    R.write(ref, k, v, tables, lens, counts)
    h.kv_write_(cache, _bf(k), _bf(v), _i32(tables), _i32(lens), counts=_i32(counts))
    assert ref.same(cache) == []
    h.kv_write_(cache, _bf(k[:, :0]), _bf(v[:, :0]), _i32(tables), _i32(lens))
    h.kv_write_(cache, _bf(k[:0]), _bf(v[:0]), _i32(tables[:0]), _i32(lens[:0]))
    assert ref.same(cache) == []


@pytest.mark.parametrize("heads,dim", [(3, 64), (2, 128), (5, 256)])
@pytest.mark.parametrize("length,starts", [(1, None), (64, None), (200, None), (65, [3, 64, 127]), (130, [-10, 60, 1000]),
                                           (10, [-100, 2147483640, -2147483648])])
def test_read(heads, dim, length, starts):
    h = _h()
    rng = np.random.default_rng(13)
    ref = R.Cache(11, heads, dim, seed=5)
    tables, lens = _tables(rng, 3, 3), np.array([192, 70, 0])
    tables[0, 1] = 11  # a page outside the pool
    k, v = h.kv_read(ref.to(), _i32(tables), _i32(lens), length, starts=None if starts is None else _i32(starts))
    for i in range(3):
        a, b, _ = R.tokens(ref, tables[i], int(lens[i]))
        first = 0 if starts is None else starts[i]
        for got, want in ((k, a), (v, b)):
            full = np.zeros((length, heads, dim))
            for r in range(length):
                if 0 <= first + r < lens[i]:
                    full[r] = want[first + r]
            # one rounding of an fp32 product of an 8-bit value and a scale
            want_bits = torch.from_numpy(full).float().to(torch.bfloat16)
            assert torch.equal(got[i].cpu(), want_bits)


def test_round_trip_error():
    """Tokens written one by one: every value within a step of its block's last scale, the newest within half of one."""
    h = _h()
    rng = np.random.default_rng(17)
    heads, dim, n = 2, 128, 150
    x = _round(rng.standard_normal((2, 1, n, heads, dim)) * np.geomspace(0.01, 30, n)[None, None, :, None, None])
    cache, tables = h.kv_cache(4, heads, dim), np.array([[2, 0, 3]], np.int32)
    for t in range(n):
        h.kv_write_(cache, _bf(x[0][:, t:t + 1]), _bf(x[1][:, t:t + 1]), _i32(tables), _i32([t + 1]))
    step = np.repeat(_np(cache.k_scale)[tables[0]], 64, 0)[:n, :, None]
    got = (_np(cache.k)[tables[0]].swapaxes(1, 2).reshape(-1, heads, dim)[:n] * step)
    off = np.abs(got - x[0][0]) / step
    assert off.max() <= 1 + 1e-5 and off[-1].max() <= 0.5 + 1e-5


# ------------------------------------------------------------------ attention


def _case(rng, heads, kv, dim, n, rows, blocks, seed):
    ref = R.Cache(n * blocks + 2, kv, dim, seed=seed)
    tables = _tables(rng, n, blocks)
    q = _round(rng.standard_normal((n, rows, heads, dim)))
    return ref, tables, q


def _check(ref, q, tables, lens, counts, causal, scale=None, blocks=None, view=None):
    h = _h()
    out = h.kv_attention(_bf(q) if view is None else view, ref.to(), _i32(tables), _i32(lens), causal=causal,
                         counts=None if counts is None else _i32(counts), scale=scale, blocks=None if blocks is None else _i32(blocks))
    if counts is None:
        counts = [q.shape[1]] * q.shape[0]
    want, mag, top = R.attention(ref, q.astype(np.float64), tables, lens, counts, causal, scale, blocks)
    got = out.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    off = np.abs(got - want) / R.bound(want, mag, top, q.shape[3])
    assert off.max(initial=0.0) <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))
    assert (got[mag == 0] == 0).all()
    return out


HEADS = [(3, 3, 64), (2, 2, 128), (3, 3, 256), (10, 2, 128), (8, 1, 64), (6, 2, 256), (20, 1, 128)]


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows,lens,counts", [
    (1, [1, 64, 65], None), (1, [700, 0, 333], None), (3, [3, 200, 130], [3, 2, 0]), (16, [16, 500, 61], [16, 15, 9]),
    (17, [400, 17, 40], None), (64, [64, 129, 700], None), (65, [65, 90, 640], [65, 1, 33]), (130, [130, 2, 600], [130, 2, 129]),
    (300, [300, 700, 299], [300, 280, 299]),
])
def test_attention(heads, kv, dim, causal, rows, lens, counts):
    rng = np.random.default_rng(rows * dim + heads)
    ref, tables, q = _case(rng, heads, kv, dim, 3, rows, 11, seed=rows)
    _check(ref, q, tables, lens, counts, causal)


@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_attention_rows_that_see_nothing(rows):
    """No tokens, rows before token 0 (more rows than tokens), lengths past the table, pages outside the pool."""
    rng = np.random.default_rng(rows)
    ref, tables, q = _case(rng, 4, 2, 128, 5, rows, 3, seed=rows)
    tables[1, :] = -1
    tables[2, 1] = 10 ** 6
    tables[3] = tables[0]  # a shared prefix
    for causal in (False, True):
        _check(ref, q, tables, [0, 150, 192, rows // 2, 500], None, causal)


@pytest.mark.parametrize("rows", [1, 30, 200])
def test_attention_does_not_read_behind_the_end(rows):
    """NaN and infinite scales in pages that no sequence has, and 8-bit values behind the last token."""
    rng = np.random.default_rng(3 * rows)
    ref, tables, q = _case(rng, 4, 4, 64, 2, rows, 4, seed=1)
    free = np.setdiff1d(np.arange(10), tables[:, :3])
    ref.ks[free], ref.vs[free] = np.nan, np.inf
    _check(ref, q, tables, [192, 140], None, False)
    _check(ref, q, tables, [192, 140], None, True)


def test_attention_poisoned_block():
    """A NaN scale reaches the rows that see its block, and no others."""
    h = _h()
    rng = np.random.default_rng(2)
    for rows in (4, 300):
        ref, tables, q = _case(rng, 2, 2, 128, 1, rows, 6, seed=2)
        ref.ks[tables[0, 3], 1] = np.nan
        out = _np(h.kv_attention(_bf(q), ref.to(), _i32(tables), _i32([384]), causal=True))
        at = 384 - rows + np.arange(rows)
        assert np.isfinite(out[0, :, 0]).all() and np.isfinite(out[0, at < 192, 1]).all() and np.isnan(out[0, at >= 192, 1]).all()


@pytest.mark.parametrize("rows", [3, 20, 150])
def test_attention_poisoned_query(rows):
    """A NaN or an infinity in a query stays in its row and head."""
    h = _h()
    rng = np.random.default_rng(12)
    ref, tables, q = _case(rng, 4, 2, 128, 1, rows, 6, seed=12)
    c, t, lens = ref.to(), _i32(tables), _i32([380])
    good = _np(h.kv_attention(_bf(q), c, t, lens))
    q[0, 1, 2, 5], q[0, 2, 0, 9] = np.nan, np.inf
    bad = _np(h.kv_attention(_bf(q), c, t, lens))
    hit = np.zeros(good.shape, bool)
    hit[0, 1, 2], hit[0, 2, 0] = True, True
    assert np.isnan(bad[hit]).all() and np.array_equal(bad[~hit], good[~hit])


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 30.0])
@pytest.mark.parametrize("rows", [2, 150])
def test_attention_scales(scale, rows):
    """Steep and negative scales; a scale of 0 is the mean of the values."""
    rng = np.random.default_rng(4)
    ref, tables, q = _case(rng, 2, 2, 64, 1, rows, 5, seed=4)
    ref.ks *= 0.2
    _check(ref, q, tables, [300], None, False, scale=scale)


@pytest.mark.parametrize("rows", [1, 200])
def test_attention_zero_and_tiny_scales(rows):
    """Blocks of zero keys or values, and scales at the ends of fp32."""
    rng = np.random.default_rng(6)
    ref, tables, q = _case(rng, 2, 2, 128, 1, rows, 6, seed=6)
    ref.ks[tables[0, 0]] = 0
    ref.k[tables[0, 0]] = 0
    ref.vs[tables[0, 1]] = 0
    ref.v[tables[0, 1]] = 0
    ref.vs[tables[0, 2]] = 1e-39
    ref.ks[tables[0, 3]] = 1e-40
    _check(ref, q, tables, [384], None, False)
    ref.vs[:] = 1e-38
    h = _h()
    out = h.kv_attention(_bf(q), ref.to(), _i32(tables), _i32([384]))
    assert np.isfinite(_np(out)).all()


@pytest.mark.parametrize("rows", [1, 3, 129])
def test_attention_of_views(rows):
    """q as a view of a projection's output."""
    rng = np.random.default_rng(8)
    ref, tables, _ = _case(rng, 4, 2, 128, 2, rows, 5, seed=8)
    qkv = _round(rng.standard_normal((2, rows, 3, 4, 128)))
    _check(ref, qkv[:, :, 1], tables, [300, 250], None, True, view=_bf(qkv)[:, :, 1])


@pytest.mark.parametrize("rows,n,heads,kv,tokens", [(1, 1, 4, 4, 20000), (1, 3, 10, 2, 9000), (24, 1, 2, 2, 12000), (200, 1, 2, 2, 9001)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_long(rows, n, heads, kv, tokens, causal):
    """Few rows over long caches: the work is split over the tokens and joined."""
    rng = np.random.default_rng(tokens)
    blocks = -(-tokens // 64)
    ref, tables, q = _case(rng, heads, kv, 128, n, rows, blocks, seed=7)
    lens = [tokens] + [tokens // 3, 100][:n - 1]
    _check(ref, q, tables, lens, None, causal)


def _check_on_gpu(c, q, table, end, causal, out):
    """out [rows, heads, dim] of one sequence whose rows are its last, against 64 bits on the GPU, head by head."""
    rows, heads, dim = q.shape
    group = heads // c.k.shape[1]
    half = torch.finfo(torch.bfloat16).eps / 2
    page = table.long()
    at = torch.arange(end, device=DEV)
    for h in range(heads):
        k = (c.k[page, h // group].double() * c.k_scale[page, h // group].double()[:, None, None]).reshape(-1, dim)[:end]
        v = (c.v[page, h // group].double() * c.v_scale[page, h // group].double()[:, None, None]).transpose(1, 2).reshape(-1, dim)[:end]
        x = q[:, h].double() @ k.t() * dim ** -0.5
        if causal:
            x.masked_fill_(at > (end - rows + torch.arange(rows, device=DEV))[:, None], -float("inf"))
        p = torch.softmax(x, 1)
        want, mag = p @ v, p @ v.abs()
        top = (q[:, h].double().abs() @ k.abs().t() * dim ** -0.5).amax(1, keepdim=True)
        # kv_ref.bound, on the GPU
        bound = half * (mag * (1 + half) + want.abs()) * (1 + 1e-3) + 2 * mag * ((dim + 8) * 2.0 ** -24 * (top + 4)) + 1e-30
        assert ((out[:, h].double() - want).abs() <= bound).all(), h


@pytest.mark.parametrize("heads,kv,dim,rows,tokens", [
    (52, 52, 128, 1100, 33000),   # 8 waves a tile, more blocks than are looked up at once
    (52, 52, 128, 1030, 8200),    # 8 waves, 129 blocks
    (60, 12, 64, 1300, 17000),    # 4 waves, more blocks than are looked up at once, the last round split
    (18, 18, 256, 1900, 16500),
    (300, 300, 128, 70, 17000),   # one tile a head
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_large(heads, kv, dim, rows, tokens, causal):
    h = _h()
    g = torch.Generator(device=DEV).manual_seed(tokens)
    blocks = -(-tokens // 64)
    shared = 40  # heads' pages: blocks of one cache in many places
    c = h.KVCache(torch.randint(-127, 128, (shared, kv, 64, dim), generator=g, device=DEV, dtype=torch.int8),
                  torch.randint(-127, 128, (shared, kv, dim, 64), generator=g, device=DEV, dtype=torch.int8),
                  torch.rand(shared, kv, generator=g, device=DEV) * 0.02 + 0.005, torch.rand(shared, kv, generator=g, device=DEV) * 0.02 + 0.005,
                  torch.zeros(shared, kv, dim, dtype=torch.int16, device=DEV))
    q = torch.randn(1, rows, heads, dim, generator=g, device=DEV).to(torch.bfloat16)
    tables = torch.randint(0, shared, (1, blocks), generator=g, device=DEV, dtype=torch.int32)
    out = h.kv_attention(q, c, tables, _i32([tokens]), causal=causal)
    _check_on_gpu(c, q[0], tables[0], tokens, causal, out[0])


@pytest.mark.parametrize("rows,dim", [(1, 128), (20, 128), (50, 64)])
def test_attention_few_rows_unsplit(rows, dim):
    """Few rows of so many sequences that a workgroup takes a whole sequence: more blocks than are looked up at once."""
    h = _h()
    n, kv, tokens, shared = 70, 8, 17000, 30
    g = torch.Generator(device=DEV).manual_seed(rows)
    c = h.KVCache(torch.randint(-127, 128, (shared, kv, 64, dim), generator=g, device=DEV, dtype=torch.int8),
                  torch.randint(-127, 128, (shared, kv, dim, 64), generator=g, device=DEV, dtype=torch.int8),
                  torch.rand(shared, kv, generator=g, device=DEV) * 0.02 + 0.005, torch.rand(shared, kv, generator=g, device=DEV) * 0.02 + 0.005,
                  torch.zeros(shared, kv, dim, dtype=torch.int16, device=DEV))
    q = torch.randn(n, rows, kv, dim, generator=g, device=DEV).to(torch.bfloat16)
    tables = torch.randint(0, shared, (n, 266), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.randint(rows, tokens + 1, (n,), generator=g, device=DEV, dtype=torch.int32)
    lens[0] = tokens
    out = h.kv_attention(q, c, tables, lens, causal=True)
    for i in (0, 1, n - 1):
        _check_on_gpu(c, q[i], tables[i], int(lens[i]), True, out[i])


def test_offsets_past_32_bits():
    """Pages whose bytes lie past 2^31 and whose elements past 2^32 in the pool, and rows past 2^31 elements."""
    h = _h()
    rng = np.random.default_rng(21)
    heads, dim = 64, 256
    pages = 4200  # 4200 * 64 * 64 * 256 = 4.4e9
    cache = h.kv_cache(pages, heads, dim)
    tables = np.array([[pages - 1, 1, pages - 2]], np.int32)
    small = R.Cache(3, heads, dim)
    k, v = (_round(rng.standard_normal((1, 150, heads, dim))) for _ in range(2))
    R.write(small, k, v, np.array([[0, 1, 2]]), [150], [150])
    h.kv_write_(cache, _bf(k), _bf(v), _i32(tables), _i32([150]))
    part = h.KVCache(*(t[tables[0].tolist()].contiguous() for t in cache))
    assert small.same(part) == []
    for rows in (1, 60):
        q = _round(rng.standard_normal((1, rows, heads, dim)))
        want, mag, top = R.attention(small, q.astype(np.float64), np.array([[0, 1, 2]]), [150], [rows], True)
        got = h.kv_attention(_bf(q), cache, _i32(tables), _i32([150]), causal=True).double().cpu().numpy()
        assert (np.abs(got - want) <= R.bound(want, mag, top, dim)).all()
        pick = h.kv_select(_bf(q), cache, _i32(tables), _i32([150]), 2).cpu().numpy()
        assert np.array_equal(pick, R.select(small, q.astype(np.float64), np.array([[0, 1, 2]]), [150], [rows], 2, False))
    rk, _ = h.kv_read(cache, _i32(tables), _i32([150]), 150)
    want = torch.from_numpy(R.tokens(small, [0, 1, 2], 150)[0]).float().to(torch.bfloat16)
    assert torch.equal(rk[0].cpu(), want)
    # a token stride that takes the last row past 2^31 elements
    wide = torch.empty(150 * 16_000_000, dtype=torch.bfloat16, device=DEV).as_strided((1, 150, heads, dim), (0, 15_999_904, dim, 1))
    wide.copy_(_bf(k))
    again = h.kv_cache(3, heads, dim)
    h.kv_write_(again, wide, _bf(v), _i32([[0, 1, 2]]), _i32([150]))
    assert small.same(again) == []


# ------------------------------------------------------------------ selection


@pytest.mark.parametrize("heads,kv,dim", [(3, 3, 64), (10, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows,lens,counts,top", [
    (1, [1, 64, 700], None, 1), (1, [2000, 0, 1337], None, 7), (5, [2048, 500, 3], [5, 0, 4], 12), (128, [128, 2000, 640], None, 3),
    (300, [300, 2048, 1000], [300, 129, 1], 5), (130, [2048, 5000, 100], None, 40), (200, [100, 150, 2048], None, 4),
])
def test_select(heads, kv, dim, causal, rows, lens, counts, top):
    rng = np.random.default_rng(rows + top + dim)
    ref, tables, q = _case(rng, heads, kv, dim, 3, rows, 32, seed=top)
    tables[2, 5] = -4
    got = _h().kv_select(_bf(q), ref.to(), _i32(tables), _i32(lens), top, causal=causal, counts=None if counts is None else _i32(counts))
    want = R.select(ref, q.astype(np.float64), tables, lens, counts or [rows] * 3, top, causal)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (10, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("rows,causal,top", [(1, True, 60), (4, False, 1), (130, True, 300), (1, False, 700)])
def test_select_over_long_tables(heads, kv, dim, rows, causal, top):
    """Few tiles over long tables, whose scores are a launch of their own: uneven sequences, pages that are not there."""
    rng = np.random.default_rng(rows + top)
    blocks = 700
    ref, tables, q = _case(rng, heads, kv, dim, 3, rows, blocks, seed=top)
    tables[1, 100:110] = -1
    tables[1, 255:258] = 10 ** 7
    lens, counts = [blocks * 64 - 7, 513 * 64, 3000], [rows, rows, max(rows - 3, 0)]
    got = _h().kv_select(_bf(q), ref.to(), _i32(tables), _i32(lens), top, causal=causal, counts=_i32(counts))
    assert np.array_equal(got.cpu().numpy(), R.select(ref, q.astype(np.float64), tables, lens, counts, top, causal))


def test_select_ties_and_specials():
    """Equal scores take the lowest blocks; NaN scales come last; a query of zeros, NaN or infinities scores all alike."""
    rng = np.random.default_rng(31)
    ref, tables, q = _case(rng, 2, 2, 64, 1, 1, 200, seed=31)
    ref.ksum[tables[0, 3:150]] = ref.ksum[tables[0, 3]]
    ref.ks[tables[0, 3:150]] = 0.01
    ref.ks[tables[0, 170:180]] = np.nan
    ref.ks[tables[0, 180:190]] = np.inf
    ref.ks[tables[0, 190:195]] = 0
    for scale in (1.0, -1.0, 0.0, np.nan, np.inf):
        with np.errstate(invalid="ignore"):
            x = _round(q * scale)
        for top in (1, 20, 100, 195, 200, 250):
            got = _h().kv_select(_bf(x), ref.to(), _i32(tables), _i32([200 * 64]), top)
            with np.errstate(invalid="ignore"):
                want = R.select(ref, x.astype(np.float64), tables, [200 * 64], [1], top, False)
            assert np.array_equal(got.cpu().numpy(), want), (scale, top)


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("blocks", [16384, 16385, 32768])
def test_select_long(dim, blocks):
    """The longest tables, and one page under many blocks: all scores equal but one."""
    ref = R.Cache(3, 1, dim, seed=32)
    ref.ksum[0], ref.ks[:] = 1, 0.01
    ref.ksum[1] = 2
    tables = np.zeros((1, blocks), np.int32)
    tables[0, 16001] = 1
    q = np.ones((1, 1, 1, dim), np.float32)
    got = _h().kv_select(_bf(q), ref.to(), _i32(tables), _i32([blocks * 64]), 100).cpu().numpy().reshape(-1)
    assert got.tolist() == list(range(99)) + [16001]


def test_select_with_more_than_there_is():
    """A pool without pages, and top at its largest."""
    h = _h()
    q = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    none = h.kv_cache(0, 2, 64)
    assert (h.kv_select(q, none, _i32([[0, 0]]), _i32([128]), 5) == -1).all()
    assert (h.kv_attention(q, none, _i32([[0, 0]]), _i32([128])) == 0).all()
    assert (h.kv_read(none, _i32([[0, 0]]), _i32([128]), 128)[0] == 0).all()
    got = h.kv_select(q, h.kv_cache(2, 2, 64), _i32([[0, 1]]), _i32([128]), 32768)
    assert got.shape == (1, 1, 2, 32768) and got[0, 0, 0, :3].tolist() == [0, 1, -1] and (got[..., 2:] == -1).all()


@pytest.mark.parametrize("heads,kv,dim", [(3, 3, 64), (10, 2, 128), (6, 2, 256), (20, 1, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows,top", [(1, 4), (2, 9), (128, 5), (300, 6), (140, 30)])
def test_sparse_attention(heads, kv, dim, causal, rows, top):
    """select, then attention over what it took."""
    h = _h()
    rng = np.random.default_rng(rows * top + dim)
    ref, tables, q = _case(rng, heads, kv, dim, 2, rows, 20, seed=rows)
    lens = [1270, 700]
    blocks = h.kv_select(_bf(q), ref.to(), _i32(tables), _i32(lens), top, causal=causal).cpu().numpy()
    assert np.array_equal(blocks, R.select(ref, q.astype(np.float64), tables, lens, [rows] * 2, top, causal))
    _check(ref, q, tables, lens, None, causal, blocks=blocks)


@pytest.mark.parametrize("rows", [1, 130])
def test_sparse_attention_any_lists(rows):
    """Lists in any order, with holes, blocks past the end and outside the table; empty lists give zeros."""
    rng = np.random.default_rng(41)
    ref, tables, q = _case(rng, 4, 2, 128, 2, rows, 12, seed=41)
    tiles = -(-rows // 128)
    blocks = np.full((2, tiles, 2, 9), -1, np.int32)
    blocks[0, :, 0] = [7, -1, 2, 11, 10, -7, 0, 12, 2147483647]
    blocks[0, :, 1] = [-1, -1, 3, -1, -1, 4, -1, -1, -2147483648]
    blocks[1, :, 0] = [5, 9, 8, 7, 6, 4, 3, 2, 1]
    for causal in (False, True):
        _check(ref, q, tables, [700, 320], None, causal, blocks=blocks)


def test_sparse_with_every_block_is_dense():
    h = _h()
    rng = np.random.default_rng(43)
    for rows in (1, 7, 260):
        ref, tables, q = _case(rng, 4, 2, 128, 2, rows, 9, seed=43)
        c, t, lens = ref.to(), _i32(tables), _i32([570, 301])
        blocks = h.kv_select(_bf(q), c, t, lens, 9, causal=True)
        a, b = h.kv_attention(_bf(q), c, t, lens, causal=True), h.kv_attention(_bf(q), c, t, lens, causal=True, blocks=blocks)
        want, mag, top = R.attention(ref, q.astype(np.float64), tables, [570, 301], [rows] * 2, True)
        for x in (a, b):
            assert (np.abs(x.double().cpu().numpy() - want) <= R.bound(want, mag, top, 128)).all()


# ------------------------------------------------------------------ together, streams, graphs


def _step(h, st):
    """A step of a block's attention: norm and rotate q and k, write, select, attend (all and selected), read back."""
    H, D, S = 4, 128, st["qkv"].shape[0]
    st["work"].copy_(st["qkv"])
    q, k, v = (st["work"][:, i * H * D:(i + 1) * H * D].view(1, S, H, D) for i in range(3))
    h.rms_rope_split_half_(q, k, st["tab"], st["qw"], st["qw"], epsilon=1e-6)
    h.kv_write_(st["cache"], k, v, st["tables"], st["lens"])
    blocks = h.kv_select(q, st["cache"], st["tables"], st["lens"], 4, causal=True)
    dense = h.kv_attention(q, st["cache"], st["tables"], st["lens"], causal=True)
    sparse = h.kv_attention(q, st["cache"], st["tables"], st["lens"], causal=True, blocks=blocks)
    rk, rv = h.kv_read(st["cache"], st["tables"], st["lens"], 100, starts=st["lens"] - 50)
    return [dense, sparse, blocks, rk, rv] + [t.clone() for t in st["cache"]]


def _state(h, S, seed):
    g = torch.Generator().manual_seed(seed)
    H, D = 4, 128
    ang = 6.28 * torch.rand(S, D // 2, generator=g)
    tab = torch.stack([ang.cos(), -ang.sin(), ang.sin(), ang.cos()], -1).reshape(1, S, D // 2, 2, 2)
    return {"qkv": torch.randn(S, 3 * H * D, generator=g).to(torch.bfloat16).to(DEV), "work": torch.empty(S, 3 * H * D, dtype=torch.bfloat16, device=DEV),
            "tab": tab.to(torch.bfloat16).to(DEV), "qw": torch.ones(D, dtype=torch.bfloat16, device=DEV),
            "cache": h.kv_cache(40, H, D), "tables": torch.randperm(40, generator=g).to(torch.int32)[None].to(DEV),
            "lens": torch.tensor([S], dtype=torch.int32, device=DEV)}


@pytest.mark.parametrize("S", [1, 20, 150])
def test_steps_captured_and_replayed(S):
    """Steps that extend a sequence, each replayed from one graph against the same step run eagerly."""
    h = _h()
    eager, st = _state(h, S, 1), _state(h, S, 1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(h, st)
    torch.cuda.synchronize()
    for t in st["cache"]:
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(h, st)
    for r in range(5):
        fresh = torch.randn(S, 3 * 512, generator=torch.Generator().manual_seed(r)).to(torch.bfloat16).to(DEV)
        for x in (eager, st):
            x["qkv"].copy_(fresh)
            x["lens"].fill_((r + 1) * S)
        want = _step(h, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_another_stream(rows):
    """Calls on a side stream, whose results and workspace are freed and reused at once, against the default stream."""
    h = _h()
    rng = np.random.default_rng(71)
    ref, tables, q = _case(rng, 4, 4, 128, 1, rows, 120, seed=71)
    c, t, lens, x = ref.to(), _i32(tables), _i32([7600]), _bf(q)
    want = h.kv_attention(x, c, t, lens)
    blocks = h.kv_select(x, c, t, lens, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            assert torch.equal(h.kv_attention(x, c, t, lens), want)
            assert torch.equal(h.kv_select(x, c, t, lens, 9), blocks)
            wide = t.repeat(1, 5)  # scores in a launch of their own
            assert torch.equal(h.kv_select(x, c, wide, lens, 9), blocks)
    torch.cuda.current_stream().wait_stream(side)


def test_two_graphs_share_no_workspace():
    """Two captured calls that split their work, replayed on two streams at once."""
    h = _h()
    rng = np.random.default_rng(51)
    ref, tables, q = _case(rng, 4, 4, 128, 1, 1, 150, seed=51)
    c, t, lens = ref.to(), _i32(tables), _i32([9600])
    qs = [_bf(q), _bf(_round(rng.standard_normal(q.shape)))]
    want = [h.kv_attention(x, c, t, lens) for x in qs]
    graphs, outs = [], []
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(h.kv_attention(x, c, t, lens))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_same_bits_every_time():
    h = _h()
    rng = np.random.default_rng(61)
    for rows, blocks in ((1, 120), (40, 60), (300, 20)):
        ref, tables, q = _case(rng, 10, 2, 128, 2, rows, blocks, seed=61)
        c, t, lens, x = ref.to(), _i32(tables), _i32([blocks * 64 - 3, blocks * 32]), _bf(q)
        a = h.kv_attention(x, c, t, lens)
        for _ in range(5):
            assert torch.equal(a, h.kv_attention(x, c, t, lens))


# ------------------------------------------------------------------ refusals


def test_refusals_of_the_python_functions():
    h = _h()
    c = h.kv_cache(4, 2, 64)
    t, lens = _i32([[0, 1]]), _i32([100])
    x = torch.zeros(1, 10, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(1, 10, 4, 64, dtype=torch.bfloat16, device=DEV)
    bad = [
        lambda: h.kv_write_(c, x.float(), x, t, lens), lambda: h.kv_write_(c, x, x[:, :5], t, lens),
        lambda: h.kv_write_(c, q, q, t, lens), lambda: h.kv_write_(c, x[0], x[0], t, lens),
        lambda: h.kv_write_(c, x.transpose(1, 2), x.transpose(1, 2), t, lens), lambda: h.kv_write_(c, x.cpu(), x, t, lens),
        lambda: h.kv_write_(c, x, x, t.long(), lens), lambda: h.kv_write_(c, x, x, t, lens.cpu()),
        lambda: h.kv_write_(c, x, x, t[0], lens), lambda: h.kv_write_(c, x, x, t, _i32([1, 2])),
        lambda: h.kv_write_(c, x, x, t, lens, counts=_i32([1, 2])), lambda: h.kv_write_(c._replace(k=c.k.float()), x, x, t, lens),
        lambda: h.kv_write_(c._replace(v=c.k), x, x, t, lens), lambda: h.kv_write_(c._replace(k_sum=c.k_sum.cpu()), x, x, t, lens),
        lambda: h.kv_write_(c._replace(k_scale=c.k_scale.t().contiguous().t()), x, x, t, lens),
        lambda: h.kv_read(c, t, lens, -1), lambda: h.kv_read(c, t, lens, 4, starts=_i32([1, 2])),
        lambda: h.kv_attention(q[..., :32], c, t, lens), lambda: h.kv_attention(q[:, :, :3], c, t, lens),
        lambda: h.kv_attention(q, c, t, lens, blocks=_i32([[[[0]]]])), lambda: h.kv_attention(q, c, t, lens, scale=float("nan")),
        lambda: h.kv_attention(q, c, t, lens, scale=float("inf")), lambda: h.kv_attention(q.expand(2, -1, -1, -1), c, t, lens),
        lambda: h.kv_select(q, c, t, lens, 0), lambda: h.kv_select(q, c, t, lens, 40000), lambda: h.kv_select(q[:, :, :3], c, t, lens, 1),
        lambda: h.kv_select(q, c, _i32(np.zeros((1, 32769))), lens, 1),
        lambda: h.kv_attention(torch.zeros(1, 10, 4 * 64 + 4, dtype=torch.bfloat16, device=DEV)[..., 4:].view(1, 10, 4, 64), c, t, lens),
        lambda: h.kv_cache(1, 1, 96),
    ]
    for n, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {n} was taken")
    with pytest.raises(RuntimeError, match="gradient"):
        h.kv_attention(q.clone().requires_grad_(), c, t, lens)
    with torch.no_grad():
        h.kv_attention(q.clone().requires_grad_(), c, t, lens)
    # a call with nothing to do
    assert h.kv_attention(q[:, :0], c, t, lens).shape == (1, 0, 4, 64)
    assert h.kv_select(q[:, :0], c, t, lens, 3).shape == (1, 0, 2, 3)
    assert h.kv_attention(q, c, t[:, :0].contiguous(), lens).abs().max() == 0
    assert (h.kv_select(q, c, t[:, :0].contiguous(), lens, 3) == -1).all()
    assert h.kv_read(c, t, lens, 0)[0].shape == (1, 0, 2, 64)


def test_lists_of_no_entry_are_refused():
    """An empty list's tensor has no address, and must not be taken for no list."""
    h = _h()
    c, t, lens = h.kv_cache(4, 2, 64), _i32([[0, 1]]), _i32([100])
    q = torch.zeros(1, 10, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="at least one"):
        h.kv_attention(q, c, t, lens, blocks=torch.empty(1, 1, 2, 0, dtype=torch.int32, device=DEV))
    assert h.kv_attention(q[:, :0], c, t, lens, blocks=torch.empty(1, 0, 2, 3, dtype=torch.int32, device=DEV)).shape == (1, 0, 4, 64)
    assert h.kv_attention(q, c, t, lens, blocks=torch.full((1, 1, 2, 1), -1, dtype=torch.int32, device=DEV)).abs().max() == 0


# ------------------------------------------------------------------ few queries of uneven sequences


@pytest.mark.parametrize("heads,kv,dim", [(3, 3, 64), (10, 2, 128), (2, 2, 256), (24, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,counts", [
    ([0, 700, 0, 64, 3000, 0], None), ([3000, 1], None), ([1, 3000], None), ([0, 0, 0], None), ([5, 0, 64, 65], [1, 0, 1, 1]),
    ([3000, 2000, 130, 0], [1, 0, 1, 1]), ([64 * 9] * 5, None), ([1 << 30, 900, -4], None)])
def test_attention_few_uneven(heads, kv, dim, causal, lens, counts):
    rng = np.random.default_rng(sum(map(abs, lens)) % 1000 + dim)
    ref, tables, q = _case(rng, heads, kv, dim, len(lens), 1, 47, seed=7)
    _check(ref, q, tables, lens, counts, causal)


@pytest.mark.parametrize("n", [255, 256, 257, 300])
def test_attention_few_many_sequences(n):
    """As many sequences as a workgroup can lay end to end, and more."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 20 * 64 + 1, n)
    lens[rng.random(n) < 0.3] = 0
    ref, tables, q = _case(rng, 2, 1, 64, n, 1, 20, seed=3)
    _check(ref, q, tables, lens, None, True)


@pytest.mark.parametrize("rows,heads,kv,dim", [(1, 4, 2, 64), (3, 10, 2, 128), (2, 2, 2, 256)])
def test_sparse_attention_few_uneven(rows, heads, kv, dim):
    """Lists over uneven sequences, some without a token, some shorter than the list."""
    rng = np.random.default_rng(rows + dim)
    n, blocks, top = 7, 60, 24
    lens = [3840, 0, 100, 2000, 64 * 24, 0, 1]
    ref, tables, q = _case(rng, heads, kv, dim, n, rows, blocks, seed=rows)
    lists = np.full((n, 1, kv, top), -1, np.int32)
    for i in range(n):
        for h in range(kv):
            lists[i, 0, h, :] = rng.permutation(blocks)[:top]
    _check(ref, q, tables, lens, None, True, blocks=lists)


@pytest.mark.parametrize("rows,kv,dim", [(1, 2, 64), (2, 8, 128), (1, 3, 256)])
def test_few_uneven_captured_and_replayed(rows, kv, dim):
    """A captured call follows the lengths that it finds, as an eager call does."""
    h = _h()
    rng = np.random.default_rng(rows)
    n, blocks = 6, 80
    ref, tables, q = _case(rng, 2 * kv, kv, dim, n, rows, blocks, seed=9)
    c, t, x, lens = ref.to(), _i32(tables), _bf(q), _i32([64 * blocks] * n)
    call = lambda: h.kv_attention(x, c, t, lens, causal=True)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(6):
        lens.copy_(_i32(rng.integers(0, 64 * blocks + 1, n) * (rng.random(n) < 0.8)))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want), r
        _check(ref, q, tables, lens.cpu().numpy(), None, True)
