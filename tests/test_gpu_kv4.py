"""The 4-bit key/value cache against plain forms on the CPU: written bytes are pinned, reading is exact, attention is within
the bounds that kv_ref.bound derives, NaNs reach the rows and elements that they belong to."""
import numpy as np
import pytest
import torch

import kv4_ref as R4
import kv_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _h():
    import h3mi
    return h3mi


def _bf(a):
    """float32 array of bf16 values -> bf16 GPU tensor"""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16).to(DEV)


def _round(a):
    return torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16).float().numpy()


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _tables(rng, n, blocks, spare=2):
    return rng.permutation(n * blocks + spare)[:n * blocks].reshape(n, blocks).astype(np.int32)


# ------------------------------------------------------------------ writing and reading


@pytest.mark.parametrize("heads,dim", [(3, 64), (2, 128), (5, 256)])
@pytest.mark.parametrize("steps", [[(100, 100)], [(64, 64), (1, 65), (1, 66), (70, 136)], [(1, 1), (62, 63), (1, 64), (1, 65)],
                                   [(130, 130), (3, 100), (200, 256)]])
def test_write_is_pinned(heads, dim, steps):
    """A chain of writes (rows, length after it) into pages that held other tokens."""
    h = _h()
    rng = np.random.default_rng(len(steps) * dim)
    blocks = 4
    ref = R4.Cache4(2 * blocks + 2, heads, dim, seed=1)
    cache, tables = ref.to(), _tables(rng, 2, blocks)
    for x, (rows, end) in enumerate(steps):
        k = _round(rng.standard_normal((2, rows, heads, dim)) * 3.0 ** x)
        v = _round(rng.standard_normal((2, rows, heads, dim)) * rng.choice([0.0, 1e-3, 1.0, 1e4], (2, rows, heads, 1)))
        lens, counts = np.array([end, max(end - 5, 0)]), np.array([rows, max(rows - 5, 0)])
        R4.write(ref, k, v, tables, lens, counts)
        assert h.kv_write_(cache, _bf(k), _bf(v), _i32(tables), _i32(lens), counts=_i32(counts)) is cache
        assert ref.same(cache) == []


def test_every_bf16_beside_every_largest():
    """All 65536 bf16 numbers: as the largest of a group, and as another of a group whose largest is each power of two and the
    numbers around 7 / 4 of it, down to the smallest and up to the last finite one."""
    h = _h()
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float().numpy()
    own = np.zeros((65536, 32), np.float32)
    own[:, 5] = every
    finite = every[np.isfinite(every)]
    rng = np.random.default_rng(1)
    tops = np.concatenate([np.float32(2.0) ** np.arange(-133, 128), np.float32(1.75) * np.float32(2.0) ** np.arange(-130, 128),
                           np.float32(1.7578125) * np.float32(2.0) ** np.arange(-130, 128), [3.3895314e38]]).astype(np.float32)
    tops = _round(tops)
    mixed = []
    for t in tops:
        near = finite[(np.abs(finite) <= t) & (np.abs(finite) >= t * 2.0 ** -6)]
        some = np.concatenate([rng.choice(near, 93), rng.choice(finite[np.abs(finite) <= t], 31)])
        mixed.append(np.insert(some.reshape(4, 31), 7, t, axis=1))
    x = np.concatenate([own, np.concatenate(mixed)])
    x = np.concatenate([x, np.zeros((-len(x) % 4, 32), np.float32)]).reshape(1, -1, 1, 128)
    n = x.shape[1]
    blocks = -(-n // 64)
    ref, tables = R4.Cache4(blocks, 1, 128, seed=2), np.arange(blocks, dtype=np.int32)[None]
    cache = ref.to()
    back = x[:, ::-1]
    R4.write(ref, x, back, tables, [n], [n])
    h.kv_write_(cache, _bf(x), _bf(back), _i32(tables), _i32([n]))
    assert ref.same(cache) == []
    k, v = h.kv_read(cache, _i32(tables), _i32([n]), n)
    for got, src in ((k, x), (v, back)):
        got = got.double().cpu().numpy().reshape(-1, 32)
        src = src.astype(np.float64).reshape(-1, 32)
        ok = np.isfinite(src).all(1)
        assert np.isnan(got[~ok]).all() and np.isfinite(got[ok]).all()
        top = np.abs(src[ok]).max(1, keepdims=True)
        step = 2.0 ** np.clip(np.ceil(np.log2(np.maximum(top, 2.0 ** -125) / 7)), -125, 125)
        # half the distance of the two values on either side; above 7 2^125 up to 1 / 4 of the value
        a = np.abs(src[ok]) / step
        most = np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0)) * step
        assert (np.abs(got[ok] - src[ok]) <= np.where(a <= 7, most, np.abs(src[ok]) / 4)).all()


def test_how_far_a_value_is_off():
    """A fifth of its group's largest, from 3.5 2^-125 up to 7 2^125, and what it is outside."""
    h = _h()
    rng = np.random.default_rng(17)
    tops = _round(np.exp2(rng.uniform(-133, 128, 4000)))
    edge = _round(np.array([a * 2.0 ** e for e in (-133, -127, -126, -125, -124, 0, 124, 125) for a in (1, 1.25, 1.75, 3.5, 3.515625, 5, 7)]))
    tops = np.concatenate([tops[np.isfinite(tops) & (tops > 0)], edge])
    x = _round(tops[:, None] * rng.uniform(-1, 1, (len(tops), 32)))
    x[np.arange(len(tops)), rng.integers(0, 32, len(tops))] = tops
    x = np.concatenate([x, np.zeros((-len(x) % 4, 32))]).reshape(1, -1, 1, 128)
    n = x.shape[1]
    tables = np.arange(-(-n // 64), dtype=np.int32)[None]
    cache = h.kv_cache(tables.size, 1, 128, bits=4)
    h.kv_write_(cache, _bf(x), _bf(x), _i32(tables), _i32([n]))
    src = _bf(x).double().cpu().numpy().reshape(-1, 32)
    for got in h.kv_read(cache, _i32(tables), _i32([n]), n):
        off = np.abs(got.double().cpu().numpy().reshape(-1, 32) - src)
        top = np.abs(src).max(1, keepdims=True)
        most = np.where(top <= 3.5 * 2.0 ** -125, np.where(np.abs(src) <= 2.0 ** -127, np.abs(src), 2.0 ** -126), np.where(top <= 7 * 2.0 ** 125, top / 5, top / 4))
        assert (off <= most).all()


def test_write_of_views_and_without_counts():
    h = _h()
    rng = np.random.default_rng(5)
    heads, dim, rows = 3, 128, 77
    qkv = _round(rng.standard_normal((2, rows, 3, heads, dim)))
    ref = R4.Cache4(6, heads, dim, seed=2)
    cache, tables, lens = ref.to(), _tables(rng, 2, 2), np.array([77, 100])
    t = _bf(qkv)
    h.kv_write_(cache, t[:, :, 1], t[:, :, 2], _i32(tables), _i32(lens))
    R4.write(ref, qkv[:, :, 1], qkv[:, :, 2], tables, lens, [rows, rows])
    assert ref.same(cache) == []


def test_write_drops_what_has_no_place():
    """Lengths past the table, rows before token 0, negative counts and lengths, pages outside the pool, no rows."""
    h = _h()
    rng = np.random.default_rng(11)
    heads, dim, rows = 2, 64, 90
    ref = R4.Cache4(9, heads, dim, seed=4)
    cache = ref.to()
    tables = np.array([[0, 1], [2, 9], [3, 4], [-1, 5], [6, 7], [8, 2147483647]], np.int32)
    lens, counts = np.array([140, 128, 30, 128, -5, 100]), np.array([90, 90, 90, 200, 20, -3])
    k, v = (_round(rng.standard_normal((6, rows, heads, dim))) for _ in range(2))
    R4.write(ref, k, v, tables, lens, counts)
    h.kv_write_(cache, _bf(k), _bf(v), _i32(tables), _i32(lens), counts=_i32(counts))
    assert ref.same(cache) == []
    h.kv_write_(cache, _bf(k[:, :0]), _bf(v[:, :0]), _i32(tables), _i32(lens))
    h.kv_write_(cache, _bf(k[:0]), _bf(v[:0]), _i32(tables[:0]), _i32(lens[:0]))
    assert ref.same(cache) == []


def test_two_sequences_write_into_one_page():
    """Only the tokens of a call have to be distinct: a page that sequences share takes tokens of both."""
    h = _h()
    rng = np.random.default_rng(12)
    ref = R4.Cache4(3, 2, 128, seed=6)
    cache, tables = ref.to(), np.array([[1], [1]], np.int32)
    k, v = (_round(rng.standard_normal((2, 9, 2, 128))) for _ in range(2))
    R4.write(ref, k, v, tables, [20, 29], [9, 9])
    h.kv_write_(cache, _bf(k), _bf(v), _i32(tables), _i32([20, 29]))
    assert ref.same(cache) == []


@pytest.mark.parametrize("heads,dim", [(3, 64), (2, 128), (5, 256)])
@pytest.mark.parametrize("length,starts", [(1, None), (64, None), (200, None), (65, [3, 64, 127]), (130, [-10, 60, 1000]),
                                           (10, [-100, 2147483640, -2147483648])])
def test_read(heads, dim, length, starts):
    h = _h()
    rng = np.random.default_rng(13)
    ref = R4.Cache4(11, heads, dim, seed=5)
    ref.ks[3, :, 0, 7], ref.vs[2, :, 1, 9], ref.vs[4, 0, 0, :3] = 255, 253, 254
    tables, lens = _tables(rng, 3, 3), np.array([192, 70, 0])
    tables[0, 1] = 11  # a page outside the pool
    k, v = h.kv_read(ref.to(), _i32(tables), _i32(lens), length, starts=None if starts is None else _i32(starts))
    plain = ref.plain()
    for i in range(3):
        a, b, _ = R.tokens(plain, tables[i], int(lens[i]))
        first = 0 if starts is None else starts[i]
        for got, want in ((k, a), (v, b)):
            full = np.zeros((length, heads, dim))
            for r in range(length):
                if 0 <= first + r < lens[i]:
                    full[r] = want[first + r]
            assert np.array_equal(got[i].double().cpu().numpy(), full, equal_nan=True)


# ------------------------------------------------------------------ attention


def _check(ref, q, tables, lens, counts, causal, scale=None, blocks=None, view=None):
    h = _h()
    out = h.kv_attention(_bf(q) if view is None else view, ref.to(), _i32(tables), _i32(lens), causal=causal,
                         counts=None if counts is None else _i32(counts), scale=scale, blocks=None if blocks is None else _i32(blocks))
    if counts is None:
        counts = [q.shape[1]] * q.shape[0]
    want, mag, top = R.attention(ref.plain(), q.astype(np.float64), tables, lens, counts, causal, scale, blocks)
    got = out.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    off = np.abs(got - want) / R.bound(want, mag, top, q.shape[3])
    assert off.max(initial=0.0) <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))
    assert (got[mag == 0] == 0).all()
    return out


def _case(rng, heads, kv, dim, n, rows, blocks, seed):
    return R4.Cache4(n * blocks + 2, kv, dim, seed=seed), _tables(rng, n, blocks), _round(rng.standard_normal((n, rows, heads, dim)))


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (6, 2, 64), (3, 3, 128), (10, 2, 128), (2, 2, 256), (5, 1, 256)])
@pytest.mark.parametrize("rows,blocks,lens,counts", [
    (1, 5, [320, 1, 0], None), (1, 40, [2500, 777, 64], None), (3, 6, [384, 200, 2], [3, 1, 0]), (17, 6, [380, 129, 17], [17, 9, 17]),
    (33, 3, [192, 64, 40], [33, 20, 33]), (70, 9, [576, 300, 65], [70, 3, 65]), (130, 4, [256, 250, 130], [130, 129, 1]),
    (200, 30, [1900, 1000, 200], None),
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention(heads, kv, dim, rows, blocks, lens, counts, causal):
    rng = np.random.default_rng(rows * 7 + dim + heads)
    ref, tables, q = _case(rng, heads, kv, dim, 3, rows, blocks, seed=rows)
    _check(ref, q, tables, lens, counts, causal)


@pytest.mark.parametrize("rows,blocks", [(1, 6), (20, 64), (150, 6), (300, 40), (1100, 130)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_with_holes(rows, blocks, causal):
    """Pages outside the pool, lengths past the table and below 0, rows before token 0, and what pages hold behind a
    sequence's end: codes of no number, and the largest of factors."""
    rng = np.random.default_rng(rows)
    ref, tables, q = _case(rng, 2, 2, 128, 4, rows, blocks, seed=rows + 1)
    lens, counts = np.array([blocks * 64 + 10, rows // 2, -3, blocks * 64 - 37]), np.array([rows, rows, rows, rows // 2 + 1])
    tables[0, 1], tables[3, blocks - 2] = -1, 2 ** 31 - 1
    last = tables[3, blocks - 1]
    ref.ks[last, :, :, 27:], ref.vs[last, :, :, 27:40], ref.vs[last, :, :, 40:] = 255, 255, 252
    ref.vs[tables[2]] = 255
    mine = tables[1, rows // 2 // 64]
    ref.vs[mine, :, :, rows // 2 % 64:] = 254
    _check(ref, q, tables, lens, counts, causal)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40, 150])
def test_every_code(dim, rows):
    """Every scale code with every 4-bit value, read back and as the one token that a sequence's rows see, whose values are
    then the result: exact where they are normal numbers (codes of 2 and more; what is written has no others)."""
    h = _h()
    ref = R4.Cache4(256, 1, dim)
    ref.v[:] = np.tile(np.arange(0x10, 0x100, 0x22, dtype=np.uint8), dim // 16 + 1)[:dim // 2]
    ref.k[:, :, 0] = ref.v[:, :, 0]
    ref.ks[:] = np.arange(256, dtype=np.uint8)[:, None, None, None]
    ref.vs[:] = ref.ks
    assert set(np.concatenate([ref.v & 15, ref.v >> 4], None)) == set(range(16))
    cache, tables, lens = ref.to(), _i32(np.arange(256)[:, None]), _i32([1] * 256)
    want = R4.values(ref.v[:, :, 0], ref.vs[:, :, :, 0])[:, None]
    k, v = h.kv_read(cache, tables, lens, 1)
    for x in (k, v):
        assert np.array_equal(x.double().cpu().numpy(), want, equal_nan=True)
    cache.k_scale.fill_(127)
    out = h.kv_attention(_bf(np.ones((256, rows, 1, dim))), cache, tables, lens).double().cpu().numpy()
    assert np.array_equal(out[2:], np.broadcast_to(want, out.shape)[2:], equal_nan=True)
    assert (np.abs(out[:2] - want[:2]) <= 2.0 ** -126).all()


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 30.0])
@pytest.mark.parametrize("rows", [2, 140])
def test_scales_and_views(rows, scale):
    rng = np.random.default_rng(rows)
    ref, tables, q = _case(rng, 6, 2, 128, 2, rows, 5, seed=8)
    wide = torch.zeros(2, rows, 11, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, :, 3:9] = _bf(q)
    _check(ref, q, tables, [300, 200], None, True, scale=scale, view=wide[:, :, 3:9])


@pytest.mark.parametrize("heads,kv,dim,rows,blocks", [(4, 4, 64, 300, 30), (10, 2, 128, 1, 50), (2, 2, 128, 500, 12), (2, 1, 256, 140, 9)])
@pytest.mark.parametrize("causal", [False, True])
def test_lists(heads, kv, dim, rows, blocks, causal):
    """Distinct blocks in any order, with entries of no block, past the sequence and past the table."""
    rng = np.random.default_rng(rows + dim)
    ref, tables, q = _case(rng, heads, kv, dim, 2, rows, blocks, seed=3)
    top = 7
    lists = np.stack([rng.permutation(blocks + 3)[:top] - 1 for _ in range(2 * -(-rows // 128) * kv)]).reshape(2, -1, kv, top)
    lists[1, 0, 0] = -1
    _check(ref, q, tables, [blocks * 64 - 5, blocks * 40], None, causal, blocks=lists)


@pytest.mark.parametrize("plan", [(1, 6), (32, 6), (1, 64), (20, 64), (300, 6), (300, 24), (300, 64), (200, 300)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [float("nan"), -float("inf")])
def test_a_number_that_is_none_reaches_what_sees_it(plan, dim, value):
    """Of a key: all of the rows that see its token, of its head; of a value: their 32 elements; however little it weighs."""
    h = _h()
    rows, blocks = plan
    g = torch.Generator().manual_seed(rows + blocks)
    end, bad = blocks * 64, (blocks - 2) * 64 + 5
    level = torch.zeros(blocks)
    level[1], level[blocks - 2] = 1.0, -1.0
    k = torch.randn(1, end, 2, dim, generator=g) * 0.01 + 8 * level.repeat_interleave(64)[None, :, None, None]
    v = torch.randn(1, end, 2, dim, generator=g)
    q = (torch.randn(1, rows, 2, dim, generator=g) * 0.01 + 8).to(torch.bfloat16).to(DEV)
    tables = torch.randperm(blocks, generator=g).to(torch.int32)[None].to(DEV)
    lens = torch.tensor([end], dtype=torch.int32, device=DEV)
    for what in ("k", "v"):
        kx, vx = k.clone(), v.clone()
        (kx if what == "k" else vx)[0, bad, 1, 39] = value
        cache = h.kv_write_(h.kv_cache(blocks, 2, dim, bits=4), kx.to(torch.bfloat16).to(DEV), vx.to(torch.bfloat16).to(DEV), tables, lens)
        for causal in (False, True):
            want = torch.zeros(1, rows, 2, dim, dtype=torch.bool)
            want[:, :, 1, :] = True
            if what == "v":
                want[..., :32] = want[..., 64:] = False
            if causal:
                want[:, end - rows + torch.arange(rows) < bad] = False
            out = h.kv_attention(q, cache, tables, lens, causal=causal).float().cpu()
            assert torch.equal(out.isnan(), want), (what, causal)
            assert out[~want].isfinite().all()
        take = torch.tensor([b for b in range(blocks) if b != blocks - 2], dtype=torch.int32, device=DEV)
        lists = take.repeat(1, -(-rows // 128), 2, 1)
        assert h.kv_attention(q, cache, tables, lens, blocks=lists).isfinite().all()


@pytest.mark.parametrize("rows,blocks", [(1, 6), (20, 64), (300, 6), (300, 64)])
def test_a_query_that_is_none_stays_in_its_row_and_head(rows, blocks):
    h = _h()
    g = torch.Generator(device=DEV).manual_seed(rows * blocks)
    draw = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    tables = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)[None]
    lens = torch.tensor([blocks * 64 - 3], dtype=torch.int32, device=DEV)
    cache = h.kv_write_(h.kv_cache(blocks, 2, 128, bits=4), draw(1, blocks * 64 - 3, 2, 128), draw(1, blocks * 64 - 3, 2, 128), tables, lens)
    q = draw(1, rows, 2, 128)
    hit = torch.zeros(rows, 2, dtype=torch.bool, device=DEV)
    hit[rows // 2, 1] = hit[0, 0] = True
    for value in (float("nan"), float("inf")):
        bad = q.clone()
        bad[0, :, :, 17] = torch.where(hit, torch.tensor(value, device=DEV, dtype=torch.bfloat16), q[0, :, :, 17])
        want, got = (h.kv_attention(x, cache, tables, lens, causal=True)[0] for x in (q, bad))
        assert got[hit].isnan().all() and want.isfinite().all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("rows,blocks", [(8, 6), (8, 64), (300, 6), (300, 64)])
def test_padding_is_not_read(rows, blocks):
    """NaN in the padding rows of a batch changes no page and no output."""
    h = _h()
    g = torch.Generator(device=DEV).manual_seed(rows + blocks)
    draw = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    n = 3
    counts, lens = _i32([rows, rows // 2 + 1, 0]), _i32([blocks * 64, blocks * 40 + 7, 0])
    tables = torch.randperm(n * blocks, generator=g, device=DEV).reshape(n, blocks).to(torch.int32)
    k, v, before, q = draw(n, rows, 2, 128), draw(n, rows, 2, 128), draw(n, blocks * 64, 2, 128), draw(n, rows, 4, 128)
    pad = (torch.arange(rows, device=DEV) >= counts[:, None])[..., None, None]
    got = []
    for fill in (0.0, float("nan")):
        kx, vx, qx = (torch.where(pad, torch.tensor(fill, dtype=torch.bfloat16, device=DEV), x) for x in (k, v, q))
        c = h.kv_write_(h.kv_cache(n * blocks, 2, 128, bits=4), before, before, tables, lens)
        h.kv_write_(c, kx, vx, tables, lens, counts=counts)
        got.append([*c, h.kv_attention(qx, c, tables, lens, causal=True, counts=counts)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_steep_factors():
    """Codes from the least to the largest in one sequence: keys of 2^-125, values of 2^125 that weigh nothing or all."""
    h = _h()
    rng = np.random.default_rng(2)
    for rows in (1, 150):
        ref, tables, q = _case(rng, 2, 2, 128, 1, rows, 4, seed=9)
        ref.ks[tables[0, 0]] = 2
        ref.vs[tables[0, 1]] = rng.integers(2, 60, ref.vs[tables[0, 1]].shape)
        ref.vs[tables[0, 2]] = rng.integers(150, 235, ref.vs[tables[0, 2]].shape)
        _check(ref, q, tables, [250], None, False)
    # 6 2^125 with all the weight is read back whole
    cache = h.kv_cache(1, 1, 64, bits=4)
    x = torch.full((1, 1, 1, 64), 6 * 2.0 ** 125, dtype=torch.bfloat16, device=DEV)
    h.kv_write_(cache, x, x, _i32([[0]]), _i32([1]))
    for rows in (1, 200):
        out = h.kv_attention(torch.zeros(1, rows, 1, 64, dtype=torch.bfloat16, device=DEV), cache, _i32([[0]]), _i32([1]))
        assert torch.equal(out, x.expand(1, rows, 1, 64))


def test_pages_past_32_bits():
    """A cache of more than 2^32 bytes of keys gives what a small one with the same pages gives."""
    h = _h()
    rng = np.random.default_rng(32)
    heads, dim, blocks = 56, 128, 9
    pages = 2 ** 32 // (heads * 64 * dim // 2) + 2 * blocks
    small, far = h.kv_cache(2 * blocks, heads, dim, bits=4), h.kv_cache(pages, heads, dim, bits=4)
    near = _i32(rng.permutation(2 * blocks).reshape(2, blocks))
    tables, lens = near + (pages - 2 * blocks), _i32([blocks * 64, 400])
    k, v = (torch.randn((2, 400, heads, dim), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    got = []
    for cache, t in ((small, near), (far, tables)):
        h.kv_write_(cache, k, v, t, lens)
        got.append([*h.kv_read(cache, t, lens, blocks * 64)] + [h.kv_attention(k[:, :rows], cache, t, lens, True) for rows in (1, 40, 300)])
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert torch.equal(small.k, far.k[pages - 2 * blocks:]) and torch.equal(small.v_scale, far.v_scale[pages - 2 * blocks:])


def test_rows_past_32_bits():
    """Of tensors of more than 2^32 bytes the last rows are what they are alone."""
    h = _h()
    rows, heads, dim, some = 300_000, 56, 128, 1280
    blocks = -(-rows // 64)
    x = torch.empty((1, rows, heads, dim), device=DEV, dtype=torch.bfloat16).normal_()
    assert x.numel() * 2 > 2 ** 32
    cache, tables, lens = h.kv_cache(blocks, heads, dim, bits=4), _i32(np.arange(blocks)[None]), _i32([rows])
    h.kv_write_(cache, x, x, tables, lens)
    assert torch.equal(cache.k, cache.v) and torch.equal(cache.k_scale, cache.v_scale)
    k, _ = h.kv_read(cache, tables, lens, rows)
    tail, _ = h.kv_read(cache, tables, lens, some, starts=_i32([rows - some]))
    assert torch.equal(k[:, -some:], tail)
    del k
    alone = h.kv_cache(blocks, heads, dim, bits=4)
    h.kv_write_(alone, x[:, -some:], x[:, -some:], tables, lens)
    assert torch.equal(h.kv_read(alone, tables, lens, some, starts=_i32([rows - some]))[0], tail)
    few = _i32([37])  # one block: a row's result is its own, whatever rows share its tile
    out = h.kv_attention(x, cache, tables[:, :1].contiguous(), few)
    assert torch.equal(out[:, -some:], h.kv_attention(x[:, -some:], cache, tables[:, :1].contiguous(), few))


def test_other_streams_and_devices_tensors():
    """Calls on a side stream follow what it did before; a native call and the checked one give the same."""
    h = _h()
    g = torch.Generator(device=DEV).manual_seed(4)
    k, v, q = (torch.randn(2, 70, 4, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3))
    tables, lens = _i32([[0, 2], [3, 1]]), _i32([70, 70])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = h.kv_write_(h.kv_cache(4, 4, 128, bits=4), k, v, tables, lens)
        a = h.kv_attention(q, c, tables, lens, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    c2 = h.kv_write_(h.kv_cache(4, 4, 128, bits=4), k, v, tables, lens, counts=None)
    assert all(torch.equal(x, y) for x, y in zip(c, c2))
    # lists of every block take the same path through Python's checks where the causal flag is no bool
    b = h.kv_attention(q, c2, tables, lens, causal=1)
    assert torch.equal(a, b)


def test_refusals():
    h = _h()
    c = h.kv_cache(2, 2, 64, bits=4)
    tables, lens = _i32([[0, 1]]), _i32([10])
    x = torch.zeros(1, 10, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="8-bit cache"):
        h.kv_select(x, c, tables, lens, 1)
    with pytest.raises(ValueError, match="k_scale"):
        h.kv_attention(x, c._replace(k_scale=c.v), tables, lens)
    with pytest.raises(ValueError, match="uint8"):
        h.kv_write_(c._replace(k=c.k.to(torch.int8)), x, x, tables, lens)
    with pytest.raises(ValueError, match="64"):
        h.kv_write_(c, x[..., :32], x[..., :32], tables, lens)
    with pytest.raises(ValueError, match="contiguous"):
        h.kv_read(c._replace(v=c.v.transpose(0, 1).contiguous().transpose(0, 1)), tables, lens, 3)
    with pytest.raises(h._lib.H3miError, match="overlap"):
        h.kv_write_(c._replace(v=c.k), x, x, tables, lens)
    with pytest.raises(RuntimeError, match="no gradient"):
        h.kv_attention(x.requires_grad_(), c, tables, lens)


@pytest.mark.parametrize("n,rows,heads,kv,dim,blocks", [
    (1, 1, 8, 2, 256, 40), (2, 200, 30, 6, 256, 30), (2, 300, 2, 2, 256, 7), (3, 1030, 18, 18, 128, 140), (2, 150, 2, 2, 64, 64),
])
def test_captured(n, rows, heads, kv, dim, blocks):
    """A captured write and attention, replayed with other tokens and lengths, beside an eager cache."""
    h = _h()
    g = torch.Generator(device=DEV).manual_seed(rows)
    caches = [h.kv_cache(n * blocks, kv, dim, bits=4) for _ in range(2)]
    q, k, v = (torch.empty(n, rows, x, dim, dtype=torch.bfloat16, device=DEV) for x in (heads, kv, kv))
    tables = torch.randperm(n * blocks, generator=g, device=DEV).reshape(n, blocks).to(torch.int32)
    lens = torch.zeros(n, dtype=torch.int32, device=DEV)

    def call(c):
        h.kv_write_(c, k, v, tables, lens)
        return [h.kv_attention(q, c, tables, lens, causal=True), *c]

    call(caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(caches[0])
    for r in range(5):
        lens.copy_(torch.randint(0, blocks * 64 + 1, (n,), generator=g, device=DEV))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        want = call(caches[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r
