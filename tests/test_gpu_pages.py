"""Pages taken and given back on the GPU against one sequence after the other on the CPU: every number is equal."""
import numpy as np
import pytest
import torch

from pages_ref import Pool

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(a):
    return None if a is None else torch.from_numpy(np.array(a, np.int32)).to(DEV)


def _start(rng, n, blocks, spare, most):
    """Sequences of 0 to `most` tokens whose pages are off a shuffled stack with `spare` pages left."""
    lens = rng.integers(0, min(most, 64 * blocks) + 1, n)
    lens[rng.random(n) < 0.2] = 0
    held = -(-lens // 64)
    stack = rng.permutation(int(held.sum()) + spare)
    tables, at = np.full((n, blocks), -1), len(stack)
    for i in range(n):
        tables[i, :held[i]] = stack[at - held[i]:at]
        at -= held[i]
    return Pool(stack, at, tables, lens)


def _extend(ref, pool, tables, lens, rows, counts=None):
    import h3mi
    got = h3mi.kv_extend_(pool, tables, lens, rows, counts=_i32(counts))
    want = ref.extend(rows, counts)
    for name, a, b in zip(("granted", "positions", "slots"), got, want):
        assert a.shape == b.shape and np.array_equal(a.cpu().numpy(), b), name
    assert got[0].dtype == got[1].dtype == torch.int32 and got[2].dtype == torch.int64
    assert ref.same(pool, tables, lens) == []


def _release(ref, pool, tables, lens, keep=None):
    import h3mi
    assert h3mi.kv_release_(pool, tables, lens, _i32(keep)) is pool
    ref.release(keep)
    assert ref.same(pool, tables, lens) == []


@pytest.mark.parametrize("n,blocks,rows,spare,most", [
    (1, 1, 1, 1, 0), (1, 309, 19200, 400, 521), (7, 40, 100, 300, 1000), (64, 20, 1, 40, 1200), (65, 5, 64, 200, 250), (256, 40, 1, 3, 2477),
    (1000, 8, 3, 100, 500), (1024, 3, 5, 2000, 100), (1025, 3, 4, 2000, 100), (2500, 4, 70, 3000, 100), (33, 2000, 4097, 9000, 100000), (3, 2, 0, 5, 100),
])
def test_steps(n, blocks, rows, spare, most):
    """Tokens come and go for a few steps, until the pool has too few pages and again after some are back."""
    rng = np.random.default_rng(n + rows)
    ref = _start(rng, n, blocks, spare, most)
    state = ref.to()
    for step in range(6):
        counts = None if step == 1 else rng.integers(-2, rows + 3, n)
        _extend(ref, *state, rows, counts)
        keep = rng.integers(-3, 64 * blocks, n)
        keep[rng.random(n) < 0.5] = 2 ** 31 - 1
        if step % 2:
            _release(ref, *state, keep)
    _release(ref, *state)
    assert ref.count == len(ref.free) and sorted(ref.free) == list(range(len(ref.free)))


def test_sequences_are_served_in_order_until_one_is_not():
    ref = Pool([9, 8, 7, 6, 5, 4, 3, 2, 1, 0], 4, np.full((6, 4), -1), [0, 0, 0, 0, 0, 0])
    ref.tables[3, 0], ref.lens[3] = 9, 10  # needs no page
    state = ref.to()
    _extend(ref, *state, 200, [100, 65, 64, 54, 1, 0])
    assert ref.lens.tolist() == [100, 65, 0, 64, 0, 0] and ref.count == 0
    _release(ref, *state, [100, 1, 0, 0, 0, 0])
    assert ref.count == 2
    _extend(ref, *state, 200, [0, 0, 64, 64, 0, 0])
    assert ref.lens.tolist() == [100, 1, 64, 64, 0, 0]


def test_tables_too_narrow():
    """A sequence that its table has no blocks for gets nothing, and takes nothing from those after it."""
    rng = np.random.default_rng(3)
    ref = _start(rng, 5, 3, 20, 190)
    state = ref.to()
    _extend(ref, *state, 300, [300, 193, 1, 64, 0])
    ref = Pool([0, 1], 2, np.zeros((2, 0), np.int32), [0, 0])
    _extend(ref, *ref.to(), 1, [0, 1])
    ref = Pool([0, 1], 2, [[0], [1]], [2 ** 31 - 1, 2 ** 31 - 1])
    state = ref.to()
    _extend(ref, *state, 5)
    _release(ref, *state, [2 ** 31 - 1, 64])


def test_what_is_no_page():
    """Counts past the stack and below 0, lengths below 0 and past the table, entries of no page, a stack that is full."""
    for count in (-5, 0, 3, 50):
        ref = Pool([4, 1, 2, 3, 7, -1, 99], count, [[0, -1, 7], [2 ** 31 - 1, -2 ** 31, 6], [1, 2, 3]], [-7, 150, 500])
        state = ref.to()
        _extend(ref, *state, 70, [70, 30, 2])
        _release(ref, *state, [5, 64, -1])
        _extend(ref, *state, 130, [130, 60, 130])
        _release(ref, *state)


def test_empty():
    ref = Pool(np.zeros(0), 0, np.full((3, 2), -1), [0, 0, 0])
    state = ref.to()
    _extend(ref, *state, 5, [0, 5, 1])
    _release(ref, *state)
    import h3mi
    pool = h3mi.kv_pool(4)
    assert pool.free.tolist() == [3, 2, 1, 0] and pool.count.tolist() == [4]
    got = h3mi.kv_extend_(pool, _i32(np.zeros((0, 2))), _i32([]), 7)
    assert [t.shape for t in got] == [(0,), (0, 7), (0, 7)]
    h3mi.kv_release_(pool, _i32(np.zeros((0, 2))), _i32([]))
    assert pool.count.tolist() == [4]


def test_slots_past_32_bits():
    import h3mi
    pages = 1 << 26
    pool = h3mi.kv_pool(pages)
    pool.free[-1], pool.free[-2] = pages - 1, pages - 2
    tables, lens = torch.full((1, 2), -1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    granted, positions, slots = h3mi.kv_extend_(pool, tables, lens, 100)
    want = torch.cat([(pages - 1) * 64 + torch.arange(64), (pages - 2) * 64 + torch.arange(36)])
    assert torch.equal(slots[0].cpu(), want) and positions[0].tolist() == list(range(100)) and granted.tolist() == [100]


def test_many_pages_come_back():
    """More entries than one pass of the workgroup takes, some of no page."""
    rng = np.random.default_rng(8)
    ref = _start(rng, 40, 3000, 10, 192000)
    ref.tables[rng.random(ref.tables.shape) < 0.01] = -1
    state = ref.to()
    _release(ref, *state, rng.integers(0, 30000, 40))


def test_shared_prefix():
    """Whole blocks that three sequences hold: the owner's pages stay out of the pool until it is released, and come back once."""
    import h3mi
    pool = h3mi.kv_pool(12)
    tables, lens = torch.full((4, 4), -1, dtype=torch.int32, device=DEV), _i32([0, 0, 0, 0])
    h3mi.kv_extend_(pool, tables, lens, 150, _i32([150, 0, 0, 0]))
    shared = tables[0, :2].clone()
    for i in (1, 2):
        tables[i, :2] = shared
        lens[i] = 128
    granted, positions, slots = h3mi.kv_extend_(pool, tables, lens, 70, _i32([1, 22, 70, 0]))
    assert granted.tolist() == [1, 22, 70, 0] and positions[:, 0].tolist() == [150, 128, 128, -1]
    held = [set(row) - {-1} for row in tables.tolist()]
    assert held[1] & held[0] == held[2] & held[0] == set(shared.tolist()) and slots[:3, 0].unique().numel() == 3

    def free():
        return pool.free[:int(pool.count)].tolist()

    for i in (1, 2):  # one at a time: the others' tables stay out of the call
        tables[i, :2] = -1
        h3mi.kv_release_(pool, tables[i:i + 1], lens[i:i + 1])
        assert not held[0] & set(free()) and (tables[i] == -1).all()
        # what is handed out meanwhile is none of the owner's
        h3mi.kv_extend_(pool, tables, lens, 200, _i32([0, 0, 0, 200 if i == 1 else 0]))
        assert not held[0] & set(tables[3].tolist())
    h3mi.kv_release_(pool, tables, lens)
    assert sorted(free()) == list(range(12)) and lens.tolist() == [0] * 4


@pytest.mark.parametrize("n,rows", [(5, 3), (300, 40)])
def test_captured(n, rows):
    """A captured step, replayed with other counts, beside the CPU's."""
    import h3mi
    rng = np.random.default_rng(n)
    ref = _start(rng, n, 30, 4 * n, 500)
    pool, tables, lens = ref.to()
    counts, keep = _i32(np.zeros(n)), _i32(np.zeros(n))

    def call():
        out = h3mi.kv_extend_(pool, tables, lens, rows, counts=counts)
        h3mi.kv_release_(pool, tables, lens, keep)
        return out

    keep.fill_(2 ** 31 - 1)
    call()  # nothing changes: no counts, all is kept
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(6):
        c, k = rng.integers(0, rows + 1, n), np.where(rng.random(n) < 0.3, rng.integers(0, 500, n), 2 ** 31 - 1)
        counts.copy_(_i32(c)), keep.copy_(_i32(k))
        graph.replay()
        torch.cuda.synchronize()
        want = ref.extend(rows, c)
        ref.release(k)
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(out, want)), r
        assert ref.same(pool, tables, lens) == [], r


def test_refusals():
    import h3mi
    pool, tables, lens = h3mi.kv_pool(5), _i32(np.zeros((2, 3))), _i32([0, 0])
    for bad, msg in (((pool, tables[0], lens, 1), "tables"), ((pool, tables.long(), lens, 1), "tables"), ((pool, tables, lens[:1], 1), "lens"),
                     ((pool, tables, lens, -1), "rows"), ((pool._replace(count=lens), tables, lens, 1), "pool.count"),
                     ((pool._replace(free=pool.free.cpu()), tables, lens, 1), "pool.free"), ((pool, tables.t().contiguous().t(), lens, 1), "contiguous")):
        with pytest.raises(ValueError, match=msg):
            h3mi.kv_extend_(*bad)
    with pytest.raises(ValueError, match="counts"):
        h3mi.kv_extend_(pool, tables, lens, 1, counts=_i32([1]))
    with pytest.raises(ValueError, match="keep"):
        h3mi.kv_release_(pool, tables, lens, keep=_i32([1, 2, 3]))
    for call in (lambda: h3mi.kv_extend_(pool, tables, lens, 1, counts=lens), lambda: h3mi.kv_release_(pool, tables, lens, keep=lens),
                 lambda: h3mi.kv_release_(pool._replace(free=tables.reshape(-1)), tables, lens)):
        with pytest.raises(h3mi._lib.H3miError, match="overlap"):
            call()
    with pytest.raises(ValueError, match="pages"):
        h3mi.kv_pool(-1)
