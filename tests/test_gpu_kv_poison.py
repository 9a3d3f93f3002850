"""Blocks that a NaN or an infinity was written to: every row that sees one is NaN, however little the block weighs in it, and
no other row is, in each of the kernels and of the joins of their parts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

# rows, blocks: what runs, for 2 heads of 128 elements of one sequence (parts: partial rows that its workspace holds, 0 for
# none; the pieces' join takes two rows' worth of spans at most)
PLANS = {
    "few": (1, 6), "few, 32 rows": (32, 6), "few, pieces joined": (1, 64), "few, 20 rows, pieces joined": (20, 64),
    "tiles": (300, 6), "tiles, 6 splits": (300, 24), "tiles, 16 splits": (300, 64), "tiles, 64 splits": (200, 300),
}
SPLITS = {"tiles, 6 splits": 6, "tiles, 16 splits": 16, "tiles, 64 splits": 64}


def _parts(n, rows, heads, kv, dim, blocks, top=0):
    from h3mi import _lib
    need = _lib.lib.h3mi_kv_attention_workspace(n, rows, heads, kv, dim, blocks, top)
    assert need % (dim * 4 + 8) == 0
    return need // (dim * 4 + 8)


def _check_plan(name):
    rows, blocks = PLANS[name]
    parts = _parts(1, rows, 2, 2, 128, blocks)
    if name in SPLITS:
        assert parts == 2 * -(-rows // 128) * SPLITS[name] * 128
    else:
        assert (parts > 0) == ("joined" in name)


def _levels(blocks, hot, bad, low):
    """Which way each block's keys point: the hot one along the query, the bad one against it, the others neither way, or
    (low) against it too."""
    to = torch.full((blocks,), -1.0 if low else 0.0)
    to[hot], to[bad] = 1.0, -1.0
    return to


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("low", [False, True])
@pytest.mark.parametrize("plan", list(PLANS))
def test_a_poisoned_block_reaches_every_row_that_sees_it(plan, low, value, what):
    """Scores 1448 apart: the block's probabilities are 0 in 32 bits, within its split and against the others."""
    import h3mi
    _check_plan(plan)
    rows, blocks = PLANS[plan]
    bad, hot, end = blocks - 2, 1, blocks * 64
    g = torch.Generator().manual_seed(rows + blocks)
    k = torch.randn(1, end, 2, 128, generator=g) * 0.01 + 8 * _levels(blocks, hot, bad, low).repeat_interleave(64)[None, :, None, None]
    v = torch.randn(1, end, 2, 128, generator=g)
    (k if what == "k" else v)[0, bad * 64 + 5, 1, 7] = value
    q = torch.randn(1, rows, 2, 128, generator=g) * 0.01 + 8
    k, v, q = (t.to(torch.bfloat16).to(DEV) for t in (k, v, q))
    tables = torch.randperm(blocks, generator=g).to(torch.int32)[None].to(DEV)
    lens = torch.tensor([end], dtype=torch.int32, device=DEV)
    cache = h3mi.kv_write_(h3mi.kv_cache(blocks, 2, 128), k, v, tables, lens)
    bad_row = torch.zeros(1, rows, 2, 128, dtype=torch.bool)
    for causal in (False, True):
        bad_row[:, :, 1] = True
        if causal:  # rows before the bad block, of which 300 rows have some
            bad_row[:, end - rows + torch.arange(rows) < bad * 64, 1] = False
        out = h3mi.kv_attention(q, cache, tables, lens, causal=causal).float().cpu()
        assert torch.equal(out.isnan(), bad_row), causal
    # a list without it
    take = torch.tensor([b for b in range(blocks) if b != bad], dtype=torch.int32, device=DEV)
    lists = take.repeat(1, -(-rows // 128), 2, 1)
    assert h3mi.kv_attention(q, cache, tables, lens, blocks=lists).isfinite().all()
    # and one with it
    lists[..., blocks - 2] = bad
    got = h3mi.kv_attention(q, cache, tables, lens, blocks=lists).isnan().cpu()
    assert got[:, :, 1].all() and not got[:, :, 0].any()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("plan", list(PLANS))
def test_a_poisoned_query_stays_in_its_row_and_head(plan, value):
    import h3mi
    _check_plan(plan)
    rows, blocks = PLANS[plan]
    g = torch.Generator(device=DEV).manual_seed(rows * blocks)
    draw = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    tables = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)[None]
    lens = torch.tensor([blocks * 64 - 3], dtype=torch.int32, device=DEV)
    cache = h3mi.kv_write_(h3mi.kv_cache(blocks, 2, 128), draw(1, blocks * 64 - 3, 2, 128), draw(1, blocks * 64 - 3, 2, 128), tables, lens)
    q = draw(1, rows, 2, 128)
    hit = torch.zeros(rows, 2, dtype=torch.bool, device=DEV)
    hit[rows // 2, 1] = hit[0, 0] = True
    bad = q.clone()
    bad[0, :, :, 17] = torch.where(hit, torch.tensor(value, device=DEV, dtype=torch.bfloat16), q[0, :, :, 17])
    for causal in (False, True):
        want, got = (h3mi.kv_attention(x, cache, tables, lens, causal=causal)[0] for x in (q, bad))
        assert got[hit].isnan().all() and want.isfinite().all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("rows,blocks", [(8, 6), (8, 64), (300, 6), (300, 64)])
def test_rows_behind_a_sequences_own_are_not_read(rows, blocks):
    """NaN in the padding of a batch changes no page, no selection and no output."""
    import h3mi
    g = torch.Generator(device=DEV).manual_seed(rows + blocks)
    draw = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    n = 3
    counts = torch.tensor([rows, rows // 2 + 1, 0], dtype=torch.int32, device=DEV)
    lens = torch.tensor([blocks * 64, blocks * 40 + 7, 0], dtype=torch.int32, device=DEV)
    tables = torch.randperm(n * blocks, generator=g, device=DEV).reshape(n, blocks).to(torch.int32)
    k, v, before = draw(n, rows, 2, 128), draw(n, rows, 2, 128), draw(n, blocks * 64, 2, 128)
    q = draw(n, rows, 4, 128)
    pad = (torch.arange(rows, device=DEV) >= counts[:, None])[..., None, None]
    got = []
    for fill in (0.0, float("nan")):
        kx, vx, qx = (torch.where(pad, torch.tensor(fill, dtype=torch.bfloat16, device=DEV), x) for x in (k, v, q))
        c = h3mi.kv_write_(h3mi.kv_cache(n * blocks, 2, 128), before, before, tables, lens)
        h3mi.kv_write_(c, kx, vx, tables, lens, counts=counts)
        pick = h3mi.kv_select(qx, c, tables, lens, 3, causal=True, counts=counts)
        got.append([*c, pick, h3mi.kv_attention(qx, c, tables, lens, causal=True, counts=counts),
                    h3mi.kv_attention(qx, c, tables, lens, counts=counts, blocks=pick)])
    for a, b in zip(*got):
        assert torch.equal(a, b) and (not a.is_floating_point() or a.isfinite().all())
    assert (got[0][6][pad.expand(n, rows, 4, 128)] == 0).all()
