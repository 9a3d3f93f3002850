"""Attention by tiles in each of the ways that a call's sizes can divide it, over batches that make every part of it count:
uneven lengths, none among them, padding rows, pages that are not there (whole look-ups of them), value scales of zero and of
no ordinary size, and poisoned blocks.  A case's parts, the partial rows that its workspace holds, say that it is divided as it
is meant to be (256 CUs)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGES, ZERO, SMALL, NAN_K, NAN_V = 40, 36, 37, 38, 39  # the last four pages are special, and only where a case puts them

# n, rows, heads, kv, dim, blocks, top, parts: partial rows = split items x splits x rows of an item
CASES = {
    "64 elements: 768 whole items, 32 in 10 splits": (2, 900, 50, 10, 64, 40, 0, 32 * 10 * 128),
    "64 elements: 768 whole items, 192 in 4 splits": (2, 900, 60, 60, 64, 40, 0, 192 * 4 * 128),
    "64 elements: 768 whole items, 192 in 4 splits, lists": (2, 900, 60, 60, 64, 90, 40, 192 * 4 * 128),
    "64 elements: 4 items in 16 splits": (2, 100, 2, 2, 64, 64, 0, 4 * 16 * 128),
    "64 elements: 12 items in 64 splits": (3, 200, 2, 2, 64, 300, 0, 12 * 64 * 128),
    "128 elements: 512 whole items, 208 in 2 splits": (3, 700, 40, 8, 128, 60, 0, 208 * 2 * 128),
    "128 elements: 512 whole items, 208 in 2 splits, lists": (3, 700, 40, 8, 128, 90, 30, 208 * 2 * 128),
    "128 elements: 512 whole items of heads in common, 128 in 4 splits": (4, 100, 200, 40, 128, 30, 0, 128 * 4 * 128),
    "128 elements: 672 whole items": (4, 300, 56, 56, 128, 7, 0, 0),
    "128 elements, 8 waves: 256 whole items, 14 in 18 splits": (3, 1100, 18, 18, 128, 1100, 0, 14 * 18 * 256),
    "128 elements, 8 waves: 256 whole items, 104 in 2 splits": (4, 1030, 18, 6, 128, 140, 0, 104 * 2 * 256),
    "256 elements: 120 items in 2 splits": (2, 200, 30, 6, 256, 30, 0, 120 * 2 * 128),
    "256 elements: 256 whole items, 44 in 5 splits, lists": (1, 1900, 20, 20, 256, 100, 40, 44 * 5 * 128),
    "256 elements: 256 whole items, 5 in 12 splits": (3, 300, 29, 29, 256, 50, 0, 5 * 12 * 128),
}


def _make(n, rows, heads, kv, dim, blocks, top, seed):
    import h3mi
    g = torch.Generator(device=DEV).manual_seed(seed)
    ints = lambda *s: torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    scales = lambda: torch.rand(PAGES, kv, generator=g, device=DEV) * 0.02 + 0.005  # noqa: E731
    c = h3mi.KVCache(ints(PAGES, kv, 64, dim), ints(PAGES, kv, dim, 64), scales(), scales(),
                     torch.zeros(PAGES, kv, dim, dtype=torch.int16, device=DEV))
    c.v_scale[ZERO], c.v[ZERO], c.v_scale[SMALL] = 0, 0, 2.0 ** -100
    c.k_scale[NAN_K, 0] = c.v_scale[NAN_V, kv - 1] = float("nan")
    q = torch.randn(n, rows, heads, dim, generator=g, device=DEV).to(torch.bfloat16)
    tables = torch.randint(0, ZERO, (n, blocks), generator=g, device=DEV, dtype=torch.int32)
    tables[:, 1], tables[:, blocks // 3] = ZERO, SMALL
    # the first sequence is whole but for a hole, the second ends in the middle and has padding rows, the third has fewer tokens
    # than rows, the fourth none
    lens = torch.tensor([blocks * 64 - 5, blocks * 33 + 1, rows // 2, 0][:n], dtype=torch.int32, device=DEV)
    counts = torch.tensor([rows, rows - rows // 3, rows, rows][:n], dtype=torch.int32, device=DEV)
    look = 512 if blocks > 1024 else 256  # blocks that a workgroup looks up at once
    if blocks > look:
        tables[0, blocks - blocks % look - look:blocks - blocks % look] = -1
        tables[n - 1, :look] = -1
    else:
        tables[0, 2:5] = -1
    if n > 1:
        tables[1, 3:6] = torch.tensor([PAGES, -7, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    lists = None
    if top:
        lists = torch.stack([torch.randperm(blocks, generator=g, device=DEV)[:top] for _ in range(n * -(-rows // 128) * kv)])
        lists = lists.to(torch.int32).reshape(n, -(-rows // 128), kv, top).contiguous()
    return c, q, tables, lens, counts, lists


def _check(out, c, q, tables, lens, counts, causal, lists):
    """Against 64 bits, a sequence and a head at a time, under kv_ref.bound; rows that see a NaN scale are NaN."""
    n, rows, heads, dim = q.shape
    kv, blocks = c.k.shape[1], tables.shape[1]
    half = torch.finfo(torch.bfloat16).eps / 2
    for i in range(n):
        size, count = min(int(lens[i]), blocks * 64), int(counts[i])
        assert (out[i, count:] == 0).all()
        page = tables[i].long()
        there = ((page >= 0) & (page < PAGES)).repeat_interleave(64)[:size]
        page = torch.where((page >= 0) & (page < PAGES), page, 0)
        at, row = torch.arange(size, device=DEV), int(lens[i]) - count + torch.arange(count, device=DEV)
        for h in range(kv):
            seen = there.expand(count, size).clone()
            if causal:
                seen &= at <= row[:, None]
            if lists is not None:
                took = torch.zeros(lists.shape[1], blocks, dtype=torch.bool, device=DEV)
                took.scatter_(1, lists[i, :, h].long(), True)
                seen &= took.repeat_interleave(64, 1)[:, :size].repeat_interleave(128, 0)[:count]
            ks, vs = c.k_scale[page, h].double(), c.v_scale[page, h].double()
            bad = (ks.isnan() | vs.isnan()).repeat_interleave(64)[:size]
            poisoned = (seen & bad).any(1)
            k = (c.k[page, h].double() * ks.nan_to_num()[:, None, None]).reshape(-1, dim)[:size]
            v = (c.v[page, h].double() * vs.nan_to_num()[:, None, None]).transpose(1, 2).reshape(-1, dim)[:size]
            any_seen = seen.any(1)
            for j in range(h * heads // kv, (h + 1) * heads // kv):
                got = out[i, :count, j].double()
                assert (got[~any_seen] == 0).all(), (i, j)
                assert got[poisoned].isnan().all(), (i, j)
                use = any_seen & ~poisoned
                x = (q[i, :count, j][use].double() @ k.t() * dim ** -0.5).masked_fill_(~seen[use], -float("inf"))
                p = torch.softmax(x, 1)
                want, mag = p @ v, p @ v.abs()
                top = (q[i, :count, j][use].double().abs() @ k.abs().t() * dim ** -0.5).masked_fill_(~seen[use], 0).amax(1, keepdim=True) \
                    if size else mag
                bound = half * (mag * (1 + half) + want.abs()) * (1 + 1e-3) + 2 * mag * ((dim + 8) * 2.0 ** -24 * (top + 4)) + 1e-30
                off = (got[use] - want).abs() / bound
                assert off.numel() == 0 or off.max() <= 1, (i, j, float(off.max()))


@pytest.mark.parametrize("poison", [False, True])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", list(CASES))
def test_attention_divided(case, causal, poison):
    import h3mi
    from h3mi import _lib
    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("the cases are made for 256 CUs")
    n, rows, heads, kv, dim, blocks, top, parts = CASES[case]
    assert _lib.lib.h3mi_kv_attention_workspace(n, rows, heads, kv, dim, blocks, top) == parts * (dim * 4 + 8)
    c, q, tables, lens, counts, lists = _make(n, rows, heads, kv, dim, blocks, top, seed=len(case))
    if poison:  # the last block of the first sequence, and one in the middle of the second
        tables[0, blocks - 1] = NAN_K
        tables[n - 1 if n < 3 else 1, blocks // 4] = NAN_V
    out = h3mi.kv_attention(q, c, tables, lens, causal=causal, counts=counts, blocks=lists)
    _check(out, c, q, tables, lens, counts, causal, lists)
