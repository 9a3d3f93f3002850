"""Attention over the 4-bit cache in each of the ways that a call's sizes can divide it, over batches that make every part of it
count: uneven lengths, none among them, padding rows, pages that are not there (whole look-ups of them), factors from the least
up, what is no number behind a sequence's end, and within it.  A case's parts, the partial rows that its workspace holds, say
that it is divided as it is meant to be (256 CUs)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGES, LEAST, SPARE = 40, 36, 37  # pages that are special: factors of 2^-125; not numbered in any table

# n, rows, heads, kv, dim, blocks, top, parts: partial rows (tiles: split items x splits x rows of an item; few queries: pieces)
CASES = {
    "64 elements, whole rounds and splits": (2, 900, 50, 10, 64, 40, 0, 32 * 10 * 128),
    "64 elements, lists": (2, 900, 60, 60, 64, 90, 40, 192 * 4 * 128),
    "64 elements, many splits": (3, 200, 2, 2, 64, 300, 0, 12 * 60 * 128),
    "64 elements, more pieces than one round": (3, 271, 24, 24, 64, 500, 0, 216 * 14 * 128),
    "128 elements, whole rounds and splits": (3, 700, 40, 8, 128, 60, 0, 208 * 2 * 128),
    "128 elements, lists": (3, 700, 40, 8, 128, 90, 30, 208 * 2 * 128),
    "128 elements, heads in common": (4, 100, 200, 40, 128, 30, 0, 128 * 4 * 128),
    "128 elements, whole rounds": (4, 300, 56, 56, 128, 7, 0, 0),
    "128 elements, 8 waves, more than a look-up": (3, 1100, 18, 18, 128, 1100, 0, 14 * 18 * 256),
    "128 elements, 8 waves, more pieces than one round": (4, 1030, 18, 6, 128, 140, 0, 104 * 7 * 256),
    "256 elements": (2, 200, 30, 6, 256, 30, 0, 120 * 2 * 128),
    "256 elements, lists": (1, 1900, 20, 20, 256, 100, 40, 44 * 5 * 128),
    "256 elements, one sequence in rounds": (1, 1000, 20, 20, 256, 63, 0, 160 * 3 * 128),
    "256 elements, whole rounds and splits": (3, 300, 29, 29, 256, 50, 0, 5 * 10 * 128),
    "few, 64 elements, 64 queries": (2, 13, 10, 2, 64, 70, 0, None),
    "few, 128 elements, 32 queries": (4, 8, 8, 2, 128, 300, 0, None),
    "few, 256 elements": (3, 4, 8, 2, 256, 90, 0, None),
    "few, a sequence each": (40, 1, 40, 40, 128, 5, 0, 0),
    "few, lists": (2, 3, 10, 2, 128, 90, 20, None),
}


def _make(n, rows, heads, kv, dim, blocks, top, seed):
    import h3mi
    g = torch.Generator(device=DEV).manual_seed(seed)
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=DEV, dtype=torch.uint8)  # noqa: E731
    c = h3mi.KVCache4(draw(0, 256, PAGES, kv, 64, dim // 2), draw(0, 256, PAGES, kv, 64, dim // 2), draw(122, 127, PAGES, kv, dim // 32, 64),
                      draw(118, 130, PAGES, kv, dim // 32, 64))
    c.k_scale[LEAST], c.v_scale[LEAST] = 2, 2
    q = torch.randn(n, rows, heads, dim, generator=g, device=DEV).to(torch.bfloat16)
    tables = torch.randint(0, LEAST, (n, blocks), generator=g, device=DEV, dtype=torch.int32)
    tables[:, blocks // 3] = LEAST
    # whole but for a hole; ends in the middle, with padding rows; fewer tokens than rows; none
    lens, counts = (torch.tensor((a * n)[:n], dtype=torch.int32, device=DEV) for a in (
        [blocks * 64 - 5, blocks * 33 + 1, rows // 2, 0], [rows, rows - rows // 3, rows, rows]))
    look = 512 if blocks > 1024 else 256
    if blocks > look:
        tables[0, blocks - blocks % look - look:blocks - blocks % look] = -1
        tables[n - 1, :look] = -1
    elif blocks > 6:
        tables[0, 2:5] = -1
        if n > 1:
            tables[1, 3:6] = torch.tensor([PAGES, -7, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    # the first sequence's last block: not numbers behind its end
    tables[0, blocks - 1] = SPARE
    c.k_scale[SPARE, :, :, 59:], c.v_scale[SPARE, :, :, 59:] = 255, 253
    lists = None
    if top:
        lists = torch.stack([torch.randperm(blocks, generator=g, device=DEV)[:top] for _ in range(n * -(-rows // 128) * kv)])
        lists = lists.to(torch.int32).reshape(n, -(-rows // 128), kv, top).contiguous()
    return c, q, tables, lens, counts, lists


def _values(q, codes):
    """bytes [.., 64, dim / 2], codes [.., dim / 32, 64] -> (64-bit values, whether each is no number) [.., 64, dim]."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=DEV)
    x = grid[torch.stack([q & 15, q >> 4], -1).flatten(-2).long()]
    bad = (codes >= 253).transpose(-1, -2).repeat_interleave(32, -1)
    f = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEV), codes.double() - 127).transpose(-1, -2).repeat_interleave(32, -1)
    return torch.where(bad, 0.0, x * f), bad


def _check(out, c, q, tables, lens, counts, causal, lists):
    """Against 64 bits, a sequence and a head at a time, under kv_ref.bound; NaNs exactly where a row sees what is no number."""
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
            (k, k_bad), (v, v_bad) = ([t.flatten(0, 1)[:size] for t in _values(a[page, h], s[page, h])] for a, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
            none = (seen & k_bad.any(1)).any(1)[:, None] | ((seen.float() @ v_bad.float()) > 0)  # [count, dim]
            any_seen = seen.any(1)
            for j in range(h * heads // kv, (h + 1) * heads // kv):
                got = out[i, :count, j].double()
                assert (got[~any_seen] == 0).all(), (i, j)
                assert torch.equal(got.isnan(), none & any_seen[:, None]), (i, j)
                x = (q[i, :count, j][any_seen].double() @ k.t() * dim ** -0.5).masked_fill_(~seen[any_seen], -float("inf"))
                p = torch.softmax(x, 1)
                want, mag = p @ v, p @ v.abs()
                top = (q[i, :count, j][any_seen].double().abs() @ k.abs().t() * dim ** -0.5).masked_fill_(~seen[any_seen], 0)
                top = top.amax(1, keepdim=True) if size else mag
                bound = half * (mag * (1 + half) + want.abs()) * (1 + 1e-3) + 2 * mag * ((dim + 8) * 2.0 ** -24 * (top + 4)) + 1e-30
                off = torch.where(none[any_seen], 0.0, (got[any_seen] - want).abs() / bound)
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
    need = _lib.lib.h3mi_kv_attention_mx4_workspace(n, rows, heads, kv, dim, blocks, top)
    assert need > 0 if parts is None else need == parts * (dim * 4 + 8)
    c, q, tables, lens, counts, lists = _make(n, rows, heads, kv, dim, blocks, top, seed=len(case))
    if poison:  # a value's group in the last block of the first sequence, a key's in the middle of the second
        c.v_scale[SPARE, kv - 1, dim // 32 - 1, 7] = 254
        tables[n - 1 if n < 3 else 1, blocks // 4] = SPARE + 1
        c.k_scale[SPARE + 1, 0, 0, 11] = 253
    out = h3mi.kv_attention(q, c, tables, lens, causal=causal, counts=counts, blocks=lists)
    _check(out, c, q, tables, lens, counts, causal, lists)
