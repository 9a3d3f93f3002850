"""The C entry points of rotary positions and of the page pool refuse bad arguments before touching a device: every pointer
here is made up."""
import ctypes

import pytest

P = ctypes.c_void_p


def _rope(q=None, k=None, **kw):
    from h3mi import _lib
    base = dict(heads=4, ld_in=512, bs_in=1 << 14, ld_out=512, bs_out=1 << 14)
    sides = [None if x is False else _lib.RopeRowsC(**{**base, **at, **(x or {})})
             for x, at in ((q, dict(in_=1 << 20, out=1 << 20)), (k, dict(in_=1 << 21, out=1 << 21)))]
    a = dict(positions=1 << 22, freqs=1 << 23, n=2, rows=3, dim=128, rot=128, interleaved=0, inverse=0, amplitude=1.0)
    a.update(kw)
    rc = _lib.lib.h3mi_rope_bf16(*(None if s is None else ctypes.byref(s) for s in sides), P(a["positions"]), P(a["freqs"]), a["n"], a["rows"],
                                 a["dim"], a["rot"], a["interleaved"], a["inverse"], ctypes.c_float(a["amplitude"]), None)
    return rc, _lib.lib.h3mi_last_error().decode()


@pytest.mark.parametrize("q,k,kw,code,msg", [
    (False, None, {}, 1, "null q"), (None, None, dict(dim=4), 1, "dim=4"), (None, None, dict(dim=100), 1, "dim=100"), (None, None, dict(dim=520), 1, "dim=520"),
    (None, None, dict(rot=0), 1, "rot=0"), (None, None, dict(rot=130), 1, "rot=130"), (None, None, dict(rot=63), 1, "rot=63"),
    (None, None, dict(n=-1), 1, "n=-1"), (None, None, dict(rows=-1), 1, "rows=-1"), (None, None, dict(n=1 << 16, rows=1 << 16), 1, "bad sizes"),
    (None, None, dict(amplitude=float("nan")), 1, "amplitude"), (None, None, dict(positions=None), 1, "null positions"), (None, None, dict(freqs=None), 1, "null"),
    (None, None, dict(positions=6), 2, "4-byte"), (None, None, dict(freqs=(1 << 23) + 4), 2, "8-byte"), (dict(in_=None), None, {}, 1, "null q"),
    (None, dict(out=None), {}, 1, "null k"), (dict(heads=0), None, {}, 1, "heads"), (dict(ld_in=256, ld_out=256), None, {}, 1, "shorter"),
    (None, dict(bs_in=8, bs_out=8), {}, 1, "shorter"), (None, dict(ld_in=516, ld_out=516), {}, 2, "multiples of 8"), (dict(in_=(1 << 20) + 8), None, {}, 2, "aligned"),
    (dict(bs_in=1024, bs_out=1024), None, {}, 3, "rows of q overlap"), (dict(ld_out=1024), None, {}, 3, "other strides"),
    (dict(out=(1 << 20) + 1024), None, {}, 3, "overlaps its result"), (None, dict(in_=1 << 20, out=1 << 20), {}, 3, "q and k overlap"),
    (None, dict(in_=(1 << 20) + 512, out=(1 << 20) + 512), {}, 3, "q and k overlap"), (None, None, dict(positions=(1 << 20) + 64), 3, "positions or freqs"),
    (None, None, dict(freqs=1 << 21), 3, "positions or freqs"), (dict(out=1 << 25), None, {}, 1, "both be in place"),
    (dict(out=1 << 25), dict(out=1 << 20), {}, 3, "overlap"),
])
def test_rope(q, k, kw, code, msg):
    rc, m = _rope(q, k, **kw)
    assert rc == code and msg in m, (rc, m)


def test_rope_of_nothing():
    assert _rope(n=0, positions=None, freqs=None)[0] == 0 and _rope(rows=0)[0] == 0


def test_rope_rows_between_each_other():
    """Heads behind heads of one buffer are apart, by any strides, unless one head is in both."""
    wide = dict(ld_in=1536, bs_in=1 << 14, ld_out=1536, bs_out=1 << 14)
    for strides, ok in ((wide, False), (dict(wide, bs_in=1536 * 8, bs_out=1536 * 8), True), (dict(ld_in=1536 * 8, ld_out=1536 * 8, bs_in=1536, bs_out=1536), True)):
        for heads, want in ((4, ok), (5, False)):
            # k in place and q not is refused after the overlap, so that nothing is launched
            rc, m = _rope(dict(strides, heads=heads, out=1 << 28), dict(strides, in_=(1 << 20) + 1024, out=(1 << 20) + 1024), rows=8)
            assert (rc, "both be in place" in m, "q and k overlap" in m) == ((1, True, False) if want else (3, False, True)), (strides, heads, m)


def _apart(qs, ks, at, n, rows, qh=4, kh=4):
    """(whether q and k in place, k `at` elements behind q, are taken for apart, whether they are), dim 128.  q's result goes
    elsewhere and k's does not, which is refused once the rows have been looked at, so that nothing is launched."""
    base = 1 << 24
    sides = [dict(ld_in=ld, ld_out=ld, bs_in=bs, bs_out=bs) for ld, bs in (qs, ks)]
    # the other order has the same rows: k's result beside q's rows
    rc, m = _rope(dict(sides[0], heads=qh, in_=base, out=1 << 40), dict(sides[1], heads=kh, in_=base + 2 * at, out=base + 2 * at), n=n, rows=rows)
    assert (rc, "both be in place" in m) == (1, True) or (rc == 3 and "q and k overlap" in m), (rc, m)
    taken = set()
    for (ld, bs), h, off in ((qs, qh, 0), (ks, kh, at)):
        runs = {off + i * bs + r * ld + x for i in range(n) for r in range(rows) for x in range(0, 128 * h, 8)}
        if taken & runs:
            return rc == 1, False
        taken |= runs
    return rc == 1, True


@pytest.mark.parametrize("n,rows", [(2, 5), (3, 4), (1, 5), (4, 1), (2, 2)])
def test_rope_rows_of_one_buffer(n, rows):
    """q and k of one buffer are taken as long as no element is in both: side by side in a row, all of a sequence's q rows before
    its k rows, tokens before sequences, and with heads of their own."""
    e, w = 512, 1024  # 4 heads, 8 heads
    layouts = [
        ((2 * e, 2 * e * rows), (2 * e, 2 * e * rows), e, 4, 4),              # [n, rows, 2, e]
        ((e, 2 * e * rows), (e, 2 * e * rows), e * rows, 4, 4),               # [n, 2, rows, e]
        ((e * n, e), (e * n, e), e * n * rows, 4, 4),                         # [2, rows, n, e]
        ((2 * e * n, e), (2 * e * n, e), e * n, 4, 4),                        # [rows, 2, n, e]
        ((w, (w + e) * rows), (e, (w + e) * rows), w * rows, 8, 4),           # [n, (rows of 8 heads, rows of 4)]
        ((e, (w + e) * rows), (w, (w + e) * rows), e * rows, 4, 8),           # [n, (rows of 4, rows of 8)]
        (((w + e) * n, w), ((w + e) * n, e), w * n, 8, 4),                    # [rows, (n of 8 heads, n of 4)]
        ((e, 2 * e * rows + 64), (e, 2 * e * rows + 64), e * rows + 32, 4, 4),  # sequences with room between them
    ]
    for qs, ks, at, qh, kh in layouts:
        for order in (1, -1):
            a, b = ((qs, qh), (ks, kh)) if order == 1 else ((ks, kh), (qs, qh))
            got = _apart(a[0], b[0], order * at, n, rows, a[1], b[1])
            assert got == (True, True), (qs, ks, at, order, got)
    # and never where an element is in both
    for qs, ks, at, qh, kh in layouts:
        for shift in (-8, 8, e // 2, -e // 2, e, -e):
            taken, apart = _apart(qs, ks, at + shift, n, rows, qh, kh)
            assert apart or not taken, (qs, ks, at, shift)


def _pages(fn, pool=None, **kw):
    from h3mi import _lib
    p = {**dict(free=1 << 20, count=1 << 21, pages=100), **(pool or {})}
    a = dict(tables=1 << 22, lens=1 << 23, counts=1 << 24, n=5, blocks=7, rows=3, granted=1 << 25, positions=1 << 26, slots=1 << 27)
    a.update(kw)
    c = ctypes.byref(_lib.KvPoolC(**p))
    L = _lib.lib
    if fn == "extend":
        rc = L.h3mi_kv_extend(c, P(a["tables"]), P(a["lens"]), P(a["counts"]), a["n"], a["blocks"], a["rows"], P(a["granted"]), P(a["positions"]),
                              P(a["slots"]), None)
    else:
        rc = L.h3mi_kv_release(c, P(a["tables"]), P(a["lens"]), P(a["counts"]), a["n"], a["blocks"], None)
    return rc, L.h3mi_last_error().decode()


@pytest.mark.parametrize("fn", ["extend", "release"])
@pytest.mark.parametrize("pool,kw,code,msg", [
    (dict(pages=-1), {}, 1, "pages=-1"), (dict(pages=(1 << 30) + 1), {}, 1, "pages"), (None, dict(n=-1), 1, "n=-1"), (None, dict(blocks=1 << 25), 1, "blocks"),
    (None, dict(n=0x7FFFFFFF), 1, "n="), (None, dict(n=1 << 11, blocks=1 << 20), 1, "2^31 entries"), (dict(free=None), {}, 1, "null free"), (dict(count=None), {}, 1, "null free or count"), (None, dict(tables=None), 1, "null tables"),
    (None, dict(lens=None), 1, "null tables or lens"), (dict(free=(1 << 20) + 2), {}, 2, "4-byte"), (None, dict(lens=(1 << 23) + 1), 2, "4-byte"),
    (None, dict(counts=(1 << 24) + 2), 2, "4-byte"), (dict(free=(1 << 22) + 136), {}, 3, "overlap"), (dict(count=(1 << 20) + 396), {}, 3, "overlap"),
    (None, dict(lens=(1 << 22) + 4), 3, "overlap"), (None, dict(counts=1 << 23), 3, "overlap"), (None, dict(counts=(1 << 20) - 4), 3, "overlap"),
])
def test_pages(fn, pool, kw, code, msg):
    rc, m = _pages(fn, pool, **kw)
    assert rc == code and msg in m, (rc, m)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows=-1"), (dict(rows=1 << 30, n=3), 1, "too many rows"), (dict(granted=None), 1, "null granted"), (dict(slots=None), 1, "null granted, positions or slots"),
    (dict(slots=(1 << 27) + 4), 2, "8-byte"), (dict(positions=(1 << 26) + 2), 2, "4-byte"), (dict(granted=1 << 24), 3, "overlap"), (dict(positions=(1 << 22) + 100), 3, "overlap"),
    (dict(slots=(1 << 26) - 112), 3, "overlap"),
])
def test_extend(kw, code, msg):
    rc, m = _pages("extend", **kw)
    assert rc == code and msg in m, (rc, m)


def test_null_pool_and_no_sequences():
    from h3mi import _lib
    L = _lib.lib
    assert L.h3mi_kv_extend(None, P(64), P(64), None, 1, 1, 1, P(64), P(64), P(64), None) == 1
    assert L.h3mi_kv_release(None, P(64), P(64), None, 1, 1, None) == 1
    for fn in ("extend", "release"):
        assert _pages(fn, n=0, tables=None, lens=None, granted=None)[0] == 0


def test_cpu_tensors_are_refused():
    import torch

    import h3mi
    pool = h3mi.kv_pool(3, device="cpu")
    tables, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: h3mi.kv_extend_(pool, tables, lens, 1), lambda: h3mi.kv_release_(pool, tables, lens)):
        with pytest.raises(ValueError, match="GPU"):
            f()
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    freqs, _ = h3mi.rotary_frequencies(64, device="cpu")
    for f in (h3mi.rotary, h3mi.rotary_):
        with pytest.raises(ValueError, match="GPU"):
            f(q, q.clone(), lens[None], freqs)


def test_the_modules_keep_their_names():
    """No function of the package hides the module that it is in."""
    import inspect

    import h3mi
    for name in ("fused", "gemm", "kvcache", "kvpages", "linear", "quant", "rope"):
        __import__(f"h3mi.{name}")
        assert inspect.ismodule(getattr(h3mi, name)), name
