"""The C entry points of the 8-bit cache refuse bad arguments before touching a device: every pointer here is made up."""
import ctypes

import pytest

P = ctypes.c_void_p
BASE = dict(k=4096, v=1 << 19, k_scale=12288, v_scale=16384, k_sum=20480, pages=10, heads=2, dim=128)
SEQS = dict(tables=24576, lens=28672, counts=None, n=2, blocks=5)


def _call(fn, cache=None, seqs=None, **kw):
    from h3mi import _lib
    c, s = _lib.KvCacheC(**{**BASE, **(cache or {})}), _lib.KvSeqsC(**{**SEQS, **(seqs or {})})
    c, s = ctypes.byref(c), ctypes.byref(s)
    a = dict(p=1 << 20, p2=1 << 21, rows=4, heads=4, ld=512, bs=2048, top=3, length=9, out=1 << 22, scale=1.0, starts=None, blocks=None,
             work=None, size=0)
    a.update(kw)
    L = _lib.lib
    if fn == "write":
        rc = L.h3mi_kv_write_i8(P(a["p"]), P(a["p2"]), a["rows"], a["ld"], a["bs"], a["ld"], a["bs"], c, s, None)
    elif fn == "read":
        rc = L.h3mi_kv_read_bf16(P(a["p"]), P(a["p2"]), P(a["starts"]), a["length"], c, s, None)
    elif fn == "select":
        rc = L.h3mi_kv_select(P(a["p"]), a["rows"], a["heads"], a["ld"], a["bs"], c, s, a["top"], 0, P(a["out"]), P(a["work"]),
                              a["size"], None)
    else:
        rc = L.h3mi_kv_attention_bf16(P(a["p"]), a["rows"], a["heads"], a["ld"], a["bs"], c, s, ctypes.c_float(a["scale"]), 0,
                                      P(a["blocks"]), a["top"], P(a["out"]), P(a["work"]), a["size"], None)
    return rc, L.h3mi_last_error().decode()


EVERY = ["write", "read", "select", "attention"]


@pytest.mark.parametrize("fn", EVERY)
@pytest.mark.parametrize("cache,seqs,code,msg", [
    (dict(dim=96), None, 1, "dim=96"), (dict(dim=0), None, 1, "dim=0"), (dict(heads=0), None, 1, "heads=0"), (dict(pages=-1), None, 1, "pages=-1"),
    (dict(pages=1 << 31), None, 1, "pages"), (None, dict(n=-1), 1, "n=-1"), (None, dict(blocks=-1), 1, "blocks=-1"),
    (None, dict(blocks=1 << 25), 1, "blocks"), (dict(k=None), None, 1, "null cache"), (dict(k_sum=None), None, 1, "null cache"),
    (None, dict(lens=None), 1, "null tables or lens"), (None, dict(tables=None), 1, "null tables or lens"), (dict(v=(1 << 19) + 8), None, 2, "aligned"), (dict(v=8192), None, 3, "k and v overlap"),
    (dict(k_scale=2), None, 2, "aligned"), (None, dict(lens=6), 2, "4-byte"),
])
def test_cache_and_sequences(fn, cache, seqs, code, msg):
    rc, m = _call(fn, cache, seqs)
    assert rc == code and msg in m, (rc, m)


@pytest.mark.parametrize("fn", ["write", "select", "attention"])
@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows=-1"), (dict(p=None), 1, "null"), (dict(p=(1 << 20) + 8), 2, "aligned"), (dict(ld=8), 1, "shorter"),
    (dict(bs=8), 1, "shorter"), (dict(ld=516), 2, "multiples of 8"), (dict(bs=2052), 2, "multiples of 8"), (dict(bs=-2048), 1, "shorter"),
])
def test_rows(fn, kw, code, msg):
    rc, m = _call(fn, **kw)
    assert rc == code and msg in m, (rc, m)


@pytest.mark.parametrize("fn,kw,code,msg", [
    ("read", dict(length=-1), 1, "length=-1"), ("read", dict(p=None), 1, "null k or v"), ("read", dict(p2=8), 2, "aligned"),
    ("read", dict(starts=2), 2, "aligned"), ("select", dict(heads=3), 1, "multiple of the cache's"), ("select", dict(heads=0), 1, "multiple"),
    ("attention", dict(heads=5), 1, "multiple of the cache's"), ("select", dict(top=0), 1, "top=0"), ("select", dict(top=32769), 1, "top=32769"),
    ("select", dict(out=None), 1, "null blocks"), ("select", dict(out=2), 2, "aligned"), ("attention", dict(out=None), 1, "null out"),
    ("attention", dict(out=8), 2, "aligned"), ("attention", dict(scale=float("nan")), 1, "scale"), ("attention", dict(scale=float("inf")), 1, "scale"),
    ("attention", dict(out=1 << 20), 3, "overlaps"), ("attention", dict(out=(1 << 20) + 2048), 3, "overlaps"),
    ("attention", dict(out=1 << 19), 3, "overlaps"), ("attention", dict(out=20480), 3, "overlaps"), ("select", dict(out=1 << 20), 3, "overlaps"),
    ("select", dict(out=12288), 3, "overlaps"), ("read", dict(p2=1 << 20), 3, "overlap"), ("read", dict(p=1 << 19), 3, "overlap"),
    ("write", dict(p=1 << 19), 3, "overlap"), ("write", dict(p2=(1 << 19) + 4096), 3, "overlap"),
    ("attention", dict(blocks=4096, top=0), 1, "top=0"), ("attention", dict(blocks=4096, top=1 << 25), 1, "top="), ("attention", dict(blocks=4098), 2, "aligned"),
])
def test_each(fn, kw, code, msg):
    rc, m = _call(fn, **kw)
    assert rc == code and msg in m, (rc, m)


def test_sizes_past_a_launch():
    assert _call("write", dict(heads=65536, dim=256, v=1 << 50), dict(blocks=(1 << 25) - 1), rows=1 << 30, ld=65536 * 256, bs=1 << 60)[0] == 1
    assert _call("read", dict(heads=65536, v=1 << 50), dict(n=1 << 30), length=1 << 30)[0] == 1
    assert _call("select", dict(heads=65536, v=1 << 50), dict(n=1 << 20), rows=1 << 20, heads=65536, ld=65536 * 128, bs=1 << 60)[0] == 1
    assert _call("select", None, dict(blocks=32769))[0] == 1
    assert _call("attention", dict(heads=65536, v=1 << 50), dict(n=1 << 20), rows=1 << 20, heads=65536, ld=65536 * 128, bs=1 << 60)[0] == 1


@pytest.mark.parametrize("fn", EVERY)
def test_nothing_to_do(fn):
    assert _call(fn, None, dict(n=0, lens=None, tables=None))[0] == 0
    assert _call(fn, rows=0, length=0, p=None, p2=None, out=None)[0] == 0


@pytest.mark.parametrize("fn", EVERY)
def test_null_structures(fn):
    from h3mi import _lib
    L = _lib.lib
    rc = {"write": lambda: L.h3mi_kv_write_i8(P(4096), P(8192), 1, 256, 256, 256, 256, None, None, None),
          "read": lambda: L.h3mi_kv_read_bf16(P(4096), P(8192), None, 1, None, None, None),
          "select": lambda: L.h3mi_kv_select(P(4096), 1, 2, 256, 256, None, None, 1, 0, P(8192), None, 0, None),
          "attention": lambda: L.h3mi_kv_attention_bf16(P(4096), 1, 2, 256, 256, None, None, ctypes.c_float(1), 0, None, 0, P(8192), None, 0, None)}[fn]()
    assert rc == 1 and "null cache or sequences" in L.h3mi_last_error().decode()


@pytest.mark.parametrize("rows,heads,kv,dim,blocks,top", [(1, 56, 56, 128, 309, 0), (1, 40, 8, 128, 2048, 64), (40, 40, 8, 128, 141, 0),
                                                          (4800, 56, 56, 128, 309, 0), (2401, 56, 56, 128, 609, 100)])
def test_workspace(rows, heads, kv, dim, blocks, top):
    """A call that splits its work asks for whole partial rows, and refuses less than it asked for."""
    from h3mi import _lib
    need = _lib.lib.h3mi_kv_attention_workspace(1, rows, heads, kv, dim, blocks, top)
    assert need > 0 and need % (dim * 4 + 8) == 0
    kw = dict(rows=rows, heads=heads, ld=heads * dim, bs=rows * heads * dim, blocks=4096 if top else None, top=top, p=1 << 41, out=1 << 43)
    seqs = dict(n=1, blocks=blocks)
    cache = dict(heads=kv, dim=dim, v=1 << 40)
    for work, size in ((None, need), (1 << 30, need - 1), (1 << 30, 0)):
        rc, m = _call("attention", cache, seqs, work=work, size=size, **kw)
        assert rc == 1 and "workspace" in m
    rc, m = _call("attention", cache, seqs, work=(1 << 30) + 8, size=need, **kw)
    assert rc == 2 and "workspace" in m


def test_workspace_of_a_selection():
    from h3mi import _lib
    f = _lib.lib.h3mi_kv_select_workspace
    need = f(4, 1, 8, 2048)
    assert need == 4 * 8 * 2048 * 4
    assert f(4, 1, 8, 100) == 0 and f(1, 2401, 56, 2048) == 0 and f(0, 1, 8, 2048) == 0 and f(1, 1, 8, 32769) == 0 and f(1 << 62, 1, 8, 2048) == 0
    kw = dict(rows=1, heads=8, ld=1024, bs=1024, p=1 << 41, out=1 << 43)
    for work, size in ((None, need), (1 << 30, need - 1)):
        rc, m = _call("select", dict(heads=8, v=1 << 40), dict(n=4, blocks=2048), work=work, size=size, **kw)
        assert rc == 1 and "workspace" in m
    assert _call("select", dict(heads=8, v=1 << 40), dict(n=4, blocks=2048), work=(1 << 30) + 2, size=need, **kw)[0] == 2


@pytest.mark.parametrize("a", [(0, 1, 2, 2, 128, 5, 0), (1, 0, 2, 2, 128, 5, 0), (-1, 1, 2, 2, 128, 5, 0), (1, 1, 3, 2, 128, 5, 0),
                               (1, 1, 2, 0, 128, 5, 0), (1, 1, 2, 2, 96, 5, 0), (1 << 62, 1 << 30, 65536, 1, 256, 5, 0), (1, 1, 2, 2, 128, -5, 0)])
def test_workspace_of_nothing(a):
    from h3mi import _lib
    assert _lib.lib.h3mi_kv_attention_workspace(*a) == 0


def test_cpu_tensors_are_refused():
    """The Python functions refuse host tensors before a kernel could see their addresses."""
    import torch

    import h3mi
    c = h3mi.kv_cache(2, 2, 64, device="cpu")
    t, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for f in (lambda: h3mi.kv_write_(c, x, x, t, lens), lambda: h3mi.kv_read(c, t, lens, 1), lambda: h3mi.kv_select(x, c, t, lens, 1),
              lambda: h3mi.kv_attention(x, c, t, lens)):
        with pytest.raises(ValueError, match="GPU"):
            f()
    with pytest.raises(ValueError, match="dim"):
        h3mi.kv_cache(2, 2, 100, device="cpu")


@pytest.mark.parametrize("at", [12288, 16384, 20480])
@pytest.mark.parametrize("name", ["p", "p2"])
def test_written_rows_over_the_scales_and_sums(name, at):
    rc, m = _call("write", dict(k=1 << 23, v=1 << 24), **{name: at})
    assert rc == 3 and "overlap" in m, (rc, m)


# a cache, sequences and rows that do not overlap
APART = dict(k=1 << 23, v=1 << 24, k_scale=1 << 25, v_scale=1 << 26, k_sum=1 << 27)
APART_SEQS = dict(tables=1 << 28, lens=1 << 29, counts=1 << 30)


@pytest.mark.parametrize("cache", [
    dict(v_scale=1 << 25), dict(v_scale=(1 << 25) + 76), dict(k_scale=(1 << 26) + 4), dict(k_sum=1 << 25), dict(k_sum=(1 << 23) + 4096),
    dict(k_scale=(1 << 24) + 163836), dict(v_scale=(1 << 27) + 5116),
])
def test_written_cache_over_itself(cache):
    """Two workgroups, or two of a thread's stores, would write the same bytes."""
    rc, m = _call("write", {**APART, **cache}, APART_SEQS)
    assert rc == 3 and "the cache's tensors overlap" in m, (rc, m)


@pytest.mark.parametrize("seqs", [
    dict(tables=1 << 23), dict(tables=(1 << 25) - 36), dict(lens=1 << 26), dict(lens=(1 << 27) + 5116), dict(counts=(1 << 24) + 8),
])
def test_written_cache_over_the_sequences(seqs):
    rc, m = _call("write", APART, {**APART_SEQS, **seqs})
    assert rc == 3 and "tables, lens or counts overlap the cache" in m, (rc, m)


@pytest.mark.parametrize("fn,kw,msg", [
    ("read", dict(p=1 << 28), "tables, lens"), ("read", dict(p2=1 << 29), "tables, lens"), ("read", dict(p2=(1 << 28) - 2 * 9 * 256 * 2 + 16), "tables, lens"),
    ("read", dict(p=(1 << 31) - 16, starts=1 << 31), "starts"), ("read", dict(p2=1 << 31, starts=1 << 31), "starts"),
    ("select", dict(out=1 << 28), "tables, lens"), ("select", dict(out=(1 << 29) - 8), "tables, lens"), ("select", dict(out=(1 << 30) + 4), "tables, lens"),
    ("attention", dict(out=1 << 28), "tables, lens"), ("attention", dict(out=(1 << 29) - 16), "tables, lens"), ("attention", dict(out=1 << 30), "tables, lens"),
    ("attention", dict(out=1 << 31, blocks=1 << 31), "blocks"), ("attention", dict(out=(1 << 31) - 8192 + 16, blocks=1 << 31), "blocks"),
    ("attention", dict(out=(1 << 31) + 32, blocks=1 << 31), "blocks"),
])
def test_outputs_over_what_is_read(fn, kw, msg):
    """A workgroup's output would change what another has yet to read."""
    rc, m = _call(fn, APART, APART_SEQS, **kw)
    assert rc == 3 and "overlap" in m and msg in m, (rc, m)


@pytest.mark.parametrize("fn,at", [(fn, at) for fn in ("select", "attention") for at in (
    "p", "out", "k", "v", "k_scale", "v_scale", "k_sum", "tables", "lens", "counts")] + [("attention", "blocks")])
def test_workspace_over_what_a_call_reads_or_writes(fn, at):
    from h3mi import _lib
    seqs = dict(APART_SEQS, n=4, blocks=2048)
    cache = dict(APART, k=1 << 33, v=1 << 34, heads=8)
    kw = dict(rows=1, heads=8, ld=1024, bs=1024, p=1 << 35, out=1 << 36, top=64 if fn == "attention" else 3)
    if fn == "attention" and at == "blocks":
        kw["blocks"] = 1 << 37
    need = _lib.lib.h3mi_kv_select_workspace(4, 1, 8, 2048) if fn == "select" else \
        _lib.lib.h3mi_kv_attention_workspace(4, 1, 8, 8, 128, 2048, 64 if "blocks" in kw else 0)
    assert need > 0
    where = {**cache, **seqs, **kw}[at]
    for work in (where, where - (need - 1) // 16 * 16):
        rc, m = _call(fn, cache, seqs, work=work, size=need, **kw)
        assert rc == 3 and "workspace overlaps" in m, (rc, m)


def test_tangents_are_refused():
    """As a gradient is: a dual tensor's tangent would be dropped.  Its primal and a dual of a level that has ended pass on."""
    import torch
    from torch.autograd import forward_ad as fwd

    import h3mi
    c = h3mi.kv_cache(2, 2, 64, device="cpu")
    t, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)

    def calls(y):
        return (lambda: h3mi.kv_write_(c, y, x, t, lens), lambda: h3mi.kv_write_(c, x, y, t, lens), lambda: h3mi.kv_select(y, c, t, lens, 1),
                lambda: h3mi.kv_attention(y, c, t, lens))

    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for f in calls(dual):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                f()
        for f in calls(fwd.unpack_dual(dual).primal):
            with pytest.raises(ValueError, match="GPU"):
                f()
    for f in calls(dual):
        with pytest.raises(ValueError, match="GPU"):
            f()
