"""The C entry points of the 4-bit cache refuse bad arguments before touching a device: every pointer here is made up."""
import ctypes

import pytest

P = ctypes.c_void_p
# a cache, sequences and rows that do not overlap
BASE = dict(k=1 << 23, v=1 << 24, k_scale=1 << 25, v_scale=1 << 26, pages=10, heads=2, dim=128)
SEQS = dict(tables=1 << 28, lens=1 << 29, counts=1 << 30, n=2, blocks=5)
EVERY = ["write", "read", "attention"]


def _call(fn, cache=None, seqs=None, **kw):
    from h3mi import _lib
    c, s = _lib.KvCache4C(**{**BASE, **(cache or {})}), _lib.KvSeqsC(**{**SEQS, **(seqs or {})})
    c, s = ctypes.byref(c), ctypes.byref(s)
    a = dict(p=1 << 20, p2=1 << 21, rows=4, heads=4, ld=512, bs=2048, top=3, length=9, out=1 << 22, scale=1.0, starts=None, blocks=None,
             work=None, size=0)
    a.update(kw)
    L = _lib.lib
    if fn == "write":
        rc = L.h3mi_kv_write_mx4(P(a["p"]), P(a["p2"]), a["rows"], a["ld"], a["bs"], a["ld"], a["bs"], c, s, None)
    elif fn == "read":
        rc = L.h3mi_kv_read_mx4_bf16(P(a["p"]), P(a["p2"]), P(a["starts"]), a["length"], c, s, None)
    else:
        rc = L.h3mi_kv_attention_mx4_bf16(P(a["p"]), a["rows"], a["heads"], a["ld"], a["bs"], c, s, ctypes.c_float(a["scale"]), 0,
                                          P(a["blocks"]), a["top"], P(a["out"]), P(a["work"]), a["size"], None)
    return rc, L.h3mi_last_error().decode()


@pytest.mark.parametrize("fn", EVERY)
@pytest.mark.parametrize("cache,seqs,code,msg", [
    (dict(dim=96), None, 1, "dim=96"), (dict(dim=0), None, 1, "dim=0"), (dict(heads=0), None, 1, "heads=0"), (dict(pages=-1), None, 1, "pages=-1"),
    (dict(pages=1 << 31), None, 1, "pages"), (None, dict(n=-1), 1, "n=-1"), (None, dict(blocks=-1), 1, "blocks=-1"),
    (None, dict(blocks=1 << 25), 1, "blocks"), (dict(k=None), None, 1, "null cache"), (dict(v_scale=None), None, 1, "null cache"),
    (None, dict(lens=None), 1, "null tables or lens"), (None, dict(tables=None), 1, "null tables or lens"), (dict(v=(1 << 24) + 8), None, 2, "aligned"),
    (dict(k_scale=(1 << 25) + 4), None, 2, "aligned"), (None, dict(lens=6), 2, "4-byte"),
    (dict(v=1 << 23), None, 3, "the cache's tensors overlap"), (dict(v=(1 << 23) + 81904), None, 3, "the cache's tensors overlap"),
    (dict(k_scale=(1 << 26) + 5104), None, 3, "the cache's tensors overlap"), (dict(v_scale=(1 << 24) - 5104), None, 3, "the cache's tensors overlap"),
])
def test_cache_and_sequences(fn, cache, seqs, code, msg):
    rc, m = _call(fn, cache, seqs)
    assert rc == code and msg in m, (rc, m)


@pytest.mark.parametrize("fn", ["write", "attention"])
@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows=-1"), (dict(p=None), 1, "null"), (dict(p=(1 << 20) + 8), 2, "aligned"), (dict(ld=8), 1, "shorter"),
    (dict(bs=8), 1, "shorter"), (dict(ld=516), 2, "multiples of 8"), (dict(bs=2052), 2, "multiples of 8"), (dict(bs=-2048), 1, "shorter"),
])
def test_rows(fn, kw, code, msg):
    rc, m = _call(fn, **kw)
    assert rc == code and msg in m, (rc, m)


@pytest.mark.parametrize("fn,kw,code,msg", [
    ("read", dict(length=-1), 1, "length=-1"), ("read", dict(p=None), 1, "null k or v"), ("read", dict(p2=8), 2, "aligned"),
    ("read", dict(starts=2), 2, "aligned"), ("attention", dict(heads=5), 1, "multiple of the cache's"), ("attention", dict(out=None), 1, "null out"),
    ("attention", dict(out=8), 2, "aligned"), ("attention", dict(scale=float("nan")), 1, "scale"), ("attention", dict(out=1 << 20), 3, "overlaps"),
    ("attention", dict(out=(1 << 24) + 81904), 3, "overlaps"), ("attention", dict(out=(1 << 25) - 16), 3, "overlaps"),
    ("attention", dict(out=(1 << 26) + 5104), 3, "overlaps"), ("read", dict(p2=1 << 20), 3, "overlap"), ("read", dict(p=(1 << 26) + 16), 3, "overlap"),
    ("write", dict(p=1 << 24), 3, "overlap"), ("write", dict(p2=(1 << 25) + 5104), 3, "overlap"), ("attention", dict(blocks=4096, top=0), 1, "top=0"),
    ("read", dict(p=1 << 28), 3, "tables, lens"), ("read", dict(p2=1 << 31, starts=1 << 31), 3, "starts"), ("attention", dict(out=1 << 30), 3, "tables, lens"),
    ("attention", dict(out=(1 << 31) + 32, blocks=1 << 31), 3, "blocks"),
])
def test_each(fn, kw, code, msg):
    rc, m = _call(fn, **kw)
    assert rc == code and msg in m, (rc, m)


@pytest.mark.parametrize("seqs", [dict(tables=1 << 23), dict(tables=(1 << 25) - 36), dict(lens=1 << 26), dict(counts=(1 << 24) + 8)])
def test_written_cache_over_the_sequences(seqs):
    rc, m = _call("write", None, seqs)
    assert rc == 3 and "tables, lens or counts overlap the cache" in m, (rc, m)


def test_sizes_past_a_launch():
    big = dict(heads=65536, dim=256, k=1 << 40, v=1 << 50, k_scale=1 << 52, v_scale=1 << 53)
    assert _call("write", big, dict(blocks=(1 << 25) - 1), rows=1 << 30, ld=65536 * 256, bs=1 << 60)[0] == 1
    assert _call("read", big, dict(n=1 << 30), length=1 << 30)[0] == 1
    assert _call("attention", big, dict(n=1 << 20), rows=1 << 20, heads=65536, ld=65536 * 256, bs=1 << 60)[0] == 1


@pytest.mark.parametrize("fn", EVERY)
def test_nothing_to_do(fn):
    assert _call(fn, None, dict(n=0, lens=None, tables=None))[0] == 0
    assert _call(fn, rows=0, length=0, p=None, p2=None, out=None)[0] == 0


@pytest.mark.parametrize("fn", EVERY)
def test_null_structures(fn):
    from h3mi import _lib
    L = _lib.lib
    rc = {"write": lambda: L.h3mi_kv_write_mx4(P(4096), P(8192), 1, 256, 256, 256, 256, None, None, None),
          "read": lambda: L.h3mi_kv_read_mx4_bf16(P(4096), P(8192), None, 1, None, None, None),
          "attention": lambda: L.h3mi_kv_attention_mx4_bf16(P(4096), 1, 2, 256, 256, None, None, ctypes.c_float(1), 0, None, 0, P(8192), None, 0, None)}[fn]()
    assert rc == 1 and "null cache or sequences" in L.h3mi_last_error().decode()


def test_workspace():
    """A call that splits its work refuses less than h3mi_kv_attention_mx4_workspace asks for, and one over what it reads or writes."""
    from h3mi import _lib
    need = _lib.lib.h3mi_kv_attention_mx4_workspace(1, 1, 56, 56, 128, 309, 0)
    assert need > 0
    cache, seqs = dict(heads=56, k=1 << 40, v=1 << 41, k_scale=1 << 42, v_scale=1 << 43), dict(n=1, blocks=309)
    kw = dict(rows=1, heads=56, ld=7168, bs=7168, p=1 << 44, out=1 << 45)
    for work, size in ((None, need), (1 << 33, need - 1)):
        rc, m = _call("attention", cache, seqs, work=work, size=size, **kw)
        assert rc == 1 and "workspace" in m
    for at in (1 << 40, 1 << 41, 1 << 42, 1 << 43, 1 << 44, 1 << 45, 1 << 28, 1 << 29, 1 << 30):
        rc, m = _call("attention", cache, seqs, work=at, size=need, **kw)
        assert rc == 3 and "workspace overlaps" in m, (at, rc, m)


def test_cpu_tensors_are_refused():
    """The Python functions refuse host tensors before a kernel could see their addresses."""
    import torch

    import h3mi
    c = h3mi.kv_cache(2, 2, 64, device="cpu", bits=4)
    assert isinstance(c, h3mi.KVCache4) and c.k.shape == (2, 2, 64, 32) and c.v_scale.shape == (2, 2, 2, 64)
    t, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for f in (lambda: h3mi.kv_write_(c, x, x, t, lens), lambda: h3mi.kv_read(c, t, lens, 1), lambda: h3mi.kv_attention(x, c, t, lens)):
        with pytest.raises(ValueError, match="GPU"):
            f()
    with pytest.raises(ValueError, match="8-bit cache"):
        h3mi.kv_select(x, c, t, lens, 1)
    for bad, what in ((dict(dim=100), "dim"), (dict(dim=64, bits=5), "bits")):
        with pytest.raises(ValueError, match=what):
            h3mi.kv_cache(2, 2, device="cpu", **bad)
