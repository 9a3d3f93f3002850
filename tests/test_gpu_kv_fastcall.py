"""The native calls of the 8-bit cache give the bytes of the Python path, leave every other form of a call to it, and raise
what it raises."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class _Never:
    def __getattr__(self, name):
        return lambda *a: None


def _both(monkeypatch, f):
    import h3mi
    from h3mi import kvcache

    def outcome():
        try:
            return f(h3mi)
        except Exception as e:  # noqa: BLE001
            return type(e)

    fast = outcome()
    with monkeypatch.context() as m:
        m.setattr(kvcache, "_fast", _Never())
        return fast, outcome()


def _same(a, b):
    if isinstance(a, type) or isinstance(b, type):
        return a is b
    a, b = (a,) if torch.is_tensor(a) else a, (b,) if torch.is_tensor(b) else b
    return len(a) == len(b) and all(x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
                                    and torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
                                    for x, y in zip(a, b))


def test_forms(monkeypatch):
    import h3mi
    g = torch.Generator(device="cuda").manual_seed(1)
    n, rows, heads, kv, dim = 2, 40, 4, 2, 64
    qkv = torch.randn(n, rows, heads + 2 * kv, dim, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :, :heads], qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:]
    tables = torch.tensor([[3, 0], [1, 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([100, 41], dtype=torch.int32, device="cuda")
    counts = torch.tensor([40, 7], dtype=torch.int32, device="cuda")
    full = h3mi.kv_write_(h3mi.kv_cache(5, kv, dim), k, v, tables, lens)

    def write(*a, **kw):
        def f(h):
            cache = h.KVCache(*(t.clone() for t in full))
            assert h.kv_write_(cache, *a, **kw) is cache
            return tuple(cache)
        return f

    sel = h3mi.kv_select(q, full, tables, lens, 1)
    forms = [
        write(k, v, tables, lens), write(k, v, tables, lens, counts=counts), write(k.contiguous(), v, tables, lens, counts),
        write(k[:, :0], v[:, :0], tables, lens), write(k, v[:, :3], tables, lens), write(k.float(), v, tables, lens),
        write(k, v, tables.long(), lens), write(k, v, tables, lens.cpu()), write(k.transpose(1, 2), v.transpose(1, 2), tables, lens),
        write(torch.nn.Parameter(k.clone(), requires_grad=False), v, tables, lens), write(k.clone().requires_grad_(), v, tables, lens),
        lambda h: h.kv_read(full, tables, lens, 70), lambda h: h.kv_read(full, tables, lens, 70, starts=counts),
        lambda h: h.kv_read(full, tables, lens, torch.tensor(70)), lambda h: h.kv_read(full, tables, lens, True),
        lambda h: h.kv_read(full, tables, lens, -1), lambda h: h.kv_read(tuple(full)[:4], tables, lens, 3),
        lambda h: h.kv_read(full._replace(v=full.k.float()), tables, lens, 3), lambda h: h.kv_read(full, tables, lens, 0),
        lambda h: h.kv_read(full, tables[:, :1].contiguous(), lens, 70), lambda h: h.kv_read(full, tables[:, :1], lens, 70),
        lambda h: h.kv_select(q, full, tables, lens, 2), lambda h: h.kv_select(q, full, tables, lens, 2, True, counts),
        lambda h: h.kv_select(q, full, tables, lens, 0), lambda h: h.kv_select(q, full, tables, lens, 1 << 40),
        lambda h: h.kv_select(q, full, tables, lens, 1 << 70), lambda h: h.kv_select(q[:, :, :3], full, tables, lens, 2),
        lambda h: h.kv_select(q, full, tables, lens, 2, causal=1), lambda h: h.kv_select(q[:, :0], full, tables, lens, 2),
        lambda h: h.kv_attention(q, full, tables, lens), lambda h: h.kv_attention(q, full, tables, lens, causal=True, counts=counts),
        lambda h: h.kv_attention(q, full, tables, lens, scale=0.3), lambda h: h.kv_attention(q, full, tables, lens, scale=1),
        lambda h: h.kv_attention(q, full, tables, lens, scale=torch.tensor(0.3)), lambda h: h.kv_attention(q, full, tables, lens, blocks=sel),
        lambda h: h.kv_attention(q, full, tables, lens, blocks=sel.long()), lambda h: h.kv_attention(q, full, tables, lens, blocks=sel[..., :0]),
        lambda h: h.kv_attention(q, full, tables, lens, blocks=sel[:, :, :1]), lambda h: h.kv_attention(q[:, :0], full, tables, lens),
        lambda h: h.kv_attention(q, full, tables, lens, scale=float("nan")), lambda h: h.kv_attention(q.clone().requires_grad_(), full, tables, lens),
        lambda h: h.kv_attention(q.cpu(), full, tables, lens), lambda h: h.kv_attention(q[:, ::2], full, tables, lens),
        lambda h: h.kv_attention(q[..., :32], full, tables, lens), lambda h: h.kv_attention(q[:1], full, tables, lens),
    ]
    for n, f in enumerate(forms):
        a, b = _both(monkeypatch, f)
        assert _same(a, b), (n, a, b)


def test_native_path_is_taken():
    import h3mi
    from h3mi._lib import _fast
    cache = h3mi.kv_cache(2, 2, 64)
    t, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert _fast.kv_write_(cache, x, x, t, lens, None) is cache
    assert _fast.kv_read(cache, t, lens, 1, None) is not None
    assert _fast.kv_select(x, cache, t, lens, 1, False, None) is not None
    assert _fast.kv_attention(x, cache, t, lens, False, None, None, None) is not None
    assert _fast.kv_attention(x.requires_grad_(), cache, t, lens, False, None, None, None) is None


def test_tangents_are_left_to_the_python_path(monkeypatch):
    from torch.autograd import forward_ad as fwd

    import h3mi
    full = h3mi.kv_cache(2, 2, 64)
    t, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        forms = [lambda h: tuple(h.kv_write_(full, dual, x, t, lens)), lambda h: tuple(h.kv_write_(full, x, dual, t, lens)),
                 lambda h: h.kv_select(dual, full, t, lens, 1), lambda h: h.kv_attention(dual, full, t, lens)]
        for f in forms:
            assert _both(monkeypatch, f) == (RuntimeError, RuntimeError)
        a, b = _both(monkeypatch, lambda h: h.kv_attention(fwd.unpack_dual(dual).primal, full, t, lens))
        assert _same(a, b)
    a, b = _both(monkeypatch, lambda h: h.kv_attention(dual, full, t, lens))
    assert torch.is_tensor(a) and _same(a, b)
