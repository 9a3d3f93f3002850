"""The native calls of rotary positions, of the page pool and of the 4-bit cache give the bytes of the checked path, leave every
other form of a call to it, and raise what it raises."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Never:
    def __getattr__(self, name):
        return lambda *a: None


def _outcome(f):
    import h3mi
    try:
        return f(h3mi)
    except Exception as e:  # noqa: BLE001
        return type(e)


def _both(monkeypatch, f):
    import h3mi
    fast = _outcome(f)
    with monkeypatch.context() as m:
        for module in (h3mi.kvcache, h3mi.kvpages, h3mi.rope):
            m.setattr(module, "_fast", _Never())
        return fast, _outcome(f)


def _same(a, b):
    if isinstance(a, type) or isinstance(b, type):
        return a is b
    a, b = (a,) if torch.is_tensor(a) else a, (b,) if torch.is_tensor(b) else b
    return len(a) == len(b) and all((x is None and y is None) or (
        x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
        and torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))) for x, y in zip(a, b))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _check(monkeypatch, forms, refused=()):
    """Every form the same by both paths; of those that run, a result; of `refused`, an error."""
    for n, f in enumerate(forms):
        a, b = _both(monkeypatch, f)
        assert not isinstance(a, type) and _same(a, b), (n, *(x if isinstance(x, type) else "ran" for x in (a, b)))
    for n, f in enumerate(refused):
        a, b = _both(monkeypatch, f)
        assert isinstance(a, type) and a is b, (n, *(x if isinstance(x, type) else "ran" for x in (a, b)))


def test_rotary(monkeypatch):
    g = torch.Generator(device=DEV).manual_seed(2)
    n, rows, hq, hk, dim = 2, 9, 3, 2, 64
    qkv = torch.randn(n, rows, hq + 2 * hk, dim, generator=g, device=DEV).to(torch.bfloat16)
    positions = torch.randint(-1, 5000, (n, rows), generator=g, device=DEV, dtype=torch.int32)
    import h3mi
    freqs, amp = h3mi.rotary_frequencies(dim, scaling="yarn", factor=4.0)
    half, pairs = freqs[:16].contiguous(), freqs[:31].contiguous()

    def place(f, **kw):
        """In place on views of a copy: all of it."""
        def call(h):
            x = qkv.clone()
            q, k = x[:, :, :hq], x[:, :, hq:hq + hk] if kw.get("two", True) else None
            got = h.rotary_(q, k, positions, f, **{a: b for a, b in kw.items() if a != "two"})
            assert got[0] is q and got[1] is k
            return x
        return call

    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    turn = lambda *a, **kw: lambda h: h.rotary(*a, **kw)  # noqa: E731
    forms = [place(f, **kw) for f in (freqs, half, pairs) for kw in ({}, dict(two=False), dict(interleaved=True), dict(inverse=True, amplitude=amp),
                                                                    dict(interleaved=True, inverse=True, amplitude=2, two=False))]
    forms += [turn(q, k, positions, f, i, j, amp) for f in (freqs, half, pairs) for i in (False, True) for j in (False, True)]
    forms += [turn(q, None, positions, half), turn(q.contiguous(), k.contiguous(), positions, freqs), turn(q, k, positions, freqs, 1, 0, 1),
              turn(q, k, positions, freqs, amplitude=torch.tensor(1.5)), turn(q[:1, :1], k[:1, :1], positions[:1, :1].contiguous(), freqs),
              turn(q[:, :0], k[:, :0], positions[:, :0].contiguous(), freqs), turn(q[:0], None, positions[:0], freqs),
              turn(q.transpose(0, 1), k.transpose(0, 1), positions.t().contiguous(), freqs),
              turn(torch.nn.Parameter(q.clone(), requires_grad=False), k, positions, freqs)]
    grad = q.clone().requires_grad_()
    refused = [turn(grad, k, positions, freqs), turn(q, k.clone().requires_grad_(), positions, freqs), turn(q.float(), k, positions, freqs),
               turn(q, k[..., :32], positions, freqs), turn(q, k[:1], positions, freqs), turn(q[0], None, positions, freqs),
               turn(q, k, positions.long(), freqs), turn(q, k, positions[:, ::2], freqs), turn(q, k, positions[0], freqs), turn(q, k, positions, freqs.float()),
               turn(q, k, positions, freqs[::2]), turn(q, k, positions.cpu(), freqs), turn(q, k, positions, freqs.cpu()), turn(q.cpu(), k, positions, freqs),
               turn(q, k, positions, freqs[:0]), turn(q, k, positions, freqs, amplitude=float("nan")), turn(q[..., :60], None, positions, freqs),
               turn(q[:, :, :0], k, positions, freqs), turn(q, k[:, :, :0], positions, freqs), turn(q.transpose(2, 3), None, positions, freqs),
               turn(q[:, :1].expand(-1, rows, -1, -1), None, positions, freqs), turn(q, k, positions, torch.cat([freqs, freqs])),
               lambda h: h.rotary_(q, q, positions, freqs), lambda h: h.rotary_(q, q[:, :, 1:], positions, freqs)]
    _check(monkeypatch, forms, refused)
    with torch.no_grad():
        _check(monkeypatch, [turn(grad, k, positions, freqs)])


def test_pages(monkeypatch):
    def state(h):
        pool = h.kv_pool(12)
        tables, lens = torch.full((4, 5), -1, dtype=torch.int32, device=DEV), _i32([0, 0, 0, 0])
        h.kv_extend_(pool, tables, lens, 70, _i32([70, 3, 64, 0]))
        return pool, tables, lens

    def extend(*a, plain=False, **kw):
        def call(h):
            pool, tables, lens = state(h)
            got = h.kv_extend_(tuple(pool) if plain else pool, tables, lens, *a, **kw)
            return (*got, *pool, tables, lens)
        return call

    def release(*a, plain=False, **kw):
        def call(h):
            pool, tables, lens = state(h)
            p = tuple(pool) if plain else pool
            assert h.kv_release_(p, tables, lens, *a, **kw) is p
            return (*pool, tables, lens)
        return call

    counts = _i32([1, 100, 0, 65])
    _check(monkeypatch, [
        extend(1), extend(3, counts), extend(130, counts=counts), extend(5000), extend(0), extend(0, counts), extend(torch.tensor(7)), extend(True),
        extend(3, counts, plain=True), extend(100), release(), release(None), release(counts), release(keep=_i32([64, -5, 2 ** 31 - 1, 1])),
        release(counts, plain=True)],
        [extend(-1), extend(3, counts[:2]), extend(3, counts.long()), extend(3, counts.cpu()), extend(3, counts[None]), release(counts[:3]),
         release(counts.float()), release(counts.cpu()), lambda h: h.kv_extend_(h.kv_pool(3), _i32([[0, 0]]).t(), _i32([0]), 1),
         lambda h: h.kv_extend_(h.kv_pool(3), _i32([[0, 0]]), _i32([0, 0]), 1), lambda h: h.kv_extend_(h.kv_pool(3, device="cpu"), _i32([[0, 0]]), _i32([0]), 1),
         lambda h: h.kv_extend_(h.kv_pool(3)[:1], _i32([[0, 0]]), _i32([0]), 1)])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_cache(monkeypatch, dim):
    import h3mi
    g = torch.Generator(device=DEV).manual_seed(dim)
    n, rows, heads, kv = 2, 40, 4, 2
    qkv = torch.randn(n, rows, heads + 2 * kv, dim, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = qkv[:, :, :heads], qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:]
    tables, lens, counts = _i32([[3, 0], [1, 2]]), _i32([100, 41]), _i32([40, 7])
    full = h3mi.kv_write_(h3mi.kv_cache(5, kv, dim, bits=4), k, v, tables, lens)
    full8 = h3mi.kv_write_(h3mi.kv_cache(5, kv, dim), k, v, tables, lens)
    lists = _i32([0, 1]).repeat(n, 1, kv, 1)

    def write(*a, plain=False, bits=4, **kw):
        def call(h):
            cache = h.KVCache4(*(t.clone() for t in full)) if bits == 4 else h.KVCache(*(t.clone() for t in full8))
            c = tuple(cache) if plain else cache
            assert h.kv_write_(c, *a, **kw) is c
            return tuple(cache)
        return call

    attend = lambda *a, **kw: lambda h: h.kv_attention(*a, **kw)  # noqa: E731
    read = lambda *a, **kw: lambda h: h.kv_read(*a, **kw)  # noqa: E731
    forms = [
        write(k, v, tables, lens), write(k, v, tables, lens, counts=counts), write(k.contiguous(), v, tables, lens, counts), write(k[:, :0], v[:, :0], tables, lens),
        write(torch.nn.Parameter(k.clone(), requires_grad=False), v, tables, lens), write(k, v, tables, lens, plain=True), write(k, v, tables, lens, plain=True, bits=8),
        read(full, tables, lens, 70), read(full, tables, lens, 70, starts=counts), read(full, tables, lens, torch.tensor(70)), read(full, tables, lens, True),
        read(full, tables, lens, 0), read(full, tables[:, :1].contiguous(), lens, 70), read(tuple(full), tables, lens, 70), read(tuple(full8), tables, lens, 70),
        attend(q, full, tables, lens), attend(q, full, tables, lens, causal=True, counts=counts), attend(q[:, :1], full, tables, lens), attend(q, full, tables, lens, scale=0.3),
        attend(q, full, tables, lens, scale=torch.tensor(0.3)), attend(q, full, tables, lens, blocks=lists), attend(q, full, tables, lens, blocks=lists[..., :1].contiguous()),
        attend(q[:, :0], full, tables, lens), attend(q, tuple(full), tables, lens, True), attend(q, tuple(full8), tables, lens, True),
        lambda h: h.kv_select(q, tuple(full8), tables, lens, 1)]
    refused = [
        write(k, v[:, :3], tables, lens), write(k.float(), v, tables, lens), write(k, v, tables.long(), lens), write(k, v, tables, lens.cpu()),
        write(k.transpose(1, 2), v.transpose(1, 2), tables, lens), write(k.clone().requires_grad_(), v, tables, lens), read(full, tables, lens, -1),
        read(tuple(full)[:3], tables, lens, 3), read(full._replace(v=full.k.float()), tables, lens, 3), read(full._replace(k_scale=full.v), tables, lens, 3),
        read(full, tables[:, :1], lens, 70), attend(q, full, tables, lens, blocks=lists.long()), attend(q, full, tables, lens, blocks=lists[..., :0]),
        attend(q, full, tables, lens, scale=float("nan")), attend(q.clone().requires_grad_(), full, tables, lens), attend(q.cpu(), full, tables, lens),
        attend(q[..., :32], full, tables, lens), attend(q[:1], full, tables, lens), attend(q[:, :, :3], full, tables, lens),
        lambda h: h.kv_select(q, full, tables, lens, 1), lambda h: h.kv_select(q, tuple(full), tables, lens, 1), lambda h: h.kv_read(None, tables, lens, 1)]
    _check(monkeypatch, forms, refused)


def test_native_path_is_taken():
    import h3mi
    from h3mi._lib import _fast
    cache, pool = h3mi.kv_cache(2, 2, 64, bits=4), h3mi.kv_pool(2)
    t, lens = torch.full((1, 1), -1, dtype=torch.int32, device=DEV), _i32([0])
    freqs, _ = h3mi.rotary_frequencies(64)
    x = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    got = _fast.kv_extend_(pool, t, lens, 1, None)
    assert got is not None and _fast.kv_extend_(pool, t, lens, 1, _i32([0])) is not None
    for inside in (False, True):
        assert _fast.rotary(x, x.clone(), got[1], freqs, False, False, 1.0, inside) is not None
        assert _fast.rotary(x, None, got[1], freqs, True, True, 2, inside) is not None
    assert _fast.kv_write_(cache, x, x, t, lens, None) is cache and _fast.kv_write_(cache, x, x, t, lens, lens) is cache
    assert _fast.kv_read(cache, t, lens, 1, None) is not None and _fast.kv_read(cache, t, lens, 1, lens) is not None
    assert _fast.kv_attention(x, cache, t, lens, True, None, None, None) is not None
    assert _fast.kv_attention(x, cache, t, lens, False, None, None, _i32([[[[0], [0]]]])) is not None
    assert _fast.kv_release_(pool, t, lens, None) is pool and _fast.kv_release_(pool, t, lens, lens.clone()) is pool
    assert _fast.kv_select(x, cache, t, lens, 1, False, None) is None


def test_tangents_are_refused(monkeypatch):
    from torch.autograd import forward_ad as fwd

    import h3mi
    cache = h3mi.kv_cache(2, 2, 64, bits=4)
    t, lens, freqs = _i32([[0]]), _i32([1]), h3mi.rotary_frequencies(64)[0]
    x = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda h: h.rotary(dual, None, t, freqs), lambda h: h.rotary(x, dual, t, freqs), lambda h: h.rotary_(dual, None, t, freqs),
                  lambda h: h.kv_write_(cache, dual, x, t, lens), lambda h: h.kv_write_(cache, x, dual, t, lens), lambda h: h.kv_attention(dual, cache, t, lens)):
            assert _both(monkeypatch, f) == (RuntimeError, RuntimeError)
        a, b = _both(monkeypatch, lambda h: h.rotary(fwd.unpack_dual(dual).primal, None, t, freqs))
        assert not isinstance(a, type) and _same(a, b)
