"""Captured calls of the 8-bit cache against eager ones: the kernels with the most LDS, the ones with parts, and selection over
the longest tables, replayed between eager work on the same and on another stream, with lengths and queries that change."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _setup(n, rows, heads, kv, dim, blocks, seed):
    import h3mi
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = 50
    c = h3mi.KVCache(torch.randint(-127, 128, (pages, kv, 64, dim), generator=g, device=DEV, dtype=torch.int8),
                     torch.randint(-127, 128, (pages, kv, dim, 64), generator=g, device=DEV, dtype=torch.int8),
                     torch.rand(pages, kv, generator=g, device=DEV) * 0.02 + 0.005, torch.rand(pages, kv, generator=g, device=DEV) * 0.02 + 0.005,
                     torch.randint(-500, 500, (pages, kv, dim), generator=g, device=DEV, dtype=torch.int16))
    q = torch.randn(n, rows, heads, dim, generator=g, device=DEV).to(torch.bfloat16)
    tables = torch.randint(0, pages, (n, blocks), generator=g, device=DEV, dtype=torch.int32)
    return g, c, q, tables, torch.full((n,), blocks * 64, dtype=torch.int32, device=DEV)


def _replays(call, change):
    """Every replay gives what the eager call gives; an eager call on another stream runs beside it."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(5):
        change(r)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = call()
        want = call()
        torch.cuda.synchronize()
        for a, b, s in zip(out, want, beside):
            assert torch.equal(a, b) and torch.equal(s, b), r


@pytest.mark.parametrize("n,rows,heads,kv,dim,blocks", [
    (1, 1, 8, 2, 256, 40), (2, 200, 30, 6, 256, 30), (2, 300, 2, 2, 256, 7), (3, 1030, 18, 18, 128, 140), (2, 150, 2, 2, 64, 64),
])
def test_attention(n, rows, heads, kv, dim, blocks):
    import h3mi
    g, c, q, tables, lens = _setup(n, rows, heads, kv, dim, blocks, seed=rows)

    def change(r):
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        lens.copy_(torch.randint(0, blocks * 64 + 1, (n,), generator=g, device=DEV))

    _replays(lambda: [h3mi.kv_attention(q, c, tables, lens, causal=True)], change)


@pytest.mark.parametrize("rows,dim,blocks", [(1, 128, 32768), (1, 256, 32768), (1, 64, 700), (200, 256, 900), (20000, 64, 16000)])
def test_selection(rows, dim, blocks):
    import h3mi
    g, c, q, tables, lens = _setup(2, rows, 2, 2, dim, blocks, seed=blocks)

    def change(r):
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        lens.copy_(torch.randint(0, blocks * 64 + 1, (2,), generator=g, device=DEV))

    _replays(lambda: [h3mi.kv_select(q, c, tables, lens, 77, causal=True)], change)


def test_write_and_read():
    """Each replay writes the next tokens of sequences that grow unevenly; an eager cache is written beside."""
    import h3mi
    g = torch.Generator(device=DEV).manual_seed(3)
    n, rows, heads, dim, blocks = 3, 50, 4, 256, 8
    caches = [h3mi.kv_cache(n * blocks, heads, dim) for _ in range(2)]
    k, v = (torch.empty(n, rows, heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    tables = torch.randperm(n * blocks, generator=g, device=DEV).reshape(n, blocks).to(torch.int32)
    lens, counts = (torch.zeros(n, dtype=torch.int32, device=DEV) for _ in range(2))

    def call(c):
        h3mi.kv_write_(c, k, v, tables, lens, counts=counts)
        return [*h3mi.kv_read(c, tables, lens, 130, starts=lens - 70), *c]

    call(caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(caches[0])
    for r in range(6):
        counts.copy_(torch.randint(0, rows + 1, (n,), generator=g, device=DEV))
        lens.add_(counts)
        k.copy_(torch.randn(k.shape, generator=g, device=DEV) * 1.5 ** r)
        v.copy_(torch.randn(v.shape, generator=g, device=DEV))
        want = call(caches[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r
