"""Pages for the tokens of many requests, handed out on the GPU (HIP, gfx950).

No counterpart in the reference, which keeps no keys and values beyond a call.  A pool
holds the free pages of a cache; a step asks it for room for its new tokens and gets,
beside the tables and lengths that kv_write_ and kv_attention take, the position and the
slot of every row, without the host knowing a length:

  pool = kv_pool(pages)
  granted, positions, slots = kv_extend_(pool, tables, lens, rows, counts)
  rotary_(q, k, positions, freqs)
  kv_write_(cache, k, v, tables, lens, counts=granted)
  kv_attention(q, cache, tables, lens, causal=True, counts=granted)
  kv_release_(pool, tables, lens, keep)

tables int32 [n, blocks] and lens int32 [n] are changed in place, as the pool is, so that a
captured step follows them.  Calls on one pool have to run in order.
"""
import ctypes
import typing

import torch

from ._lib import KvPoolC, _fast, check, lib, ptr, same_gpu, stream_of, wrote
from .kvcache import _ints


class KVPool(typing.NamedTuple):
    """Free pages: free[0 .. count - 1], taken from the end."""
    free: torch.Tensor   # int32 [pages]
    count: torch.Tensor  # int32 [1]


def kv_pool(pages, device="cuda"):
    """A KVPool with pages 0 .. pages - 1 free, the first taken first."""
    pages = int(pages)
    if not 0 <= pages <= 1 << 30:
        raise ValueError("pages must be 0 to 2^30")
    return KVPool(torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device), torch.full((1,), pages, dtype=torch.int32, device=device))


def _pool(pool, tables, lens):
    if type(pool) is tuple and len(pool) == 2:  # as the native calls do
        pool = KVPool(*pool)
    if tables.dim() != 2:
        raise ValueError("tables must be [n, blocks]")
    n, blocks = tables.shape
    for t, shape, name in ((pool.free, (pool.free.numel(),), "pool.free"), (pool.count, (1,), "pool.count"),
                           (tables, (n, blocks), "tables"), (lens, (n,), "lens")):
        _ints(t, shape, name)
    same_gpu(tables, **{"pool.free": pool.free, "pool.count": pool.count, "lens": lens})
    return KvPoolC(pool.free.data_ptr(), pool.count.data_ptr(), pool.free.numel()), n, blocks


def kv_extend_(pool, tables, lens, rows, counts=None):
    """Room for counts[i] (default rows) more tokens of each sequence -> (granted, positions, slots).

    granted int32 [n]: counts[i] (taken as 0 to rows), or 0 where the pool has too few pages for the sequence and those
    before it, or its table too few blocks: nothing of such a sequence changes, and later ones are served that need no
    page.  tables gets the new blocks' pages, lens grows by granted.
    positions int32 [n, rows]: the token that each row is, -1 behind a sequence's own; slots int64 [n, rows]: 64 times its
    page and its place there, or -1."""
    rows = int(rows)
    got = _fast.kv_extend_(pool, tables, lens, rows, counts)
    if got is not None:
        return got
    p, n, blocks = _pool(pool, tables, lens)
    if rows < 0:
        raise ValueError("rows must not be negative")
    _ints(counts, (n,), "counts")
    same_gpu(tables, counts=counts)
    granted = torch.empty(n, dtype=torch.int32, device=tables.device)
    positions = torch.empty((n, rows), dtype=torch.int32, device=tables.device)
    slots = torch.empty((n, rows), dtype=torch.int64, device=tables.device)
    with torch.cuda.device(tables.device):
        check(lib.h3mi_kv_extend(ctypes.byref(p), ptr(tables), ptr(lens), ptr(counts), n, blocks, rows, ptr(granted), ptr(positions),
                                 ptr(slots), stream_of(tables)))
    wrote(*pool, tables, lens)
    return granted, positions, slots


def kv_release_(pool, tables, lens, keep=None):
    """Drops all but the first keep[i] (int32 [n]; default none) tokens of each sequence; returns the pool.

    The pages of blocks wholly behind go back to the pool, their entries in tables become -1 and lens what is kept (a
    sequence shorter than keep[i] stays as it is).  A page that two released tables hold goes back twice, and later to two
    sequences: of sequences that share pages one is their owner, released last, and the others' entries for them are set to
    -1 before, which a release passes over."""
    done = _fast.kv_release_(pool, tables, lens, keep)
    if done is not None:
        return done
    p, n, blocks = _pool(pool, tables, lens)
    _ints(keep, (n,), "keep")
    same_gpu(tables, keep=keep)
    with torch.cuda.device(tables.device):
        check(lib.h3mi_kv_release(ctypes.byref(p), ptr(tables), ptr(lens), ptr(keep), n, blocks, stream_of(tables)))
    wrote(*pool, tables, lens)
    return pool
