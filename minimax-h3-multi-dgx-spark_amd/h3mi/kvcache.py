"""Keys and values held in 8 bits, and attention over them (HIP, gfx950).

No counterpart in the reference, which computes its attention in the host program
(comfyui_nodes/minimax-h3-sp/minimax_sp/sp_forward.py:276-318).  Keys and values
that outlive a call (the finished chunks' of a long clip, the tokens before a step's,
a prompt's or reference frames' whose own rows attend to nothing that changes) stay in
a KVCache, at half of bf16's size.  Rows of one bidirectional sequence change with
every denoising step, its text rows among them: their keys are written anew for each.

  kv_cache(pages, heads, dim)                          an empty pool of pages of 64 tokens
  kv_write_(cache, k, v, tables, lens)                 quantize new tokens into it
  kv_read(cache, tables, lens, length)                 tokens back as bf16
  kv_attention(q, cache, tables, lens, causal)         attention over all of it
  kv_select(q, cache, tables, lens, top, causal)       the blocks worth attending to,
  kv_attention(..., blocks=...)                        and attention over those alone

tables int32 [n, blocks] gives the page of each block of 64 tokens of n sequences and
lens int32 [n] their tokens, those of the call among them; counts int32 [n] says how
many of a call's rows a sequence has (the rest is padding), and row r of sequence i is
token lens[i] - counts[i] + r.  All stay on the GPU and are read there, so that a
captured call follows them.  How a call's work is split goes by the tables' width, so
tables no wider than the sequences need serve best.  Rows are [n, rows, heads, dim] bf16
with contiguous heads, 16-byte aligned, with token and sequence strides that are multiples
of 8 elements and no shorter than a row: views of a projection's output serve, as after
rms_rope_split_half_.
"""
import ctypes
import typing

import torch
from torch.autograd import forward_ad

from ._lib import KvCacheC, KvSeqsC, _fast, check, lib, ptr, same_gpu, stream_of

KV_BLOCK = 64   # tokens of a block, one scale per block and head, and of a page
KV_TILE = 128   # query rows that share a selection


class KVCache(typing.NamedTuple):
    """A pool of pages, and their scales and sums."""
    k: torch.Tensor        # int8 [pages, heads, 64, dim]
    v: torch.Tensor        # int8 [pages, heads, dim, 64]: each block's values transposed
    k_scale: torch.Tensor  # fp32 [pages, heads]
    v_scale: torch.Tensor  # fp32 [pages, heads]
    k_sum: torch.Tensor    # int16 [pages, heads, dim]: sum of the block's 8-bit keys


def kv_cache(pages, heads, dim, device="cuda"):
    """An empty KVCache (zeros)."""
    if dim not in (64, 128, 256):
        raise ValueError("dim must be 64, 128 or 256")
    z = lambda *s, t: torch.zeros(*s, dtype=t, device=device)  # noqa: E731
    return KVCache(z(pages, heads, KV_BLOCK, dim, t=torch.int8), z(pages, heads, dim, KV_BLOCK, t=torch.int8),
                   z(pages, heads, t=torch.float32), z(pages, heads, t=torch.float32), z(pages, heads, dim, t=torch.int16))


# The functions below first offer the call to native code, which takes it in the
# plain form (csrc/fastcall.cpp) or returns None; the checks here then decide every
# other form.


def _cache(c):
    k = c.k
    if k.dim() != 4 or k.shape[2] != KV_BLOCK or k.dtype != torch.int8:
        raise ValueError(f"cache.k must be int8 [pages, heads, {KV_BLOCK}, dim]")
    pages, heads, _, dim = k.shape
    for name, shape, dtype in (("v", (pages, heads, dim, KV_BLOCK), torch.int8), ("k_scale", (pages, heads), torch.float32),
                               ("v_scale", (pages, heads), torch.float32), ("k_sum", (pages, heads, dim), torch.int16)):
        t = getattr(c, name)
        if t.shape != shape or t.dtype != dtype:
            raise ValueError(f"cache.{name} must be {dtype} {list(shape)}")
    if not all(t.is_contiguous() for t in c):
        raise ValueError("the cache's tensors must be contiguous")
    same_gpu(k, **{name: t for name, t in zip(c._fields[1:], c[1:])})
    return KvCacheC(*(t.data_ptr() for t in c), pages, heads, dim)


def _ints(t, shape, name):
    if t is not None and (t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}")


def _seqs(c, tables, lens, counts):
    if tables.dim() != 2:
        raise ValueError("tables must be [n, blocks]")
    n, blocks = tables.shape
    _ints(tables, (n, blocks), "tables")
    _ints(lens, (n,), "lens")
    _ints(counts, (n,), "counts")
    same_gpu(c.k, tables=tables, lens=lens, counts=counts)
    return KvSeqsC(tables.data_ptr(), lens.data_ptr(), None if counts is None else counts.data_ptr(), n, blocks)


def _rows(t, c, n, name, heads=None):
    """(rows, token stride, sequence stride) of [n, rows, heads, dim]."""
    if t.dtype != torch.bfloat16 or t.dim() != 4:
        raise ValueError(f"{name} must be bfloat16 [n, rows, heads, dim]")
    _, rows, h, d = t.shape
    if t.shape[0] != n or d != c.k.shape[3] or (heads is not None and h != heads):
        raise ValueError(f"{name} must be [{n}, rows, {'heads' if heads is None else heads}, {c.k.shape[3]}]")
    if t.numel() and (t.stride(3) != 1 or (h > 1 and t.stride(2) != d)):
        raise ValueError(f"{name}: heads must be contiguous (strides [*, *, dim, 1])")
    same_gpu(c.k, **{name: t})
    return rows, t.stride(1) if rows > 1 else h * d, t.stride(0) if n > 1 else rows * h * d


def _no_grad(*ts):
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError("attention over an 8-bit cache has no gradient: call it under torch.no_grad()")
    if any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError("attention over an 8-bit cache has no forward-mode gradient: call it with the primal tensors")


def kv_write_(cache, k, v, tables, lens, counts=None):
    """Quantizes k and v, the last counts[i] tokens of each sequence, into the cache's pages; returns the cache.

    A block's scale is max|x| / 127 of its first write.  A later write of tokens that do not fit doubles it as often
    as they need and halves the block's older 8-bit values as often, so that an error stays within one step.  A NaN or
    an infinity makes its block read back as NaN until the block's first token is written again.  The pages that a call
    writes have to be distinct."""
    done = _fast.kv_write_(cache, k, v, tables, lens, counts)
    if done is not None:
        return done
    _no_grad(k, v)
    c = _cache(cache)
    s = _seqs(cache, tables, lens, counts)
    rows, ldk, bsk = _rows(k, cache, s.n, "k", c.heads)
    rv, ldv, bsv = _rows(v, cache, s.n, "v", c.heads)
    if rv != rows:
        raise ValueError("k and v must have the same number of rows")
    with torch.cuda.device(k.device):
        check(lib.h3mi_kv_write_i8(ptr(k), ptr(v), rows, ldk, bsk, ldv, bsv, ctypes.byref(c), ctypes.byref(s), stream_of(k)))
    return cache


def kv_read(cache, tables, lens, length, starts=None):
    """(k, v) bf16 [n, length, heads, dim]: tokens starts[i] (default 0) on of each sequence, zeros where it has none."""
    got = _fast.kv_read(cache, tables, lens, length, starts)
    if got is not None:
        return got
    c = _cache(cache)
    s = _seqs(cache, tables, lens, None)
    _ints(starts, (s.n,), "starts")
    same_gpu(cache.k, starts=starts)
    length = int(length)
    if length < 0:
        raise ValueError("length must not be negative")
    k = torch.empty((s.n, length, c.heads, c.dim), dtype=torch.bfloat16, device=cache.k.device)
    v = torch.empty_like(k)
    with torch.cuda.device(k.device):
        check(lib.h3mi_kv_read_bf16(ptr(k), ptr(v), ptr(starts), length, ctypes.byref(c), ctypes.byref(s), stream_of(k)))
    return k, v


def kv_select(q, cache, tables, lens, top, causal=False, counts=None):
    """int32 [n, ceil(rows / 128), kv heads, top]: the blocks that each tile of 128 query rows takes for each kv head,
    ascending, -1 behind the last.

    A block's score is the product of its mean key with the mean of the tile's queries (of all heads that share the kv
    head), formed from 8-bit keys and 11-bit queries in whole numbers.  With causal, the blocks of the tile's own tokens
    are taken first and later ones never.  Equal scores go to the lowest block: of a tile with a NaN or an infinity in any
    of its queries all scores are equal."""
    out = _fast.kv_select(q, cache, tables, lens, top, causal, counts)
    if out is not None:
        return out
    _no_grad(q)
    c = _cache(cache)
    s = _seqs(cache, tables, lens, counts)
    rows, ld, bs = _rows(q, cache, s.n, "q")
    top = int(top)
    out = torch.empty((s.n, -(-rows // KV_TILE), c.heads, max(top, 0)), dtype=torch.int32, device=q.device)
    with torch.cuda.device(q.device):
        need = lib.h3mi_kv_select_workspace(s.n, rows, c.heads, s.blocks)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        check(lib.h3mi_kv_select(ptr(q), rows, q.shape[2], ld, bs, ctypes.byref(c), ctypes.byref(s), top, int(bool(causal)),
                                 ptr(out), ptr(work), need, stream_of(q)))
    return out


def kv_attention(q, cache, tables, lens, causal=False, counts=None, scale=None, blocks=None):
    """softmax(scale q k^T) v over each sequence's tokens -> bf16 [n, rows, heads, dim].

    q bf16 [n, rows, heads, dim]; query head h reads kv head h / (heads / kv heads); scale defaults to dim ** -0.5.
    causal: a row sees tokens up to its own.  blocks (from kv_select, or any distinct ones in its shape): a row sees the
    tokens of its tile's blocks alone.  Rows that see no token, and padding rows, are 0."""
    out = _fast.kv_attention(q, cache, tables, lens, causal, counts, scale, blocks)
    if out is not None:
        return out
    _no_grad(q)
    c = _cache(cache)
    s = _seqs(cache, tables, lens, counts)
    rows, ld, bs = _rows(q, cache, s.n, "q")
    heads, top = q.shape[2], 0
    if blocks is not None:
        top = blocks.shape[-1]
        _ints(blocks, (s.n, -(-rows // KV_TILE), c.heads, top), "blocks")
        if top < 1:  # an empty tensor has no address, which would say: all blocks
            raise ValueError("blocks must name at least one block a tile (-1: none)")
        same_gpu(q, blocks=blocks)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    with torch.cuda.device(q.device):
        need = lib.h3mi_kv_attention_workspace(s.n, rows, heads, c.heads, c.dim, s.blocks, top)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        check(lib.h3mi_kv_attention_bf16(ptr(q), rows, heads, ld, bs, ctypes.byref(c), ctypes.byref(s),
                                         float(c.dim ** -0.5 if scale is None else scale), int(bool(causal)), ptr(blocks), top,
                                         ptr(out), ptr(work), max(need, 0), stream_of(q)))
    return out
