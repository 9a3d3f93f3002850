"""Plain forms of the 8-bit key/value cache on the CPU: the writer in its own fp32 steps (its bytes are pinned), reading,
selection and attention in 64 bits."""
import math

import numpy as np
import torch

BLOCK, TILE = 64, 128


class Cache:
    """A cache as numpy arrays, values not transposed: k, v int8 [pages, heads, 64, dim]."""

    def __init__(self, pages, heads, dim, seed=None):
        self.k = np.zeros((pages, heads, BLOCK, dim), np.int8)
        self.v = np.zeros_like(self.k)
        self.ks = np.zeros((pages, heads), np.float32)
        self.vs = np.zeros_like(self.ks)
        if seed is not None:
            r = np.random.default_rng(seed)
            self.k[:] = r.integers(-127, 128, self.k.shape)
            self.v[:] = r.integers(-127, 128, self.v.shape)
            self.ks[:] = r.uniform(0.005, 0.03, self.ks.shape)
            self.vs[:] = r.uniform(0.005, 0.03, self.ks.shape)
        self.ksum = self.k.sum(2, dtype=np.int16)

    def to(self, device="cuda"):
        import h3mi
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)  # noqa: E731
        return h3mi.KVCache(t(self.k), t(self.v.swapaxes(2, 3)), t(self.ks), t(self.vs), t(self.ksum))

    def same(self, c):
        """The names of the tensors in which a KVCache differs from this one."""
        mine = {"k": self.k, "v": self.v.swapaxes(2, 3), "k_scale": self.ks, "v_scale": self.vs, "k_sum": self.ksum}
        return [n for n, a in mine.items() if not np.array_equal(a, getattr(c, n).cpu().numpy(), equal_nan=a.dtype == np.float32)]


def _grow(new, old, fresh):
    """(scale, power by which the old 8-bit values shrink, or None where they go) of one block and head."""
    with np.errstate(all="ignore"):
        a = np.float32(np.abs(new).max() if not np.isnan(new).any() else np.nan) * (np.float32(1) / np.float32(127))
        if fresh or old == 0:
            return a, None
        if not np.isfinite(old):
            return old, None
        r = a / old
    if not r <= 256:
        return a, None
    k = 0
    while np.float32(2.0 ** k) < r:
        k += 1
    return np.float32(np.ldexp(old, k)), k


def write(c, k, v, tables, lens, counts):
    """k, v float32 arrays [n, rows, heads, dim] of bf16 values."""
    for i in range(k.shape[0]):
        end, count = max(0, int(lens[i])), min(max(0, int(counts[i])), k.shape[1])
        start = end - count
        for b in range(max(start, 0) // BLOCK, -(-end // BLOCK)):
            lo, hi = max(start, b * BLOCK), min(end, (b + 1) * BLOCK)
            if b >= tables.shape[1] or lo >= hi or not 0 <= tables[i, b] < c.k.shape[0]:
                continue
            page, off = tables[i, b], lo - b * BLOCK
            for ints, scale, src in ((c.k, c.ks, k), (c.v, c.vs, v)):
                for h in range(k.shape[2]):
                    new = src[i, lo - start:hi - start, h]
                    s, fold = _grow(new, scale[page, h], start <= b * BLOCK)
                    tile = np.zeros((BLOCK, k.shape[3]), np.float32)
                    if s > 0 and np.isfinite(s):
                        if fold is not None:
                            tile[:off] = np.rint(ints[page, h, :off] * np.float32(2.0 ** -fold))
                        tile[off:off + hi - lo] = np.clip(np.rint(new / s), -127, 127)
                    ints[page, h], scale[page, h] = tile.astype(np.int8), s
            c.ksum[page] = c.k[page].sum(1, dtype=np.int16)


def tokens(c, table, end):
    """(k, v) float64 [end, heads, dim] of a sequence and which of its tokens are there."""
    heads, dim = c.k.shape[1], c.k.shape[3]
    k, v = np.zeros((end, heads, dim)), np.zeros((end, heads, dim))
    there = np.zeros(end, bool)
    for b in range(min(-(-end // BLOCK), len(table))):
        if not 0 <= table[b] < c.k.shape[0]:
            continue
        n = min(BLOCK, end - b * BLOCK)
        for out, ints, scale in ((k, c.k, c.ks), (v, c.v, c.vs)):
            with np.errstate(invalid="ignore"):
                tile = ints[table[b]].astype(np.float64) * scale[table[b]].astype(np.float64)[:, None, None]
            out[b * BLOCK:b * BLOCK + n] = tile[:, :n].swapaxes(0, 1)
        there[b * BLOCK:b * BLOCK + n] = True
    return k, v, there


def select(c, q, tables, lens, counts, top, causal):
    """q float64 [n, rows, heads, dim] -> int32 [n, tiles, kv heads, top]."""
    n, rows, heads, dim = q.shape
    kv = c.k.shape[1]
    g = heads // kv
    out = np.full((n, -(-rows // TILE), kv, top), -1, np.int32)
    for i in range(n):
        end, count = max(0, int(lens[i])), min(max(0, int(counts[i])), rows)
        size = min(end, tables.shape[1] * BLOCK)
        for t in range(out.shape[1]):
            live = min(count - t * TILE, TILE)
            if live <= 0:
                continue
            first = end - count + t * TILE
            last = first + live - 1
            seen = -(-size // BLOCK)
            if causal and last < size:
                seen = 0 if last < 0 else last // BLOCK + 1
            for h in range(kv):
                p = q[i, t * TILE:t * TILE + live, h * g:(h + 1) * g].sum((0, 1))
                m = np.abs(p).max()
                qi = np.rint(p * 1023.0 / m) if m > 0 and np.isfinite(m) else np.zeros(dim)
                order = []
                for b in range(seen):
                    page = tables[i, b]
                    if not 0 <= page < c.k.shape[0]:
                        continue
                    with np.errstate(all="ignore"):
                        s = np.float32(int((qi.astype(np.int64) * c.ksum[page, h]).sum())) * (
                            c.ks[page, h] / np.float32(min(BLOCK, size - b * BLOCK)))
                    own = causal and b >= max(first, 0) // BLOCK
                    rank = (2, 0.0) if own else (0, 0.0) if np.isnan(s) else (1, float(s))
                    order.append((-rank[0], -rank[1], b))
                got = sorted(b for _, _, b in sorted(order)[:top])
                out[i, t, h, :len(got)] = got
    return out


def attention(c, q, tables, lens, counts, causal, scale=None, blocks=None):
    """(out, weight of |v|, largest sum of |q k| scale) float64 [n, rows, heads, dim], the latter two for bounds of error."""
    n, rows, heads, dim = q.shape
    g = heads // c.k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3] + (1,))
    for i in range(n):
        end, count = max(0, int(lens[i])), min(max(0, int(counts[i])), rows)
        size = min(end, tables.shape[1] * BLOCK)
        k, v, there = tokens(c, tables[i], size)
        at = np.arange(size)
        for h in range(heads):
            kh, vh = torch.from_numpy(k[:, h // g].copy()), torch.from_numpy(v[:, h // g].copy())
            qh = torch.from_numpy(q[i, :count, h].copy())
            seen = np.broadcast_to(there, (count, size)).copy()
            if causal:
                seen &= at <= (end - count + np.arange(count))[:, None]
            if blocks is not None:
                for t in range(-(-count // TILE)):
                    took = np.zeros(max(tables.shape[1], 1), bool)
                    mine = blocks[i, t, h // g]
                    took[mine[(mine >= 0) & (mine < tables.shape[1])]] = True
                    seen[t * TILE:(t + 1) * TILE] &= took[at // BLOCK]
            if size == 0 or count == 0:
                continue
            seen = torch.from_numpy(seen)
            s = (qh @ kh.t() * scale).masked_fill(~seen, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
            p = p / torch.where(p.sum(1, keepdim=True) == 0, 1.0, p.sum(1, keepdim=True))
            p = torch.where(seen, p, 0.0)
            held = seen.any(0)
            vh = torch.where(held[:, None], vh, 0.0)  # tokens that no row sees have no part in a row
            out[i, :count, h] = (p @ vh).numpy()
            mag[i, :count, h] = (p @ vh.abs()).numpy()
            big = torch.where(seen, qh.abs() @ torch.where(held[:, None], kh, 0.0).abs().t(), 0.0)
            top[i, :count, h] = (big.amax(1, keepdim=True) * abs(scale)).numpy()
    return out, mag, top


def bound(out, mag, top, dim):
    """How far a correct result may be off: probabilities rounded to bf16 (half a step, 2^-8 relative) and the result's own
    rounding; 32-bit scores, whose sums of dim products are off by at most (dim + 8) 2^-24 of the sum of magnitudes, which
    the exponential turns into as much relative to both sums; and as many 32-bit roundings of the sums."""
    half = torch.finfo(torch.bfloat16).eps / 2
    return half * (mag * (1 + half) + np.abs(out)) * (1 + 1e-3) + 2 * mag * ((dim + 8) * 2.0 ** -24 * (top + 4)) + 1e-30
