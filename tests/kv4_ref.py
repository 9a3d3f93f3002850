"""Plain forms of the 4-bit key/value cache on the CPU: the writer's bytes from the values themselves, reading and (with
kv_ref's) attention in 64 bits."""
import types

import numpy as np
import torch

BLOCK, GROUP = 64, 32
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(x):
    """float64 array [..., dim] of bf16 values -> (bytes [..., dim / 2], codes [..., dim / 32])."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        top = np.abs(g).max(-1)
        bad = ~np.isfinite(top)
        # the least e with top <= 7 2^e, from the exponents that could be it
        e = np.full(top.shape, -125)
        for x2 in range(-125, 125):
            e = np.where(top > 7 * 2.0 ** x2, x2 + 1, e)
        y = np.where(bad[..., None], 0.0, g / 2.0 ** e[..., None].astype(np.float64))
    # nearest of the grid, between two as near the even place
    mid = (GRID[1:] + GRID[:-1]) / 2
    a = np.abs(y)
    place = np.searchsorted(mid, a, side="left")  # places whose upper neighbour's middle is below a
    tie = (place < 7) & (a == mid[np.minimum(place, 6)])
    place = np.where(tie & (place % 2 == 1), place + 1, place)
    nib = (place | (np.signbit(y) << 3)).astype(np.uint8).reshape(x.shape)
    return nib[..., 0::2] | nib[..., 1::2] << 4, np.where(bad, 255, e + 127).astype(np.uint8)


def values(q, codes):
    """bytes [..., dim / 2] and codes [..., dim / 32] -> float64 [..., dim]."""
    nib = np.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1)
    x = np.where(nib & 8, -1.0, 1.0) * GRID[nib & 7]
    f = np.where(codes >= 253, np.nan, 2.0 ** (codes.astype(np.float64) - 127))
    return x * np.repeat(f, GROUP, -1)


class Cache4:
    """A cache as numpy arrays."""

    def __init__(self, pages, heads, dim, seed=None):
        self.k = np.zeros((pages, heads, BLOCK, dim // 2), np.uint8)
        self.v = np.zeros_like(self.k)
        self.ks = np.zeros((pages, heads, dim // GROUP, BLOCK), np.uint8)
        self.vs = np.zeros_like(self.ks)
        if seed is not None:
            r = np.random.default_rng(seed)
            self.k[:] = r.integers(0, 256, self.k.shape)
            self.v[:] = r.integers(0, 256, self.v.shape)
            self.ks[:] = r.integers(123, 128, self.ks.shape)
            self.vs[:] = r.integers(120, 130, self.ks.shape)

    def to(self, device="cuda"):
        import h3mi
        return h3mi.KVCache4(*(torch.from_numpy(a.copy()).to(device) for a in (self.k, self.v, self.ks, self.vs)))

    def same(self, c):
        """The names of the tensors in which a KVCache4 differs from this one."""
        mine = {"k": self.k, "v": self.v, "k_scale": self.ks, "v_scale": self.vs}
        return [n for n, a in mine.items() if not np.array_equal(a, getattr(c, n).cpu().numpy())]

    def plain(self):
        """What kv_ref's reader and attention take: values in 64 bits, with scales of 1."""
        k, v = (values(q, s.swapaxes(2, 3)) for q, s in ((self.k, self.ks), (self.v, self.vs)))
        one = np.ones(k.shape[:2])
        return types.SimpleNamespace(k=k, v=v, ks=one, vs=one)


def write(c, k, v, tables, lens, counts):
    """k, v arrays [n, rows, heads, dim] of bf16 values."""
    for i in range(k.shape[0]):
        end, count = max(0, int(lens[i])), min(max(0, int(counts[i])), k.shape[1])
        for r in range(count):
            at = end - count + r
            if at < 0 or at // BLOCK >= tables.shape[1] or not 0 <= tables[i, at // BLOCK] < c.k.shape[0]:
                continue
            page, off = tables[i, at // BLOCK], at % BLOCK
            for q, s, x in ((c.k, c.ks, k), (c.v, c.vs, v)):
                q[page, :, off], s[page, :, :, off] = quantize(x[i, r].astype(np.float64))
