"""Plain form of the page pool on the CPU: one sequence after the other."""
import numpy as np

BLOCK = 64


class Pool:
    """Tables, lengths and a stack of free pages as numpy arrays."""

    def __init__(self, free, count, tables, lens):
        self.free, self.count = np.array(free, np.int32), int(count)
        self.tables, self.lens = np.array(tables, np.int32), np.array(lens, np.int32)

    def to(self, device="cuda"):
        import torch

        import h3mi
        t = lambda a: torch.from_numpy(np.array(a, np.int32)).to(device)  # noqa: E731
        return h3mi.KVPool(t(self.free), t([self.count])), t(self.tables), t(self.lens)

    def same(self, pool, tables, lens):
        """The names of what differs from this."""
        mine = {"free": (self.free, pool.free), "count": ([self.count], pool.count), "tables": (self.tables, tables), "lens": (self.lens, lens)}
        return [n for n, (a, t) in mine.items() if not np.array_equal(a, t.cpu().numpy())]

    def _clip(self):
        self.count = min(max(self.count, 0), len(self.free))

    def extend(self, rows, counts=None):
        n, blocks = self.tables.shape
        self._clip()
        granted = np.zeros(n, np.int32)
        positions, slots = np.full((n, rows), -1, np.int32), np.full((n, rows), -1, np.int64)
        had, upto = self.count, 0
        for i in range(n):
            c = min(max(rows if counts is None else int(counts[i]), 0), rows)
            old = max(int(self.lens[i]), 0)
            self.lens[i] = old
            held = -(-old // BLOCK)
            if old + c > BLOCK * blocks:
                continue
            want = -(-(old + c) // BLOCK) - held
            upto += want
            if want and upto > had:
                continue
            for b in range(held, held + want):
                self.count -= 1
                self.tables[i, b] = self.free[self.count]
            granted[i] = c
            self.lens[i] = old + c
            for r in range(c):
                positions[i, r] = old + r
                page = int(self.tables[i, (old + r) // BLOCK])
                if 0 <= page < len(self.free):
                    slots[i, r] = page * BLOCK + (old + r) % BLOCK
        return granted, positions, slots

    def release(self, keep=None):
        n, blocks = self.tables.shape
        self._clip()
        for i in range(n):
            old = max(int(self.lens[i]), 0)
            left = min(max(0 if keep is None else int(keep[i]), 0), old)
            for b in range(-(-left // BLOCK), min(-(-old // BLOCK), blocks)):
                page = int(self.tables[i, b])
                self.tables[i, b] = -1
                if 0 <= page < len(self.free) and self.count < len(self.free):
                    self.free[self.count] = page
                    self.count += 1
            self.lens[i] = left
