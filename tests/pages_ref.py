"""Pages of a cache in plain Python, by the definition: one row and one entry at a time.  Returns the device's error bits."""

import numpy as np

EXHAUSTED, BAD_LENGTH, BAD_PARENT, BAD_BLOCK, BAD_COUNT, NO_ROOM = 1, 2, 4, 8, 16, 32


class Pool:
    """planes: arrays [layers][blocks][bytes]."""

    def __init__(self, blocks, width, planes):
        self.blocks, self.width, self.planes = blocks, width, planes
        self.refs = np.zeros(blocks, np.int32)

    def free_mask(self):
        words = np.zeros(-(-self.blocks // 32), np.uint32)
        for i in np.flatnonzero(self.refs == 0):
            words[i // 32] |= np.uint32(1 << (i % 32))
        return words

    def valid(self, b):
        return 0 <= b < self.blocks

    def fork(self, tables, lens, rows_out, parents=None, reserve=0, appended=0, keep_inputs=False):
        """-> tables, lens, error bits"""
        error, rows_in = 0, len(tables)
        want = []
        for r in range(rows_out):
            p = int(parents[r]) if parents is not None else (r if r < rows_in else -1)
            if not -1 <= p < rows_in:
                error |= BAD_PARENT
                p = -1
            length = 0
            if p >= 0:
                length = int(lens[p]) + appended
                if not 0 <= length <= self.width * 16:
                    error |= BAD_LENGTH
                    length = 0
            room = max(0, int(reserve[r]) if np.ndim(reserve) else int(reserve))
            if length + room > self.width * 16:
                error |= NO_ROOM
            want.append((p, length, min(-(-(length + room) // 16), self.width)))
        before = self.refs.copy()
        free = [int(b) for b in np.flatnonzero(before == 0)]
        out, taken, copies, seen = [], [], [], set()
        for p, length, need in want:
            row = [-1] * self.width
            filled, kept = length // 16, length // 16
            for j in range(filled):
                if self.valid(tables[p][j]):
                    row[j] = int(tables[p][j])
                else:
                    error |= BAD_BLOCK
            if p >= 0 and not keep_inputs and p not in seen:
                while kept < need and self.valid(tables[p][kept]) and before[tables[p][kept]] == 1:
                    row[kept] = int(tables[p][kept])
                    kept += 1
            seen.add(p)
            for j in range(kept, need):
                row[j] = ("fresh", len(taken))
                taken.append(j)
            if p >= 0 and length % 16 and kept == filled:
                if self.valid(tables[p][filled]):
                    copies.append((int(tables[p][filled]), row[filled][1]))
                else:
                    error |= BAD_BLOCK
            out.append(row)
        if len(taken) > len(free):
            return (np.full((rows_out, self.width), -1, np.int32), np.full(rows_out, -1, np.int32), error & ~BAD_BLOCK | EXHAUSTED)
        out = np.array([[free[b[1]] if isinstance(b, tuple) else b for b in row] for row in out], np.int32).reshape(rows_out, self.width)
        for src, k in copies:
            for plane in self.planes:
                plane[:, free[k]] = plane[:, src]
        if not keep_inputs:
            for row in tables:
                for b in row:
                    if self.valid(b):
                        self.refs[b] -= 1
                    elif b != -1:
                        error |= BAD_BLOCK
        for row in out:
            for b in row:
                if b >= 0:
                    self.refs[b] += 1
        return out, np.array([w[1] for w in want], np.int32), error

    def compact(self, tables):
        """-> tables, forward"""
        live = int((self.refs > 0).sum())
        holes = [b for b in range(live) if self.refs[b] == 0]
        movers = [b for b in range(live, self.blocks) if self.refs[b] > 0]
        forward = np.arange(self.blocks, dtype=np.int32)
        for src, dst in zip(movers, holes):
            forward[src] = dst
            self.refs[dst], self.refs[src] = self.refs[src], 0
            for plane in self.planes:
                plane[:, dst] = plane[:, src]
        return np.array([[forward[b] if self.valid(b) else b for b in row] for row in tables], np.int32).reshape(np.shape(tables)), forward
