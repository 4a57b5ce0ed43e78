"""Batches over paged caches in plain numpy: rows of several sequences appended to fp16 or 8-bit pages, and attention over
what is held, in 64 bits.  Independent of the library."""

import numpy as np

import q8_ref as R
from pvlc_testlib import key_slot, pvlc

F16 = 2
_T, _D = np.meshgrid(np.arange(16), np.arange(128), indexing="ij")
KEY_AT, VALUE_AT = (_D // 8) * 128 + key_slot(_T) * 8 + _D % 8, _D * 16 + _T  # [token][dim] of an fp16 slab


class HalfCache:
    """fp16 planes [blocks][2][2048] as bits, filled with NaN where no row is."""

    def __init__(self, blocks, fill=0xFFFF):
        self.key = np.full((blocks, 2, 2048), fill, np.uint16)
        self.value = np.full((blocks, 2, 2048), fill, np.uint16)

    def put_rows(self, table, first, rows_k, rows_v):
        for i, (k, v) in enumerate(zip(rows_k, rows_v)):
            block, slot = table[(first + i) // 16], (first + i) % 16
            for h in range(2):
                self.key[block, h, KEY_AT[slot]] = np.asarray(k[h], np.float16).view(np.uint16)
                self.value[block, h, VALUE_AT[slot]] = np.asarray(v[h], np.float16).view(np.uint16)

    def rows(self, table, tokens):
        ids = np.asarray(table)[:-(-tokens // 16)]
        return [plane[ids][:, :, at].view(np.float16).astype(np.float64).transpose(0, 2, 1, 3).reshape(-1, 2, 128)[:tokens]
                for plane, at in ((self.key, KEY_AT), (self.value, VALUE_AT))]


def cache(blocks, code):
    return HalfCache(blocks) if code == F16 else R.Cache(blocks, code, fill=0xFF)


class Batch:
    """Sequences with `held` rows in a pool of shuffled blocks (or contiguous ones), and `counts` more for each as rows of
    one matrix: alone, or slices of q|k|v."""

    def __init__(self, counts, held, code=F16, f32=False, seed=0, paged=True, fused=False, spare=0, room=0, positions=False, rope=True, scale=1.0):
        g = self.g = np.random.default_rng(seed)
        self.counts, self.held, self.code, self.f32, self.paged, self.rope = list(counts), list(held), code, f32, paged, rope
        self.n = len(counts)
        self.width = max(1, max(-(-(c + h + room) // 16) for c, h in zip(counts, held)))
        self.blocks = self.n * self.width + 3
        ids = g.permutation(self.blocks) if paged else np.arange(self.blocks)
        self.table = ids[:self.n * self.width].reshape(self.n, self.width).astype(np.int32)
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.offsets[-1]) + spare
        kind = np.float32 if f32 else np.float16
        wide = (g.standard_normal((max(1, self.rows), 20, 128)) * scale).astype(kind)
        self.q, self.k, self.v = wide[:, :16], wide[:, 16:18], wide[:, 18:]
        self.wide, self.fused = wide, fused
        self.table_rows = max(c + h for c, h in zip(counts, held)) + room + 9
        self.cos, self.sin = pvlc.rope_table(500000.0, self.table_rows)
        self.positions = g.integers(0, self.table_rows, self.rows).astype(np.int32) if positions else None
        self.cache = cache(self.blocks, code)
        for i, t in enumerate(self.held):
            if t:
                k = (g.standard_normal((t, 2, 128)) * np.exp(0.5 * g.standard_normal((2, 128)))).astype(np.float16)
                self.cache.put_rows(self.table[i], 0, k, g.standard_normal((t, 2, 128)).astype(np.float16))

    def place(self, row):
        """Sequence of a row and its place in it."""
        s = int(np.searchsorted(self.offsets, row, "right")) - 1
        return s, self.held[s] + row - int(self.offsets[s])

    def turned(self, x, row):
        """A row [heads][128] as it is rotated, in fp16's values (f64)."""
        if not self.rope:
            return x.astype(np.float16).astype(np.float64)
        pos = self.place(row)[1] if self.positions is None else int(self.positions[row])
        return R.rotate(x, self.cos[pos], self.sin[pos])

    def upload(self):
        import torch
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        bits = lambda a: put(a.view(np.int16) if a.dtype == np.uint16 else a)  # noqa: E731
        self.planes = [bits(self.cache.key.copy()), bits(self.cache.value.copy())]
        self.exponents = None if self.code == F16 else put(self.cache.exponents.copy())
        self.dtable, self.dlens, self.doffsets = put(self.table), put(np.asarray(self.held, np.int32)), put(self.offsets)
        self.dcos, self.dsin = put(self.cos), put(self.sin)
        self.dpositions = None if self.positions is None else put(self.positions)
        if self.fused:
            wide = put(self.wide).flatten(1)
            self.dq, self.dk, self.dv = wide[:, :2048], wide[:, 2048:2304], wide[:, 2304:]
        else:
            self.dq, self.dk, self.dv = (put(x).flatten(1) for x in (self.q, self.k, self.v))
        self.out = torch.full((max(1, self.rows), 16, 128), 9.0, dtype=self.dq.dtype, device="cuda")
        self.error = torch.zeros(1, dtype=torch.int32, device="cuda")
        return self

    def common(self):
        return dict(num_blocks=self.blocks, max_blocks_per_seq=self.width, key_cache=self.planes[0], value_cache=self.planes[1],
                    block_tables=self.dtable if self.paged else None, rope_cos=self.dcos if self.rope else None,
                    rope_sin=self.dsin if self.rope else None, rope_rows=self.table_rows if self.rope else 0, positions=self.dpositions)

    def packed(self):
        return dict(num_seqs=self.n, rows=self.rows, row_offsets=self.doffsets, cache_lens=self.dlens, key_stride=self.dk.stride(0),
                    value_stride=self.dv.stride(0), **self.common())

    def append_args(self, **change):
        self.keep = change  # (the arguments hold addresses alone)
        base = dict(self.packed(), code=self.code, exponents=self.exponents, error_word=self.error)
        return pvlc.kv_append_args(**{**base, **change})

    def append(self, args, stream=None):
        (pvlc.kv_append_f32 if self.f32 else pvlc.kv_append_f16)(args, self.dk, self.dv, stream)

    def put(self):
        """The rows into self.cache."""
        for s in range(self.n):
            at, c = int(self.offsets[s]), self.counts[s]
            if c:
                k = np.stack([self.turned(self.k[at + i], at + i) for i in range(c)])
                self.cache.put_rows(self.table[s], self.held[s], k, self.v[at:at + c].astype(np.float16).astype(np.float64))

    def check_planes(self, label):
        import torch
        torch.cuda.synchronize()
        names = ("key", "value") if self.code == F16 else ("key", "value", "exponents")
        for name, d in zip(names, self.planes + [self.exponents]):
            want = getattr(self.cache, name)
            got = d.cpu().numpy().view(want.dtype)
            same = got == want
            if self.code == R.E4M3 and name != "exponents":  # a NaN is a NaN, of either sign
                same |= (got & 0x7F == 0x7F) & (want & 0x7F == 0x7F)
            bad = np.argwhere(~same)
            assert bad.size == 0, f"{label}: {name} differs at {bad[0]} ({len(bad)} places)"


def attend(q, k, v, limits):
    """q [rows][16][128], row i over the first limits[i] of the rows k, v [t][2][128], in 64 bits; and for every row the largest
    sum of |q k| / sqrt(128) and the largest value size."""
    out, big, most = np.empty(q.shape), np.zeros(len(q)), np.zeros(len(q))
    for i, t in enumerate(limits):
        out[i], big[i] = R.attend(q[i], k[:t], v[:t])
        most[i] = np.abs(v[:t]).max()
    return out, big, most


def bound(out, big, most, tokens, f32, code=F16):
    """How far an evaluation in 32 bits may be off (see q8_ref.attend_bound).  A weight is rounded by 2^-11 of itself to fp16, 2^-22
    as a pair, 2^-17 as two bf16 terms, 2^-25 as three (or, where it is tiny, by 2^-25 of the largest one), and so is its part
    of the sum: twice that of the largest value.  Parts joined round their factors once more: 4 u."""
    u = 2.0 ** -24
    d = 131 * u * big + 2 * u * (1.5 * big + 40) + 8 * u
    weight = {True: 2.0 ** -22, False: 2.0 ** -11}[f32] if code == F16 else {True: 2.0 ** -24, False: 2.0 ** -17}[f32]
    b = (2 * (d + weight) + tokens * 2.0 ** -24 + 3 * tokens * u) * most
    b = b[:, None, None] * np.ones_like(out)
    return b if f32 else b * (1 + 2.0 ** -11) + np.abs(out) * 2.0 ** -11 + 2.0 ** -25


def check(label, got, want, limit):
    ratio = np.abs(np.asarray(got, np.float64) - want) / limit
    print(f"[batches] {label}: error / bound {ratio.max() if ratio.size else 0:.3g}", flush=True)
    assert np.isfinite(got).all(), label
    assert ratio.size == 0 or ratio.max() <= 1, f"{label}: {ratio.max()} at {np.unravel_index(ratio.argmax(), ratio.shape)}"
