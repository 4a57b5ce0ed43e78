"""The 8-bit cache in plain numpy: codes, exponents, slabs, the append and the attention over what is held, in 64 bits.
Independent of the library; rotary's products and sum are rounded to 32 bits and the row to fp16, as the cache's
definition says."""

import numpy as np

E4M3, INT8 = 0, 1
LARGEST = {E4M3: 448.0, INT8: 127.0}
BIAS, LEAST = 127, -32


def e4m3_value(code):
    """e4m3 bytes as f64 (0x7F and 0xFF are NaN)."""
    c = np.asarray(code, np.uint8).astype(np.int64)
    sign, exp, frac = np.where(c & 0x80, -1.0, 1.0), (c >> 3) & 15, c & 7
    value = np.where(exp == 0, frac * 2.0 ** -9, (8 + frac) * np.ldexp(1.0, exp - 10))
    return np.where((c & 0x7F) == 0x7F, np.nan, sign * value)


E4M3_VALUES = e4m3_value(np.arange(256))


def value_of(code, byte):
    if code == E4M3:
        return E4M3_VALUES[np.asarray(byte, np.uint8)]
    return np.asarray(byte, np.uint8).view(np.int8).astype(np.float64)


def exponent_for(size, code):
    """The least e >= LEAST with size <= LARGEST 2^e (by search, not by taking numbers apart)."""
    size = np.asarray(size, np.float64)
    e = np.full(size.shape, LEAST, np.int64)
    for _ in range(64):
        e = np.where(size > LARGEST[code] * np.ldexp(1.0, e), e + 1, e)
    return e


def encode(x, e, code):
    """Bytes of f64 values at exponents e: the nearest code, ties to the even one."""
    y = np.asarray(x, np.float64) / np.ldexp(1.0, np.asarray(e, np.int64))
    nan = np.isnan(y)
    y = np.clip(np.where(nan, 0.0, y), -LARGEST[code], LARGEST[code])
    if code == INT8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    grid = E4M3_VALUES[:0x7F]  # the sizes, ascending; neighbours differ in the last bit of their code
    a = np.abs(y)
    lo = np.clip(np.searchsorted(grid, a, "right") - 1, 0, 0x7D)
    down, up = a - grid[lo], grid[lo + 1] - a
    pick = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, lo + 1)
    byte = (pick | np.where(np.signbit(y), 0x80, 0)).astype(np.uint8)
    return np.where(nan, np.uint8(0x7F), byte)


def held(x):
    """fp16 values as the cache takes them: infinities as 65504."""
    return np.clip(np.asarray(x, np.float64), -65504.0, 65504.0)


def key_index(t, d):
    """Byte of (token, dim) in a key slab."""
    return (t // 4) * 512 + (d // 16) * 64 + (t % 4) * 16 + d % 16


def value_index(t, d):
    return d * 16 + t


_T, _D = np.meshgrid(np.arange(16), np.arange(128), indexing="ij")
KEY_AT, VALUE_AT = key_index(_T, _D), value_index(_T, _D)  # [token][dim]


class Cache:
    """Planes [blocks][2][2048] and exponents [blocks][2][2], as bytes."""

    def __init__(self, blocks, code, fill=0):
        self.code = code
        self.key = np.full((blocks, 2, 2048), fill, np.uint8)
        self.value = np.full((blocks, 2, 2048), fill, np.uint8)
        self.exponents = np.full((blocks, 2, 2), fill, np.uint8)

    def put(self, block, first, rows_k, rows_v):
        """Rows [n][2][128] (fp16 values) as the tokens first.. of a block that holds `first` rows."""
        n = len(rows_k)
        for which, (plane, at, rows) in enumerate(((self.key, KEY_AT, rows_k), (self.value, VALUE_AT, rows_v))):
            for h in range(2):
                x = held(rows[:, h])
                e = int(exponent_for(np.nan_to_num(np.abs(x)).max(), self.code))
                if first:
                    old = int(self.exponents[block, h, which]) - BIAS
                    e = max(e, old)
                    if e > old:
                        before = value_of(self.code, plane[block, h, at[:first]]) * 2.0 ** old
                        plane[block, h, at[:first]] = encode(before, e, self.code)
                plane[block, h, at[first:first + n]] = encode(x, e, self.code)
                self.exponents[block, h, which] = e + BIAS

    def put_rows(self, table, first, rows_k, rows_v):
        """Rows as the tokens first.. of the sequence whose blocks are `table`."""
        done, n = 0, len(rows_k)
        while done < n:
            t = first + done
            take = min(16 - t % 16, n - done)
            self.put(table[t // 16], t % 16, rows_k[done:done + take], rows_v[done:done + take])
            done += take

    def rows(self, table, tokens):
        """What is held of the first tokens: [tokens][2][128] f64, twice."""
        out = []
        ids = np.asarray(table)[:-(-tokens // 16)]
        for which, (plane, at) in enumerate(((self.key, KEY_AT), (self.value, VALUE_AT))):
            power = np.ldexp(1.0, self.exponents[ids, :, which].astype(np.int64) - BIAS)  # [block][2]
            x = value_of(self.code, plane[ids][:, :, at]) * power[:, :, None, None]  # [block][2][token][dim]
            out.append(x.transpose(0, 2, 1, 3).reshape(-1, 2, 128)[:tokens])
        return out


def rotate(row, cos, sin):
    """Rotate-half of [heads][128] f32: products and sum rounded to 32 bits, the result to fp16 (as f64)."""
    x = np.asarray(row, np.float32)
    lo, hi = x[:, :64], x[:, 64:]
    c, s = np.float32(cos), np.float32(sin)
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.concatenate([lo * c + (-hi) * s, hi * c + lo * s], 1)
        return r.astype(np.float16).astype(np.float64)


def attend(q, k, v):
    """q [16][128] over rows [t][2][128], in 64 bits; and the largest sum of |q k| / sqrt(128), for error bounds."""
    out, big = np.empty((16, 128)), 0.0
    for g in range(2):
        h = slice(g * 8, g * 8 + 8)
        s = q[h] @ k[:, g].T / np.sqrt(128.0)
        big = max(big, float((np.abs(q[h]) @ np.abs(k[:, g]).T / np.sqrt(128.0)).max()))
        p = np.exp(s - s.max(1, keepdims=True))
        out[h] = (p / p.sum(1, keepdims=True)) @ v[:, g]
    return out, big


def attend_bound(big, k_tokens, v):
    """How far an f32 evaluation may be off, element by element.

    A score is 128 exact products summed in f32 and two more roundings: at most 131 u of the sum of sizes `big` (u =
    2^-24); the subtraction of the reference and exp2's own error add 2 u of its size and 4 u.  A weight's relative
    error d moves the quotient by at most 2 d of the largest value.  The pair of fp16 weights keeps 22 bits or, where a
    weight is tiny, 2^-25 of the largest one, for each token; and the sums over the tokens round once a token."""
    u = 2.0 ** -24
    d = 131 * u * big + 2 * u * (1.5 * big + 40) + 4 * u
    return (2 * d + 2.0 ** -21 + 3 * k_tokens * u) * float(np.abs(v).max())
