"""The weights of the decode over the 8-bit cache, each head and dim by itself: against the 64-bit result, within what
its own terms sum p |v| allow, however large other dims of other rows are."""

import numpy as np
import pytest

import q8_ref as R
from pvlc_testlib import log
from test_gpu_decode_q8 import CODES, Case, workspace

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def weighted(q, k, v):
    """attend's output, the sums of p |v| by head and dim, and the largest sum of |q k| / sqrt(128)."""
    out, big = R.attend(q, k, v)
    return out, R.attend(q, k, np.abs(v))[0], big


def bound_of(sizes, big, tokens, f32):
    """How far the quotient may be off before its output is rounded.

    A score is 128 exact products summed in f32 and two more roundings, so off by at most 131 u of `big`; the
    subtraction of the reference and exp2 add 2 u of its size (1.5 big + 40 log2 units) and 4 u.  A weight that is off
    by a factor 1 + d moves numerator and denominator, 2 d of sum p |v|.  Weights go to the products in 16 bits (2^-16)
    for fp16 operands, whole for f32 ones.  The sums have up to three terms a token, each added at 2^-23, and there are
    a few roundings for each join of waves and partitions."""
    d = 131 * U * big + 2 * U * (1.5 * big + 40) + 4 * U
    return (2 * d + (0.0 if f32 else 2.0 ** -16) + (6 * tokens + 100) * U) * sizes


def rounded_within(got, want, bound):
    """Whether fp16 outputs are the rounding of a value within bound of want."""
    with np.errstate(over="ignore"):
        return ((want - bound).astype(np.float16) <= got) & (got <= (want + bound).astype(np.float16))


def expect(c, i):
    """Appends sequence i's new row and attends: output, its bound."""
    t = int(c.lens[i])
    half = lambda x: x.astype(np.float16).astype(np.float64)  # noqa: E731
    c.cache.put_rows(c.table[i], t, half(c.nk[i])[None], half(c.nv[i])[None])
    keys, values = c.cache.rows(c.table[i], t + 1)
    out, sizes, big = weighted(half(c.q[i]), keys, values)
    return out, bound_of(sizes, big, t + 1, c.f32)


def check(c, ws, label, **how):
    import torch
    c.launch(c.args(ws, rope=False, rotate_query=False, **how))
    torch.cuda.synchronize()
    got = c.out.cpu().numpy()
    worst = 0.0
    for i in range(c.n):
        want, bound = expect(c, i)
        assert np.isfinite(got[i]).all(), f"{label}, sequence {i}"
        if c.f32:
            ratio = np.abs(got[i] - want) / bound
            worst = max(worst, ratio.max())
            assert ratio.max() <= 1, f"{label}, sequence {i}: {ratio.max():.3g} bounds off at {np.unravel_index(ratio.argmax(), ratio.shape)}"
        else:
            ok = rounded_within(got[i], want, bound)
            assert ok.all(), f"{label}, sequence {i}: {(~ok).sum()} outputs not a rounding of the result, first {np.argwhere(~ok)[0]}"
    print(f"[q8 weights] {label}: worst {worst:.3g} of the bound", flush=True)


@CODES
def test_fp16_outputs_are_rounded_once(code):
    """fp16 operands: what is returned is the rounding of the result, not of one whose weights were rounded as coarsely.
    Small queries, so that the scores' own error is far below the output's step."""
    log(f"case: q8 decode fp16 outputs, code={code}")
    c = Case(list(range(1, 49)), code, False, seed=101 + code)
    c.q = (c.q * 0.03).astype(np.float16)
    c.upload()
    check(c, workspace(c.n, c.width * 16), "short sequences")


def outlying(tokens, code, f32, size, others, score, seed):
    """Sequences with one large value: `size` in one dim of one row of each kv head, values of scale `others` elsewhere,
    and a score of about `score` for that row."""
    c = Case(tokens, code, f32, seed=seed)
    for i, t in enumerate(c.lens):
        t = int(t)
        k, v = c.rows(t)
        v = (v.astype(np.float64) * others).astype(np.float16)
        q = c.q[i].astype(np.float64).reshape(2, 8, 128) * 0.2 + c.g.standard_normal((2, 1, 128))
        c.q[i] = q.reshape(16, 128).astype(c.q.dtype)
        row = t // 3
        for h in range(2):
            mean = q[h].mean(0)
            k[row, h] = (mean * (score * np.sqrt(128.0) / (mean @ mean))).astype(np.float16)
            v[row, h, 5 + 60 * h] = size
        c.cache.put_rows(c.table[i], 0, k, v)
        c.nv[i] = (c.nv[i] * others).astype(c.nv.dtype)
    return c


@CODES
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("size,others,score", [(3, 1, 0), (3000, 1, 6), (30000, 1, 0), (60000, 1, 6), (30000, 0.05, 0), (60000, 0.002, -3)])
def test_one_large_value(code, f32, size, others, score):
    """A value far larger than the rest leaves the other dims as exact as they are without it."""
    log(f"case: q8 decode one large value {size} among {others}, score {score}, code={code} f32={f32}")
    c = outlying([40, 75, 130, 300], code, f32, size, others, score, seed=int(size) + code).upload()
    check(c, workspace(c.n, c.width * 16), "short")
    c = outlying([1200, 700], code, f32, size, others, score, seed=int(size) + 7 + code).upload()
    check(c, workspace(c.n, c.width * 16, 64), "partitions of 64", partition=64)
    c = outlying([900] * 3, code, f32, size, others, score, seed=int(size) + 9 + code).upload()
    check(c, workspace(c.n, c.width * 16, 1024), "streaming", partition=1024)
