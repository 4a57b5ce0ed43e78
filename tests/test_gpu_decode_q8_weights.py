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
