"""Appended rows that raise their block's exponents where the wave that appends reads the block in a later turn of its
loop, and where it reads it first: planes and exponents byte for byte, and the output."""

import numpy as np
import pytest

import q8_ref as R
from pvlc_testlib import log, pvlc
from test_gpu_decode_q8 import CODES, WIDTHS, Case, workspace

pytestmark = pytest.mark.gpu


def grown(c):
    """The case's new rows, 30 times larger than those before: the exponents that each sequence's last block then has
    must be larger than they were."""
    c.operands(scale=30.0)
    last = [int(c.table[i][int(t) // 16]) for i, t in enumerate(c.lens) if t % 16]
    before = c.cache.exponents[last].astype(int)

    def check():
        assert last and (c.cache.exponents[last].astype(int) > before).all(), "an exponent did not grow"
    return check


@CODES
@WIDTHS
@pytest.mark.parametrize("partition", [1024, 4096])
def test_in_a_later_turn_of_the_walk(code, f32, partition):
    """The walk's workgroups take 256 tokens a turn: rows appended in turns 0 to 3, at slots 1 to 15, on and off the
    last tile of a wave, and one that starts a block."""
    log(f"case: q8 decode grows in a later turn partition={partition} code={code} f32={f32}")
    c = Case([300, 523, 1009, 1025 + 767, 2047, 3500, 514 + 1024, 257, 130, 1024 + 496], code, f32, seed=partition + 2 * code + f32).upload()
    check = grown(c)
    ws = workspace(c.n, c.width * 16, partition)
    c.launch(c.args(ws, partition=partition))
    c.check(f"P={partition}")
    check()
    c.lens += 1
    c.dlens += 1
    c.operands(scale=1000.0)  # and again, over rows rounded twice
    c.launch(c.args(ws, partition=partition))
    c.check(f"P={partition}, again")
    assert pvlc.workspace_error(*ws) == 0


def test_in_a_later_turn_of_the_widest_workgroup():
    """More sequences than the walk numbers: 768 tokens a turn, the row in the second."""
    log("case: q8 decode grows in a later turn of twelve waves")
    c = Case([905, 770] + [3] * 2098, R.E4M3, True, seed=17, paged=False).upload()
    check = grown(c)
    ws = workspace(c.n, c.width * 16, 1024)
    c.launch(c.args(ws, partition=1024))
    c.check("2100 sequences")
    check()
