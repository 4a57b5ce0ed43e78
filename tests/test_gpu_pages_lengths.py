"""Lengths that a fork refuses: negative ones, whatever is appended, and those beyond the table."""

import numpy as np
import pytest

import pages_ref as P
from pvlc_testlib import log, pvlc
from test_gpu_pages import Both

pytestmark = pytest.mark.gpu


class Pool(P.Pool):
    """The plain form, in which a negative length stays one however many rows were appended."""

    def fork(self, tables, lens, *a, **k):
        return super().fork(tables, np.where(np.asarray(lens) < 0, -(1 << 40), np.asarray(lens, np.int64)), *a, **k)


def both(*a, **k):
    b = Both(*a, **k)
    b.ref.__class__ = Pool
    return b


@pytest.mark.parametrize("appended", [0, 1, 16, 1 << 31])
@pytest.mark.parametrize("length", [-1, -16, -(1 << 31)])
def test_a_negative_length_is_an_error(length, appended):
    """Its row is taken as empty and reported; the others are as they would be without it."""
    log(f"case: pages length {length} with {appended} appended")
    b = both(40, 8)
    b.step(3, "admission", parents=[-1, -1, -1], reserve=[40, 33, 20])
    beyond = appended > 8 * 16  # then the lengths of the others are out of range too
    b.lens = np.array([length, 30, length], np.int32)
    b.step(4, "children", parents=[1, 0, 2, 1], reserve=1, appended=appended, errors=pvlc.PAGES_BAD_LENGTH)
    assert (b.lens == ([0] * 4 if beyond else [30 + appended, 0, 0, 30 + appended])).all()


@pytest.mark.parametrize("keep_inputs", [False, True])
def test_rows_of_a_fork_that_found_too_few_pages(keep_inputs):
    """The next step's fork of rows that were left at -1 reports them."""
    log("case: pages after a fork that found too few")
    b = both(10, 8)
    b.step(2, "admission", parents=[-1, -1], reserve=64)
    b.lens = np.array([50, 33], np.int32)
    tables, lens = b.fork(5, "exhausted", parents=[0, 0, 1, 1, 0], reserve=40, errors=pvlc.PAGES_EXHAUSTED)
    assert (tables == -1).all() and (lens == -1).all()
    b.fork(2, "its rows, a row appended", parents=[0, 3], reserve=1, appended=1, tables=tables, lens=lens, keep_inputs=keep_inputs,
           errors=pvlc.PAGES_BAD_LENGTH)


def test_an_unused_negative_row_is_no_error():
    """A row that no output row continues is let go, whatever its length says."""
    log("case: pages negative length without children")
    b = both(40, 8)
    b.step(3, "admission", parents=[-1, -1, -1], reserve=[40, 33, 20])
    b.lens = np.array([17, -1, 5], np.int32)
    b.step(2, "without it", parents=[2, 0], reserve=1, appended=1)
