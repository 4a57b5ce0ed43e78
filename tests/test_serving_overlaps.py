"""Outputs over one another are refused before any GPU effect."""

import pytest

from pvlc_testlib import pvlc
from test_serving_abi import P, pool, refused


@pytest.mark.parametrize("change", [dict(parents=P * 5), dict(tokens=P * 6 + 28), dict(next_finished=P * 7 - 28), dict(tokens=P * 5 + 4)])
def test_beam_outputs(change):
    base = dict(batch=2, beams=4, vocab=1000, best=4, logits=P * 16, scores=P * 2, next_scores=P * 5, parents=P * 6, tokens=P * 7,
                next_finished=P * 9, workspace=P * 8, workspace_bytes=1)
    refused(lambda: pvlc.beam_select(pvlc.beam_select_args(**{**base, **change})), "InvalidActivationLayout")
    # side by side they pass this check and reach the next
    refused(lambda: pvlc.beam_select(pvlc.beam_select_args(**{**base, "parents": P * 5 + 32, "tokens": P * 5 + 64})), "LengthMismatch")


def test_a_compaction_map_over_the_tables():
    c = pool()
    tables = 3 * P
    for forward in (tables, tables + c.max_blocks_per_seq * 4 - 4, tables - c.num_blocks * 4 + 4):
        refused(lambda: pvlc.kv_pages_compact(c, rows=1, tables=tables, forward=forward), "InvalidActivationLayout")
