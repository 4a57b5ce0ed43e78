"""A row's scores are its own: the same bits whatever else is in the batch."""

import numpy as np
import pytest

from pvlc_testlib import log, pvlc
from test_gpu_beam import Device, logits_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,beams,vocab,best", [(16, 4, 103424, 8), (1, 24, 103424, 16), (150, 4, 5000, 8), (40, 1, 103424, 4), (3, 8, 300007, 4)])
def test_an_entry_alone_and_in_a_batch(batch, beams, vocab, best):
    """Scores near 0, where f32 shows the last bits of the sum: likely tokens over a wide tail."""
    import torch
    log(f"case: beam entries alone and in a batch of {batch} x {beams}, vocab={vocab}")
    g = np.random.default_rng(vocab + batch)
    logits = logits_of(g, 4 * beams, vocab)
    logits[np.arange(4 * beams), g.integers(0, vocab, 4 * beams)] += np.float32(np.log(vocab) + 7)
    logits = np.tile(logits, (-(-batch // 4), 1))[:batch * beams]  # four entries, again and again
    scores = np.zeros((batch, beams), np.float32)
    whole = Device(batch, beams, vocab, best)
    pvlc.beam_select(whole.args(logits, scores))
    torch.cuda.synchronize()
    got = [o.cpu().numpy() for o in whole.out]
    for b in sorted({0, 1, 2, batch - 1} & set(range(batch))):
        one = Device(1, beams, vocab, best)
        pvlc.beam_select(one.args(logits[b * beams:(b + 1) * beams], scores[:1]))
        torch.cuda.synchronize()
        alone = [o.cpu().numpy()[0] for o in one.out]
        np.testing.assert_array_equal(got[0][b].view(np.int32), alone[0].view(np.int32), f"scores of entry {b}")
        np.testing.assert_array_equal(got[1][b] - b * beams, alone[1], f"parents of entry {b}")
        np.testing.assert_array_equal(got[2][b], alone[2], f"tokens of entry {b}")
    # and a beam in an entry of its own
    single = Device(beams, 1, vocab, best)
    pvlc.beam_select(single.args(logits[:beams], scores[:1].reshape(beams, 1)))
    torch.cuda.synchronize()
    rows = [o.cpu().numpy() for o in single.out]
    for i in range(best):
        p, t = int(got[1][0, i]), int(got[2][0, i])
        at = np.flatnonzero(rows[2][p] == t)
        assert at.size == 1 and rows[0][p, at[0]] == got[0][0, i], f"candidate {i}"
