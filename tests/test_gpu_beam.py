"""Beam selection against the plain form in 64 bits: parents, tokens and flags equal, scores to the rounding of f32 and
the error of the sum of exponentials."""

import numpy as np
import pytest

from pvlc_testlib import log, pvlc

pytestmark = pytest.mark.gpu


def order_key(x):
    """f32 as whole numbers in the order of the greedy top-1 (-0 below +0)."""
    b = np.asarray(x, np.float32).view(np.int32).astype(np.int64)
    return b ^ ((b >> 31) & 0x7FFFFFFF)


def plain(logits, scores, best, finished=None, end=-1):
    batch, beams = scores.shape
    out = [np.full((batch, best), v, t) for v, t in ((-np.inf, np.float64), (-1, np.int64), (-1, np.int64), (0, np.int64))]
    gap = np.inf
    for b in range(batch):
        cand = []
        for w in range(beams):
            r, s = b * beams + w, float(scores[b, w])
            if not s > -np.inf:
                continue
            if finished is not None and finished[b, w]:
                cand.append((s, w, 0, end, 1))
                continue
            x = np.where(np.isnan(logits[r]) | (logits[r] < -2.0 ** 127), np.float32(-np.inf), np.minimum(logits[r], np.float32(2.0 ** 127)))
            if not (x > -np.inf).any():
                continue
            m = x.max().astype(np.float64)
            log_sum = np.log(np.exp(x.astype(np.float64) - m).sum())
            k = order_key(x)
            top = np.lexsort((np.arange(x.size), -k))[:best]
            cand += [(s + ((float(x[t]) - m) - log_sum), w, i, int(t), int(t == end)) for i, t in enumerate(top) if x[t] > -np.inf]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for a, c in zip(cand[:best], cand[1:]):
            if a[1] != c[1] and a[0] != c[0]:
                gap = min(gap, a[0] - c[0])
        for i, c in enumerate(cand[:best]):
            for o, v in zip(out, (c[0], b * beams + c[1], c[3], c[4])):
                o[b, i] = v
    return out, gap


class Device:
    def __init__(self, batch, beams, vocab, best):
        import torch
        self.shape = batch, beams, vocab, best
        self.nbytes = pvlc.beam_workspace_bytes(batch, beams, vocab, best)
        self.ws = torch.empty(self.nbytes, dtype=torch.uint8, device="cuda")
        pvlc.workspace_init(self.ws, self.nbytes)

    def args(self, logits, scores, finished=None, end=-1, stride=None, offset=0):
        import torch
        batch, beams, vocab, best = self.shape
        stride = stride or vocab
        buf = np.full(batch * beams * stride + offset, 1e30, np.float32)  # what lies between rows would win
        for r in range(batch * beams):
            buf[offset + r * stride:offset + r * stride + vocab] = logits[r]
        self.logits = torch.from_numpy(buf).cuda()[offset:]
        self.scores = torch.from_numpy(np.ascontiguousarray(scores, np.float32)).cuda()
        self.finished = None if finished is None else torch.from_numpy(np.ascontiguousarray(finished, np.int32)).cuda()
        self.out = [torch.full((batch, best), 55, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32, torch.int32)]
        return pvlc.beam_select_args(batch=batch, beams=beams, vocab=vocab, best=best, logits=self.logits, row_stride=stride,
                                     scores=self.scores, finished=self.finished, end_token=end, next_scores=self.out[0],
                                     parents=self.out[1], tokens=self.out[2], next_finished=self.out[3], workspace=self.ws,
                                     workspace_bytes=self.nbytes)

    def run(self, logits, scores, finished=None, end=-1, label="", **how):
        import torch
        args = self.args(logits, scores, finished, end, **how)
        pvlc.beam_select(args)
        torch.cuda.synchronize()
        self.check(logits, scores, finished, end, label)

    def check(self, logits, scores, finished, end, label):
        want, gap = plain(logits, np.asarray(scores, np.float32), self.shape[3], finished, end)
        # terms of the sum are off by 2^-23 + 2^-24 |x - m| log2(e) <= 2e-6 each at most, in either direction; here the
        # candidates of two beams lie further apart than that
        assert gap > 4e-6, f"{label}: candidates {gap} apart"
        got = [o.cpu().numpy() for o in self.out]
        for name, a, b in zip(("parents", "tokens", "finished"), got[1:], want[1:]):
            np.testing.assert_array_equal(a, b, f"{label} {name}")
        fine = np.isfinite(want[0])
        np.testing.assert_array_equal(np.isfinite(got[0]), fine, label)
        with np.errstate(invalid="ignore"):
            off = np.abs(got[0][fine] - want[0][fine]) - np.abs(want[0][fine]) * 2.0 ** -24
        assert (off <= 2e-6).all(), f"{label}: {off.max()}"


def logits_of(g, rows, vocab, scale=2.5):
    x = (g.standard_normal((rows, vocab)) * scale).astype(np.float32)
    for r in range(rows):
        for t in g.integers(0, vocab, 6):
            x[r, t] += np.float32(6 + 2 * g.standard_normal())
    return x


@pytest.mark.parametrize("batch,beams,vocab,best", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 6), (1, 4, 97, 4), (3, 2, 2047, 4), (2, 5, 2048, 10), (1, 4, 2049, 8), (4, 8, 5000, 16),
    (1, 16, 6001, 32), (2, 64, 300, 128), (1, 1, 30011, 128), (1, 4, 103424, 4), (2, 8, 103424, 16), (1, 2, 300007, 64)])
def test_random_logits(batch, beams, vocab, best):
    log(f"case: beam batch={batch} beams={beams} vocab={vocab} best={best}")
    g = np.random.default_rng(vocab + best)
    d = Device(batch, beams, vocab, best)
    for finished in (None, (g.random((batch, beams)) < 0.3).astype(np.int32)):
        x = logits_of(g, batch * beams, vocab)
        d.run(x, -5 * g.random((batch, beams)), finished, end=vocab // 2, label=f"finished={finished is not None}")


@pytest.mark.parametrize("stride,offset", [(1003, 0), (1001, 1), (1024, 2), (1000, 3)])
def test_row_strides_and_odd_addresses(stride, offset):
    log(f"case: beam stride={stride} offset={offset}")
    g = np.random.default_rng(stride)
    Device(2, 3, 1000, 6).run(logits_of(g, 6, 1000), -g.random((2, 3)), end=3, stride=stride, offset=offset)


def test_first_step_and_dead_beams():
    """Only beam 0 alive (the step after a prompt), none alive, and scores of NaN."""
    log("case: beam dead rows")
    g = np.random.default_rng(5)
    x = logits_of(g, 12, 3000)
    x[1:4] = np.nan
    scores = np.full((3, 4), -np.inf, np.float32)
    scores[0, 0] = 0
    scores[2] = [-1, np.nan, -2.5, -np.inf]
    Device(3, 4, 3000, 8).run(x, scores, label="dead")


def test_masks():
    """Tokens masked by -inf and NaN, whole rows of them, rows of the type's lowest value, fewer candidates than asked
    for, +inf, and rows whose only token lies in the last place."""
    log("case: beam masks")
    g = np.random.default_rng(6)
    low = np.finfo(np.float32).min
    x = logits_of(g, 8, 4500)
    x[0] = -np.inf
    x[0, [7, 4499]] = [1.0, 2.0]
    x[1] = -np.inf
    x[2] = np.nan
    x[3] = low
    x[4, g.random(4500) < 0.9] = -np.inf
    x[5, ::2] = np.nan
    x[6, :2100] = low
    x[7] = -np.inf
    x[7, 4499] = -3.0
    scores = np.array([[-1.0, -2, -3, -4], [-0.5, -0.25, -0.125, -9]], np.float32)
    Device(2, 4, 4500, 12).run(x, scores, label="masks")
    y = logits_of(g, 2, 100)
    y[0, 50], y[1, 60] = np.inf, np.inf
    y[1, 61] = np.inf
    Device(1, 2, 100, 3).run(y, np.array([[-1.0, -1.5]]), label="inf")
    z = np.full((2, 50), -np.inf, np.float32)
    Device(1, 2, 50, 3).run(z, np.array([[-1.0, -1.5]]), label="nothing")


def test_ties():
    """Equal logits go by token, within a thread, a segment and over segments; equal beams by beam; -0 below +0; a row of
    one value everywhere."""
    log("case: beam ties")
    g = np.random.default_rng(7)
    x = np.full((4, 9000), -4.0, np.float32)
    x[:, [8999, 17, 5000, 18, 2048, 2047, 0]] = 1.0
    x[:, 100], x[:, 99] = 0.0, -0.0
    d = Device(2, 2, 9000, 9)
    d.run(x, np.array([[-1.0, -1.0], [-2.0, -2.0]]), label="equal beams")
    x[:] = 0.25
    Device(2, 2, 9000, 20).run(x, np.array([[-1.0, -1.0], [-2.0, -7.0]]), label="one value")
    y = logits_of(g, 1, 5000)
    y = np.concatenate([y, y])
    Device(1, 2, 5000, 10).run(y, np.array([[-3.0, -3.0]]), label="the same beam twice")


def test_finished_beams_compete():
    log("case: beam finished")
    g = np.random.default_rng(8)
    x = logits_of(g, 4, 700)
    x[1] = np.nan  # a finished row's logits are not read
    for finished in ([[0, 1, 0, 0]], [[1, 1, 1, 1]], [[1, 0, 1, 0]]):
        Device(1, 4, 700, 6).run(x if finished[0][1] else logits_of(g, 4, 700), np.array([[-1.0, -0.5, -3.0, -2.0]]), np.array(finished), end=11,
                                 label=str(finished))


def test_large_and_small_logits():
    log("case: beam sizes of logits")
    g = np.random.default_rng(9)
    x = (g.standard_normal((4, 3000)) * np.array([[1e4], [1e-3], [30.0], [1e30]])).astype(np.float32)
    Device(4, 1, 3000, 5).run(x, -g.random((4, 1)), label="sizes")


def test_another_stream_and_a_graph():
    import torch
    log("case: beam graph")
    g = np.random.default_rng(10)
    d = Device(2, 4, 20000, 8)
    x, s = logits_of(g, 8, 20000), -g.random((2, 4))
    args = d.args(x, s, end=5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    pvlc.beam_select(args, side)
    side.synchronize()
    d.check(x, s, None, 5, "side stream")
    first = [o.clone() for o in d.out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pvlc.beam_select(args, torch.cuda.current_stream())
    other = Device(2, 4, 20000, 8)
    for _ in range(4):
        for o in d.out:
            o.zero_()
        pvlc.beam_select(other.args(x, s))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(d.out, first))


def test_rows_beyond_32_bits_of_offset():
    import torch
    log("case: beam rows 4 GiB apart")
    g = np.random.default_rng(12)
    x, stride = logits_of(g, 2, 5000), (1 << 30) + 5
    d = Device(1, 2, 5000, 4)
    args = d.args(x, np.array([[-1.0, -2.0]]))
    far = torch.empty(stride + 5000, dtype=torch.float32, device="cuda")
    far[:5000], far[stride:] = torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda()
    args.logits, args.row_stride = far.data_ptr(), stride
    pvlc.beam_select(args)
    torch.cuda.synchronize()
    d.check(x, np.array([[-1.0, -2.0]]), None, -1, "far rows")


def test_rows_of_one_low_value_but_a_few():
    """What a constrained step gives: all but a few tokens at one large negative value; every selection is exact."""
    log("case: beam constrained rows")
    g = np.random.default_rng(13)
    x = np.full((4, 20011), -1e9, np.float32)
    for r in range(4):
        x[r, g.choice(20011, 3 + 9 * r, replace=False)] = g.standard_normal(3 + 9 * r) * 3
    for best in (4, 16, 70):
        Device(2, 2, 20011, best).run(x, -g.random((2, 2)), label=f"best={best}")


def test_calls_of_other_shapes_share_a_workspace():
    """A workspace of any content, used by selections whose layouts of it differ, eagerly and from two graphs."""
    import torch
    log("case: beam shapes on one workspace")
    g = np.random.default_rng(14)
    wide, deep = Device(130, 2, 300, 4), Device(1, 8, 40000, 16)
    ws = torch.full((max(wide.nbytes, deep.nbytes),), 0xA5, dtype=torch.uint8, device="cuda")
    runs = []
    for d in (wide, deep):
        d.ws, d.nbytes = ws, ws.numel()
        batch, beams, vocab, _ = d.shape
        x, s = logits_of(g, batch * beams, vocab), -g.random((batch, beams))
        args = d.args(x, s, end=7)
        torch.cuda.synchronize()
        runs.append((d, args, x, s, torch.cuda.CUDAGraph()))
    for d, args, x, s, _ in runs + runs:
        for o in d.out:
            o.fill_(55)
        pvlc.beam_select(args)
        torch.cuda.synchronize()
        d.check(x, s, None, 7, f"batch {d.shape[0]}")
    for d, args, _, _, graph in runs:
        with torch.cuda.graph(graph):
            pvlc.beam_select(args, torch.cuda.current_stream())
    for _ in range(3):
        for d, _, _, _, graph in runs:
            for o in d.out:
                o.fill_(55)
            graph.replay()
        torch.cuda.synchronize()
        for d, args, x, s, _ in runs:
            d.check(x, s, None, 7, f"batch {d.shape[0]}, replayed")
            pvlc.beam_select(args)
