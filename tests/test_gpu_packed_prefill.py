"""Packed prompts and chunks of prompts against the plain form in 64 bits; planes bit for bit."""

import numpy as np
import pytest

import batches_ref as B
from pvlc_testlib import log, pvlc

pytestmark = pytest.mark.gpu
WIDTHS = pytest.mark.parametrize("f32", [False, True])


def workspace(b, context):
    import torch
    nbytes = pvlc.packed_prefill_workspace_bytes(b.n, b.rows, context)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, nbytes)
    return ws, nbytes


def args_of(b, ws, **change):
    b.keep = change
    base = dict(b.packed(), max_context=b.width * 16, query_stride=b.dq.stride(0), workspace=ws[0], workspace_bytes=ws[1])
    return pvlc.packed_prefill_args(**{**base, **change})


def launch(b, args, stream=None):
    (pvlc.packed_prefill_f32io if b.f32 else pvlc.packed_prefill_f16)(args, b.dq, b.dk, b.dv, b.out, stream)


def wanted(b, some=None):
    """Outputs of the rows (or of some of them) and their bounds, after the rows have been put into the cache."""
    rows = np.arange(int(b.offsets[-1])) if some is None else some
    want, limit = np.empty((len(rows), 16, 128)), np.empty((len(rows), 16, 128))
    for s in range(b.n):
        mine = np.flatnonzero((rows >= b.offsets[s]) & (rows < b.offsets[s + 1]))
        if mine.size == 0:
            continue
        k, v = b.cache.rows(b.table[s], b.held[s] + b.counts[s])
        limits = [b.place(int(r))[1] + 1 for r in rows[mine]]
        q = np.stack([b.turned(b.q[r], int(r)) for r in rows[mine]])
        out, big, most = B.attend(q, k, v, limits)
        want[mine] = out
        limit[mine] = B.bound(out, big, most, max(limits), b.f32)
    return want, limit


def check(b, label, some=None):
    import torch
    torch.cuda.synchronize()
    b.put()
    b.check_planes(label)
    want, limit = wanted(b, some)
    got = b.out.float().cpu().numpy()
    rows = np.arange(int(b.offsets[-1])) if some is None else some
    B.check(label, got[rows], want, limit)
    assert (got[int(b.offsets[-1]):] == 9.0).all(), "rows behind the last sequence stay as they were"


BATCHES = {
    "one": ([1], [0]), "few": ([5, 0, 97, 16], [0, 0, 0, 0]), "behind": ([3, 33, 1, 40], [17, 100, 64, 31]), "ends": ([16, 32, 48, 64, 15, 17], [0, 16, 0, 1, 49, 15]),
    "many": ([1 + i % 5 for i in range(70)], [i * 11 % 70 for i in range(70)]), "long": ([300], [0]), "chunk": ([20, 1], [3000, 700]),
}


@WIDTHS
@pytest.mark.parametrize("name", list(BATCHES))
def test_batches(f32, name):
    """Planes hold NaN wherever no row is: values behind a sequence's last row carry no weight."""
    log(f"case: packed prefill {name} f32={f32}")
    counts, held = BATCHES[name]
    b = B.Batch(counts, held, f32=f32, seed=len(name), paged=name != "ends", fused=name in ("few", "chunk"), spare=3, positions=name == "behind",
                rope=name != "many").upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    check(b, name)
    assert pvlc.workspace_error(*ws) == 0


@WIDTHS
def test_items_are_cut_and_joined(f32):
    """Few rows on long histories, and a long prompt beside short ones: items in parts."""
    log(f"case: packed prefill in parts f32={f32}")
    b = B.Batch([40, 1500, 7], [6000, 0, 2047], f32=f32, seed=31).upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    some = np.unique(np.concatenate([np.arange(0, 40, 3), 40 + np.array([0, 15, 16, 31, 500, 1023, 1024, 1300, 1499]), 1540 + np.arange(7)]))
    check(b, "parts", some)


@WIDTHS
def test_rising_scores_move_the_reference(f32):
    """Scores that grow along the sequence by far more than the reference may lag."""
    log(f"case: packed prefill, rising scores f32={f32}")
    b = B.Batch([200], [90], f32=f32, seed=12, rope=False)
    b.q[:] = 1.0
    b.k[:, :, :] = (np.arange(b.rows)[:, None, None] * 0.05).astype(b.k.dtype)
    b.upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    check(b, "rising")


def test_without_offsets_lengths_and_table():
    log("case: packed prefill without offsets")
    b = B.Batch([21] * 3, [0] * 3, seed=6, paged=False).upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws, row_offsets=None, cache_lens=None))
    check(b, "equal prompts")


def test_many_sequences():
    """More sequences than are planned, the last ones without rows."""
    log("case: packed prefill, many sequences")
    n = 1100
    b = B.Batch([(i % 3) if i < 1000 else 0 for i in range(n)], [0] * n, seed=7).upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    check(b, "many")


def test_a_sequence_beyond_the_context_is_skipped():
    import torch
    log("case: packed prefill, beyond the context")
    b = B.Batch([20, 8, 6], [30, 3, 0], seed=9, room=16).upload()
    ws = workspace(b, 48)
    launch(b, args_of(b, ws, max_context=48))
    torch.cuda.synchronize()
    assert pvlc.workspace_error(*ws) == 1
    got = b.out.float().cpu().numpy()
    assert (got[:20] == 9.0).all()
    b.counts = [0, 8, 6]
    b.put()
    b.check_planes("skipped")
    some = np.arange(20, 34)
    want, limit = wanted(b, some)
    B.check("the others", got[some], want, limit)


def test_graphs_that_share_a_workspace():
    """Two captured calls of different shapes over one workspace, replayed in turn with direct calls between."""
    import torch
    log("case: packed prefill from graphs")
    one, two = (B.Batch(c, h, f32=f, seed=s).upload() for c, h, f, s in (([50, 9], [700, 0], False, 1), ([7] * 20, [40] * 20, True, 2)))
    sizes = [pvlc.packed_prefill_workspace_bytes(b.n, b.rows, b.width * 16) for b in (one, two)]
    ws = torch.empty(max(sizes), dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, max(sizes))
    args = [args_of(b, (ws, max(sizes))) for b in (one, two)]
    for b, a in zip((one, two), args):
        launch(b, a)
    torch.cuda.synchronize()
    want = [b.out.clone() for b in (one, two)]
    check(one, "direct")
    check(two, "direct")
    stream, graphs = torch.cuda.Stream(), []
    for b, a in zip((one, two), args):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            launch(b, a, stream)
    for _ in range(3):
        for g, b, w in zip(graphs, (one, two), want):
            b.out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(b.out, w)
        launch(one, args[0])
        torch.cuda.synchronize()
        assert torch.equal(one.out, want[0])
    assert pvlc.workspace_error(ws, max(sizes)) == 0


@WIDTHS
@pytest.mark.parametrize("n", [3, 1100])
def test_rows_before_the_first_sequence(f32, n):
    """The first sequence need not begin at row 0, among those that are planned and those that are not."""
    import torch
    log(f"case: packed prefill, rows before the first sequence, f32={f32} n={n}")
    b = B.Batch([60] + [1 + i % 3 for i in range(n)], [0] + [40 + i % 7 for i in range(n)], f32=f32, seed=n, spare=3).upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws, num_seqs=n, row_offsets=b.doffsets[1:], cache_lens=b.dlens[1:], block_tables=b.dtable[1:]))
    torch.cuda.synchronize()
    assert pvlc.workspace_error(*ws) == 0
    assert (b.out[:60] == 9.0).all() and (b.out[int(b.offsets[-1]):] == 9.0).all()
    b.counts[0] = 0
    b.put()
    b.check_planes("behind row 60")
    some = np.arange(60, int(b.offsets[-1]))
    want, limit = wanted(b, some)
    B.check("behind row 60", b.out.float().cpu().numpy()[some], want, limit)


@WIDTHS
@pytest.mark.parametrize("name", list(BATCHES))
def test_batches_in_wide_tables(f32, name):
    """Small calls give a workgroup one head; with room for longer sequences the same ones give it eight."""
    log(f"case: packed prefill {name} in wide tables f32={f32}")
    counts, held = BATCHES[name]
    b = B.Batch(counts, held, f32=f32, seed=len(name) + 40, fused=name in ("few", "chunk"), spare=3, positions=name == "behind", rope=name != "many")
    b.width = 300
    b.table = np.pad(b.table, ((0, 0), (0, 300 - b.table.shape[1])), constant_values=-1)
    b.upload()
    ws = workspace(b, 4800)
    launch(b, args_of(b, ws))
    check(b, name)
    assert pvlc.workspace_error(*ws) == 0


@WIDTHS
@pytest.mark.parametrize("name", ["equal", "one_more", "tiles"])
def test_small_calls(f32, name):
    """Without offsets and tables, one token behind whole pieces of keys, and prompts that end at tiles."""
    log(f"case: packed prefill, small calls, {name} f32={f32}")
    counts, held = {"equal": ([16] * 5, [0] * 5), "one_more": ([1] * 6, [31, 32, 127, 128, 129, 1000]), "tiles": ([128, 127, 129], [0, 1, 0])}[name]
    b = B.Batch(counts, held, f32=f32, seed=77, paged=name != "equal", spare=0 if name == "equal" else 5).upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws, **(dict(row_offsets=None, cache_lens=None) if name == "equal" else {})))
    check(b, name)
    assert pvlc.workspace_error(*ws) == 0


@WIDTHS
def test_rising_scores_over_eight_heads(f32):
    """As above, where a workgroup has eight heads, and parts of the keys to join."""
    log(f"case: packed prefill, rising scores, eight heads f32={f32}")
    b = B.Batch([100], [5000], f32=f32, seed=13, rope=False)
    b.q[:] = 1.0
    b.k[:, :, :] = (np.arange(b.rows)[:, None, None] * 0.05).astype(b.k.dtype)
    b.upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    check(b, "rising", np.arange(0, 100, 7))


@WIDTHS
@pytest.mark.parametrize("wide", [False, True])
def test_histories_on_the_same_pages(f32, wide):
    """Three requests behind one instruction: the same blocks in every table, rows of their own behind them."""
    log(f"case: packed prefill, one history, f32={f32} wide={wide}")
    b = B.Batch([5, 40, 17], [64, 64, 64], f32=f32, seed=21, room=5000 if wide else 0)
    for s in (1, 2):
        b.table[s, :4] = b.table[0, :4]
    b.upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    check(b, "one history")
    assert pvlc.workspace_error(*ws) == 0


@pytest.mark.parametrize("wide", [False, True])
def test_replays_follow_the_lengths(wide):
    """Offsets, lengths and tables are read by the launches: what lies there at a replay counts, not what lay there at the capture."""
    import torch
    log(f"case: packed prefill, replays with other lengths, wide={wide}")
    b = B.Batch([30, 7, 50], [20, 0, 33], seed=22, room=5000 if wide else 64, spare=6).upload()
    other = B.Batch([1, 80, 6], [0, 40, 17], seed=23, room=b.width * 16 - 120, spare=6)
    assert other.width == b.width and other.rows == b.rows and other.blocks == b.blocks
    ws = workspace(b, b.width * 16)
    args = args_of(b, ws, rope_rows=min(b.table_rows, other.table_rows))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        launch(b, args, stream)
    graph.replay()
    check(b, "as captured")
    other.upload()
    for name in ("planes", "dtable", "dlens", "doffsets", "dq", "dk", "dv"):
        for to, of in zip(*([getattr(x, name)] if name != "planes" else x.planes for x in (b, other))):
            to.copy_(of)
    b.out.fill_(9.0)
    graph.replay()
    torch.cuda.synchronize()
    other.planes, other.out = b.planes, b.out
    check(other, "with other lengths")
    assert pvlc.workspace_error(*ws) == 0


@WIDTHS
@pytest.mark.parametrize("held,wide", [(0, False), (21, False), (0, True), (21, True), (4500, True)])
def test_values_that_are_not_finite(f32, held, wide):
    """An infinity or NaN among the values reaches the rows that see it, in its head and dim, and no other."""
    import torch
    log(f"case: packed prefill, values that are not finite, held={held} f32={f32} wide={wide}")
    b = B.Batch([70, 33], [held, held // 2], f32=f32, seed=held + 5, room=4600 - held if wide else 0)
    for row, head, dim, value in ((3, 0, 5, np.inf), (37, 0, 5, -np.inf), (40, 1, 127, np.nan), (63, 1, 64, -np.inf), (69, 0, 0, np.nan), (70 + 32, 1, 9, np.inf)):
        b.v[row, head, dim] = value
    b.upload()
    ws = workspace(b, b.width * 16)
    launch(b, args_of(b, ws))
    torch.cuda.synchronize()
    got = b.out.float().cpu().numpy()
    with np.errstate(invalid="ignore"):
        b.put()
        seen = np.zeros((103, 16, 128), bool)
        bad = ~np.isfinite(b.v.astype(np.float64))
        for row, head, dim in np.argwhere(bad):
            seen[row:70 if row < 70 else 103, head * 8:head * 8 + 8, dim] = True
        for plane in (b.cache.value,):  # the finite values' attention: 0 in the places of the others
            plane[(plane & 0x7C00) == 0x7C00] = 0
        want, limit = wanted(b)
    assert np.array_equal(~np.isfinite(got), seen)
    B.check("finite ones", np.where(seen, 0, got), np.where(seen, 0, want), limit)
    assert pvlc.workspace_error(*ws) == 0


@WIDTHS
@pytest.mark.parametrize("counts,held,wide", [([40, 9, 17], [100, 64, 0], False), ([40, 9, 17], [100, 64, 0], True), ([50, 20], [6000, 700], True)])
def test_blocks_outside_the_planes(f32, counts, held, wide):
    """A block id outside the planes, among the rows that are held or the call's own, is reported and block 0 read; other
    sequences are as ever, and the rows of a block that is not there are not written."""
    import torch
    log(f"case: packed prefill, blocks outside the planes, held={held} f32={f32} wide={wide}")
    for bad, at in ((-1, 2), (None, 0), (-1, (held[0] + counts[0] - 1) // 16), (None, held[0] // 16 - 1)):
        b = B.Batch(counts, held, f32=f32, seed=41, room=5000 if wide else 0)
        b.upload()
        ws = workspace(b, b.width * 16)
        table = b.dtable.clone()
        table[0, at] = b.blocks if bad is None else bad
        launch(b, args_of(b, ws, block_tables=table))
        torch.cuda.synchronize()
        assert pvlc.workspace_error(*ws) == 2, at
        kept = [x[b.table[0, at]].copy() for x in (b.cache.key, b.cache.value)]
        b.put()
        for x, k in zip((b.cache.key, b.cache.value), kept):
            x[b.table[0, at]] = k
        b.check_planes(f"block {at}")
        some = np.arange(counts[0], int(b.offsets[-1]))
        want, limit = wanted(b, some)
        B.check("the others", b.out.float().cpu().numpy()[some], want, limit)
