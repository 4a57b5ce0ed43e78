"""Forks, compaction and copies of pages against the plain form (pages_ref): tables, lengths, counts, free bits, error
bits and every byte of every plane."""

import numpy as np
import pytest

import pages_ref as P
from pvlc_testlib import log, pvlc

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Both:
    """A pool on the device and its plain form; every call is made on both and compared."""

    def __init__(self, blocks, width, layers=2, sizes=(64, 32, 4), rows=64, seed=0):
        import torch
        g = np.random.default_rng(seed)
        self.ref = P.Pool(blocks, width, [g.integers(0, 256, (layers, blocks, n)).astype(np.uint8) for n in sizes])
        self.planes = [dev(p) for p in self.ref.planes]
        self.refs, self.mask = torch.full((blocks,), 7, dtype=torch.int32, device="cuda"), torch.zeros(-(-blocks // 32), dtype=torch.int32, device="cuda")
        nbytes = pvlc.kv_pages_workspace_bytes(blocks, rows)
        self.ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        pvlc.workspace_init(self.ws, nbytes)
        self.pool = pvlc.kv_page_pool(num_blocks=blocks, max_blocks_per_seq=width, num_layers=layers, planes=self.planes,
                                      ref_counts=self.refs, free_mask=self.mask, workspace=self.ws, workspace_bytes=nbytes)
        self.nbytes, self.width, self.blocks = nbytes, width, blocks
        pvlc.kv_pages_reset(self.pool)
        self.tables, self.lens = np.empty((0, width), np.int32), np.empty(0, np.int32)
        self.same("reset")

    def same(self, what):
        import torch
        torch.cuda.synchronize()
        np.testing.assert_array_equal(self.refs.cpu().numpy(), self.ref.refs, what)
        np.testing.assert_array_equal(self.mask.cpu().numpy().view(np.uint32), self.ref.free_mask(), what)
        for a, b in zip(self.planes, self.ref.planes):
            np.testing.assert_array_equal(a.cpu().numpy(), b, what)

    def error(self):
        e = pvlc.workspace_error(self.ws, self.nbytes)
        self.ws[:4] = 0
        return e

    def fork(self, rows_out, what, parents=None, reserve=0, appended=0, keep_inputs=False, errors=0, tables=None, lens=None, stream=None):
        import torch
        tables = self.tables if tables is None else tables
        lens = self.lens if lens is None else lens
        t_in, l_in = dev(tables.astype(np.int32)), dev(lens.astype(np.int32))
        t_out = torch.full((rows_out, self.width), 99, dtype=torch.int32, device="cuda")
        l_out = torch.full((rows_out,), 99, dtype=torch.int32, device="cuda")
        p = None if parents is None else dev(np.asarray(parents, np.int32))
        r = dev(np.asarray(reserve, np.int32)) if np.ndim(reserve) else None
        torch.cuda.synchronize()
        pvlc.kv_pages_fork(self.pool, rows_in=len(tables), rows_out=rows_out, tables_in=t_in, lens_in=l_in, tables_out=t_out,
                           lens_out=l_out, parents=p, reserve=r, reserve_tokens=0 if r is not None else reserve, appended=appended,
                           keep_inputs=keep_inputs, stream=stream)
        torch.cuda.synchronize()
        want_t, want_l, want_e = self.ref.fork(tables, lens, rows_out, parents, reserve, appended, keep_inputs)
        np.testing.assert_array_equal(t_out.cpu().numpy(), want_t, what)
        np.testing.assert_array_equal(l_out.cpu().numpy(), want_l, what)
        self.same(what)
        assert self.error() == want_e == errors, what
        return want_t, want_l

    def step(self, *a, **k):
        self.tables, self.lens = self.fork(*a, **k)

    def compact(self, what):
        import torch
        t = dev(self.tables)
        forward = torch.full((self.blocks,), -5, dtype=torch.int32, device="cuda")
        pvlc.kv_pages_compact(self.pool, rows=len(self.tables), tables=t, forward=forward)
        torch.cuda.synchronize()
        self.tables, want = self.ref.compact(self.tables)
        np.testing.assert_array_equal(t.cpu().numpy(), self.tables, what)
        np.testing.assert_array_equal(forward.cpu().numpy(), want, what)
        self.same(what)


@pytest.mark.parametrize("blocks,width,layers,sizes", [(40, 6, 1, (16,)), (97, 8, 3, (64, 32, 4)), (5000, 40, 2, (4096, 4096, 4)),
                                                       (70000, 6, 1, (4,)), (64, 6, 2, (12, 20, 8, 4))])
def test_a_page_is_searched_with_beams(blocks, width, layers, sizes):
    """Admission, a prompt's fan-out that keeps the prompt, beam steps that append and cross block borders, sequences
    that end, compaction, truncation, and everything freed."""
    log(f"case: pages blocks={blocks} width={width} layers={layers} sizes={sizes}")
    b, g = Both(blocks, width, layers, sizes, seed=blocks), np.random.default_rng(blocks)
    b.step(3, "admission", parents=[-1, -1, -1], reserve=[37, 16, 0])
    b.lens = np.array([37, 16, 0], np.int32)
    b.step(8, "fan-out", parents=[0, 1, 0, 0, 2, 1, 0, 2], reserve=1)
    for i in range(20):
        parents = g.integers(0, len(b.tables), 8)
        if i % 7 == 3:
            parents[g.integers(0, 8)] = -1
        b.step(8, f"beam step {i}", parents=parents, reserve=int(g.integers(0, 3)) or 1, appended=1 if i % 5 else 0)
        if i % 6 == 5:
            b.compact(f"compaction {i}")
    kept = b.fork(5, "fan-out beside its inputs", parents=[0, 3, 3, 1, 0], reserve=2, keep_inputs=True)
    b.tables, b.lens = np.concatenate([b.tables, kept[0]]), np.concatenate([b.lens, kept[1]])
    b.lens = np.minimum(b.lens, g.integers(0, 40, len(b.lens))).astype(np.int32)
    b.step(len(b.tables), "truncation")
    b.compact("after truncation")
    b.step(4, "identity of the first four, the others end")
    b.step(6, "two more", reserve=17)
    b.fork(0, "all freed")
    assert not b.ref.refs.any()


def test_a_shared_last_block_is_copied_for_everyone():
    """Two rows cut to a length inside a block that they share: neither may write it."""
    log("case: pages shared tail")
    b = Both(30, 4)
    b.step(1, "admission", parents=[-1], reserve=40)
    b.lens = np.array([40], np.int32)
    b.step(2, "fan-out", parents=[0, 0], reserve=1)
    b.lens = np.array([20, 25], np.int32)  # block 1 is shared
    b.step(3, "cut", parents=[0, 1, 1], reserve=1)


def test_reserved_pages_stay_with_the_first_child():
    log("case: pages reserve")
    b = Both(60, 10)
    b.step(2, "admission", parents=[-1, -1], reserve=100)
    b.lens = np.array([20, 48], np.int32)
    b.step(4, "children", parents=[1, 0, 1, 0], reserve=60)
    b.step(4, "less", reserve=5)
    b.step(4, "nothing", reserve=0)


def test_too_few_pages_change_nothing():
    log("case: pages exhausted")
    b = Both(10, 8)
    b.step(2, "admission", parents=[-1, -1], reserve=64)
    b.lens = np.array([50, 33], np.int32)
    before = b.tables.copy(), b.lens.copy()
    b.fork(8, "beyond the pool", parents=[0, 0, 0, 1, 1, 1, 0, 1], reserve=1, errors=P.EXHAUSTED)
    b.tables, b.lens = before
    b.step(3, "within it", parents=[0, 1, 0], reserve=1)


def test_exactly_all_pages():
    log("case: pages all taken")
    b = Both(33, 33)
    b.step(2, "all", parents=[-1, -1], reserve=[32 * 16, 16])
    b.compact("nothing moves")
    b.fork(3, "none left", reserve=1, errors=P.EXHAUSTED)
    b.step(1, "one frees", parents=[1])
    b.compact("a page moves")
    b.fork(0, "none")


def test_bad_rows_set_their_bits_and_hurt_no_other():
    log("case: pages bad inputs")
    b = Both(50, 5)
    b.step(4, "admission", parents=[-1] * 4, reserve=40)
    b.lens = np.array([40, 39, 38, 37], np.int32)
    good = b.tables.copy()
    b.fork(3, "parent beyond", parents=[0, 4, -2], keep_inputs=True, errors=P.BAD_PARENT)
    b.fork(3, "no room", parents=[0, 1, 2], reserve=100, keep_inputs=True, errors=P.NO_ROOM)
    bad = good.copy()
    bad[1, 0], bad[2, 2] = 50, -7
    b.fork(4, "blocks outside", tables=bad, errors=P.BAD_BLOCK)
    b = Both(50, 5)
    b.step(2, "admission", parents=[-1] * 2, reserve=40)
    b.fork(2, "lengths", lens=np.array([81, -1], np.int32), errors=P.BAD_LENGTH)


def test_a_page_in_no_count_sets_a_bit():
    import torch
    log("case: pages count below zero")
    b = Both(20, 2)
    t, n = dev(np.array([[3, 4]], np.int32)), dev(np.array([32], np.int32))
    pvlc.kv_pages_fork(b.pool, rows_in=1, rows_out=0, tables_in=t, lens_in=n)
    torch.cuda.synchronize()
    assert b.error() == P.BAD_COUNT


def test_many_rows_and_a_wide_table():
    log("case: pages 2500 rows")
    b, g = Both(12000, 70, layers=1, sizes=(4,), rows=2600), np.random.default_rng(4)
    reserve = g.integers(0, 60, 2500)
    reserve[7] = 1100
    b.step(2500, "admission", parents=np.full(2500, -1), reserve=reserve)
    b.lens = reserve.astype(np.int32)
    b.step(2600, "reorder", parents=g.integers(-1, 2500, 2600), reserve=1)
    b.compact("compaction")


def test_compaction_of_random_pools():
    for seed in range(12):
        g = np.random.default_rng(seed)
        blocks = int(g.integers(1, 400))
        log(f"case: pages compaction seed={seed} blocks={blocks}")
        b = Both(blocks, 12, layers=2, sizes=(16, 4), seed=seed)
        n = int(g.integers(1, 12))
        reserve = g.integers(0, max(1, blocks // n) * 16, n)
        reserve = np.minimum(reserve, 12 * 16)
        b.step(n, "admission", parents=[-1] * n, reserve=reserve)
        b.lens = reserve.astype(np.int32)
        b.step(n, "some end", parents=[i if g.random() < 0.5 else -1 for i in range(n)])
        b.compact("compaction")
        b.compact("again")


def test_copies_between_pools_and_on_a_stream():
    import torch
    log("case: pages copied")
    a, b = Both(20, 2, seed=1), Both(31, 3, seed=2)
    src, dst = np.array([3, 19, 0, 7], np.int32), np.array([30, 1, 5, 0], np.int32)
    side = torch.cuda.Stream()
    s, d = dev(src), dev(dst)
    side.wait_stream(torch.cuda.current_stream())
    pvlc.kv_pages_copy(a.pool, s, b.pool, d, 4, side)
    side.synchronize()
    for x, y in zip(a.ref.planes, b.ref.planes):
        y[:, dst] = x[:, src]
    b.same("copied")
    s2, d2 = dev(np.array([20, 2], np.int32)), dev(np.array([2, 31], np.int32))
    pvlc.kv_pages_copy(a.pool, s2, b.pool, d2, 2)
    torch.cuda.synchronize()
    b.same("bad ids")
    assert b.error() == P.BAD_BLOCK
    s3, d3 = dev(np.array([4, 5], np.int32)), dev(np.array([8, 9], np.int32))
    pvlc.kv_pages_copy(b.pool, s3, b.pool, d3, 2)
    for y in b.ref.planes:
        y[:, [8, 9]] = y[:, [4, 5]]
    b.same("within a pool")


def test_a_fork_and_a_compaction_replayed_from_a_graph():
    """Rows forked from a prompt that stays, then freed, then compacted: each replay, with eager work between, leaves the
    same state."""
    import torch
    log("case: pages graph")
    b = Both(200, 6)
    b.step(2, "admission", parents=[-1, -1], reserve=[45, 20])
    b.lens = np.array([45, 20], np.int32)
    t, n = dev(b.tables), dev(b.lens)
    t_out, n_out = torch.zeros((6, 6), dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    parents = dev(np.array([0, 1, 0, 0, 1, 0], np.int32))

    def steps(stream):
        pvlc.kv_pages_fork(b.pool, rows_in=2, rows_out=6, tables_in=t, lens_in=n, tables_out=t_out, lens_out=n_out, parents=parents,
                           reserve_tokens=1, keep_inputs=True, stream=stream)
        pvlc.kv_pages_fork(b.pool, rows_in=6, rows_out=0, tables_in=t_out, lens_in=n_out, stream=stream)
        pvlc.kv_pages_compact(b.pool, rows=2, tables=t, stream=stream)

    want = b.ref.fork(b.tables, b.lens, 6, [0, 1, 0, 0, 1, 0], 1, 0, True)
    b.ref.fork(want[0], want[1], 0)
    b.tables, _ = b.ref.compact(b.tables)
    steps(torch.cuda.current_stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(t_out.cpu().numpy(), want[0])
    b.same("eager")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(torch.cuda.current_stream())
    for i in range(4):
        t_out.fill_(77)
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(t_out.cpu().numpy(), want[0])
        np.testing.assert_array_equal(t.cpu().numpy(), b.tables)
        b.same(f"replay {i}")
    assert b.error() == 0


def test_pages_beyond_32_bits_of_offset_and_rows_behind_the_last():
    """Planes of more than 4 GiB; rows of the output behind rows_out stay as they were."""
    import torch
    log("case: pages in planes of more than 4 GiB")
    blocks, size = 70000, 65536
    plane = torch.zeros(1, blocks, size, dtype=torch.uint8, device="cuda")
    refs, mask = torch.ones(blocks, dtype=torch.int32, device="cuda"), torch.zeros(-(-blocks // 32), dtype=torch.int32, device="cuda")
    refs[-40:] = 0
    bits = np.zeros(-(-blocks // 32) * 32, bool)
    bits[blocks - 40:blocks] = True
    mask.copy_(dev(np.packbits(bits, bitorder="little").view(np.int32)))
    nbytes = pvlc.kv_pages_workspace_bytes(blocks, 4)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, nbytes)
    pool = pvlc.kv_page_pool(num_blocks=blocks, max_blocks_per_seq=3, num_layers=1, planes=[plane], ref_counts=refs, free_mask=mask,
                             workspace=ws, workspace_bytes=nbytes)
    last = blocks - 50
    plane[0, last] = torch.arange(size, device="cuda").to(torch.uint8) + 3
    t, n = dev(np.array([[5, last, -1]], np.int32)), dev(np.array([20], np.int32))
    out, lens = torch.full((5, 3), 44, dtype=torch.int32, device="cuda"), torch.full((5,), 44, dtype=torch.int32, device="cuda")
    pvlc.kv_pages_fork(pool, rows_in=1, rows_out=3, tables_in=t, lens_in=n, tables_out=out, lens_out=lens, parents=dev(np.zeros(3, np.int32)))
    torch.cuda.synchronize()
    first = blocks - 40
    np.testing.assert_array_equal(out.cpu().numpy(), [[5, last, -1], [5, first, -1], [5, first + 1, -1], [44] * 3, [44] * 3])
    np.testing.assert_array_equal(lens.cpu().numpy(), [20, 20, 20, 44, 44])
    assert torch.equal(plane[0, first], plane[0, last]) and torch.equal(plane[0, first + 1], plane[0, last])
    assert not plane[0, first + 2:].any() and not plane[0, :last].any()
    assert pvlc.workspace_error(ws, nbytes) == 0


def test_a_pool_of_more_pages_than_one_turn_names():
    """140000 pages: four words of the mask a thread, and free pages in more than one turn of the workgroup."""
    log("case: pages in a pool of 140000")
    b, g = Both(140000, 70, layers=1, sizes=(4,), rows=2600), np.random.default_rng(9)
    b.step(2000, "admission", parents=np.full(2000, -1), reserve=1100)
    b.lens = g.integers(0, 1100, 2000).astype(np.int32)
    b.step(1500, "reorder and truncation", parents=g.integers(-1, 2000, 1500), reserve=20)
    b.lens = np.minimum(b.lens + 20, 70 * 16).astype(np.int32)
    b.compact("compaction")
    b.step(2600, "fan-out", parents=g.integers(0, 1500, 2600), reserve=1)
    b.step(3, "most are freed")
    b.step(3, "one new, one twice", parents=[-1, 0, 0], reserve=16)


def test_two_graphs_share_a_pool():
    """A fork out, and a fork back with a compaction, captured apart on one workspace and replayed in turn."""
    import torch
    log("case: pages two graphs")
    b = Both(60, 4, rows=8)
    b.step(2, "admission", parents=[-1, -1], reserve=[30, 17])
    b.lens = np.array([30, 17], np.int32)
    t, n = dev(b.tables), dev(b.lens)
    t_out, n_out = torch.zeros((5, 4), dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    parents = dev(np.array([1, 0, 1, 0, 0], np.int32))

    def out(stream):
        pvlc.kv_pages_fork(b.pool, rows_in=2, rows_out=5, tables_in=t, lens_in=n, tables_out=t_out, lens_out=n_out, parents=parents,
                           reserve_tokens=1, keep_inputs=True, stream=stream)

    def back(stream):
        pvlc.kv_pages_fork(b.pool, rows_in=5, rows_out=0, tables_in=t_out, lens_in=n_out, stream=stream)
        pvlc.kv_pages_compact(b.pool, rows=2, tables=t, stream=stream)

    graphs = []
    torch.cuda.synchronize()
    for call in (out, back):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(torch.cuda.current_stream())
        graphs.append(graph)
    for i in range(4):
        graphs[0].replay()
        torch.cuda.synchronize()
        want = b.ref.fork(b.tables, b.lens, 5, [1, 0, 1, 0, 0], 1, 0, True)
        np.testing.assert_array_equal(t_out.cpu().numpy(), want[0])
        b.same(f"out {i}")
        graphs[1].replay()
        torch.cuda.synchronize()
        b.ref.fork(want[0], want[1], 0)
        b.tables, _ = b.ref.compact(b.tables)
        np.testing.assert_array_equal(t.cpu().numpy(), b.tables)
        b.same(f"back {i}")
    assert b.error() == 0


def test_copies_replayed_from_a_graph():
    """Pages swapped through a third one, captured: after two replays they are where they were."""
    import torch
    log("case: pages copied from a graph")
    b = Both(12, 2, seed=8)
    one, two, three = (dev(np.array(x, np.int32)) for x in ([4, 7], [9, 2], [1, 0]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for s, d in ((one, three), (two, one), (three, two)):
            pvlc.kv_pages_copy(b.pool, s, b.pool, d, 2, torch.cuda.current_stream())
    for i in range(4):
        graph.replay()
        for y in b.ref.planes:
            y[:, [1, 0]] = y[:, [4, 7]]
            y[:, [4, 7]] = y[:, [9, 2]]
            y[:, [9, 2]] = y[:, [1, 0]]
        b.same(f"replay {i}")
    assert b.error() == 0
