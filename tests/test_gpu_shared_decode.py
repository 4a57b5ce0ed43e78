"""Decode of groups with shared pages against the plain form in 64 bits; planes and exponents byte for byte."""

import numpy as np
import pytest

import batches_ref as B
import q8_ref as R
from pvlc_testlib import log, pvlc

pytestmark = pytest.mark.gpu
CODES = pytest.mark.parametrize("code", [B.F16, R.E4M3, R.INT8])
WIDTHS = pytest.mark.parametrize("f32", [False, True])
# Calls of few rows run as paged decodes: `far` makes room for more rows than those have, and the sequences as short as they were.
FAR = pytest.mark.parametrize("far", [False, True])


class Groups(B.Batch):
    """Groups of sizes whose sequences have their first `shared` rows in common (in whole blocks) and `tails` of their own."""

    def __init__(self, sizes, shared, tails, code, f32, seed=0, far=True, **how):
        self.sizes, self.shared = list(sizes), list(shared)
        group = np.repeat(np.arange(len(sizes)), sizes)
        held = [shared[g] + t for g, t in zip(group, tails)]
        super().__init__([1] * len(group), held, code, f32, seed, **how)
        firsts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.firsts = firsts
        for i, g in enumerate(group):  # the others repeat the first one's entries
            whole = shared[g] // 16
            self.table[i, :whole] = self.table[firsts[g], :whole]
        if far:
            self.width = max(self.width, -(-220000 // self.n // 16))
            self.table = np.pad(self.table, ((0, 0), (0, self.width - self.table.shape[1])), constant_values=-1)

    def shared_args(self, ws, offsets=False, **change):
        import torch
        self.keep = change
        self.dshared = torch.tensor(self.shared, dtype=torch.int32, device="cuda")
        self.dfirsts = torch.from_numpy(self.firsts).cuda() if offsets else None
        base = dict(self.common(), num_seqs=self.n, num_groups=len(self.sizes), group_offsets=self.dfirsts, shared_lens=self.dshared,
                    cache_lens=self.dlens, max_context=self.width * 16, code=self.code, exponents=self.exponents, rotate_query=True,
                    workspace=ws[0], workspace_bytes=ws[1], block_tables=self.dtable)
        return pvlc.shared_decode_args(**{**base, **change})

    def workspace(self):
        import torch
        nbytes = pvlc.shared_decode_workspace_bytes(self.n, len(self.sizes), self.width * 16)
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        pvlc.workspace_init(ws, nbytes)
        return ws, nbytes

    def launch(self, args, stream=None):
        (pvlc.shared_decode_f32io if self.f32 else pvlc.shared_decode_f16)(args, self.dq, self.dk, self.dv, self.out, stream)

    def check(self, label, rotate_query=True, skipped=()):
        import torch
        torch.cuda.synchronize()
        for i in range(self.n):
            if i not in skipped:
                self.cache.put_rows(self.table[i], self.held[i], self.turned(self.k[i], i)[None],
                                    self.v[i].astype(np.float16).astype(np.float64)[None])
        self.check_planes(label)
        got = self.out.float().cpu().numpy()
        for i in range(self.n):
            if i in skipped:
                assert (got[i] == 9.0).all(), f"{label}: sequence {i}"
                continue
            k, v = self.cache.rows(self.table[i], self.held[i] + 1)
            q = self.turned(self.q[i], i) if rotate_query else self.q[i].astype(np.float16).astype(np.float64)
            out, big, most = B.attend(q[None], k, v, [self.held[i] + 1])
            B.check(f"{label} sequence {i}", got[i:i + 1], out, B.bound(out, big, most, self.held[i] + 1, self.f32, self.code))


def tails_of(n, most, seed=1):
    return np.random.default_rng(seed).integers(0, most + 1, n).tolist()


CASES = {
    # group sizes, shared rows, own rows
    "one": ([1], [0], [0]), "alone": ([1], [300], [7]), "beams": ([4], [157], tails_of(4, 40)), "beams_no_tail": ([4], [160], [0] * 4),
    "nothing_shared": ([3, 3], [0, 15], [0, 20, 130, 1, 16, 17]), "pages": ([2] * 5, [16, 33, 64, 200, 129], tails_of(10, 33)),
    "answers": ([23], [500], tails_of(23, 60)), "long": ([5, 5], [4000, 40], tails_of(10, 300)),
}


@CODES
@WIDTHS
@FAR
@pytest.mark.parametrize("name", list(CASES))
def test_groups_of_one_size(code, f32, far, name):
    log(f"case: shared decode {name} code={code} f32={f32} far={far}")
    sizes, shared, tails = CASES[name]
    c = Groups(sizes, shared, tails, code, f32, seed=len(name), far=far, positions=name == "pages", rope=name != "answers").upload()
    ws = c.workspace()
    c.launch(c.shared_args(ws, rotate_query=name != "beams"))
    c.check(name, rotate_query=name != "beams")
    assert pvlc.workspace_error(*ws) == 0


@CODES
@pytest.mark.parametrize("sizes", [[1, 7, 0, 3, 12], [3] * 70, [0, 40, 0]])
def test_groups_of_different_sizes(code, sizes):
    log(f"case: shared decode groups of {sizes[:6]}.. code={code}")
    shared = [16 * (i % 5) + i % 7 for i in range(len(sizes))]
    c = Groups(sizes, shared, tails_of(sum(sizes), 50), code, code == R.E4M3, seed=sum(sizes)).upload()
    ws = c.workspace()
    c.launch(c.shared_args(ws, offsets=True))
    c.check("sizes")
    assert pvlc.workspace_error(*ws) == 0


@CODES
def test_rows_that_are_not_shared_by_all(code):
    """A shared length beyond the group's shortest sequence counts as that one's."""
    log(f"case: shared decode, lengths beyond, code={code}")
    c = Groups([3], [96], [0, 5, 40], code, True, seed=2).upload()
    c.shared = [4000]
    ws = c.workspace()
    c.launch(c.shared_args(ws))
    c.check("beyond")
    assert pvlc.workspace_error(*ws) == 0


@CODES
@FAR
def test_errors_are_reported_and_skipped(code, far):
    import torch
    log(f"case: shared decode errors, code={code} far={far}")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    c = Groups([3, 2], [48, 16], [0, 5, 20, 3, 4], code, False, seed=3, far=far).upload()
    ws = c.workspace()
    lens = list(c.held)
    lens[1], lens[3] = -1, c.width * 16
    c.launch(c.shared_args(ws, offsets=True, cache_lens=ints(lens)))
    c.check("lengths", skipped=(1, 3))
    assert pvlc.workspace_error(*ws) == 1
    c = Groups([2], [32], [5, 9], code, False, seed=4, far=far).upload()  # a position outside the tables: no rotation
    ws = c.workspace()
    c.launch(c.shared_args(ws, positions=ints([c.table_rows, -1])))
    c.rope = False
    c.check("positions")
    assert pvlc.workspace_error(*ws) == 4


def test_steps_from_a_graph_beside_direct_calls():
    """A captured step replayed, and direct calls of another shape on the same workspace between the replays."""
    import torch
    log("case: shared decode from a graph")
    for code in (B.F16, R.E4M3):
        one = Groups([4], [700], [3, 9, 0, 40], code, True, seed=5).upload()
        two = Groups([2] * 9, [40] * 9, tails_of(18, 20), code, True, seed=6, far=False).upload()  # (a paged decode on the same words)
        nbytes = max(pvlc.shared_decode_workspace_bytes(c.n, len(c.sizes), c.width * 16) for c in (one, two))
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        pvlc.workspace_init(ws, nbytes)
        args = [c.shared_args((ws, nbytes)) for c in (one, two)]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            one.launch(args[0], stream)
        start = [x.clone() for x in one.planes + ([] if one.exponents is None else [one.exponents])]
        outs = []
        for _ in range(3):
            for d, s in zip(one.planes + ([] if one.exponents is None else [one.exponents]), start):
                d.copy_(s)
            one.out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            outs.append(one.out.clone())
            two.launch(args[1])
            torch.cuda.synchronize()
        assert all(torch.equal(outs[0], x) for x in outs)
        one.check("replayed")
        assert pvlc.workspace_error(ws, nbytes) == 0


def test_far_blocks():
    """Shared and own blocks whose elements lie beyond 2^31."""
    import torch
    log("case: shared decode, far blocks")
    c = Groups([3], [40], [2, 20, 9], B.F16, True, seed=7).upload()
    blocks = (1 << 31) // 4096 + 300
    ids = torch.from_numpy(np.arange(blocks - c.blocks, blocks).astype(np.int32)).cuda()
    planes = [torch.zeros(blocks * 4096, dtype=torch.int16, device="cuda") for _ in range(2)]
    for p, small in zip(planes, c.planes):
        p.view(blocks, 4096)[blocks - c.blocks:] = small.view(c.blocks, 4096)
    ws = c.workspace()
    c.launch(c.shared_args(ws, num_blocks=blocks, key_cache=planes[0], value_cache=planes[1], block_tables=torch.where(c.dtable < 0, -1, ids[c.dtable.clamp_min(0).long()])))
    torch.cuda.synchronize()
    for p, small in zip(planes, c.planes):
        small.copy_(p.view(blocks, 4096)[blocks - c.blocks:].view_as(small))
    c.check("far")


@CODES
def test_sequences_before_the_first_group_have_no_output(code):
    import torch
    log(f"case: shared decode, sequences before the first group, code={code}")
    c = Groups([9, 3, 2], [48, 33, 16], tails_of(14, 30), code, False, seed=8).upload()
    nbytes = pvlc.shared_decode_workspace_bytes(14, 2, c.width * 16)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda"), nbytes
    pvlc.workspace_init(*ws)
    c.launch(c.shared_args(ws, num_groups=2, group_offsets=torch.from_numpy(c.firsts[1:]).cuda(), shared_lens=torch.tensor([33, 16], dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    assert pvlc.workspace_error(*ws) == 0
    assert (c.out[:9] == 9.0).all()
    got = c.out.float().cpu().numpy()
    for i in range(9, 14):
        c.cache.put_rows(c.table[i], c.held[i], c.turned(c.k[i], i)[None], c.v[i].astype(np.float64)[None])
        k, v = c.cache.rows(c.table[i], c.held[i] + 1)
        out, big, most = B.attend(c.turned(c.q[i], i)[None], k, v, [c.held[i] + 1])
        B.check(f"sequence {i}", got[i:i + 1], out, B.bound(out, big, most, c.held[i] + 1, False, code))


@pytest.mark.parametrize("n", [4, 90])
def test_group_offsets_that_descend_are_reported(n):
    import torch
    log(f"case: shared decode, group offsets that descend, n={n}")
    for bad in (-1, 0, 10 ** 6):
        c = Groups([2] * n, [16] * n, [1] * (2 * n), B.F16, False, seed=n).upload()
        ws = c.workspace()
        firsts = c.firsts.copy()
        firsts[n // 2] = bad
        c.launch(c.shared_args(ws, group_offsets=torch.from_numpy(firsts).cuda()))
        assert pvlc.workspace_error(*ws) == 1


@CODES
def test_two_steps_at_once(code):
    """On two streams, each with its workspace, and pools of their own."""
    import torch
    log(f"case: shared decode, two at once, code={code}")
    pair = [Groups([5, 3], [900, 40], tails_of(8, 60, seed), code, seed == 1, seed=seed).upload() for seed in (1, 2)]
    spaces = [c.workspace() for c in pair]
    args = [c.shared_args(ws) if len(set(c.sizes)) == 1 else c.shared_args(ws, offsets=True) for c, ws in zip(pair, spaces)]
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    for c, a, s in zip(pair, args, streams):
        c.launch(a, s)
    for c, ws in zip(pair, spaces):
        c.check("at once")
        assert pvlc.workspace_error(*ws) == 0


@CODES
def test_replays_follow_the_lengths(code):
    """A captured step replayed as its sequences grow: lengths, shared lengths and rows change in place."""
    import torch
    log(f"case: shared decode, replays of a growing batch, code={code}")
    c = Groups([4, 4], [100, 31], tails_of(8, 40), code, True, seed=9, room=8).upload()
    ws = c.workspace()
    args = c.shared_args(ws)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        c.launch(args, stream)
    for step in range(4):
        c.out.fill_(9.0)
        graph.replay()
        c.check(f"step {step}")
        c.held = [t + 1 for t in c.held]
        c.dlens.add_(1)
        if step == 1:
            c.dshared[1] = 0  # (shared as before, attended as rows of each one's own)
    assert pvlc.workspace_error(*ws) == 0


@CODES
@pytest.mark.parametrize("offsets", [False, True])
def test_groups_of_sequences_that_do_not_fit(code, offsets):
    """A group whose sequences are all left out shares nothing, however far beyond the tables its shared length is; the other
    group, of the first sequences, is attended."""
    import torch
    log(f"case: shared decode, groups that do not fit, code={code} offsets={offsets}")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for length, beyond in ((-1, 4000), (None, 1 << 20), (-1, 0x7FFFFFFF)):
        c = Groups([3, 3], [48, 32], [0, 5, 20, 3, 4, 17], code, False, seed=23).upload()
        ws = c.workspace()
        lens = c.held[:3] + [c.width * 16 if length is None else length] * 3
        c.shared = [48, beyond]
        c.launch(c.shared_args(ws, offsets=offsets, cache_lens=ints(lens)))
        c.check("left out", skipped=(3, 4, 5))
        assert pvlc.workspace_error(*ws) == 1


@CODES
@FAR
@pytest.mark.parametrize("out", [(0,), (0, 1), (2, 5, 6), (0, 1, 2, 3)])
def test_sequences_left_out_beside_others(code, far, out):
    """Sequences that are done, with a negative length and a table of no blocks, and the others of their groups: the shared pages
    are the others', too."""
    import torch
    log(f"case: shared decode, sequences left out, code={code} far={far} out={out}")
    c = Groups([7], [64], [0, 5, 20, 3, 4, 17, 33], code, True, seed=24, far=far).upload()
    ws = c.workspace()
    lens, table = list(c.held), c.dtable.clone()
    for i in out:
        lens[i], table[i] = -1, -1
    c.launch(c.shared_args(ws, cache_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), block_tables=table))
    c.check("beside others", skipped=out)
    assert pvlc.workspace_error(*ws) == 1


# (8-bit pages hold an infinity as the largest code, and int8 no NaN; a paged decode gives NaN, too, where all that a wave has
# are scores of -infinity)
ODD = [(code, far, kind) for code, kinds in ((B.F16, ("nan", "cancel", "plus", "minus", "value")), (R.E4M3, ("nan",))) for far in (False, True)
       for kind in kinds if far or kind != "minus"]


@WIDTHS
@pytest.mark.parametrize("tail", [0, 1, 40])
@pytest.mark.parametrize("code,far,kind", ODD)
def test_new_rows_that_are_not_finite(code, f32, far, tail, kind):
    """A new key with a NaN, or with infinities whose products cancel, makes its head's outputs NaN, and so does one whose score
    is +infinity; a score of -infinity is a weight of 0.  An infinite value is infinite or NaN in its dim."""
    import torch
    log(f"case: shared decode, new row {kind} code={code} f32={f32} far={far} tail={tail}")
    c = Groups([3, 3], [64, 32], [tail] * 6, code, f32, seed=25, far=far, rope=False)
    c.q[:, :, :2] = np.abs(c.q[:, :, :2]) + np.asarray(0.5, c.q.dtype)
    if kind == "value":
        c.v[1, 1, 3] = np.inf
    else:
        c.k[1, 1, :2] = {"nan": (np.nan, 1), "cancel": (np.inf, -np.inf), "plus": (np.inf, 1), "minus": (-np.inf, 1)}[kind]
    c.upload()
    ws = c.workspace()
    c.launch(c.shared_args(ws))
    torch.cuda.synchronize()
    got, odd = c.out.float().cpu().numpy(), np.zeros((6, 16, 128), bool)
    if kind == "value":
        odd[1, 8:, 3] = True
    elif kind != "minus":
        odd[1, 8:] = True
    assert np.array_equal(~np.isfinite(got), odd)
    with np.errstate(invalid="ignore"):
        for i in range(6):
            c.cache.put_rows(c.table[i], c.held[i], c.k[i].astype(np.float16).astype(np.float64)[None], c.v[i].astype(np.float16).astype(np.float64)[None])
    c.check_planes(kind)
    for i in range(6):
        q = c.q[i].astype(np.float16).astype(np.float64)[None]
        k, v = (np.where(np.isfinite(x), x, 0) for x in c.cache.rows(c.table[i], c.held[i] + 1))
        out, big, most = B.attend(q, k, v, [c.held[i] + 1])
        if i == 1 and kind == "minus":
            out[:, 8:] = B.attend(q, k, v, [c.held[i]])[0][:, 8:]
        mine = ~odd[i:i + 1]
        B.check(f"{kind} sequence {i}", np.where(mine, got[i:i + 1], 0), np.where(mine, out, 0), B.bound(out, big, most, c.held[i] + 1, f32, code))


@pytest.mark.parametrize("code", [B.F16, R.E4M3])
@FAR
def test_shared_rows_that_are_not_finite(code, far):
    """Keys of NaN among the shared rows make every output of their head NaN, one or all of them."""
    import torch
    log(f"case: shared decode, shared rows that are not finite, code={code} far={far}")
    for rows in ([5], range(64)):
        c = Groups([3], [64], [0, 5, 20], code, True, seed=26, far=far, rope=False)
        bad = 0x7F if code == R.E4M3 else 0x7E00
        at = R.KEY_AT if code == R.E4M3 else B.KEY_AT
        for r in rows:
            c.cache.key[c.table[0, r // 16], 1, at[r % 16]] = bad
        c.upload()
        ws = c.workspace()
        c.launch(c.shared_args(ws))
        torch.cuda.synchronize()
        got = c.out.cpu().numpy()
        assert np.isnan(got[:, 8:]).all() and np.isfinite(got[:, :8]).all(), (len(rows))


@CODES
@FAR
@pytest.mark.parametrize("where", ["shared", "own"])
def test_blocks_outside_the_planes(code, far, where):
    """A block id outside the planes among the rows that are held is reported, block 0 read; others' outputs and all new rows are
    as ever."""
    import torch
    log(f"case: shared decode, blocks outside the planes, code={code} far={far} where={where}")
    for bad in (-1, None):
        c = Groups([3, 2], [64, 160], [40, 33, 70, 20, 0], code, False, seed=27, far=far).upload()
        ws = c.workspace()
        table = c.dtable.clone()
        if where == "shared":
            table[0:3, 2] = c.blocks if bad is None else bad
        else:
            table[2, 5] = c.blocks if bad is None else bad
        c.launch(c.shared_args(ws, offsets=True, block_tables=table))
        torch.cuda.synchronize()
        assert pvlc.workspace_error(*ws) == 2
        got = c.out.float().cpu().numpy()
        for i in range(5):
            c.cache.put_rows(c.table[i], c.held[i], c.turned(c.k[i], i)[None], c.v[i].astype(np.float64)[None])
        c.check_planes(where)
        for i in (3, 4) if where == "shared" else (0, 1, 3, 4):
            k, v = c.cache.rows(c.table[i], c.held[i] + 1)
            out, big, most = B.attend(c.turned(c.q[i], i)[None], k, v, [c.held[i] + 1])
            B.check(f"{where} sequence {i}", got[i:i + 1], out, B.bound(out, big, most, c.held[i] + 1, False, code))
