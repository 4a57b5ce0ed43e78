"""Decode over the 8-bit cache against the plain form in 64 bits: the attention within the error bound of its f32
evaluation (q8_ref.attend_bound, plus fp16's rounding of the output), the planes and exponents byte for byte."""

import numpy as np
import pytest

import q8_ref as R
from pvlc_testlib import log, pvlc, to_dev_f32, to_dev_i32

pytestmark = pytest.mark.gpu

BASE = 500000.0


def workspace(n, context, partition=0):
    import torch
    nbytes = pvlc.decode_workspace_bytes(n, context, partition)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, nbytes)
    return ws, nbytes


class Case:
    """Sequences of `lens` cached rows in a pool of shuffled blocks (or contiguous ones), filled with NaN codes and
    exponents of 255 where no row is."""

    def __init__(self, lens, code, f32, seed, paged=True, spare=2, scale=1.0, room=1):
        g = self.g = np.random.default_rng(seed)
        self.lens, self.code, self.f32 = np.asarray(lens, np.int32), code, f32
        n = self.n = len(lens)
        self.width = max(-(-(int(t) + room) // 16) for t in lens)
        self.blocks = n * self.width + spare
        ids = g.permutation(self.blocks) if paged else np.arange(self.blocks)
        self.table = ids[:n * self.width].reshape(n, self.width).astype(np.int32)
        self.paged = paged
        self.cache = R.Cache(self.blocks, code, fill=0xFF)
        self.cos, self.sin = pvlc.rope_table(BASE, max(self.lens) + 70)
        for i, t in enumerate(self.lens):
            if t:
                k, v = self.rows(int(t), scale)
                self.cache.put_rows(self.table[i], 0, k, v)
        self.operands()

    def rows(self, t, scale=1.0):
        k = (self.g.standard_normal((t, 2, 128)) * np.exp(0.7 * self.g.standard_normal((2, 128))) * scale).astype(np.float16)
        return k, (self.g.standard_normal((t, 2, 128)) * scale).astype(np.float16)

    def operands(self, scale=1.0):
        kind = np.float32 if self.f32 else np.float16
        self.q = self.g.standard_normal((self.n, 16, 128)).astype(kind)
        self.nk = (self.g.standard_normal((self.n, 2, 128)) * scale).astype(kind)
        self.nv = (self.g.standard_normal((self.n, 2, 128)) * scale).astype(kind)

    def upload(self):
        import torch
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.dev = [put(a.copy()) for a in (self.cache.key, self.cache.value, self.cache.exponents)]
        self.dtable, self.dlens = to_dev_i32(self.table), to_dev_i32(self.lens)
        self.dcos, self.dsin = to_dev_f32(self.cos), to_dev_f32(self.sin)
        return self

    def args(self, ws, *, ragged=True, rope=True, rotate_query=True, partition=0, positions=None, context=None):
        import torch
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.dq, self.dk, self.dv = put(self.q), put(self.nk), put(self.nv)
        self.out = torch.full((self.n, 16, 128), 9.0, dtype=self.dq.dtype, device="cuda")
        self.positions = None if positions is None else to_dev_i32(positions)
        operands = dict.fromkeys(("query", "new_key", "new_value", "out")) if self.f32 else dict(
            query=self.dq, new_key=self.dk, new_value=self.dv, out=self.out)
        lens = dict(cache_lens=self.dlens) if ragged else dict(uniform_cache_len=int(self.lens[0]))
        return pvlc.paged_decode_q8_args(
            num_seqs=self.n, num_blocks=self.blocks, max_blocks_per_seq=self.width, code=self.code,
            block_tables=self.dtable if self.paged else None, key_cache=self.dev[0], value_cache=self.dev[1],
            exponents=self.dev[2], workspace=ws[0], workspace_bytes=ws[1], max_context=context or self.width * 16,
            rope_cos=self.dcos if rope else None, rope_sin=self.dsin if rope else None,
            rope_rows=self.cos.shape[0] if rope else 0, rotate_query=rotate_query, partition_tokens=partition,
            positions=self.positions, **operands, **lens)

    def launch(self, args, stream=None):
        if self.f32:
            pvlc.paged_decode_q8_f32io(args, self.dq, self.dk, self.dv, self.out, stream)
        else:
            pvlc.paged_decode_q8_f16(args, stream)

    def want(self, rope=True, rotate_query=True, positions=None):
        """Appends to self.cache and attends: outputs [n][16][128] f64 and their bounds."""
        outs, bounds = [], []
        for i, t in enumerate(self.lens):
            pos = int(t if positions is None else positions[i])
            turn = (lambda x: R.rotate(x, self.cos[pos], self.sin[pos])) if rope else (lambda x: x.astype(np.float16).astype(np.float64))
            k = turn(self.nk[i])
            q = turn(self.q[i]) if rotate_query else self.q[i].astype(np.float16).astype(np.float64)
            v = self.nv[i].astype(np.float16).astype(np.float64)
            self.cache.put_rows(self.table[i], int(t), k[None], v[None])
            keys, values = self.cache.rows(self.table[i], int(t) + 1)
            out, big = R.attend(q, keys, values)
            bound = R.attend_bound(big, int(t) + 1, values)
            outs.append(out)
            bounds.append(np.full_like(out, bound) if self.f32 else bound * (1 + 2.0 ** -11) + np.abs(out) * 2.0 ** -11 + 2.0 ** -25)
        return np.stack(outs), np.stack(bounds)

    def check(self, label, **how):
        import torch
        torch.cuda.synchronize()
        want, bound = self.want(**how)
        got = self.out.cpu().numpy().astype(np.float64)
        ratio = np.abs(got - want) / bound
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        print(f"[q8] {label}: error / bound {ratio.max():.3g}, rel {rel:.3g}", flush=True)
        assert np.isfinite(got).all(), label
        assert ratio.max() <= 1, label
        for name, d in zip(("key", "value", "exponents"), self.dev):
            bad = np.argwhere(d.cpu().numpy() != getattr(self.cache, name))
            assert bad.size == 0, f"{label}: {name} differs at {bad[0]} ({len(bad)} places)"
        return got


CODES = pytest.mark.parametrize("code", [R.E4M3, R.INT8])
WIDTHS = pytest.mark.parametrize("f32", [False, True])


@CODES
@WIDTHS
@pytest.mark.parametrize("t", [0, 1, 15, 16, 17, 63, 64, 130, 300, 1157, 2047])
def test_one_sequence(code, f32, t):
    log(f"case: q8 decode one sequence t={t} code={code} f32={f32}")
    c = Case([t], code, f32, seed=t * 4 + code * 2 + f32, paged=t % 2 == 0).upload()
    ws = workspace(1, c.width * 16)
    c.launch(c.args(ws, ragged=False, rotate_query=t != 300))
    c.check(f"t={t}", rotate_query=t != 300)
    assert pvlc.workspace_error(*ws) == 0


@CODES
def test_layers_of_one_length_in_one_launch(code):
    log(f"case: q8 decode 18 caches, code={code}")
    c = Case([700] * 18, code, code == R.INT8, seed=5, paged=False).upload()
    ws = workspace(18, c.width * 16)
    c.launch(c.args(ws, ragged=False, rope=False))
    c.check("18 caches", rope=False, rotate_query=False)


@CODES
@WIDTHS
def test_ragged_batch(code, f32):
    log(f"case: q8 decode ragged batch code={code} f32={f32}")
    c = Case([0, 1, 15, 16, 31, 32, 100, 257, 511, 900, 64, 3, 48], code, f32, seed=11 + code).upload()
    positions = [int(t) + 3 for t in c.lens]
    ws = workspace(c.n, c.width * 16)
    c.launch(c.args(ws, positions=positions))
    c.check("ragged", positions=positions)


@CODES
@WIDTHS
def test_streaming_batch(code, f32):
    """More workgroups than two rounds: the persistent kernel and its merge; up to 64 sequences are numbered in lanes,
    more in LDS."""
    for n, hi in ((40, 1500), (70, 700)):
        log(f"case: q8 decode streaming batch n={n} code={code} f32={f32}")
        lens = np.random.default_rng(n).integers(0, hi, n)
        lens[0], lens[1] = hi, 0
        c = Case(lens, code, f32, seed=21 + code).upload()
        ws = workspace(c.n, c.width * 16, 32)
        c.launch(c.args(ws, partition=32 if hi < 2048 else 0))
        c.check(f"streaming n={n}")


@pytest.mark.parametrize("t,partition", [(5000, 0), (5000, 512), (9001, 4096), (20000, 0)])
def test_long_caches(t, partition):
    log(f"case: q8 decode t={t} partition={partition}")
    c = Case([t, 77], R.E4M3 if t == 5000 else R.INT8, True, seed=t).upload()
    ws = workspace(2, c.width * 16, partition)
    c.launch(c.args(ws, partition=partition))
    c.check(f"t={t} P={partition}")


@pytest.mark.parametrize("partition", [16, 48, 64, 80, 128, 192, 208, 320, 384])
def test_partitions(partition):
    log(f"case: q8 decode partition={partition}")
    c = Case([partition * 3 + 5, partition, partition - 1, 1], R.INT8, True, seed=partition).upload()
    ws = workspace(4, c.width * 16, partition)
    c.launch(c.args(ws, partition=partition))
    c.check(f"P={partition}")


@CODES
@WIDTHS
def test_growing_a_sequence_row_by_row(code, f32):
    """Rows of very different sizes, so that exponents grow within a block (all four bits of growth and none), from an
    empty cache over two block borders; one workspace, one set of buffers."""
    log(f"case: q8 decode grows row by row code={code} f32={f32}")
    c = Case([0, 13], code, f32, seed=31, room=40).upload()
    ws = workspace(2, c.width * 16)
    for step in range(36):
        c.operands(scale=[1.0, 1.0, 7.0, 1e-3, 30.0, 0.0, 2.0, 900.0, 1.0][step % 9])
        c.launch(c.args(ws))
        c.check(f"step {step}")
        c.lens += 1
        c.dlens += 1
    assert pvlc.workspace_error(*ws) == 0


@CODES
def test_values_of_very_different_blocks(code):
    """Blocks whose values differ by 2^24: one reference serves the weights and the sum."""
    log(f"case: q8 decode value scales code={code}")
    c = Case([90], code, True, seed=41)
    for b in range(5):
        k, v = c.rows(16)
        c.cache.put(c.table[0][b], 0, k, (v.astype(np.float64) * 2.0 ** (8 - 6 * b)).astype(np.float16))
    c.upload()
    ws = workspace(1, c.width * 16)
    c.launch(c.args(ws))
    c.check("scales")


def test_device_errors():
    """A length without room, a block outside the planes and a position outside the tables set their bits; the other
    sequences are right, and a bad block's row is not written."""
    import torch
    log("case: q8 decode device errors")
    c = Case([40, 33, 20, 50], R.E4M3, True, seed=51).upload()
    c.dlens[0] = c.width * 16
    bad = c.dtable.clone()
    bad[1, 2] = c.blocks
    c.dtable = bad
    ws = workspace(4, c.width * 16)
    before = [d.clone() for d in c.dev]
    c.launch(c.args(ws, positions=[40, 33, 10 ** 6, 50]))
    torch.cuda.synchronize()
    assert pvlc.workspace_error(*ws) == 7
    assert (c.out[0] == 9).all()
    last = int(c.table[1][2])
    for d, b in zip(c.dev, before):
        assert torch.equal(d[last], b[last])
    want, bound = c.want(positions=[40, 33, 20, 50])
    assert (np.abs(c.out[3].cpu().numpy() - want[3]) <= bound[3]).all()


def test_stream_workspace_and_graph():
    """A launch on another stream, the fp16 decode's workspace shared, and replays of a captured launch with eager work
    between them: every result the same bits."""
    import torch
    log("case: q8 decode from a graph")
    c = Case([300, 20, 999], R.INT8, False, seed=61).upload()
    ws = workspace(3, c.width * 16)
    args = c.args(ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.launch(args, side)
    side.synchronize()
    first = torch.from_numpy(c.check("side stream")).clone()
    rows = torch.zeros(3 * 16 * 128, dtype=torch.float16, device="cuda")
    planes = [torch.zeros(c.blocks * 4096, dtype=torch.float16, device="cuda") for _ in range(2)]
    f16 = pvlc.paged_decode_args(
        num_seqs=3, num_blocks=c.blocks, max_blocks_per_seq=c.width, block_tables=c.dtable, cache_lens=c.dlens,
        key_cache=planes[0], value_cache=planes[1], query=c.dq, new_key=c.dk, new_value=c.dv, out=rows, workspace=ws[0],
        workspace_bytes=ws[1], max_context=c.width * 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.launch(args, torch.cuda.current_stream())
    for _ in range(4):
        c.out.zero_()
        pvlc.paged_decode_f16(f16)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out.cpu().double(), first)


@CODES
@WIDTHS
def test_infinite_and_nan_rows(code, f32):
    """An appended infinity is held as 65504; a NaN as the e4m3 NaN, which its head's output shows, or as 0."""
    import torch
    log(f"case: q8 decode non-finite rows code={code} f32={f32}")
    c = Case([20, 20, 20], code, f32, seed=71).upload()
    c.nk[0, 0, 3], c.nv[0, 1, 7] = np.inf, -np.inf
    c.nk[1, 1, 100], c.nv[1, 0, 64] = np.nan, np.nan
    ws = workspace(3, c.width * 16)
    c.launch(c.args(ws, rope=False, rotate_query=False))
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        want, bound = c.want(rope=False, rotate_query=False)
    got = c.out.cpu().numpy().astype(np.float64)
    nan = lambda a: np.where((a & 0x7F) == 0x7F, 0x7F, a) if code == R.E4M3 else a  # noqa: E731
    for name, d in zip(("key", "value"), c.dev):
        np.testing.assert_array_equal(nan(d.cpu().numpy()), nan(getattr(c.cache, name)))
    np.testing.assert_array_equal(c.dev[2].cpu().numpy(), c.cache.exponents)
    for s in (0, 2):
        assert (np.abs(got[s] - want[s]) <= bound[s]).all(), s
    if code == R.INT8:
        assert (np.abs(got[1] - want[1]) <= bound[1]).all()
    else:
        assert np.isnan(got[1, 8:]).all(), "the NaN key reaches every score of its head's group"
        assert np.isnan(got[1, :8, 64]).all() and not np.isnan(got[1, :8, :64]).any()


def test_blocks_beyond_32_bits_of_offset():
    """A pool whose planes exceed 4 GiB, the sequences in its last blocks."""
    import torch
    log("case: q8 decode in planes of more than 4 GiB")
    c = Case([100, 37], R.E4M3, True, seed=81)
    blocks = (1 << 20) + 5000
    far = c.table + (blocks - c.blocks)
    planes = [torch.zeros(blocks, 2, n, dtype=torch.uint8, device="cuda") for n in (2048, 2048, 2)]
    for d, a in zip(planes, (c.cache.key, c.cache.value, c.cache.exponents)):
        d[blocks - c.blocks:] = torch.from_numpy(a).cuda()
    c.upload()
    c.dev, c.dtable = planes, torch.from_numpy(far.astype(np.int32)).cuda()
    ws = workspace(2, c.width * 16)
    args = c.args(ws)
    args.num_blocks = blocks
    c.launch(args)
    torch.cuda.synchronize()
    want, bound = c.want()
    assert (np.abs(c.out.cpu().numpy() - want) <= bound).all()
    for d, a in zip(planes, (c.cache.key, c.cache.value, c.cache.exponents)):
        np.testing.assert_array_equal(d[blocks - c.blocks:].cpu().numpy(), a)
        assert not d[:blocks - c.blocks].any()


def test_more_sequences_than_the_walk_numbers():
    """More ragged sequences than the persistent kernel numbers: a workgroup for each partition."""
    log("case: q8 decode 2100 sequences")
    c = Case(np.random.default_rng(5).integers(0, 40, 2100), R.INT8, True, seed=92).upload()
    ws = workspace(c.n, c.width * 16)
    c.launch(c.args(ws))
    c.check("2100 sequences")
    c = Case([1200] + [3] * 2099, R.INT8, True, seed=93, paged=False)
    c.upload()
    ws = workspace(c.n, c.width * 16, 1024)
    c.launch(c.args(ws, partition=1024))
    c.check("2100 sequences, a long one")


@CODES
@WIDTHS
@pytest.mark.parametrize("partition", [400, 512, 528, 640, 768])
def test_the_widest_workgroups(code, f32, partition):
    """Eight and twelve waves of 64 tokens, partitions that end inside the last wave's."""
    log(f"case: q8 decode partition={partition} code={code} f32={f32}")
    c = Case([partition * 2 + 70, partition, partition - 1, 0], code, f32, seed=partition + code).upload()
    ws = workspace(4, c.width * 16, partition)
    c.launch(c.args(ws, partition=partition))
    c.check(f"P={partition}")
    assert pvlc.workspace_error(*ws) == 0


@pytest.mark.parametrize("n,t", [(18, 4000), (8, 6500), (4, 6000)])
def test_one_round_of_long_caches(n, t):
    """Lengths at which the automatic partition of a uniform launch takes six, eight and twelve waves."""
    log(f"case: q8 decode {n} caches of {t} rows")
    c = Case([t] * n, R.E4M3 if n == 18 else R.INT8, n == 4, seed=t, paged=n != 18).upload()
    ws = workspace(n, c.width * 16)
    c.launch(c.args(ws, ragged=False))
    c.check(f"{n} x {t}")


def test_two_graphs_share_a_workspace():
    """Captured launches of different shapes (single, ragged, streaming) on one workspace, replayed in turn."""
    import torch
    log("case: q8 decode two graphs")
    cases = [Case([500, 33, 900], R.E4M3, True, seed=71).upload(), Case([1157], R.INT8, False, seed=72).upload(),
             Case(np.random.default_rng(73).integers(0, 600, 70), R.INT8, True, seed=73).upload()]
    ws = workspace(70, 37 * 16, 32)  # the largest of the three
    runs = []
    for c in cases:
        partition = 32 if c.n == 70 else 0
        assert pvlc.decode_workspace_bytes(c.n, c.width * 16, partition) <= ws[1]
        args = c.args(ws, ragged=c.n > 1, partition=partition)
        c.launch(args)
        c.check(f"{c.n} sequences, eager")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.launch(args, torch.cuda.current_stream())
        runs.append((c, args, graph, c.out.clone()))
    for i in range(4):
        for c, _, graph, _ in runs:
            c.out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for c, args, _, first in runs:
            assert torch.equal(c.out, first), f"replay {i}, {c.n} sequences"
            c.launch(args)
    assert pvlc.workspace_error(*ws) == 0
