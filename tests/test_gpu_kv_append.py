"""Rows of several sequences appended to fp16 and 8-bit pages: planes and exponents byte for byte, what they held before among
them."""

import numpy as np
import pytest

import batches_ref as B
import q8_ref as R
from pvlc_testlib import log, pvlc

pytestmark = pytest.mark.gpu

CODES = pytest.mark.parametrize("code", [B.F16, R.E4M3, R.INT8])
WIDTHS = pytest.mark.parametrize("f32", [False, True])
BATCHES = {
    "one": ([1], [0]), "one_into_block": ([1], [5]), "drafts": ([1, 3, 2, 4, 1], [15, 16, 13, 0, 31]), "empty": ([0, 5, 0, 17, 0], [3, 0, 0, 30, 16]),
    "prompt": ([211], [0]), "prompts": ([33, 1, 100, 16, 15], [0, 0, 7, 16, 1]), "many": ([i % 4 for i in range(150)], [i * 7 % 40 for i in range(150)]),
    "a_block_ends": ([16, 32, 15], [16, 0, 1]),
}


@CODES
@WIDTHS
@pytest.mark.parametrize("name", list(BATCHES))
def test_batches(code, f32, name):
    log(f"case: append {name} code={code} f32={f32}")
    counts, held = BATCHES[name]
    b = B.Batch(counts, held, code, f32, seed=len(name), paged=name != "prompts", fused=name in ("drafts", "prompts"), spare=2,
                positions=name == "prompts", rope=name != "a_block_ends").upload()
    b.append(b.append_args())
    b.put()
    b.check_planes(name)
    assert int(b.error) == 0


@CODES
def test_without_offsets_and_lengths(code):
    log(f"case: append without offsets, code={code}")
    b = B.Batch([19] * 4, [0] * 4, code, code != R.INT8, seed=2).upload()
    b.append(b.append_args(row_offsets=None, cache_lens=None))
    b.put()
    b.check_planes("equal rows")


@CODES
def test_values_out_of_range(code):
    """Infinities and NaN, and rows far larger and smaller than what their block holds."""
    log(f"case: append odd values, code={code}")
    b = B.Batch([6, 20, 3], [4, 9, 14], code, True, seed=3, rope=False)
    b.k[0, 0, :3] = np.inf, -np.inf, 1e9
    b.v[1, 1, 5] = -np.inf
    b.k[7] *= 1000.0
    b.v[8] *= 1e-6
    b.k[26] *= 3000.0
    if code != B.F16:
        b.v[3, 0, 7] = np.nan
    b.upload()
    with np.errstate(over="ignore", invalid="ignore"):
        b.put()
    b.append(b.append_args())
    b.check_planes("odd values")


def test_calls_in_turn_and_from_a_graph():
    """Appends to the same pages one after the other, captured and replayed on another stream: the second call's block holds
    the first one's rows."""
    import torch
    log("case: append from a graph")
    for code in (B.F16, R.E4M3, R.INT8):
        b = B.Batch([5, 0, 30], [3, 12, 20], code, False, seed=8, room=40).upload()
        first = b.append_args()
        lens = b.later = torch.from_numpy(np.asarray(b.held, np.int32) + np.asarray(b.counts, np.int32)).cuda()
        second = b.append_args(cache_lens=lens)
        start = [x.clone() for x in b.planes + ([] if b.exponents is None else [b.exponents])]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            b.append(first, stream)
            b.append(second, stream)
        b.put()
        b.held = [h + c for h, c in zip(b.held, b.counts)]
        b.put()
        for _ in range(3):
            for d, s in zip(b.planes + ([] if b.exponents is None else [b.exponents]), start):
                d.copy_(s)
            graph.replay()
            b.check_planes(f"replay, code {code}")


def test_far_blocks():
    """Block ids whose elements lie beyond 2^31, and beyond 2^32 bytes."""
    import torch
    log("case: append to far blocks")
    b = B.Batch([20, 3], [0, 14], B.F16, True, seed=4).upload()
    blocks = (1 << 31) // 4096 + 9
    planes = [torch.zeros(blocks * 4096, dtype=torch.int16, device="cuda") for _ in range(2)]
    ids = torch.tensor([[blocks - 1, blocks - 5], [blocks - 2, blocks - 8]], dtype=torch.int32, device="cuda")
    held = torch.from_numpy(np.stack([b.cache.key, b.cache.value])[:, b.table].view(np.int16)).cuda()
    for which, p in enumerate(planes):
        p.view(blocks, 4096)[ids.long()] = held[which].view(2, 2, 4096)
    b.append(b.append_args(num_blocks=blocks, key_cache=planes[0], value_cache=planes[1], block_tables=ids))
    b.put()
    torch.cuda.synchronize()
    for which, p in enumerate(planes):
        got = p.view(blocks, 4096)[ids.long()].cpu().numpy().view(np.uint16).reshape(2, 2, 2, 2048)
        assert np.array_equal(got, np.stack([b.cache.key, b.cache.value])[which][b.table])


def test_errors_are_reported_and_skipped():
    import torch
    log("case: append errors")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for code in (B.F16, R.INT8):
        fresh = lambda: B.Batch([5, 7, 9], [3, 0, 20], code, False, seed=5).upload()  # noqa: E731
        b = fresh()  # a length that leaves no room, and a negative one
        b.append(b.append_args(cache_lens=ints([b.width * 16 - 4, 0, -1])))
        b.counts = [0, 7, 0]
        b.put()
        b.check_planes("lengths")
        assert int(b.error) == 1
        b = fresh()  # a block outside the planes
        table = b.dtable.clone()
        table[1, 0] = b.blocks
        table[0, 0] = -1
        b.append(b.append_args(block_tables=table))
        b.counts = [0, 0, 9]
        b.put()
        b.check_planes("blocks")
        assert int(b.error) == 2
        b = fresh()  # positions outside the tables: as given
        b.append(b.append_args(positions=ints([b.table_rows] * 21)))
        b.rope = False
        b.put()
        b.check_planes("positions")
        assert int(b.error) == 4
        b = fresh()  # offsets that pass the rows: nothing outside the matrices is read
        b.append(b.append_args(row_offsets=ints([0, 5, 12, 400])))
        b.counts = [5, 7, 0]
        b.put()
        b.check_planes("offsets")
        assert int(b.error) == 1


@CODES
@pytest.mark.parametrize("n", [3, 100])
def test_rows_before_the_first_sequence(code, n):
    """The first sequence need not begin at row 0: rows before it are not used, as those behind the last one are not."""
    log(f"case: append, rows before the first sequence, code={code} n={n}")
    counts, held = [60] + [1 + i % 3 for i in range(n)], [0] + [40 + i % 7 for i in range(n)]
    b = B.Batch(counts, held, code, False, seed=n, spare=2)
    b.upload()
    b.append(b.append_args(num_seqs=n, row_offsets=b.doffsets[1:], cache_lens=b.dlens[1:], block_tables=b.dtable[1:]))
    b.counts[0] = 0
    b.put()
    b.check_planes("behind row 60")
    assert int(b.error) == 0


@CODES
@pytest.mark.parametrize("n", [3, 100, 5000])
def test_offsets_that_descend_are_reported(code, n):
    """Wherever they descend; other sequences' rows may be skipped, but nothing else is written."""
    import torch
    log(f"case: append, offsets that descend, code={code} n={n}")
    for at in sorted({1, n // 2, n - 1}):
        b = B.Batch([4] * n, [2] * n, code, False, seed=n + at).upload()
        bad = b.offsets.copy()
        bad[at] = bad[at + 1] + 3 if at % 2 else bad[at - 1] - 3
        b.append(b.append_args(row_offsets=torch.from_numpy(bad).cuda()))
        torch.cuda.synchronize()
        assert int(b.error) == 1, at
        unused = np.setdiff1d(np.arange(b.blocks), b.table)
        assert np.array_equal(b.planes[0].cpu().numpy().view(b.cache.key.dtype)[unused], b.cache.key[unused])
