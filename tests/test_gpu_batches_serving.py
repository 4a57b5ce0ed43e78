"""Batches served as a program does: prompts admitted to a page pool and prefilled together, in chunks, fanned out to beams,
decoded with their shared pages, reordered by a fork at every step.  Every
call against the one-sequence and unshared entry points: pages bit for bit, outputs within the sums' rounding."""

import numpy as np
import pytest

import q8_ref as R
from pvlc_testlib import log, pvlc

pytestmark = pytest.mark.gpu
PROMPTS, BEAMS, ROOM, STEPS = (75, 33, 130), 3, 40, 5


class Pool:
    """fp16 (one plane pair) or 8-bit pages of one layer, with its tables."""

    def __init__(self, blocks, width, code):
        import torch
        self.blocks, self.width, self.code = blocks, width, code
        zeros = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        element = torch.float16 if code == pvlc.KV_F16 else torch.uint8
        self.planes = [zeros(1, blocks, 4096, t=element) for _ in range(2)]
        if code != pvlc.KV_F16:
            self.planes.append(zeros(1, blocks, 4, t=torch.uint8))
        self.refs, self.mask = zeros(blocks), zeros(-(-blocks // 32))
        nbytes = pvlc.kv_pages_workspace_bytes(blocks, 64)
        self.ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        pvlc.workspace_init(self.ws, nbytes)
        self.pool = pvlc.kv_page_pool(num_blocks=blocks, max_blocks_per_seq=width, num_layers=1, planes=self.planes, ref_counts=self.refs,
                                      free_mask=self.mask, workspace=self.ws, workspace_bytes=nbytes)
        pvlc.kv_pages_reset(self.pool)

    def fork(self, tables, lens, parents, **how):
        import torch
        n = len(parents)
        out, out_lens = torch.empty(n, self.width, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        self.parents = torch.tensor(parents, dtype=torch.int32, device="cuda")
        pvlc.kv_pages_fork(self.pool, rows_in=0 if tables is None else len(tables), rows_out=n, tables_in=tables, lens_in=lens, tables_out=out,
                           lens_out=out_lens, parents=self.parents, **how)
        torch.cuda.synchronize()
        return out, out_lens

    def held(self):
        return dict(key_cache=self.planes[0], value_cache=self.planes[1])


@pytest.mark.parametrize("code", [pvlc.KV_F16, R.E4M3, R.INT8])
@pytest.mark.parametrize("context", [0, 60000])  # 0: the tables' own reach, decoded alone; far: with the shared pages once
def test_admit_and_search(code, context):
    import torch
    log(f"case: batches served code={code} context={context}")
    g = torch.Generator(device="cuda").manual_seed(11)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    n, width = len(PROMPTS), max(-(-(max(PROMPTS) + ROOM) // 16), context // 16)
    cos, sin = (torch.from_numpy(x).cuda() for x in pvlc.rope_table(500000.0, max(PROMPTS) + ROOM))
    rope = dict(rope_cos=cos, rope_sin=sin, rope_rows=cos.shape[0])
    blocks = 200
    prompts = Pool(blocks, width, pvlc.KV_F16)
    pages = prompts if code == pvlc.KV_F16 else Pool(blocks, width, code)
    rows = [[normal(t, h, 128) for h in (16, 2, 2)] for t in PROMPTS]

    # Admission, and both chunks of all prompts, against one prompt at a time over planes of its own.
    tables, lens = prompts.fork(None, None, [-1] * n, reserve=ints(PROMPTS))
    nbytes = pvlc.packed_prefill_workspace_bytes(n, sum(PROMPTS), width * 16)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, nbytes)
    halves, done = [t // 2 for t in PROMPTS], [0] * n
    got = [torch.empty(t, 16, 128, device="cuda") for t in PROMPTS]
    for counts in (halves, [t - h for t, h in zip(PROMPTS, halves)]):
        q, k, v = (torch.cat([rows[i][w][done[i]:done[i] + c] for i, c in enumerate(counts)]) for w in range(3))
        out, offsets, held = torch.empty_like(q), ints([0] + np.cumsum(counts).tolist()), ints(done)
        args = pvlc.packed_prefill_args(num_seqs=n, rows=len(q), num_blocks=blocks, max_blocks_per_seq=width, max_context=width * 16,
                                        row_offsets=offsets, block_tables=tables, cache_lens=held, workspace=ws, workspace_bytes=nbytes,
                                        **prompts.held(), **rope)
        pvlc.packed_prefill_f32io(args, q, k, v, out)
        torch.cuda.synchronize()
        at = 0
        for i, c in enumerate(counts):
            got[i][done[i]:done[i] + c] = out[at:at + c]
            at, done[i] = at + c, done[i] + c
    assert pvlc.workspace_error(ws, nbytes) == 0
    alone = [torch.zeros_like(x) for x in prompts.planes]
    for i, t in enumerate(PROMPTS):
        out = torch.empty(t, 16, 128, device="cuda")
        pvlc.paged_prefill_f32io(tokens=t, num_blocks=blocks, key_cache=alone[0], value_cache=alone[1], query=rows[i][0], key=rows[i][1],
                                 value=rows[i][2], out=out, block_table=tables[i], **rope)
        torch.cuda.synchronize()
        # (both are off by the f32 sums and the pairs of weights alone)
        assert (got[i] - out).abs().max() <= 2e-5 * rows[i][2].abs().max(), i
    assert all(torch.equal(a, b) for a, b in zip(prompts.planes, alone))

    # The prompts' rows into 8-bit pages, all in one call, against one at a time.
    if code != pvlc.KV_F16:
        tables, lens = pages.fork(None, None, [-1] * n, reserve=ints(PROMPTS))
        offsets, k, v = ints([0] + np.cumsum(PROMPTS).tolist()), *(torch.cat([r[w] for r in rows]) for w in (1, 2))
        pvlc.kv_append_f32(pvlc.kv_append_args(num_seqs=n, rows=len(k), num_blocks=blocks, max_blocks_per_seq=width, code=code,
                                               exponents=pages.planes[2], row_offsets=offsets, block_tables=tables, **pages.held(), **rope), k, v)
        torch.cuda.synchronize()
        packed = [torch.zeros_like(x) for x in pages.planes]
        for i, t in enumerate(PROMPTS):  # (the fp16 pages hold the rotated rows)
            kr, vr = (torch.empty(t, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
            pvlc.kv_unpack_f16(prompts.planes[0], prompts.planes[1], t, kr, vr, blocks, prompt_table(prompts, i))
            pvlc.kv_pack_q8(kr, vr, t, *packed, blocks, code, tables[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pages.planes, packed))

    # Beams: the prompts fanned out, then steps against the unshared decode on a copy of the pages.
    rows_in = ints(PROMPTS)
    tables, lens = pages.fork(tables, rows_in, np.repeat(np.arange(n), BEAMS).tolist(), reserve_tokens=1)
    beams = n * BEAMS
    shared = ints(PROMPTS)  # (a prompt's last block may be a copy: whole blocks are taken)
    nbytes = pvlc.shared_decode_workspace_bytes(beams, n, width * 16)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, nbytes)
    other = torch.empty(pvlc.decode_workspace_bytes(beams, width * 16), dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(other, other.numel())
    choose = np.random.default_rng(5)
    for step in range(STEPS):
        q, k, v = normal(beams, 16, 128), normal(beams, 2, 128), normal(beams, 2, 128)
        out, want, copy = torch.empty_like(q), torch.empty_like(q), [x.clone() for x in pages.planes]
        common = dict(num_seqs=beams, num_blocks=blocks, max_blocks_per_seq=width, block_tables=tables, cache_lens=lens,
                      max_context=width * 16, rotate_query=True, **rope)
        pvlc.shared_decode_f32io(pvlc.shared_decode_args(num_groups=n, shared_lens=shared, code=code, workspace=ws, workspace_bytes=nbytes,
                                                         exponents=None if code == pvlc.KV_F16 else pages.planes[2], **pages.held(), **common),
                                 q, k, v, out)
        one = dict(common, workspace=other, workspace_bytes=other.numel(), query=None, new_key=None, new_value=None, out=None)
        if code == pvlc.KV_F16:
            pvlc.paged_decode_f32io(pvlc.paged_decode_args(key_cache=copy[0], value_cache=copy[1], **one), q, k, v, want)
        else:
            pvlc.paged_decode_q8_f32io(pvlc.paged_decode_q8_args(code=code, key_cache=copy[0], value_cache=copy[1], exponents=copy[2], **one),
                                       q, k, v, want)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pages.planes, copy)), step
        assert (out - want).abs().max() <= 2e-5 * 5.0, step  # (values below 5 standard deviations)
        parents = [b * BEAMS + int(choose.integers(BEAMS)) for b in range(n) for _ in range(BEAMS)]
        tables, lens = pages.fork(tables, lens, parents, reserve_tokens=1, appended=1)
    assert pvlc.workspace_error(ws, nbytes) == 0 and pvlc.workspace_error(pages.ws, pages.ws.numel()) == 0


def prompt_table(pool, i):
    """The table that the first fork of an empty pool gives its row i: the lowest pages, rows in order."""
    import torch
    first = sum(-(-t // 16) for t in PROMPTS[:i])
    return torch.arange(first, first + -(-PROMPTS[i] // 16), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("code", [pvlc.KV_F16, R.E4M3])
def test_one_workspace(code):
    """Packed prompts (whose values are not all finite, whose items are many), groups' decodes of either route and paged decodes in
    turn over one workspace."""
    import torch

    import batches_ref as B
    from test_gpu_packed_prefill import args_of, launch, wanted
    from test_gpu_shared_decode import Groups, tails_of
    log(f"case: one workspace code={code}")

    def prompts(seed, room):
        b = B.Batch([70, 33] + [20] * 40, [9, 0] + [3] * 40, f32=True, seed=seed, room=room)
        b.v[3, 0, 5] = np.inf
        return b.upload()

    def groups(seed):
        return [Groups([4] * 10, [400 + 16 * i for i in range(10)], tails_of(40, 60), code, True, seed=seed, far=False).upload(),
                Groups([2], [4000], [5, 90], code, False, seed=seed + 1, far=False).upload(),
                Groups([5, 5], [700, 40], tails_of(10, 90), code, True, seed=seed + 2).upload()]

    def needs(c):
        if isinstance(c, Groups):
            return pvlc.shared_decode_workspace_bytes(c.n, len(c.sizes), c.width * 16)
        return pvlc.packed_prefill_workspace_bytes(c.n, c.rows, c.width * 16)
    steps = [prompts(31, 5000)] + groups(32) + [prompts(36, 0)] + groups(37) + [prompts(41, 5000)] + groups(42)
    nbytes = max(needs(c) for c in steps)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(ws, nbytes)
    for c in steps:
        if isinstance(c, Groups):
            c.launch(c.shared_args((ws, nbytes)))
        else:
            launch(c, args_of(c, (ws, nbytes)))
    torch.cuda.synchronize()
    for i, c in enumerate(steps):
        if isinstance(c, Groups):
            c.check(f"step {i}")
            continue
        with np.errstate(invalid="ignore"):
            c.put()
        some = np.arange(70, c.rows)
        want, limit = wanted(c, some)
        B.check(f"step {i}", c.out.cpu().numpy()[some], want, limit)
    assert pvlc.workspace_error(ws, nbytes) == 0
