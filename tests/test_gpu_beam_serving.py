"""The operators of beam-searched serving together, as a program uses them: prompts packed into 8-bit pages, fanned out to
beams, then steps of projections, decode over the pages of every layer, logits, selection and the fork of the pages, with
compactions between.  Each step's attention, selection and pages against the plain forms, and the whole search again from
a captured graph, bit for bit."""

import numpy as np
import pytest

import pages_ref as P
import q8_ref as R
from pvlc_testlib import log, pvlc
from test_gpu_beam import plain as plain_selection

pytestmark = pytest.mark.gpu

LAYERS, HIDDEN, VOCAB, BASE = 2, 64, 404, 500000.0
PROMPTS, BEAMS, ROOM = (21, 48), 3, 24


class Serving:
    def __init__(self, code, seed):
        import torch
        self.code = code
        g = np.random.default_rng(seed)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        half = lambda *s: put((g.standard_normal(s) / np.sqrt(s[-1])).astype(np.float16))  # noqa: E731
        self.n, self.batch = len(PROMPTS) * BEAMS, len(PROMPTS)
        self.width = -(-(max(PROMPTS) + ROOM) // 16)
        self.blocks = self.n * self.width + 5
        self.embedding = put((g.standard_normal((VOCAB, HIDDEN))).astype(np.float32))
        self.w_qkv, self.w_o = [half(2560, HIDDEN) for _ in range(LAYERS)], [half(HIDDEN, 2048) for _ in range(LAYERS)]
        self.w_head = put((g.standard_normal((VOCAB, HIDDEN)) * 0.4).astype(np.float16))
        self.prompts = [[[(g.standard_normal((t, 2, 128))).astype(np.float16) for _ in range(2)] for _ in range(LAYERS)] for t in PROMPTS]
        self.cos, self.sin = pvlc.rope_table(BASE, self.width * 16)
        self.dcos, self.dsin = put(self.cos), put(self.sin)
        zeros = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        i32 = torch.int32
        self.planes = [zeros(LAYERS, self.blocks, k, t=torch.uint8) for k in (4096, 4096, 4)]
        self.refs, self.mask = zeros(self.blocks, t=i32), zeros(-(-self.blocks // 32), t=i32)
        self.tables, self.lens = [zeros(self.n, self.width, t=i32) for _ in range(2)], [zeros(self.n, t=i32) for _ in range(2)]
        self.qkv = [zeros(self.n, 2560) for _ in range(LAYERS)]
        self.q, self.k, self.v = ([zeros(self.n, h * 128) for _ in range(LAYERS)] for h in (16, 2, 2))
        self.attention, self.o = [zeros(self.n, 2048) for _ in range(LAYERS)], zeros(self.n, HIDDEN)
        self.logits = zeros(self.n, VOCAB)
        self.scores, self.finished = ([zeros(self.batch, BEAMS, t=t) for _ in range(2)] for t in (torch.float32, i32))
        self.parents, self.tokens = zeros(self.batch, BEAMS, t=i32), zeros(self.batch, BEAMS, t=i32)
        self.bias = zeros(4096)

        def workspace(nbytes):
            w = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
            pvlc.workspace_init(w, nbytes)
            return w, nbytes

        self.decode_ws = workspace(pvlc.decode_workspace_bytes(self.n, self.width * 16))
        self.page_ws = workspace(pvlc.kv_pages_workspace_bytes(self.blocks, self.n))
        self.beam_ws = workspace(pvlc.beam_workspace_bytes(self.batch, BEAMS, VOCAB, BEAMS))
        self.proj_ws = workspace(max(pvlc.linear_projection_workspace_bytes(self.n, w) for w in (HIDDEN, 2048)))
        self.pool = pvlc.kv_page_pool(num_blocks=self.blocks, max_blocks_per_seq=self.width, num_layers=LAYERS, planes=self.planes,
                                      ref_counts=self.refs, free_mask=self.mask, workspace=self.page_ws[0], workspace_bytes=self.page_ws[1])

    def start(self):
        """Prompts into pages, one row each, then fanned out to their beams; beam 0 of each begins."""
        import torch
        put = lambda a, t=np.int32: torch.from_numpy(np.asarray(a, t)).cuda()  # noqa: E731
        for p in self.planes:
            p.zero_()
        pvlc.kv_pages_reset(self.pool)
        rows, lens = torch.zeros(self.batch, self.width, dtype=torch.int32, device="cuda"), torch.zeros(self.batch, dtype=torch.int32, device="cuda")
        new, reserve, fan = put([-1] * self.batch), put(PROMPTS), put(np.repeat(np.arange(self.batch), BEAMS))
        pvlc.kv_pages_fork(self.pool, rows_in=0, rows_out=self.batch, tables_out=rows, lens_out=lens, parents=new, reserve=reserve)
        for b, t in enumerate(PROMPTS):
            for l in range(LAYERS):
                k, v = (torch.from_numpy(x.view(np.int16)).cuda() for x in self.prompts[b][l])
                pvlc.kv_pack_q8(k, v, t, self.planes[0][l], self.planes[1][l], self.planes[2][l], self.blocks, self.code, rows[b])
        pvlc.kv_pages_fork(self.pool, rows_in=self.batch, rows_out=self.n, tables_in=rows, lens_in=reserve, tables_out=self.tables[0],
                           lens_out=self.lens[0], parents=fan, reserve_tokens=1)
        self.scores[0].fill_(-np.inf)
        self.scores[0][:, 0] = 0
        self.finished[0].zero_()
        self.tokens.copy_(put(np.arange(self.n).reshape(self.batch, BEAMS) + 7))
        torch.cuda.synchronize()

    def step(self, a, stream=None):
        """One step of every beam, state a to state 1 - a."""
        x = self.embedding[self.tokens.view(-1).clamp_min(0).long()]
        for l in range(LAYERS):
            pvlc.linear_projection_f16(x, self.w_qkv[l], self.bias, self.qkv[l], self.n, HIDDEN, 2560, *self.proj_ws, stream)
            self.q[l].copy_(self.qkv[l][:, :2048])
            self.k[l].copy_(self.qkv[l][:, 2048:2304])
            self.v[l].copy_(self.qkv[l][:, 2304:])
            args = pvlc.paged_decode_q8_args(
                num_seqs=self.n, num_blocks=self.blocks, max_blocks_per_seq=self.width, code=self.code, block_tables=self.tables[a],
                cache_lens=self.lens[a], key_cache=self.planes[0][l], value_cache=self.planes[1][l], exponents=self.planes[2][l], query=None,
                new_key=None, new_value=None, out=None, workspace=self.decode_ws[0], workspace_bytes=self.decode_ws[1],
                max_context=self.width * 16, rope_cos=self.dcos, rope_sin=self.dsin, rope_rows=self.width * 16, rotate_query=True)
            pvlc.paged_decode_q8_f32io(args, self.q[l], self.k[l], self.v[l], self.attention[l], stream)
            pvlc.linear_projection_f16(self.attention[l], self.w_o[l], self.bias, self.o, self.n, 2048, HIDDEN, *self.proj_ws, stream)
            x = x + self.o
        pvlc.linear_projection_f16(x, self.w_head, self.bias, self.logits, self.n, HIDDEN, VOCAB, *self.proj_ws, stream)
        pvlc.beam_select(pvlc.beam_select_args(
            batch=self.batch, beams=BEAMS, vocab=VOCAB, best=BEAMS, logits=self.logits, scores=self.scores[a], finished=self.finished[a],
            end_token=3, next_scores=self.scores[1 - a], parents=self.parents, tokens=self.tokens, next_finished=self.finished[1 - a],
            workspace=self.beam_ws[0], workspace_bytes=self.beam_ws[1]), stream)
        pvlc.kv_pages_fork(self.pool, rows_in=self.n, rows_out=self.n, tables_in=self.tables[a], lens_in=self.lens[a], tables_out=self.tables[1 - a],
                           lens_out=self.lens[1 - a], parents=self.parents, reserve_tokens=1, appended=1, stream=stream)

    def compact(self, a, stream=None):
        pvlc.kv_pages_compact(self.pool, rows=self.n, tables=self.tables[a], stream=stream)

    def state(self, a):
        import torch
        torch.cuda.synchronize()
        return [x.clone() for x in (self.tables[a], self.lens[a], self.scores[a], self.finished[a], self.tokens, self.refs, self.mask, *self.planes)]


@pytest.mark.parametrize("code", [R.E4M3, R.INT8])
def test_a_search_step_by_step(code):
    import torch
    log(f"case: beam search over 8-bit pages, code={code}")
    s = Serving(code, 3 + code)
    s.start()
    # The plain program: a cache of its own for every row and layer, pages in pages_ref.
    pages = P.Pool(s.blocks, s.width, [])
    table, lens, _ = pages.fork([], [], s.batch, [-1] * s.batch, PROMPTS)
    rows = []
    for b, t in enumerate(PROMPTS):
        caches = [R.Cache(s.width, code) for _ in range(LAYERS)]
        for l in range(LAYERS):
            caches[l].put_rows(range(s.width), 0, *s.prompts[b][l])
        rows.append((caches, t))
    fan = np.repeat(np.arange(s.batch), BEAMS)
    table, lens, _ = pages.fork(table, np.array(PROMPTS), s.n, fan, 1)

    def copied(row):
        caches = []
        for c in row[0]:
            d = R.Cache(s.width, code)
            d.key, d.value, d.exponents = c.key.copy(), c.value.copy(), c.exponents.copy()
            caches.append(d)
        return caches, row[1]

    rows = [copied(rows[b]) for b in fan]
    scores = np.full((s.batch, BEAMS), -np.inf, np.float32)
    scores[:, 0] = 0
    finished = np.zeros((s.batch, BEAMS), np.int32)
    a, worst = 0, 0.0
    for step in range(ROOM - 2):
        if step == 8:  # a program may end a beam by itself
            s.finished[a][1, 0] = 1
            finished[1, 0] = 1
        s.step(a)
        torch.cuda.synchronize()
        for r in range(s.n):
            caches, t = rows[r]
            for l in range(LAYERS):
                turn = lambda x: R.rotate(x, s.cos[t], s.sin[t])  # noqa: E731
                q, k, v = (x[l][r].cpu().numpy().reshape(-1, 128) for x in (s.q, s.k, s.v))
                caches[l].put_rows(range(s.width), t, turn(k)[None], v.astype(np.float16).astype(np.float64)[None])
                keys, values = caches[l].rows(range(s.width), t + 1)
                want, big = R.attend(turn(q), keys, values)
                off = np.abs(s.attention[l][r].cpu().numpy().reshape(16, 128) - want).max() / R.attend_bound(big, t + 1, values)
                worst = max(worst, off)
                assert off <= 1, (step, r, l, off)
            rows[r] = caches, t + 1
        want, gap = plain_selection(s.logits.cpu().numpy(), scores, BEAMS, finished, 3)
        assert gap > 4e-6, gap
        parents, tokens = s.parents.cpu().numpy(), s.tokens.cpu().numpy()
        np.testing.assert_array_equal(parents, want[1], f"step {step}")
        np.testing.assert_array_equal(tokens, want[2], f"step {step}")
        np.testing.assert_array_equal(s.finished[1 - a].cpu().numpy(), want[3])
        assert np.allclose(s.scores[1 - a].cpu().numpy(), want[0], atol=4e-6, rtol=0)
        scores, finished = s.scores[1 - a].cpu().numpy(), want[3].astype(np.int32)
        table, lens, error = pages.fork(table, lens, s.n, parents.ravel(), 1, 1)
        assert error == 0
        rows = [copied(rows[p]) for p in parents.ravel()]
        a = 1 - a
        if step % 7 == 4:
            s.compact(a)
            table, _ = pages.compact(table)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(s.tables[a].cpu().numpy(), table, f"step {step}")
        np.testing.assert_array_equal(s.lens[a].cpu().numpy(), lens)
        np.testing.assert_array_equal(s.refs.cpu().numpy(), pages.refs)
    assert finished[1].any()
    print(f"[serving] worst attention error / bound {worst:.2g}")
    # What the pages hold of every row, byte for byte.
    key, value, exponents = (p.cpu().numpy().reshape(LAYERS, s.blocks, 2, -1) for p in s.planes)
    for r, (caches, t) in enumerate(rows):
        n = -(-t // 16)
        for l in range(LAYERS):
            ids = table[r][:n]
            full, tail = t // 16, t % 16
            np.testing.assert_array_equal(key[l][ids[:full]], caches[l].key[:full])
            np.testing.assert_array_equal(value[l][ids[:full]], caches[l].value[:full])
            np.testing.assert_array_equal(exponents[l][ids], caches[l].exponents[:n])
            if tail:
                np.testing.assert_array_equal(key[l][ids[full]][:, R.KEY_AT[:tail]], caches[l].key[full][:, R.KEY_AT[:tail]])
                np.testing.assert_array_equal(value[l][ids[full]][:, R.VALUE_AT[:tail]], caches[l].value[full][:, R.VALUE_AT[:tail]])
    assert pvlc.workspace_error(*s.page_ws) == 0 and pvlc.workspace_error(*s.decode_ws) == 0


def test_a_search_from_a_graph():
    """Two steps and a compaction captured once and replayed, with eager work between, against the same calls made
    eagerly."""
    import torch
    log("case: beam search from a graph")
    s = Serving(R.INT8, 9)
    steps = 10

    def two(stream=None):
        s.step(0, stream)
        s.step(1, stream)
        s.compact(0, stream)

    s.start()
    eager = []
    for _ in range(steps):
        two()
        eager.append(s.state(0))
    s.start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two(side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two(torch.cuda.current_stream())
    s.start()
    for i in range(steps):
        graph.replay()
        got = s.state(0)
        assert all(torch.equal(x, y) for x, y in zip(got, eager[i])), f"replay {i}"
        torch.randn(1000, 1000, device="cuda").sum().item()
