"""Operators of beam-searched serving over a paged cache in 8 bits, and their plain forms.

``own`` says which side ``run`` takes: the package's entry points, or elementary torch operations in 32 bits.
Kinds of work, and the ranges that ``draw`` takes its sizes from:

* ``decode``    one decode step (rotary, append, attention) over 8-bit pages with a power-of-two scale for each block of
                16 tokens and head: 1 to 18 caches of one length of 16 to 16384 rows, or 2 to 256 sequences of different
                lengths up to 32768 rows; e4m3 or int8 codes, fp16 or f32 operands;
* ``move``      fp16 rows into 8-bit pages and back, 1 to 65536 tokens;
* ``beam``      the best candidates over beams and vocabulary, 1 to 16 batch entries of 1 to 16 beams, 97 to 160000 logits;
* ``fork``      pages reordered by beam parents: shared, copied where a beam writes, freed, two steps a pass;
* ``turnover``  finished sequences freed, the pages compacted, new sequences admitted.
"""

import math
import random

import torch

own = False

HEADS, KV, DIM, BLOCK = 16, 2, 128, 16
GROUP = HEADS // KV
SLAB = KV * DIM * BLOCK  # elements of one block of one plane
ROPE_BASE = 500000.0
LAYERS, VOCAB = 18, 103424
LARGEST = {"e4m3": 448.0, "int8": 127.0}
LEAST_EXPONENT, BIAS = -32, 127


def listed():
    return [
        # the smallest call of a decode loop: one layer of one page being recognised, on its projections' f32 operands
        dict(name="decode_layer", kind="decode", seqs=1, lo=1157, hi=1157, ragged=False, io="f32", format="e4m3"),
        # the attention of a whole decode step: 18 caches of one length in one launch
        dict(name="decode_step18", kind="decode", seqs=18, lo=2048, hi=2048, ragged=False, io="f16", format="int8"),
        # a small serving batch: pages in different states of recognition, permuted block tables
        dict(name="decode_batch", kind="decode", seqs=13, lo=90, hi=2010, ragged=True, io="f16", format="e4m3"),
        # the largest batch: 256 sequences of up to 32768 rows
        dict(name="decode_long", kind="decode", seqs=256, lo=1024, hi=32768, ragged=True, io="f16", format="e4m3"),
        # a prompt's rows taken into 8-bit pages and read back; a long document's
        dict(name="move_page", kind="move", tokens=1157, format="int8"),
        dict(name="move_long", kind="move", tokens=65536, format="e4m3"),
        # one page searched with four beams; a full batch with eight, two candidates a beam, the finished ones among them
        dict(name="beam_page", kind="beam", batch=1, beams=4, vocab=VOCAB, best=4, finished=False),
        dict(name="beam_batch", kind="beam", batch=16, beams=8, vocab=VOCAB, best=16, finished=True),
        # the page's beams reordered, all layers of an fp16 cache; the full batch's, 8-bit pages
        dict(name="fork_page", kind="fork", batch=1, beams=4, lo=1157, hi=1157, width=16),
        dict(name="fork_batch", kind="fork", batch=32, beams=8, lo=300, hi=2010, width=8),
        # a few sequences end and others take their place; the same in a large pool
        dict(name="turnover_page", kind="turnover", seqs=8, lo=90, hi=2010, width=16),
        dict(name="turnover_long", kind="turnover", seqs=64, lo=256, hi=8192, width=8),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "move", "beam", "beam", "fork", "turnover"])
    code = rng.choice(["e4m3", "int8"])
    if kind == "decode":
        io, ragged = rng.choice(["f16", "f32"]), rng.random() < 0.6
        if not ragged:
            context = _log(rng, 16, 16384)
            return dict(kind=kind, seqs=rng.choice([1, 1, 18, _log(rng, 2, 17)]), lo=context, hi=context, ragged=False, io=io, format=code)
        seqs = _log(rng, 2, 256)
        hi = min(_log(rng, 64, 32768), (1 << 21) // seqs)
        return dict(kind=kind, seqs=seqs, lo=_log(rng, max(1, hi // 32), hi), hi=hi, ragged=True, io=io, format=code)
    if kind == "move":
        return dict(kind=kind, tokens=_log(rng, 1, 65536), format=code)
    if kind == "beam":
        beams = _log(rng, 1, 16)
        best = rng.choice([beams, 2 * beams])
        vocab = rng.choice([VOCAB, _log(rng, 97, 160000)])
        return dict(kind=kind, batch=_log(rng, 1, min(16, 128 // beams)), beams=beams, vocab=vocab, best=best, finished=rng.random() < 0.5)
    width = rng.choice([8, 16])
    if kind == "fork":
        beams = _log(rng, 2, 16)
        hi = _log(rng, 40, 2500)
        return dict(kind=kind, batch=_log(rng, 1, 256 // beams), beams=beams, lo=_log(rng, max(1, hi // 16), hi), hi=hi, width=width)
    seqs = _log(rng, 4, 64)
    hi = _log(rng, 64, 8192 if width == 8 else 4096)
    return dict(kind=kind, seqs=seqs, lo=_log(rng, max(1, hi // 32), hi), hi=hi, width=width)


def _blocks(tokens):
    return -(-tokens // BLOCK)


def _lengths(n, lo, hi):
    """Lengths of n sequences, evenly spread over the logarithm of lo..hi."""
    return [min(hi, max(lo, int(round(lo * (hi / lo) ** ((i + 0.5) / n))))) for i in range(n)]


# ---------------------------------------------------------------------------
# Inputs, made from the seed alone
# ---------------------------------------------------------------------------

def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _code_type(code):
    return torch.float8_e4m3fn if code == "e4m3" else torch.int8


def _power(e):
    """2 to whole exponents, exactly (a power function may round)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _exponent(most, code):
    """The least power of two that brings `most`, the largest size in a block, within the codes' range."""
    fraction, power = torch.frexp(most)
    whole, border = (9, 0.875) if code == "e4m3" else (7, 127.0 / 128.0)
    return torch.where(most > 0, power - whole + (fraction > border).to(power.dtype), LEAST_EXPONENT).clamp_min(LEAST_EXPONENT)


def _codes(x, exponent, code):
    """Values divided by their block's power of two, rounded to the codes."""
    y = (x * _power(-exponent)).clamp(-LARGEST[code], LARGEST[code])
    return y.to(torch.float8_e4m3fn) if code == "e4m3" else y.round().to(torch.int8)


def _key_order(x):
    """[..., token 16, dim 128] as a key block keeps it: [..., token / 4, dim / 16, token % 4, dim % 16]."""
    return x.unflatten(-1, (8, 16)).unflatten(-3, (4, 4)).transpose(-3, -2)


def _key_rows(x):
    """The inverse of _key_order."""
    return x.transpose(-3, -2).flatten(-4, -3).flatten(-2)


def _raw(x):
    return x.view(torch.uint8)


def _cache(g, blocks, code):
    """Planes of codes and their exponents; keys with channels of different scales."""
    planes, exponents = [], torch.empty(blocks, KV, 2, dtype=torch.uint8, device="cuda")
    for which in range(2):
        channels = torch.exp(0.6 * _normal(g, KV, 1, DIM)) if which == 0 else 1.0
        plane = torch.empty(blocks, SLAB, dtype=torch.uint8, device="cuda")
        for at in range(0, blocks, 16384):  # (in pieces: the f32 values of a large pool would take its room many times)
            x = _normal(g, min(16384, blocks - at), KV, BLOCK, DIM, dtype=torch.float16).float() * channels
            e = _exponent(x.abs().amax((-2, -1)), code)
            x = _codes(x, e[..., None, None], code)
            plane[at:at + x.shape[0]] = _raw((_key_order(x) if which == 0 else x.transpose(-1, -2)).contiguous()).flatten(1)
            exponents[at:at + x.shape[0], :, which] = (e + BIAS).to(torch.uint8)
        planes.append(plane.view(_code_type(code)))
    return planes[0], planes[1], exponents


def _table(g, lens, blocks, width):
    """Block tables of sequences of `lens` rows over a pool in any order, -1 behind each one's last block."""
    ids = torch.randperm(blocks, generator=g, device="cuda", dtype=torch.int32)
    rows, at = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"), 0
    for i, t in enumerate(lens):
        rows[i, :_blocks(t)] = ids[at:at + _blocks(t)]
        at += _blocks(t)
    return rows


def _free_mask(refs):
    """One bit a block, set where it is free, in words of 32."""
    bits = torch.nn.functional.pad((refs == 0).to(torch.int64), (0, -refs.numel() % 32)).view(-1, 32)
    return (bits << torch.arange(32, device="cuda")).sum(1).to(torch.int32)


def _page_planes(g, blocks, width):
    """Keys, values (and, in 8 bits, the exponents) of all layers: [layers][blocks][elements]."""
    if width == 16:
        return [_normal(g, LAYERS, blocks, SLAB, dtype=torch.float16) for _ in range(2)]
    make = lambda n: torch.randint(0, 256, (LAYERS, blocks, n), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    return [make(SLAB), make(SLAB), make(4)]


def _parents(case):
    """Two steps of beam parents: a few beams of each batch entry lead on, some rows end."""
    rng, steps = random.Random("%d %d %d" % (case["batch"], case["beams"], case["hi"])), []
    for _ in range(2):
        rows = []
        for b in range(case["batch"]):
            leading = rng.sample(range(case["beams"]), -(-case["beams"] // 2))
            rows += [b * case["beams"] + rng.choice(leading) for _ in range(case["beams"])]
        steps.append(rows)
    return steps


def _inputs(case, seed):
    g, kind, s = torch.Generator(device="cuda").manual_seed(seed), case["kind"], dict(case)
    if kind == "decode":
        n, f32 = case["seqs"], case["io"] == "f32"
        lens = _lengths(n, case["lo"], case["hi"])
        if case["ragged"]:
            order = torch.randperm(n, generator=g, device="cuda").tolist()
            lens = [lens[i] for i in order]
            s["row_blocks"] = _blocks(case["hi"])
            s["blocks"] = sum(_blocks(t) for t in lens) + 7
            s["table"] = _table(g, lens, s["blocks"], s["row_blocks"])
        else:
            s["row_blocks"] = _blocks(case["hi"] + 64)
            s["blocks"] = n * s["row_blocks"]
            s["table"] = torch.arange(s["blocks"], dtype=torch.int32, device="cuda").view(n, -1)
        s["lens"] = _ints([t - 1 for t in lens])
        angle = torch.arange(case["hi"] + 1, device="cuda", dtype=torch.float64)[:, None] * ROPE_BASE ** (
            -torch.arange(0, DIM, 2, device="cuda", dtype=torch.float64) / DIM)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["k"], s["v"], s["exponents"] = _cache(g, s["blocks"], case["format"])
        s["q"], s["nk"], s["nv"] = (_normal(g, n, h, DIM, dtype=torch.float32 if f32 else torch.float16) for h in (HEADS, KV, KV))
    elif kind == "move":
        n = case["tokens"]
        s["blocks"] = _blocks(n) + 5
        s["table"] = torch.randperm(s["blocks"], generator=g, device="cuda", dtype=torch.int32)[:_blocks(n)].contiguous()
        channels = torch.exp(0.6 * _normal(g, KV, DIM))
        s["rows_k"], s["rows_v"] = (_normal(g, n, KV, DIM) * channels).half(), _normal(g, n, KV, DIM, dtype=torch.float16)
        s["k"], s["v"] = (torch.zeros(s["blocks"], SLAB, dtype=torch.uint8, device="cuda").view(_code_type(case["format"])) for _ in range(2))
        s["exponents"] = torch.zeros(s["blocks"], KV, 2, dtype=torch.uint8, device="cuda")
    elif kind == "beam":
        rows = case["batch"] * case["beams"]
        # a peaked distribution over a wide tail, as a head gives; scores of sequences of some length
        s["logits"] = _normal(g, rows, case["vocab"]).mul_(2.5)
        peaks = torch.randint(0, case["vocab"], (rows, 24), generator=g, device="cuda")
        s["logits"].scatter_add_(1, peaks, 9.0 + 2.0 * _normal(g, rows, 24))
        s["scores"] = -6.0 * torch.rand(case["batch"], case["beams"], generator=g, device="cuda")
        s["finished"] = (torch.rand(case["batch"], case["beams"], generator=g, device="cuda") < 0.2).to(torch.int32) if case["finished"] else None
        s["end"] = 2
    elif kind == "fork":
        beams = case["beams"]
        lens = [t for t in _lengths(case["batch"], case["lo"], case["hi"]) for _ in range(beams)]
        n, s["row_blocks"] = len(lens), _blocks(case["hi"] + 1)
        s["blocks"] = sum(_blocks(t + 1) for t in lens[::beams]) + 3 * n + 9
        # the beams of an entry share the blocks that they have filled, and each has its last one
        table = _table(g, lens[::beams], s["blocks"], s["row_blocks"]).repeat_interleave(beams, 0)
        left = torch.ones(s["blocks"], dtype=torch.bool, device="cuda")
        left[table[table >= 0].long()] = False
        spare = left.nonzero().flatten().to(torch.int32)
        rows = torch.tensor([i for i, t in enumerate(lens) if t % BLOCK], device="cuda", dtype=torch.long)
        ends = torch.tensor([t // BLOCK for t in lens if t % BLOCK], device="cuda", dtype=torch.long)
        if rows.numel():
            table[rows, ends] = spare[torch.randperm(spare.numel(), generator=g, device="cuda")[:rows.numel()]]
        s["tables"] = [table, torch.empty_like(table)]
        s["lens"] = [_ints(lens), torch.empty(n, dtype=torch.int32, device="cuda")]
        s["parents"] = [_ints(p) for p in _parents(case)]
    else:
        lens = _lengths(case["seqs"], case["lo"], case["hi"])
        n, s["row_blocks"] = case["seqs"], _blocks(case["hi"])
        s["blocks"] = sum(_blocks(t) for t in lens) * 5 // 4 + 9
        table = _table(g, lens, s["blocks"], s["row_blocks"])
        s["tables"] = [table, torch.empty_like(table)]
        s["lens"] = [_ints(lens), torch.empty(n, dtype=torch.int32, device="cuda")]
        s["full"], s["turn"] = _ints(lens), 0
        rows = torch.arange(n, dtype=torch.int32, device="cuda")
        s["stay"] = [torch.where(rows % 2 == i, rows, -1) for i in range(2)]
        s["rows"] = rows
        s["reserve"] = [torch.where(rows % 2 == i, 0, s["full"]) for i in range(2)]
    if kind in ("fork", "turnover"):
        s["refs"] = torch.bincount(table[table >= 0].long(), minlength=s["blocks"]).to(torch.int32)
        s["free"] = _free_mask(s["refs"])
        s["planes"] = _page_planes(g, s["blocks"], case["width"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # what a program keeps beside its data: outputs, workspaces and the calls' arguments
        _keep(s)
    return s


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _workspace(pvlc, nbytes):
    w = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(w, nbytes)
    return w


def _keep(s):
    from __graft_entry__ import load_package

    pvlc = s["pvlc"] = load_package()
    kind = s["kind"]
    if kind in ("decode", "move"):
        s["code"] = pvlc.KV_E4M3 if s["format"] == "e4m3" else pvlc.KV_INT8
    if kind == "decode":
        s["out"] = torch.empty_like(s["q"])
        nbytes = pvlc.decode_workspace_bytes(s["seqs"], s["row_blocks"] * BLOCK)
        s["ws"] = _workspace(pvlc, nbytes)
        caches = dict(block_tables=s["table"], cache_lens=s["lens"]) if s["ragged"] else dict(uniform_cache_len=s["hi"] - 1)
        names = ("query", "new_key", "new_value", "out")
        operands = dict.fromkeys(names) if s["io"] == "f32" else dict(zip(names, (s["q"], s["nk"], s["nv"], s["out"])))
        s["args"] = pvlc.paged_decode_q8_args(
            num_seqs=s["seqs"], num_blocks=s["blocks"], max_blocks_per_seq=s["row_blocks"], code=s["code"], key_cache=s["k"],
            value_cache=s["v"], exponents=s["exponents"], workspace=s["ws"], workspace_bytes=nbytes,
            max_context=s["row_blocks"] * BLOCK, rope_cos=s["cos"], rope_sin=s["sin"], rope_rows=s["cos"].shape[0],
            rotate_query=True, **operands, **caches)
    elif kind == "move":
        s["back_k"], s["back_v"] = torch.empty_like(s["rows_k"]), torch.empty_like(s["rows_v"])
    elif kind == "beam":
        shape = (s["batch"], s["best"])
        s["out"] = [torch.empty(shape, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32, torch.int32)]
        nbytes = pvlc.beam_workspace_bytes(s["batch"], s["beams"], s["vocab"], s["best"])
        s["ws"] = _workspace(pvlc, nbytes)
        s["args"] = pvlc.beam_select_args(
            batch=s["batch"], beams=s["beams"], vocab=s["vocab"], best=s["best"], logits=s["logits"], row_stride=s["vocab"],
            scores=s["scores"], finished=s["finished"], end_token=s["end"], next_scores=s["out"][0], parents=s["out"][1],
            tokens=s["out"][2], next_finished=s["out"][3], workspace=s["ws"], workspace_bytes=nbytes)
    else:
        nbytes = pvlc.kv_pages_workspace_bytes(s["blocks"], s["tables"][0].shape[0])
        s["ws"] = _workspace(pvlc, nbytes)
        s["pool"] = pvlc.kv_page_pool(
            num_blocks=s["blocks"], max_blocks_per_seq=s["row_blocks"], num_layers=LAYERS, planes=s["planes"],
            ref_counts=s["refs"], free_mask=s["free"], workspace=s["ws"], workspace_bytes=nbytes)


def _pages(s):
    """A pool's state: tables, lengths, what is held and free, and the pages as whole numbers (they are moved, not computed)."""
    return dict(tables=s["tables"][0], lens=s["lens"][0], ref_counts=s["refs"], free_mask=s["free"],
                planes=[p.view(torch.int16) if p.dtype == torch.float16 else p for p in s["planes"]])


def _run_own(s):
    pvlc, kind = s["pvlc"], s["kind"]
    if kind == "decode":
        if s["io"] == "f32":
            pvlc.paged_decode_q8_f32io(s["args"], s["q"], s["nk"], s["nv"], s["out"])
        else:
            pvlc.paged_decode_q8_f16(s["args"])
        return dict(out=s["out"], key_cache=s["k"], value_cache=s["v"], exponents=s["exponents"])
    if kind == "move":
        pvlc.kv_pack_q8(s["rows_k"], s["rows_v"], s["tokens"], s["k"], s["v"], s["exponents"], s["blocks"], s["code"], s["table"])
        pvlc.kv_unpack_q8(s["k"], s["v"], s["exponents"], s["tokens"], s["back_k"], s["back_v"], s["blocks"], s["code"], s["table"])
        return dict(keys=s["back_k"], values=s["back_v"], key_cache=s["k"], value_cache=s["v"], exponents=s["exponents"])
    if kind == "beam":
        pvlc.beam_select(s["args"])
        return dict(zip(("scores", "parents", "tokens", "finished"), s["out"]))
    n, (a, b), (len_a, len_b) = s["tables"][0].shape[0], s["tables"], s["lens"]
    if kind == "fork":
        pvlc.kv_pages_fork(s["pool"], rows_in=n, tables_in=a, lens_in=len_a, rows_out=n, parents=s["parents"][0], tables_out=b,
                           lens_out=len_b, reserve_tokens=1)
        pvlc.kv_pages_fork(s["pool"], rows_in=n, tables_in=b, lens_in=len_b, rows_out=n, parents=s["parents"][1], tables_out=a,
                           lens_out=len_a, reserve_tokens=1)
    else:
        turn = s["turn"]
        s["turn"] = 1 - turn
        pvlc.kv_pages_fork(s["pool"], rows_in=n, tables_in=a, lens_in=len_a, rows_out=n, parents=s["stay"][turn], tables_out=b,
                           lens_out=len_b)
        pvlc.kv_pages_compact(s["pool"], rows=n, tables=b)
        pvlc.kv_pages_fork(s["pool"], rows_in=n, tables_in=b, lens_in=len_b, rows_out=n, parents=s["rows"], tables_out=a,
                           lens_out=len_a, reserve=s["reserve"][turn])
        len_a.copy_(s["full"])  # the admitted prompts fill what was reserved for them
    return _pages(s)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _rotate(x, cos, sin):
    """Rotate-half of [n][heads][128] in 32 bits, products and sum each rounded, then the cache's fp16."""
    x, cos, sin = x.float(), cos[:, None], sin[:, None]
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat([lo * cos + (-hi) * sin, hi * cos + lo * sin], -1).half().float()


def _append(plane, e, row, ids, slot, code, which):
    """The row [n][2][128] into slot `slot` of the blocks `ids`: the block's exponent grows where the row needs it, and the
    rows before are rounded again at the new one."""
    order, rows = ((_key_order, _key_rows) if which == 0 else (lambda x: x.transpose(-1, -2),) * 2)
    n = row.shape[0]
    shape = (n, KV, 4, 8, 4, 16) if which == 0 else (n, KV, DIM, BLOCK)
    raw = _raw(plane)
    old = rows(raw[ids].view(shape)).contiguous()
    before = e[ids, :, which].int() - BIAS
    need = _exponent(row.abs().amax(-1), code)
    now = torch.where(slot[:, None] > 0, torch.maximum(before, need), need)
    value = old.view(plane.dtype).float() * _power(before)[..., None, None]
    token = torch.arange(BLOCK, device="cuda")[None, None, :, None]
    at = slot[:, None, None, None]
    value = torch.where(token == at, row[:, :, None], value)
    new = torch.where(token <= at, _raw(_codes(value, now[..., None, None], code)), old)
    raw[ids] = order(new).reshape(n, SLAB)
    e[ids, :, which] = (now + BIAS).to(torch.uint8)


def _plain_decode(s):
    n, lens, code = s["seqs"], s["lens"].long(), s["format"]
    cos, sin = s["cos"][lens], s["sin"][lens]
    q, nk, nv = _rotate(s["q"], cos, sin), _rotate(s["nk"], cos, sin), s["nv"].half().float()
    ids = s["table"].gather(1, (lens // BLOCK)[:, None])[:, 0].long()
    for which, (plane, row) in enumerate(((s["k"], nk), (s["v"], nv))):
        _append(plane, s["exponents"], row, ids, lens % BLOCK, code, which)
    every = s["table"].clamp_min(0).long()  # [n][row blocks]
    power = _power(s["exponents"][every].int() - BIAS)  # [n][blocks][2][2]
    k = s["k"].view(torch.uint8)[every].view(s["k"].dtype).float().view(n, -1, KV, 4, 8, 4, 16)
    k.mul_(power[..., 0, None, None, None, None])
    k = k.permute(0, 2, 4, 6, 1, 3, 5).reshape(n * KV, DIM, -1)  # [dim][token]
    scores = (q.view(n * KV, GROUP, DIM) @ k).mul_(1 / math.sqrt(DIM)).view(n, HEADS, -1)
    del k
    scores.masked_fill_(torch.arange(scores.shape[-1], device="cuda") > lens[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(n * KV, GROUP, -1)
    v = s["v"].view(torch.uint8)[every].view(s["v"].dtype).float().view(n, -1, KV, DIM, BLOCK)
    v.mul_(power[..., 1, None, None])
    v = v.permute(0, 2, 1, 4, 3).reshape(n * KV, -1, DIM)
    return dict(out=(p @ v).view(n, HEADS, DIM).to(s["q"].dtype), key_cache=s["k"], value_cache=s["v"], exponents=s["exponents"])


def _plain_move(s):
    n, ids, code, back = s["tokens"], s["table"].long(), s["format"], []
    for which, (rows, plane) in enumerate(((s["rows_k"], s["k"]), (s["rows_v"], s["v"]))):
        x = torch.nn.functional.pad(rows.float(), (0, 0, 0, 0, 0, -n % BLOCK)).view(-1, BLOCK, KV, DIM).transpose(1, 2)
        e = _exponent(x.abs().amax((-2, -1)), code)
        x = _codes(x, e[..., None, None], code)
        _raw(plane)[ids] = _raw((_key_order(x) if which == 0 else x.transpose(-1, -2)).contiguous()).view(-1, SLAB)
        s["exponents"][ids, :, which] = (e + BIAS).to(torch.uint8)
        codes, e = _raw(plane)[ids].view(plane.dtype).float(), s["exponents"][ids, :, which].int() - BIAS
        codes = _key_rows(codes.view(-1, KV, 4, 8, 4, 16)) if which == 0 else codes.view(-1, KV, DIM, BLOCK).transpose(-1, -2)
        x = (codes * _power(e)[..., None, None]).clamp(-65504, 65504).half()
        back.append(x.transpose(1, 2).reshape(-1, KV, DIM)[:n].contiguous())
    return dict(keys=back[0], values=back[1], key_cache=s["k"], value_cache=s["v"], exponents=s["exponents"])


def _plain_beam(s):
    batch, beams, vocab, best = s["batch"], s["beams"], s["vocab"], s["best"]
    x = s["logits"]
    most = x.amax(1, keepdim=True)
    # the sums and the candidates' scores in 64 bits: candidates of two beams may lie closer than 32 tell apart
    total = most[:, 0].double() + torch.exp(x - most).sum(1, dtype=torch.float64).log()
    # a beam's best by logit, equal ones by token: one whole number that orders both
    bits = x.view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + (0xFFFFFFFF - torch.arange(vocab, device="cuda"))
    take = min(best, vocab)
    tokens = 0xFFFFFFFF - (key.topk(take, 1).values & 0xFFFFFFFF)  # [rows][take], best first
    score = s["scores"].double().view(-1, 1) + (x.gather(1, tokens).double() - total[:, None])
    if s["finished"] is not None:  # a finished beam goes on as it is, by its end token
        done, first = s["finished"].view(-1, 1) != 0, torch.arange(take, device="cuda") == 0
        score = torch.where(done, torch.where(first, s["scores"].double().view(-1, 1), -math.inf), score)
        tokens = torch.where(done & first, s["end"], tokens)
    score, tokens = score.view(batch, -1), tokens.view(batch, -1)
    if score.shape[1] < best:
        score = torch.nn.functional.pad(score, (0, best - score.shape[1]), value=-math.inf)
        tokens = torch.nn.functional.pad(tokens, (0, best - tokens.shape[1]))
    score, at = score.sort(dim=1, descending=True, stable=True)
    score, at = score[:, :best], at[:, :best]
    none = score == -math.inf
    tokens = tokens.gather(1, at).masked_fill(none, -1)
    parents = (at // take + beams * torch.arange(batch, device="cuda")[:, None]).masked_fill(none, -1)
    finished = tokens == s["end"]
    if s["finished"] is not None:
        finished |= s["finished"].view(-1)[parents.clamp_min(0)] != 0
    finished &= ~none
    return dict(scores=score.float(), parents=parents.int(), tokens=tokens.int(), finished=finished.int())


def _plain_fork(s, source, lens, parents, target, lens_out, reserve):
    """Rows of `source` taken over by the rows of `target` that name them: filled blocks are shared, the block that a row
    writes next is the first child's own and copied for the others, blocks without a row become free."""
    n, width = source.shape
    has, p = parents >= 0, parents.clamp_min(0).long()
    length = torch.where(has, lens[p], 0)
    filled = (length // BLOCK)[:, None]
    need = ((length + reserve + BLOCK - 1) // BLOCK)[:, None]
    rows, j = torch.arange(n, device="cuda"), torch.arange(width, device="cuda")[None]
    first = torch.full((n,), n, device="cuda").scatter_reduce_(0, p[has], rows[has], "amin")
    keeper = has & (first[p] == rows)
    entry = source[p]
    sole = (entry >= 0) & (s["refs"][entry.clamp_min(0).long()] == 1) & keeper[:, None]
    kept = ((sole | (j < filled)).int().cumprod(1).sum(1, keepdim=True)).clamp_min(0)  # blocks from the first one on
    kept = torch.minimum(torch.where(has[:, None], kept, 0), need)
    fresh = (j >= kept) & (j < need)
    order = torch.argsort((s["refs"] != 0).to(torch.int8), stable=True)  # the free blocks, lowest first
    number = (fresh.flatten().cumsum(0) - 1).clamp_min(0).view(n, width)
    out = torch.where(fresh, order[number.clamp_max(order.numel() - 1)].int(), torch.where((j < kept) & has[:, None], entry, -1))
    copied = has & (length % BLOCK > 0) & (kept[:, 0] <= filled[:, 0])
    at = filled[copied]
    src, dst = entry[copied].gather(1, at.long())[:, 0].long(), out[copied].gather(1, at.long())[:, 0].long()
    for plane in s["planes"]:
        plane[:, dst] = plane[:, src]
    one = torch.ones((), dtype=torch.int32, device="cuda")
    for table, sign in ((source, -one), (out, one)):
        held = table.flatten() >= 0
        s["refs"].scatter_add_(0, table.flatten().clamp_min(0).long(), torch.where(held, sign, 0))
    s["free"].copy_(_free_mask(s["refs"]))
    target.copy_(out)
    lens_out.copy_(length)


def _plain_compact(s, table):
    """The used blocks behind as many as there are move to the free ones before, in order."""
    used, at = s["refs"] > 0, torch.arange(s["blocks"], device="cuda")
    live = used.sum()
    src, dst = at[used & (at >= live)], at[~used & (at < live)]
    forward = at.int()
    forward[src] = dst.int()
    for plane in s["planes"]:
        plane[:, dst] = plane[:, src]
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    s["free"].copy_(_free_mask(s["refs"]))
    table.copy_(torch.where(table >= 0, forward[table.clamp_min(0).long()], table))


def _run_plain(s):
    kind = s["kind"]
    if kind == "decode":
        return _plain_decode(s)
    if kind == "move":
        return _plain_move(s)
    if kind == "beam":
        return _plain_beam(s)
    (a, b), (len_a, len_b) = s["tables"], s["lens"]
    if kind == "fork":
        _plain_fork(s, a, len_a, s["parents"][0], b, len_b, 1)
        _plain_fork(s, b, len_b, s["parents"][1], a, len_a, 1)
    else:
        turn = s["turn"]
        s["turn"] = 1 - turn
        _plain_fork(s, a, len_a, s["stay"][turn], b, len_b, 0)
        _plain_compact(s, b)
        _plain_fork(s, b, len_b, s["rows"], a, len_a, s["reserve"][turn])
        len_a.copy_(s["full"])
    return _pages(s)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it gives in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "decode":
        lens, operand = _lengths(case["seqs"], case["lo"], case["hi"]), 4 if case["io"] == "f32" else 2
        # keys, values and exponents once; the query and the new row in, the row and the output out
        each = [2 * KV * DIM * (t - 1) + 2 * KV * _blocks(t) + (2 * HEADS + 2 * KV) * DIM * operand + 2 * KV * DIM for t in lens]
        return dict(bytes=sum(each), flops=4 * HEADS * DIM * sum(lens))
    if kind == "move":  # fp16 rows in and out, codes out and in
        return dict(bytes=case["tokens"] * KV * DIM * 2 * (2 + 1 + 1 + 2) + 8 * _blocks(case["tokens"]), flops=0)
    if kind == "beam":  # the logits once; a difference, an exponential, a sum and a comparison each
        count = case["batch"] * case["beams"] * case["vocab"]
        return dict(bytes=4 * count + 16 * case["batch"] * case["best"], flops=4 * count)
    page = LAYERS * (2 * SLAB * 2 if case["width"] == 16 else 2 * SLAB + 4)
    if kind == "fork":
        lens = [t for t in _lengths(case["batch"], case["lo"], case["hi"]) for _ in range(case["beams"])]
        tables = 2 * 4 * sum(_blocks(t) for t in lens)
        # every child but the first of a parent gets a copy of the last block, if that is not full
        copies = sum(len(step) - len(set(step)) - sum(lens[p] % BLOCK == 0 for i, p in enumerate(step) if p in step[:i]) for step in _parents(case))
        return dict(bytes=2 * tables + 2 * page * copies, flops=0)
    used = [_blocks(t) for t in _lengths(case["seqs"], case["lo"], case["hi"])]
    # the sequences that stay were admitted behind those that end, and move into their place
    moved = min(sum(used[0::2]), sum(used[1::2]))
    return dict(bytes=2 * page * moved + 6 * 4 * sum(used), flops=0)


def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_codes(x, e, code):
    """The nearest codes' values (ties to even) of f64 values at exponents e, times their power."""
    y = (x * _exact_power(-e)).clamp(-LARGEST[code], LARGEST[code])
    if code == "int8":
        step = torch.ones_like(y)
    else:
        step = _exact_power((torch.frexp(y).exponent - 1).clamp_min(-6) - 3)
    return (y / step).round() * step * _exact_power(e)


def _exact_exponent(most, code):
    e = torch.ceil(torch.log2((most / LARGEST[code]).clamp_min(2.0 ** LEAST_EXPONENT)))
    e = torch.where(most > LARGEST[code] * _exact_power(e), e + 1, e)  # (the logarithm is rounded)
    return torch.where((e > LEAST_EXPONENT) & (most <= LARGEST[code] * _exact_power(e - 1)), e - 1, e)


def _exact_decode(case, s):
    outs = []
    for i, last in enumerate(s["lens"].tolist()):
        ids = s["table"][i, :_blocks(last + 1)].long()
        e = s["exponents"][ids].long() - BIAS
        k = s["k"].view(torch.uint8)[ids].view(s["k"].dtype).float().double().view(-1, KV, 4, 8, 4, 16).permute(0, 2, 4, 1, 3, 5)
        v = s["v"].view(torch.uint8)[ids].view(s["v"].dtype).float().double().view(-1, KV, DIM, BLOCK).permute(0, 3, 1, 2)
        k, v = k.reshape(-1, BLOCK, KV, DIM) * _exact_power(e)[:, None, :, :1], v * _exact_power(e)[:, None, :, 1:]
        c, sn = s["cos"][last], s["sin"][last]
        turn = lambda x: torch.cat([x[:, :64] * c - x[:, 64:] * sn, x[:, 64:] * c + x[:, :64] * sn], 1).half().double()  # noqa: E731
        q, slot = turn(s["q"][i].float()), last % BLOCK  # (a rotation's products and sum are rounded to 32 bits, the result to 16)
        for which, (rows, new) in enumerate(((k, turn(s["nk"][i].float())), (v, s["nv"][i].half().double()))):
            now = _exact_exponent(new.abs().amax(1), case["format"])
            if slot:
                now = torch.maximum(now, e[-1, :, which])
            rows[-1, slot] = new
            rows[-1, :slot + 1] = _exact_codes(rows[-1, :slot + 1], now[:, None], case["format"])
        k, v = k.reshape(-1, KV, DIM)[:last + 1], v.reshape(-1, KV, DIM)[:last + 1]
        scores = torch.stack([q[h] @ k[:, h // GROUP].t() for h in range(HEADS)]) / math.sqrt(DIM)
        p = torch.softmax(scores, 1)
        outs.append(torch.stack([p[h] @ v[:, h // GROUP] for h in range(HEADS)]))
    return dict(out=torch.stack(outs), key_cache=None, value_cache=None, exponents=None)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "turnover"):
        return None  # whole numbers and moved bytes
    s = _inputs(case, seed)
    if kind == "decode":
        return _exact_decode(case, s)
    if kind == "move":
        back, n = [], case["tokens"]
        for rows in (s["rows_k"], s["rows_v"]):
            x = rows.double()
            for at in range(0, n, BLOCK * 4096):
                piece = torch.nn.functional.pad(x[at:at + BLOCK * 4096], (0, 0, 0, 0, 0, -min(n - at, BLOCK * 4096) % BLOCK)).view(-1, BLOCK, KV, DIM)
                e = _exact_exponent(piece.abs().amax((1, 3)), case["format"])
                x[at:at + BLOCK * 4096] = _exact_codes(piece, e[:, None, :, None], case["format"]).view(-1, KV, DIM)[:n - at]
            back.append(x)
        return dict(keys=back[0], values=back[1], key_cache=None, value_cache=None, exponents=None)
    scores = []
    for b in range(case["batch"]):
        each = []
        for w in range(case["beams"]):
            start = s["scores"][b, w].double()
            if s["finished"] is not None and s["finished"][b, w]:
                each.append(start.view(1))
            else:
                x = s["logits"][b * case["beams"] + w].double()
                each.append(start + x - torch.logsumexp(x, 0))
        every = torch.cat(each).sort(descending=True).values[:case["best"]]
        scores.append(torch.nn.functional.pad(every, (0, case["best"] - every.numel()), value=-math.inf))
    return dict(scores=torch.stack(scores), parents=None, tokens=None, finished=None)
