"""Operators of batched serving over a paged cache, and their plain forms.

``own`` says which side ``run`` takes: the package's entry points, or elementary torch operations in 32 bits.
Kinds of work, and the ranges that ``draw`` takes its sizes from:

* ``append``   rows of several sequences rotated into the pages behind what each holds: 1 to 65536 rows of 1 to 256
               sequences, fp16 or f32 rows, compact or slices of one q|k|v matrix; fp16, e4m3 or int8 pages;
* ``prefill``  prompts of different lengths in one call, each causal over its own pages, on what its cache holds already:
               1 to 32768 rows of 1 to 128 sequences, up to 16384 rows before them;
* ``shared``   a decode step of groups of sequences (the beams of a page, answers to one prompt) whose first pages are the
               same ones: 1 to 32 groups of 1 to 64 rows, 16 to 32768 shared rows; fp16, e4m3 or int8 pages.
"""

import math

import torch

own = False

HEADS, KV, DIM, BLOCK = 16, 2, 128, 16
GROUP, WIDTH = HEADS // KV, (HEADS + 2 * KV) * DIM  # query heads of a key head; elements of a row of q|k|v
SLAB = KV * DIM * BLOCK  # elements of one block of one plane
ROPE_BASE = 500000.0
LARGEST = {"e4m3": 448.0, "int8": 127.0}
LEAST_EXPONENT, BIAS = -32, 127


def listed():
    return [
        # a few drafted tokens for each sequence of a batch that is being recognised
        dict(name="append_drafts", kind="append", seqs=24, lo=1, hi=4, held=2010, io="f32", pages="f16", fused=False, positions=False),
        # one page's prompt into 8-bit pages, its image tokens at positions of their own
        dict(name="append_page", kind="append", seqs=1, lo=1157, hi=1157, held=0, io="f32", pages="e4m3", fused=False, positions=True),
        # a batch of pages admitted at once, their keys and values in the rows of one q|k|v projection
        dict(name="append_batch", kind="append", seqs=16, lo=90, hi=2010, held=0, io="f16", pages="f16", fused=True, positions=False),
        # long documents, in chunks on what was taken before
        dict(name="append_long", kind="append", seqs=8, lo=4096, hi=14336, held=16384, io="f16", pages="int8", fused=False, positions=False),
        # short instructions, no images
        dict(name="prefill_few", kind="prefill", seqs=3, lo=5, hi=97, held=0, io="f32", fused=False, positions=False),
        # a batch of pages admitted at once
        dict(name="prefill_pages", kind="prefill", seqs=12, lo=211, hi=2010, held=0, io="f16", fused=True, positions=True),
        # chunks of long documents, each on thousands of rows before it
        dict(name="prefill_chunks", kind="prefill", seqs=6, lo=256, hi=512, held=16384, io="f32", fused=False, positions=False),
        # the largest: whole documents
        dict(name="prefill_long", kind="prefill", seqs=4, lo=4096, hi=8192, held=0, io="f16", fused=False, positions=False),
        # one page searched with four beams, on its projections' f32 operands
        dict(name="shared_page", kind="shared", groups=1, rows=4, lo=1157, hi=1157, tail=64, io="f32", pages="f16"),
        # a batch of pages with eight beams each, 8-bit pages
        dict(name="shared_batch", kind="shared", groups=16, rows=8, lo=300, hi=2010, tail=200, io="f16", pages="e4m3"),
        # many answers to one long document
        dict(name="shared_document", kind="shared", groups=1, rows=64, lo=16384, hi=16384, tail=500, io="f32", pages="int8"),
        # the largest: many long documents, eight beams each
        dict(name="shared_long", kind="shared", groups=32, rows=8, lo=8192, hi=32768, tail=500, io="f16", pages="f16"),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "prefill", "prefill", "shared", "shared"])
    io, pages = rng.choice(["f16", "f32"]), rng.choice(["f16", "e4m3", "int8"])
    if kind == "append":
        seqs = _log(rng, 1, 256)
        hi = _log(rng, 1, min(16384, 65536 // seqs))
        return dict(kind=kind, seqs=seqs, lo=_log(rng, max(1, hi // 32), hi), hi=hi, held=rng.choice([0, _log(rng, 1, 8192)]), io=io,
                    pages=pages, fused=rng.random() < 0.5, positions=rng.random() < 0.5)
    if kind == "prefill":
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, min(8192, 32768 // seqs))
        held = rng.choice([0, _log(rng, 1, 16384)])
        while seqs * hi * (held + (hi + 1) // 2) > 1 << 26:
            held, hi = held * 3 // 4, hi if held > hi else hi * 3 // 4
        return dict(kind=kind, seqs=seqs, lo=_log(rng, max(1, hi // 32), hi), hi=hi, held=held, io=io, fused=rng.random() < 0.5,
                    positions=rng.random() < 0.5)
    groups = _log(rng, 1, 32)
    hi = _log(rng, 16, 32768)
    return dict(kind=kind, groups=groups, rows=_log(rng, 1, min(64, 256 // groups, (1 << 22) // (groups * hi))), lo=_log(rng, max(16, hi // 32), hi), hi=hi,
                tail=_log(rng, 1, 500), io=io, pages=pages)


def _blocks(tokens):
    return -(-tokens // BLOCK)


def _spread(n, lo, hi):
    """Whole numbers evenly spread over the logarithm of lo..hi, every fifth of the way through them, so not in order."""
    every = [min(hi, max(lo, int(round(lo * (hi / lo) ** ((i + 0.5) / n))))) for i in range(n)]
    step = next(k for k in (5, 7, 11, 1) if n % k or k == 1)
    return [every[i * step % n] for i in range(n)]


def _held(case):
    """Rows that each sequence's cache holds before the call; the last of several has none."""
    n = case["seqs"]
    if not case["held"]:
        return [0] * n
    return [case["held"]] if n == 1 else _spread(n - 1, max(1, case["held"] // 8), case["held"]) + [0]


def _tails(case):
    """Rows of its own that each sequence of a shared decode holds."""
    n = case["groups"] * case["rows"]
    return [int((i - 0.5) * case["tail"] / n) for i in _spread(n, 1, n)]


# ---------------------------------------------------------------------------
# Inputs, made from the seed alone
# ---------------------------------------------------------------------------

def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


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


_SWAP = [(t & 3) | ((t & 4) << 1) | ((t & 8) >> 1) for t in range(BLOCK)]  # the slot of a token in an fp16 key block


def _raw(x):
    return x.view(torch.int16) if x.dtype == torch.float16 else x.view(torch.uint8)


def _to_block(x, pages, which):
    """[..., token 16, dim 128] in the order in which a block keeps keys (which 0) or values (1)."""
    if which:
        return x.transpose(-1, -2)
    if pages == "f16":  # [dim / 8][slot][dim % 8]; the slots' order is its own inverse
        return x[..., _SWAP, :].unflatten(-1, (16, 8)).transpose(-3, -2)
    return x.unflatten(-1, (8, 16)).unflatten(-3, (4, 4)).transpose(-3, -2)  # [token / 4][dim / 16][token % 4][dim % 16]


def _from_block(x, pages, which):
    """[..., elements of a block of one head] as [..., token 16, dim 128]."""
    if which:
        return x.unflatten(-1, (DIM, BLOCK)).transpose(-1, -2)
    if pages == "f16":
        return x.unflatten(-1, (16, BLOCK, 8)).transpose(-3, -2).flatten(-2)[..., _SWAP, :]
    return x.unflatten(-1, (4, 8, 4, 16)).transpose(-3, -2).flatten(-4, -3).flatten(-2)


def _cache(g, blocks, pages):
    """Planes of keys (with channels of different scales) and values, and the exponents of 8-bit ones."""
    planes, exponents = [], None if pages == "f16" else torch.empty(blocks, KV, 2, dtype=torch.uint8, device="cuda")
    for which in range(2):
        channels = torch.exp(0.6 * _normal(g, KV, 1, DIM)) if which == 0 else 1.0
        plane = torch.empty(blocks, SLAB, dtype=torch.float16 if pages == "f16" else torch.uint8, device="cuda")
        for at in range(0, blocks, 16384):  # (in pieces: the f32 values of a large pool would take its room many times)
            x = (_normal(g, min(16384, blocks - at), KV, BLOCK, DIM, dtype=torch.float16).float() * channels).half()
            if pages != "f16":
                e = _exponent(x.float().abs().amax((-2, -1)), pages)
                exponents[at:at + x.shape[0], :, which] = (e + BIAS).to(torch.uint8)
                x = _raw(_codes(x.float(), e[..., None, None], pages))
            plane[at:at + x.shape[0]] = _to_block(x, pages, which).reshape(-1, SLAB)
        planes.append(plane if pages == "f16" else plane.view(torch.float8_e4m3fn if pages == "e4m3" else torch.int8))
    return planes[0], planes[1], exponents


def _angles(rows):
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * ROPE_BASE ** (
        -torch.arange(0, DIM, 2, device="cuda", dtype=torch.float64) / DIM)
    return angle.cos().float(), angle.sin().float()


def _inputs(case, seed):
    g, s = torch.Generator(device="cuda").manual_seed(seed), dict(case)
    dtype = torch.float32 if case["io"] == "f32" else torch.float16
    s["pages"] = case.get("pages", "f16")
    if case["kind"] == "shared":
        n = case["groups"] * case["rows"]
        s["shared"] = _spread(case["groups"], case["lo"], case["hi"])
        # what each sequence holds: the shared rows, and some of its own behind them
        s["held"] = [s["shared"][i // case["rows"]] + t for i, t in enumerate(_tails(case))]
        s["counts"] = [1] * n
        s["row_blocks"] = _blocks(case["hi"] + case["tail"] + 1)
    else:
        n, s["counts"], s["held"] = case["seqs"], _spread(case["seqs"], case["lo"], case["hi"]), _held(case)
        s["row_blocks"] = _blocks(max(a + b for a, b in zip(s["counts"], s["held"])))
    ends = [a + b for a, b in zip(s["counts"], s["held"])]
    total, s["n"] = sum(s["counts"]), n
    # block tables over a pool in any order, -1 behind each sequence's last block; a group shares its first whole blocks
    same = [t // BLOCK for t in s["shared"]] if case["kind"] == "shared" else [0] * n
    each = case["rows"] if case["kind"] == "shared" else 1
    s["blocks"] = sum(same) + sum(_blocks(t) - same[i // each] for i, t in enumerate(ends)) + 7
    ids = torch.randperm(s["blocks"], generator=g, device="cuda", dtype=torch.int32).cpu()
    table, at = torch.full((n, s["row_blocks"]), -1, dtype=torch.int32), 0
    for i, t in enumerate(ends):
        m = same[i // each]
        if i % each == 0:
            table[i:i + each, :m] = ids[at:at + m]
            at += m
        table[i, m:_blocks(t)] = ids[at:at + _blocks(t) - m]
        at += _blocks(t) - m
    s["table"] = table.cuda()
    s["lens"] = _ints(s["held"])
    s["offsets"] = _ints([0] + torch.tensor(s["counts"]).cumsum(0).tolist())
    s["cos"], s["sin"] = _angles(max(ends))
    s["k"], s["v"], s["exponents"] = _cache(g, s["blocks"], s["pages"])
    # the rows: matrices of their own, or slices of one [rows][q|k|v]
    if case.get("fused"):
        rows = _normal(g, total, WIDTH, dtype=dtype)
        s["q"], s["nk"], s["nv"] = (x.unflatten(1, (-1, DIM)) for x in rows.split([HEADS * DIM, KV * DIM, KV * DIM], 1))
    else:
        s["q"], s["nk"], s["nv"] = (_normal(g, total, h, DIM, dtype=dtype) for h in (HEADS, KV, KV))
    s["positions"] = None
    if case.get("positions"):  # of an image's tokens: a few at each position, none past the sequence's length
        s["positions"] = torch.cat([(torch.arange(h, h + c) * 5 // 8).int() for c, h in zip(s["counts"], s["held"])]).cuda()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # what a program keeps beside its data: outputs, workspaces and the calls' arguments
        _keep(s)
    return s


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _keep(s):
    from __graft_entry__ import load_package

    pvlc = s["pvlc"] = load_package()
    code = {"f16": pvlc.KV_F16, "e4m3": pvlc.KV_E4M3, "int8": pvlc.KV_INT8}[s["pages"]]
    common = dict(num_blocks=s["blocks"], max_blocks_per_seq=s["row_blocks"], key_cache=s["k"], value_cache=s["v"], block_tables=s["table"],
                  cache_lens=s["lens"], rope_cos=s["cos"], rope_sin=s["sin"], rope_rows=s["cos"].shape[0], positions=s["positions"])
    context = s["row_blocks"] * BLOCK
    rows = s["q"].shape[0]
    strides = dict(key_stride=s["nk"].stride(0), value_stride=s["nv"].stride(0))
    if s["kind"] == "append":
        s["args"] = pvlc.kv_append_args(num_seqs=s["n"], rows=rows, code=code, exponents=s["exponents"], row_offsets=s["offsets"], **strides,
                                        **common)
        return
    s["out"] = torch.empty(rows, HEADS, DIM, dtype=s["q"].dtype, device="cuda")
    if s["kind"] == "prefill":
        nbytes = pvlc.packed_prefill_workspace_bytes(s["n"], rows, context)
    else:
        nbytes = pvlc.shared_decode_workspace_bytes(s["n"], s["groups"], context)
    s["ws"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    pvlc.workspace_init(s["ws"], nbytes)
    common.update(max_context=context, workspace=s["ws"], workspace_bytes=nbytes)
    if s["kind"] == "prefill":
        s["args"] = pvlc.packed_prefill_args(num_seqs=s["n"], rows=rows, row_offsets=s["offsets"], query_stride=s["q"].stride(0), **strides,
                                             **common)
    else:
        s["shared_lens"] = _ints(s["shared"])
        s["args"] = pvlc.shared_decode_args(num_seqs=s["n"], num_groups=s["groups"], shared_lens=s["shared_lens"], code=code,
                                            exponents=s["exponents"], rotate_query=True, **common)


def _run_own(s):
    pvlc, f32 = s["pvlc"], s["io"] == "f32"
    if s["kind"] == "append":
        (pvlc.kv_append_f32 if f32 else pvlc.kv_append_f16)(s["args"], s["nk"], s["nv"])
    elif s["kind"] == "prefill":
        (pvlc.packed_prefill_f32io if f32 else pvlc.packed_prefill_f16)(s["args"], s["q"], s["nk"], s["nv"], s["out"])
    else:
        (pvlc.shared_decode_f32io if f32 else pvlc.shared_decode_f16)(s["args"], s["q"], s["nk"], s["nv"], s["out"])
    return _outputs(s, s.get("out"))


def _outputs(s, out):
    every = dict(out=out, key_cache=s["k"], value_cache=s["v"], exponents=s["exponents"])
    return {name: x for name, x in every.items() if x is not None}


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _rotate(x, cos, sin):
    """Rotate-half of [n][heads][128] in 32 bits, products and sum each rounded, then the cache's fp16."""
    x, cos, sin = x.float(), cos[:, None], sin[:, None]
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat([lo * cos + (-hi) * sin, hi * cos + lo * sin], -1).half().float()


def _places(s):
    """Of every row: its sequence, its place in that, and its position."""
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["offsets"], row, right=True, out_int32=False) - 1
    place = s["lens"][seq].long() + row - s["offsets"][seq]
    return seq, place, place if s["positions"] is None else s["positions"].long()


def _plain_append(s):
    """The rows' keys rotated, and keys and values written behind what the pages hold."""
    seq, place, position = _places(s)
    k, v = _rotate(s["nk"], s["cos"][position], s["sin"][position]), s["nv"].half().float()
    # a block of values for each block that a sequence may write, numbered with room to spare
    first, count = s["lens"].long() // BLOCK, s["q"].shape[0] // BLOCK + 2 * s["n"]
    base = s["offsets"][:-1].long() // BLOCK + 2 * torch.arange(s["n"], device="cuda")
    unit, slot = base[seq] + place // BLOCK - first[seq], place % BLOCK
    ids = torch.zeros(count, dtype=torch.long, device="cuda")  # (those that none writes stand for block 0, and write it as it is)
    ids[unit] = s["table"][seq, place // BLOCK].long()
    new = torch.zeros(count, BLOCK, dtype=torch.bool, device="cuda")
    new[unit, slot] = True
    used = new.any(1)
    ids = torch.where(used, ids, ids[unit[0]])
    for which, (plane, rows) in enumerate(((s["k"], k), (s["v"], v))):
        raw = _raw(plane)
        if s["pages"] == "f16":
            index = torch.arange(SLAB, device="cuda").view(KV, -1)
            order = _from_block(index, "f16", which)  # [head][token][dim]
            raw.view(-1)[(s["table"][seq, place // BLOCK].long() * SLAB)[:, None, None] + order[:, slot].transpose(0, 1)] = _raw(rows.half())
            continue
        value = torch.zeros(count, BLOCK, KV, DIM, device="cuda")
        value[unit, slot] = rows
        value = value.transpose(1, 2)
        old = _from_block(raw[ids].view(count, KV, -1), s["pages"], which).contiguous()
        fresh, before = new.to(torch.int8).argmax(1) == 0, s["exponents"][ids, :, which].int() - BIAS
        need = _exponent(value.abs().amax((-2, -1)), s["pages"])
        now = torch.where(fresh[:, None], need, torch.maximum(before, need))
        now = torch.where(used[:, None], now, before)
        at = torch.arange(BLOCK, device="cuda")
        earlier = (at < new.to(torch.int8).argmax(1)[:, None])[:, None, :, None]
        value = torch.where(earlier, old.view(plane.dtype).float() * _power(before)[..., None, None], value)
        changed = (earlier | new[:, None, :, None]) & used[:, None, None, None]
        value = torch.where(changed, _raw(_codes(value, now[..., None, None], s["pages"])), old)
        value = _to_block(value, s["pages"], which).reshape(count, SLAB)
        # (unused numbers repeat the first used one, whose row they take)
        at = torch.where(used, torch.arange(count, device="cuda"), unit[0])
        raw[ids] = value[at]
        s["exponents"][ids, :, which] = (now + BIAS).to(torch.uint8)[at]


def _held_rows(s, ids, which):
    """Keys or values of blocks, f32 [heads][rows][128]."""
    x = _from_block(s["kv"[which]][ids].float().view(-1, KV, BLOCK * DIM), s["pages"], which)
    if s["pages"] != "f16":
        x = x * _power(s["exponents"][ids, :, which].int() - BIAS)[..., None, None]
    return x.transpose(0, 1).flatten(1, 2).contiguous()


def _softmax(scores):
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_prefill(s):
    _plain_append(s)
    _, _, position = _places(s)
    q, out, at = _rotate(s["q"], s["cos"][position], s["sin"][position]), torch.empty_like(s["q"], memory_format=torch.contiguous_format), 0
    for i, (count, held) in enumerate(zip(s["counts"], s["held"])):
        ids = s["table"][i, :_blocks(held + count)].long()
        k, v = _held_rows(s, ids, 0), _held_rows(s, ids, 1)
        for lo in range(0, count, 1024):
            hi = min(count, lo + 1024)
            end = held + hi
            piece = q[at + lo:at + hi].view(hi - lo, KV, GROUP, DIM).permute(1, 2, 0, 3).reshape(KV, -1, DIM)
            scores = (piece @ k[:, :end].transpose(1, 2).contiguous()).mul_(1 / math.sqrt(DIM)).view(KV, GROUP, hi - lo, end)
            later = torch.arange(end, device="cuda") > torch.arange(held + lo, held + hi, device="cuda")[:, None]
            p = _softmax(scores.masked_fill_(later, -math.inf)).view(KV, -1, end)
            out[at + lo:at + hi] = (p @ v[:, :end]).view(KV, GROUP, hi - lo, DIM).permute(2, 0, 1, 3).reshape(hi - lo, HEADS, DIM)
        at += count
    return _outputs(s, out)


def _plain_shared(s):
    _plain_append(s)
    _, _, position = _places(s)
    q, out, n = _rotate(s["q"], s["cos"][position], s["sin"][position]), torch.empty_like(s["q"]), s["rows"]
    for i, shared in enumerate(s["shared"]):
        whole, rows = shared // BLOCK, slice(i * n, (i + 1) * n)
        ends = s["held"][rows]
        tails = s["table"][rows, whole:_blocks(max(ends) + 1)].clamp_min(0).long()
        piece = q[rows].view(n, KV, GROUP, DIM).transpose(0, 1)
        # the shared rows for all of the group at once, then each one's own
        k = _held_rows(s, s["table"][i * n, :whole].long(), 0) if whole else q.new_empty(KV, 0, DIM)
        scores = [(piece.reshape(KV, -1, DIM) @ k.transpose(1, 2).contiguous()).view(KV, n, GROUP, -1)]
        k = _held_rows(s, tails.flatten(), 0).view(KV, n, -1, DIM)
        scores.append(piece @ k.transpose(2, 3).contiguous())
        scores = torch.cat(scores, -1).mul_(1 / math.sqrt(DIM))
        later = torch.arange(scores.shape[-1], device="cuda") > s["lens"][rows, None]
        p = _softmax(scores.masked_fill_(later[None, :, None], -math.inf))
        v = _held_rows(s, tails.flatten(), 1).view(KV, n, -1, DIM)
        total = p[..., whole * BLOCK:].contiguous() @ v
        if whole:
            v = _held_rows(s, s["table"][i * n, :whole].long(), 1)
            total = total + (p[..., :whole * BLOCK].reshape(KV, n * GROUP, -1) @ v).view(KV, n, GROUP, DIM)
        out[rows] = total.transpose(0, 1).reshape(n, HEADS, DIM).to(out.dtype)
    return _outputs(s, out)


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "append":
        _plain_append(state)
        return _outputs(state, None)
    return _plain_prefill(state) if state["kind"] == "prefill" else _plain_shared(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it gives in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    operand, kind = 4 if case["io"] == "f32" else 2, case["kind"]
    element = 2 if case.get("pages", "f16") == "f16" else 1
    token = 2 * KV * DIM  # key and value elements of a token
    if kind == "shared":  # the shared rows once a group, each sequence's own, the operands, the new rows
        n = case["groups"] * case["rows"]
        shared, tails = sum(_spread(case["groups"], case["lo"], case["hi"])), sum(_tails(case))
        return dict(bytes=(shared + tails) * token * element + n * (2 * HEADS * DIM + token) * operand + n * token * element,
                    flops=4 * HEADS * DIM * (case["rows"] * shared + tails + n))
    counts, held = _spread(case["seqs"], case["lo"], case["hi"]), _held(case)
    written = sum(counts) * token * (operand + element)
    if kind == "append":
        return dict(bytes=written, flops=6 * sum(counts) * KV * DIM // 2)
    pairs = sum(c * h + c * (c + 1) // 2 for c, h in zip(counts, held))
    return dict(bytes=written + sum(held) * token * element + sum(counts) * 2 * HEADS * DIM * operand, flops=4 * HEADS * DIM * pairs)


def _two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_exponent(most, code):
    e = torch.ceil(torch.log2((most / LARGEST[code]).clamp_min(2.0 ** LEAST_EXPONENT)))
    e = torch.where(most > LARGEST[code] * _two(e), e + 1, e)  # (the logarithm is rounded)
    return torch.where((e > LEAST_EXPONENT) & (most <= LARGEST[code] * _two(e - 1)), e - 1, e)


def _exact_codes(x, e, code):
    """The codes' values nearest to x 2^-e (ties to even)."""
    y = (x * _two(-e)).clamp(-LARGEST[code], LARGEST[code])
    step = torch.ones_like(y) if code == "int8" else _two((torch.frexp(y).exponent - 1).clamp_min(-6) - 3)
    return (y / step).round() * step


def _index(pages, which):
    """Of (token, dim) of a block of one head: where its element lies."""
    t, d = torch.arange(BLOCK, device="cuda")[:, None], torch.arange(DIM, device="cuda")[None]
    if which:
        return d * BLOCK + t
    if pages == "f16":
        return d // 8 * 128 + ((t & 3) + ((t >> 2) & 1) * 8 + (t >> 3) * 4) * 8 + d % 8
    return t // 4 * 512 + d // 16 * 64 + t % 4 * 16 + d % 16


def _exact_turn(x, cos, sin):
    """A rotation as it enters a cache of fp16 values: products and sum are rounded to 32 bits, the result to 16."""
    x, c, n = x.float(), cos[:, None], sin[:, None]
    return torch.cat([x[..., :64] * c - x[..., 64:] * n, x[..., 64:] * c + x[..., :64] * n], -1).half().double()


def exact(case, seed):
    s = _inputs(case, seed)
    pages, at, outs = s["pages"], 0, []
    where = [_index(pages, w).flatten() for w in range(2)]
    planes = [x.double().view(s["blocks"], KV, -1) for x in (s["k"], s["v"])]
    exponents = None if pages == "f16" else s["exponents"].long() - BIAS
    for i, (count, held) in enumerate(zip(s["counts"], s["held"])):
        rows = slice(at, at + count)
        at += count
        places = torch.arange(held, held + count, device="cuda")
        position = places if s["positions"] is None else s["positions"][rows].long()
        turn = _exact_turn(s["nk"][rows], s["cos"][position], s["sin"][position])
        news = (turn, s["nv"][rows].half().double())
        if case["kind"] == "append" and pages == "f16":  # (an output here: what it is before it is rounded)
            x, c, n = s["nk"][rows].double(), s["cos"][position][:, None].double(), s["sin"][position][:, None].double()
            news = (torch.cat([x[..., :64] * c - x[..., 64:] * n, x[..., 64:] * c + x[..., :64] * n], -1), s["nv"][rows].double())
        lo = held // BLOCK
        ids = s["table"][i, lo:_blocks(held + count)].long()
        for which, new in enumerate(news):
            block = planes[which][ids][..., where[which]].view(-1, KV, BLOCK, DIM)  # in the order of tokens
            flat = block.transpose(1, 2).reshape(-1, KV, DIM)
            if pages == "f16":
                flat[held - lo * BLOCK:held - lo * BLOCK + count] = new
                block = flat.view(-1, BLOCK, KV, DIM).transpose(1, 2)
            else:
                mine = torch.zeros_like(flat)
                mine[held - lo * BLOCK:held - lo * BLOCK + count] = new
                mine = mine.view(-1, BLOCK, KV, DIM).transpose(1, 2)
                e = _exact_exponent(mine.abs().amax((2, 3)), pages)
                if held % BLOCK:
                    e[0] = torch.maximum(e[0], exponents[ids[0], :, which])
                token = torch.arange(block.shape[0] * BLOCK, device="cuda").view(-1, 1, BLOCK, 1) + lo * BLOCK
                value = torch.where(token < held, block * _two(exponents[ids, :, which])[..., None, None], mine)
                block = torch.where(token < held + count, _exact_codes(value, e[..., None, None].long(), pages), block)
                exponents[ids, :, which] = e.long()
            planes[which][ids[:, None], :, where[which][None]] = block.flatten(2).transpose(1, 2)
        if case["kind"] == "append":
            continue
        every = s["table"][i, :_blocks(held + count)].long()
        k, v = (planes[w][every][..., where[w]].view(-1, KV, BLOCK, DIM) for w in range(2))
        if pages != "f16":
            k, v = (x * _two(exponents[every, :, w])[..., None, None] for w, x in enumerate((k, v)))
        k, v = (x.transpose(1, 2).reshape(-1, KV, DIM)[:held + count] for x in (k, v))
        q, out = _exact_turn(s["q"][rows], s["cos"][position], s["sin"][position]), torch.empty(count, HEADS, DIM, dtype=torch.float64, device="cuda")
        for h in range(HEADS):
            for first in range(0, count, 2048):
                last = min(count, first + 2048)
                scores = (q[first:last, h] @ k[:held + last, h // GROUP].t().contiguous()) / math.sqrt(DIM)
                scores.masked_fill_(torch.arange(held + last, device="cuda")[None] > places[first:last, None], -math.inf)
                out[first:last, h] = torch.softmax(scores, 1) @ v[:held + last, h // GROUP]
        outs.append(out)
    planes = [x.reshape(s["blocks"], SLAB) for x in planes]
    if case["kind"] != "append":  # (the caches are rounded before they are read: `append` says what they hold)
        return _outputs(dict(s, k=None, v=None, exponents=None), torch.cat(outs)) | {n: None for n in _outputs(s, None)}
    return _outputs(dict(s, k=planes[0], v=planes[1], exponents=None if exponents is None else exponents + BIAS), None)
