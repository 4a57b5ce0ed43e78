"""Refusals of the batches over paged caches, on the host: every one is an error with its code before any GPU effect (the
pointers here are numbers)."""

import numpy as np
import pytest

from pvlc_testlib import pvlc
from test_serving_abi import refused

M = 1 << 32  # addresses far apart, aligned to anything
COMMON = dict(num_seqs=3, num_blocks=64, max_blocks_per_seq=8, key_cache=M, value_cache=2 * M, block_tables=3 * M, cache_lens=4 * M)
ROWS = dict(COMMON, rows=30, row_offsets=5 * M)
QUERY, KEY, VALUE, OUT = 6 * M, 7 * M, 8 * M, 9 * M
WORKSPACE = dict(workspace=10 * M, workspace_bytes=1 << 34)


def append(change, f32=False):
    operands = [change.pop("key", KEY), change.pop("value", VALUE)]
    args = pvlc.kv_append_args(**{**dict(ROWS, code=pvlc.KV_F16), **change})
    return lambda: (pvlc.kv_append_f32 if f32 else pvlc.kv_append_f16)(args, *operands)


def prefill(change, f32=False):
    operands = [change.pop(n, at) for n, at in zip(("query", "key", "value", "out"), (QUERY, KEY, VALUE, OUT))]
    args = pvlc.packed_prefill_args(**{**dict(ROWS, max_context=128, **WORKSPACE), **change})
    return lambda: (pvlc.packed_prefill_f32io if f32 else pvlc.packed_prefill_f16)(args, *operands)


def shared(change, f32=False):
    operands = [change.pop(n, at) for n, at in zip(("query", "key", "value", "out"), (QUERY, KEY, VALUE, OUT))]
    args = pvlc.shared_decode_args(**{**dict(COMMON, num_groups=3, shared_lens=5 * M, max_context=128, **WORKSPACE), **change})
    return lambda: (pvlc.shared_decode_f32io if f32 else pvlc.shared_decode_f16)(args, *operands)


CALLS = pytest.mark.parametrize("call", [append, prefill, shared])


@CALLS
@pytest.mark.parametrize("change,code", [
    (dict(num_seqs=0), "ZeroDimension"), (dict(num_blocks=0), "ZeroDimension"), (dict(max_blocks_per_seq=0), "ZeroDimension"),
    (dict(key_cache=None), "LengthMismatch"), (dict(value_cache=2 * M + 8), "LengthMismatch"), (dict(key=None), "LengthMismatch"),
    (dict(value=VALUE + 8), "LengthMismatch"), (dict(block_tables=3 * M + 2), "LengthMismatch"), (dict(cache_lens=4 * M + 1), "LengthMismatch"),
    (dict(positions=M + 3), "LengthMismatch"), (dict(rope_cos=M, rope_rows=9), "InvalidRotaryDimension"),
    (dict(rope_cos=11 * M, rope_sin=12 * M), "InvalidRotaryDimension"), (dict(rope_cos=11 * M + 4, rope_sin=12 * M, rope_rows=9), "LengthMismatch"),
    (dict(num_blocks=1 << 31), "InvalidDecoderGeometry"), (dict(max_blocks_per_seq=1 << 28), "InvalidDecoderGeometry"),
    (dict(key=M + 64 * 8192 - 16), "InvalidActivationLayout"), (dict(value_cache=M + 4096), "InvalidActivationLayout"),
    (dict(block_tables=M + 512), "InvalidActivationLayout"), (dict(cache_lens=2 * M), "InvalidActivationLayout")])
def test_common_refusals(call, change, code):
    refused(call(dict(change)), code)
    refused(call(dict(change), True), code)


@pytest.mark.parametrize("change,code", [
    (dict(rows=0), "ZeroDimension"), (dict(code=3), "InvalidActivationLayout"), (dict(code=pvlc.KV_INT8), "LengthMismatch"),
    (dict(code=pvlc.KV_E4M3, exponents=M * 13 + 2), "LengthMismatch"), (dict(code=pvlc.KV_E4M3, exponents=M + 8), "InvalidActivationLayout"),
    (dict(row_offsets=None, rows=31), "InvalidSequenceBoundaries"), (dict(row_offsets=5 * M + 2), "LengthMismatch"),
    (dict(rows=1 << 31), "InvalidDecoderGeometry"), (dict(num_seqs=1 << 23, rows=1 << 23), "InvalidDecoderGeometry"),
    (dict(block_tables=None, num_blocks=23), "InvalidDecoderGeometry"), (dict(key_stride=255), "InvalidActivationLayout"),
    (dict(value_stride=260), "InvalidActivationLayout"), (dict(key_stride=1 << 31), "InvalidActivationLayout"),
    (dict(error_word=M * 13 + 2), "LengthMismatch"), (dict(error_word=KEY + 64), "InvalidActivationLayout")])
def test_append_refuses(change, code):
    refused(append(dict(change)), code)


def test_append_strides_are_elements():
    """A stride of 258 elements is 1032 bytes of f32, no multiple of 16; of 260, 1040 bytes, one."""
    refused(append(dict(key_stride=258), True), "InvalidActivationLayout")
    refused(append(dict(key_stride=260, value=None), True), "LengthMismatch")  # (the next check)


@pytest.mark.parametrize("change,code", [
    (dict(rows=0), "ZeroDimension"), (dict(max_context=0), "ZeroDimension"), (dict(max_context=129), "InvalidDecoderGeometry"),
    (dict(query=None), "LengthMismatch"), (dict(out=None), "LengthMismatch"), (dict(query=QUERY + 2), "LengthMismatch"),
    (dict(out=OUT + 4), "LengthMismatch"), (dict(query_stride=2047), "InvalidActivationLayout"), (dict(workspace=None), "LengthMismatch"),
    (dict(workspace=10 * M + 128), "LengthMismatch"), (dict(workspace_bytes=255), "LengthMismatch"), (dict(out=QUERY), "InvalidActivationLayout"),
    (dict(out=KEY - 16), "InvalidActivationLayout"), (dict(out=10 * M), "InvalidActivationLayout"), (dict(workspace=5 * M), "InvalidActivationLayout")])
def test_prefill_refuses(change, code):
    refused(prefill(dict(change)), code)


@pytest.mark.parametrize("change,code", [
    (dict(num_groups=0), "ZeroDimension"), (dict(num_groups=2), "InvalidSequenceBoundaries"), (dict(shared_lens=None), "LengthMismatch"),
    (dict(block_tables=None), "LengthMismatch"), (dict(cache_lens=None), "LengthMismatch"), (dict(group_offsets=M + 2), "LengthMismatch"),
    (dict(shared_lens=5 * M + 1), "LengthMismatch"), (dict(max_context=0), "ZeroDimension"), (dict(max_context=129), "InvalidDecoderGeometry"),
    (dict(num_seqs=9000, num_groups=9000, num_blocks=1 << 20), "InvalidDecoderGeometry"), (dict(code=7), "InvalidActivationLayout"),
    (dict(code=pvlc.KV_E4M3), "LengthMismatch"), (dict(query=None), "LengthMismatch"), (dict(out=OUT + 8), "LengthMismatch"),
    (dict(workspace=None), "LengthMismatch"), (dict(workspace_bytes=256), "LengthMismatch"), (dict(out=QUERY + 4096), "InvalidActivationLayout"),
    (dict(shared_lens=OUT), "InvalidActivationLayout"), (dict(group_offsets=2 * M), "InvalidActivationLayout")])
def test_shared_refuses(change, code):
    refused(shared(dict(change)), code)


def test_workspace_sizes():
    """The sizes that the helpers give are taken (a NULL output is the next refusal), none is needed for nothing, and with
    group offsets a call never needs more."""
    assert pvlc.packed_prefill_workspace_bytes(0, 5, 5) == 0 and pvlc.shared_decode_workspace_bytes(4, 0, 9) == 0
    for seqs, groups, context in ((1, 1, 1), (4, 1, 1200), (64, 16, 5000), (256, 256, 40000), (8000, 10, 64), (16000, 384, 100)):
        nbytes = pvlc.shared_decode_workspace_bytes(seqs, groups, context)
        width = -(-context // 16)
        base = dict(num_seqs=seqs, num_groups=groups, max_context=context, max_blocks_per_seq=width, num_blocks=64)
        for more in (dict(), dict(group_offsets=11 * M)):
            if not more and seqs % groups:
                continue
            message = refused(shared(dict(base, workspace_bytes=256, **more)), "LengthMismatch")
            assert int(message.rsplit(" ", 1)[1]) <= nbytes, (seqs, groups, context)
        pvlc.packed_prefill_workspace_bytes(seqs, seqs * 3, context)


@CALLS
def test_tables_of_nearly_2_31_tokens(call):
    """Positions are whole numbers of 32 bits, and so is one rounded up to the next pieces of keys."""
    refused(call(dict(max_blocks_per_seq=(1 << 27) - 15)), "InvalidDecoderGeometry")
    refused(call(dict(max_blocks_per_seq=(1 << 27) - 16, key=None)), "LengthMismatch")  # (a later check)


def test_prefill_grid():
    """Two workgroups of 256 threads for every 16 rows and for every sequence: fewer than 2^32 threads."""
    far = dict(query=1 << 44, key=2 << 44, value=3 << 44, out=4 << 44, workspace_bytes=1 << 40, row_offsets=5 << 44, cache_lens=6 << 44, block_tables=7 << 44)
    refused(prefill(dict(far, num_seqs=1 << 22, rows=1 << 26)), "InvalidDecoderGeometry")
    refused(prefill(dict(far, num_seqs=1 << 22, rows=1 << 25, workspace=None)), "LengthMismatch")  # (the next check)


def needed(call, change):
    """What a call says that it needs, given too little."""
    return int(refused(call(dict(change, workspace_bytes=256)), "LengthMismatch").rsplit(" ", 1)[1])


def test_a_shared_workspace_serves_smaller_calls():
    """A batch that shrinks, as its pages finish, keeps the workspace of its largest step."""
    far = dict(zip(("query", "key", "value", "out"), (x << 44 for x in range(1, 5))))
    g = np.random.default_rng(3)
    largest = [(64, 16, 4096), (72, 9, 32768), (256, 32, 32768), (4, 1, 1300), (7, 7, 262144), (2000, 100, 500), (12000, 4000, 40), (300, 300, 5000),
               (1, 1, 1)] + [tuple(int(np.exp(g.uniform(0, np.log(top)))) for top in (4096, 512, 1 << 18)) for _ in range(12)]
    for seqs, groups, context in largest:
        nbytes = pvlc.shared_decode_workspace_bytes(seqs, groups, context)
        smaller = [(seqs * a // b, max(1, groups * a // b), max(1, context // c)) for a, b in ((1, 1), (9, 10), (3, 4), (1, 2), (1, 3), (1, 16), (1, 100)) for c in (1, 2, 5, 64)]
        smaller += [tuple(int(g.integers(1, top + 1)) for top in (seqs, groups, context)) for _ in range(40)]
        smaller += [(n, n, c) for n in range(1, min(seqs, groups) + 1, 7) for c in (context, max(1, context // 2))]
        for n, m, c in smaller:
            base = dict(far, num_seqs=n, num_groups=m, max_context=c, max_blocks_per_seq=-(-c // 16), num_blocks=64)
            for more in (dict(), dict(group_offsets=11 * M)):
                if n and (more or n % m == 0):
                    assert needed(shared, dict(base, **more)) <= nbytes, (seqs, groups, context, n, m, c, more)


def test_a_packed_workspace_serves_smaller_calls():
    far = dict(zip(("query", "key", "value", "out"), (x << 44 for x in range(1, 5))))
    g = np.random.default_rng(4)
    largest = [(1025, 5000, 4096), (1024, 5000, 4096), (3000, 3000, 513), (72, 1152, 4096), (73, 73, 600), (4, 32768, 8192), (1, 1, 1), (40, 9000, 512)]
    largest += [tuple(int(np.exp(g.uniform(0, np.log(top)))) for top in (4096, 1 << 16, 1 << 16)) for _ in range(12)]
    for seqs, rows, context in largest:
        nbytes = pvlc.packed_prefill_workspace_bytes(seqs, rows, context)
        smaller = [(max(1, seqs * a // b), max(1, rows * d // b), max(1, context // c)) for a, b in ((1, 1), (99, 100), (1, 2), (1, 40)) for d in (a, b) for c in (1, 2, 9)]
        smaller += [tuple(int(g.integers(1, top + 1)) for top in (seqs, rows, context)) for _ in range(40)]
        for n, r, c in smaller:
            base = dict(far, num_seqs=n, rows=r, max_context=c, max_blocks_per_seq=-(-c // 16), num_blocks=64)
            assert needed(prefill, base) <= nbytes, (seqs, rows, context, n, r, c)
