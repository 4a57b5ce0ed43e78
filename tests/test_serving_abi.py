"""Refusals of the 8-bit cache, the page pool and the beam selection, on the host: every one is an error with its code
before any GPU effect (the pointers here are numbers)."""

import ctypes

import pytest

from __graft_entry__ import load_package

pvlc = load_package()
P = 0x10000  # an address, aligned to anything


def refused(call, code):
    with pytest.raises(pvlc.PvlcHipError) as e:
        call()
    assert (e.value.code, e.value.invocation_code) == ("InvalidInvocation", code), str(e.value)
    return str(e.value)


# -- 8-bit decode ------------------------------------------------------------------------------------------------

def decode(**k):
    f32 = k.pop("f32", False)
    base = dict(num_seqs=2, num_blocks=64, max_blocks_per_seq=8, code=pvlc.KV_E4M3, key_cache=P, value_cache=P, exponents=P, query=P,
                new_key=P, new_value=P, out=P, workspace=P, workspace_bytes=1 << 24, max_context=100, uniform_cache_len=50)
    if f32:
        base.update(query=None, new_key=None, new_value=None, out=None)
    args = pvlc.paged_decode_q8_args(**{**base, **k})
    return (lambda: pvlc.paged_decode_q8_f32io(args, P, P, P, P)) if f32 else (lambda: pvlc.paged_decode_q8_f16(args))


@pytest.mark.parametrize("change,code", [
    (dict(code=2), "InvalidActivationLayout"), (dict(exponents=None), "LengthMismatch"), (dict(exponents=P + 2), "LengthMismatch"),
    (dict(key_cache=None), "LengthMismatch"), (dict(value_cache=P + 8), "LengthMismatch"), (dict(num_seqs=0), "ZeroDimension"),
    (dict(query=None), "LengthMismatch"), (dict(out=P + 4), "LengthMismatch"), (dict(workspace=None), "LengthMismatch"),
    (dict(workspace_bytes=64), "LengthMismatch"), (dict(rope_cos=P), "InvalidRotaryDimension"),
    (dict(max_context=129), "InvalidDecoderGeometry"), (dict(uniform_cache_len=100), "InvalidDecoderGeometry"),
    (dict(num_blocks=15), "InvalidDecoderGeometry"), (dict(partition_tokens=24), "InvalidDecoderGeometry"),
    (dict(partition_tokens=8192), "InvalidDecoderGeometry"), (dict(num_seqs=65536, num_blocks=1 << 20, cache_lens=P), "InvalidDecoderGeometry"),
    (dict(f32=True, query=P), "LengthMismatch")])
def test_decode_q8_refuses(change, code):
    refused(decode(**change), code)


def test_decode_q8_partitions_fit_the_fp16_workspace():
    """Every automatic 8-bit launch runs in the workspace that the fp16 decode's helper sizes: a workspace one byte short
    of it may be refused, but none is refused for the size the helper gives."""
    for seqs in (1, 2, 3, 7, 18, 40, 64, 100, 129, 256, 300, 2500):
        for context in (1, 16, 65, 300, 700, 1157, 2048, 4000, 9000, 32768, 200000):
            blocks = -(-context // 16)
            nbytes = pvlc.decode_workspace_bytes(seqs, context)
            for extra in (dict(cache_lens=P), dict(uniform_cache_len=context - 1)):
                # NULL query: refused for that after the geometry, or for the geometry
                args = pvlc.paged_decode_q8_args(num_seqs=seqs, num_blocks=seqs * blocks, max_blocks_per_seq=blocks, code=pvlc.KV_INT8,
                                                 key_cache=P, value_cache=P, exponents=P, query=P, new_key=P, new_value=P, out=P,
                                                 workspace=P, workspace_bytes=256, max_context=context, **extra)
                message = refused(lambda: pvlc.paged_decode_q8_f16(args), "LengthMismatch")
                needs = int(message.rsplit(" ", 1)[1])
                assert needs <= nbytes, (seqs, context, extra, needs, nbytes)


# -- moves -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("change,code", [
    (dict(code=7), "InvalidActivationLayout"), (dict(key_rows=None), "LengthMismatch"), (dict(key_rows=P + 1), "LengthMismatch"),
    (dict(tokens=0), "ZeroDimension"), (dict(num_blocks=0), "ZeroDimension"), (dict(num_blocks=3), "InvalidDecoderGeometry"),
    (dict(key_cache=P + 8), "LengthMismatch"), (dict(exponents=P + 1), "LengthMismatch"), (dict(value_cache=None), "LengthMismatch"),
    (dict(first_token=0xFFFFFFF0, block_table=P), "ArithmeticOverflow"), (dict(first_token=20, tokens=45), "InvalidDecoderGeometry")])
def test_moves_refuse(change, code):
    base = dict(key_rows=P, value_rows=P, tokens=60, key_cache=P, value_cache=P, exponents=P, num_blocks=4, code=pvlc.KV_E4M3)
    refused(lambda: pvlc.kv_pack_q8(**{**base, **change}), code)
    if "first_token" not in change:
        refused(lambda: pvlc.kv_unpack_q8(**{**base, **change}), code)


# -- pages -------------------------------------------------------------------------------------------------------

def pool(**k):
    planes = k.pop("planes", [(P, 4096, 4096 * 100)] * 3)
    base = dict(num_blocks=100, max_blocks_per_seq=10, num_layers=2, planes=planes, ref_counts=P, free_mask=P, workspace=P, workspace_bytes=1 << 24)
    return pvlc.kv_page_pool(**{**base, **k})


def fork(p=None, **k):
    base = dict(rows_in=4, rows_out=4, tables_in=P, lens_in=P, tables_out=2 * P, lens_out=2 * P)
    return lambda: pvlc.kv_pages_fork(p or pool(), **{**base, **k})


@pytest.mark.parametrize("change,code", [
    (dict(num_blocks=0), "ZeroDimension"), (dict(num_layers=0), "ZeroDimension"), (dict(num_layers=65536), "InvalidDecoderGeometry"),
    (dict(num_blocks=1 << 31), "InvalidDecoderGeometry"), (dict(max_blocks_per_seq=1 << 28), "InvalidDecoderGeometry"),
    (dict(ref_counts=None), "LengthMismatch"), (dict(free_mask=P + 2), "LengthMismatch"), (dict(workspace=P + 128), "LengthMismatch"),
    (dict(workspace_bytes=255), "LengthMismatch"), (dict(planes=[(None, 4096, 409600)]), "LengthMismatch"),
    (dict(planes=[(P, 6, 600)]), "InvalidActivationLayout"), (dict(planes=[(P + 2, 4096, 409600)]), "InvalidActivationLayout"),
    (dict(planes=[(P, 4096, 4096 * 99)]), "InvalidActivationLayout"), (dict(planes=[(P, 1 << 32, 1 << 40)]), "ArithmeticOverflow"),
    (dict(planes=[(P, 0, 409600)]), "InvalidActivationLayout")])
def test_pools_refuse(change, code):
    refused(lambda: pvlc.kv_pages_reset(pool(**change)), code)
    refused(fork(pool(**change)), code)
    refused(lambda: pvlc.kv_pages_compact(pool(**change)), code)
    refused(lambda: pvlc.kv_pages_copy(pool(**change), P, pool(), P, 1), code)


@pytest.mark.parametrize("change,code", [
    (dict(rows_in=0, rows_out=0), "ZeroDimension"), (dict(rows_in=4097), "InvalidDecoderGeometry"), (dict(rows_out=4097), "InvalidDecoderGeometry"),
    (dict(tables_in=None), "LengthMismatch"), (dict(lens_out=None), "LengthMismatch"), (dict(parents=P + 1), "LengthMismatch"),
    (dict(tables_out=P), "InvalidActivationLayout"), (dict(tables_out=P + 4 * 39), "InvalidActivationLayout"),
    (dict(lens_out=P + 12), "InvalidActivationLayout"), (dict(rows_out=3000), "LengthMismatch")])
def test_forks_refuse(change, code):
    small = pool(workspace_bytes=pvlc.kv_pages_workspace_bytes(100, 4))
    refused(fork(small if change.get("rows_out") == 3000 else None, **change), code)


def test_forks_refuse_a_grid_of_rows_and_layers():
    refused(fork(pool(num_layers=60000, planes=[(P, 16, 1600)]), rows_out=400, tables_out=P * 100, lens_out=P * 100), "InvalidDecoderGeometry")


def test_compactions_and_copies_refuse():
    refused(lambda: pvlc.kv_pages_compact(pool(), rows=3), "LengthMismatch")
    refused(lambda: pvlc.kv_pages_compact(pool(), rows=3, tables=P + 2), "LengthMismatch")
    refused(lambda: pvlc.kv_pages_compact(pool(), forward=P + 2), "LengthMismatch")
    refused(lambda: pvlc.kv_pages_compact(pool(), rows=65536, tables=P), "InvalidDecoderGeometry")
    copy = lambda a, b, n=1, s=P, d=P: lambda: pvlc.kv_pages_copy(a, s, b, d, n)  # noqa: E731
    refused(copy(pool(), pool(), 0), "ZeroDimension")
    refused(copy(pool(), pool(), 1 << 24), "InvalidDecoderGeometry")
    refused(copy(pool(), pool(), 1, None), "LengthMismatch")
    refused(copy(pool(), pool(num_layers=3)), "InvalidActivationLayout")
    refused(copy(pool(), pool(planes=[(P, 4096, 409600)])), "InvalidActivationLayout")
    refused(copy(pool(), pool(planes=[(P, 4096, 409600)] * 2 + [(P, 16, 1600)])), "InvalidActivationLayout")


def test_page_planes_of_the_wrong_shape_refuse():
    torch = pytest.importorskip("torch")
    for p in (torch.zeros(2, 100), torch.zeros(3, 100, 8), torch.zeros(2, 99, 8), torch.zeros(2, 8, 100).transpose(1, 2)):
        refused(lambda: pool(planes=[p]), "InvalidActivationLayout")
    refused(lambda: pool(planes=[]), "InvalidDecoderGeometry")
    refused(lambda: pool(planes=[(P, 4, 400)] * 5), "InvalidDecoderGeometry")


def test_page_workspace_sizes():
    assert pvlc.kv_pages_workspace_bytes(0, 5) == 0
    assert pvlc.kv_pages_workspace_bytes(1, 0) > 0
    assert pvlc.kv_pages_workspace_bytes(1 << 20, 4096) < 14 << 20


# -- beams -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("change,code", [
    (dict(batch=0), "ZeroDimension"), (dict(best=0), "ZeroDimension"), (dict(beams=65), "InvalidDecoderGeometry"),
    (dict(best=129), "InvalidDecoderGeometry"), (dict(vocab=1 << 31), "InvalidDecoderGeometry"), (dict(batch=20000, beams=4), "InvalidDecoderGeometry"),
    (dict(batch=10000, vocab=1 << 30), "InvalidDecoderGeometry"), (dict(row_stride=999), "InvalidActivationLayout"),
    (dict(logits=None), "LengthMismatch"), (dict(scores=None), "LengthMismatch"), (dict(tokens=None), "LengthMismatch"),
    (dict(logits=P + 2), "LengthMismatch"), (dict(next_finished=P * 9 + 1), "LengthMismatch"), (dict(workspace=P + 16), "LengthMismatch"),
    (dict(workspace=None), "LengthMismatch"), (dict(workspace_bytes=1000), "LengthMismatch"), (dict(next_scores=P * 2), "InvalidActivationLayout"),
    (dict(next_scores=P * 2 + 28), "InvalidActivationLayout"), (dict(next_finished=P * 3, finished=P * 3), "InvalidActivationLayout")])
def test_beams_refuse(change, code):
    base = dict(batch=2, beams=4, vocab=1000, best=4, logits=P, scores=P * 2, next_scores=P * 5, parents=P * 6, tokens=P * 7, workspace=P * 8,
                workspace_bytes=1 << 26)
    refused(lambda: pvlc.beam_select(pvlc.beam_select_args(**{**base, **change})), code)


def test_beam_workspace_sizes():
    assert pvlc.beam_workspace_bytes(0, 4, 1000, 4) == 0
    assert pvlc.beam_workspace_bytes(1, 4, 103424, 4) < 1 << 20
    # 26 segments of 4096 logits and 16 keys, and what a row leaves
    assert pvlc.beam_workspace_bytes(16, 8, 103424, 16) < 128 * (26 * (16 * 8 + 12) + 16 * 16) + 4096


def test_null_argument_structs_refuse():
    null = None
    for name, args in (("pvlc_hip_paged_decode_q8_f16", (null, null)), ("pvlc_hip_paged_decode_q8_f32io", (null, P, P, P, P, null)),
                       ("pvlc_hip_kv_pages_reset", (null, null)), ("pvlc_hip_kv_pages_fork", (ctypes.byref(pool()), null, null)),
                       ("pvlc_hip_kv_pages_fork", (null, null, null)), ("pvlc_hip_beam_select_f32", (null, null)),
                       ("pvlc_hip_kv_pages_compact", (null, null, 0, null, null)), ("pvlc_hip_kv_pages_copy", (null, P, null, P, 1, null))):
        status = getattr(pvlc.lib, name)(*args)
        assert status == (3 << 8 | 2), name


def test_outputs_over_any_input_refuse():
    """What a call reads may not lie under what it writes, whichever operand it is."""
    for change in (dict(parents=2 * P), dict(reserve=2 * P + 8), dict(lens_in=2 * P + 32), dict(tables_out=3 * P, lens_out=3 * P + 60)):
        refused(fork(**{"tables_out": 2 * P, "lens_out": 4 * P, **change}), "InvalidActivationLayout")
    base = dict(batch=2, beams=4, vocab=1000, best=4, logits=P * 16, scores=P * 2, next_scores=P * 5, parents=P * 6, tokens=P * 7, workspace=P * 8,
                workspace_bytes=1 << 26)
    for change in (dict(tokens=P * 16), dict(next_scores=P * 16 + 7 * 4000 + 3996), dict(parents=P * 17, row_stride=(P + 2000) // 4)):
        refused(lambda: pvlc.beam_select(pvlc.beam_select_args(**{**base, **change})), "InvalidActivationLayout")


def test_sizes_beyond_the_grid_or_64_bits_refuse():
    move = dict(key_rows=P, value_rows=P, key_cache=P, value_cache=P, exponents=P, num_blocks=1 << 31, code=pvlc.KV_INT8)
    for table in (None, P):
        refused(lambda: pvlc.kv_pack_q8(tokens=1 << 28, block_table=table, **move), "InvalidDecoderGeometry")
        refused(lambda: pvlc.kv_pack_q8(tokens=100, first_token=1 << 28, block_table=table, **move), "InvalidDecoderGeometry")
        refused(lambda: pvlc.kv_unpack_q8(tokens=1 << 28, block_table=table, **move), "InvalidDecoderGeometry")
    refused(lambda: pvlc.kv_pages_reset(pool(planes=[(P, 4096, 1 << 60)])), "ArithmeticOverflow")
    refused(lambda: pvlc.beam_select(pvlc.beam_select_args(
        batch=2, beams=4, vocab=1000, best=4, logits=P, scores=P * 2, next_scores=P * 5, parents=P * 6, tokens=P * 7, workspace=P * 8,
        workspace_bytes=1 << 26, row_stride=1 << 60)), "ArithmeticOverflow")
