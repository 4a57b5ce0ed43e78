"""fp16 rows into the 8-bit cache and back (pvlc_hip_kv_pack_q8 / _unpack_q8) against the plain form: every byte of the
planes and exponents, whatever is not a row's left as it was."""

import numpy as np
import pytest

import q8_ref as R
from pvlc_testlib import log, pvlc, to_dev, to_dev_i32

pytestmark = pytest.mark.gpu


def rows(seed, n, scale=1.0):
    g = np.random.default_rng(seed)
    channels = np.exp(0.8 * g.standard_normal((2, 128)))
    k = (g.standard_normal((n, 2, 128)) * channels * scale).astype(np.float16)
    v = (g.standard_normal((n, 2, 128)) * scale).astype(np.float16)
    return k, v


class Device:
    def __init__(self, cache):
        import torch
        put = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        self.key, self.value, self.exponents = put(cache.key), put(cache.value), put(cache.exponents)
        self.blocks, self.code = cache.key.shape[0], cache.code

    def pack(self, k, v, first, table, stream=None, offset=0):
        pad = np.zeros(offset, np.uint16)
        d = [to_dev(np.concatenate([pad, np.ascontiguousarray(x).view(np.uint16).ravel()]))[offset:] for x in (k, v)]
        pvlc.kv_pack_q8(d[0], d[1], len(k), self.key, self.value, self.exponents, self.blocks, self.code, table, first, stream)
        return d

    def unpack(self, n, table, offset=0):
        import torch
        out = [torch.full((n * 256 + offset,), 7.0, dtype=torch.float16, device="cuda")[offset:] for _ in range(2)]
        pvlc.kv_unpack_q8(self.key, self.value, self.exponents, n, out[0], out[1], self.blocks, self.code, table)
        torch.cuda.synchronize()
        return [o.cpu().numpy().reshape(n, 2, 128) for o in out]

    def same(self, cache, what):
        import torch
        torch.cuda.synchronize()
        for name in ("key", "value", "exponents"):
            got, want = getattr(self, name).cpu().numpy(), getattr(cache, name)
            bad = np.argwhere(got != want)
            assert bad.size == 0, f"{what}: {name} differs at {bad[0]} ({len(bad)} places): {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"


@pytest.mark.parametrize("code", [R.E4M3, R.INT8])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 500])
@pytest.mark.parametrize("paged", [False, True])
def test_rows_into_blocks_and_back(code, tokens, paged):
    log(f"case: pack code={code} tokens={tokens} paged={paged}")
    blocks = -(-tokens // 16) + 3
    cache = R.Cache(blocks, code, fill=0xA5)
    dev = Device(cache)
    table = np.random.default_rng(tokens).permutation(blocks).astype(np.int32)[:-(-tokens // 16)] if paged else None
    k, v = rows(tokens + code, tokens)
    dev.pack(k, v, 0, to_dev_i32(table) if paged else None)
    ids = table if paged else np.arange(blocks)
    cache.put_rows(ids, 0, k, v)
    dev.same(cache, "pack")
    got = dev.unpack(tokens, to_dev_i32(table) if paged else None)
    for a, b in zip(got, cache.rows(ids, tokens)):
        np.testing.assert_array_equal(a.astype(np.float64), b)


@pytest.mark.parametrize("code", [R.E4M3, R.INT8])
def test_appended_rows_raise_the_exponent_of_the_block_they_enter(code):
    log(f"case: pack in pieces, code={code}")
    cache = R.Cache(12, code, fill=0xFF)
    dev, table = Device(cache), np.random.default_rng(3).permutation(12).astype(np.int32)
    at = 0
    for i, (n, scale) in enumerate([(1, 1.0), (3, 40.0), (5, 1e-3), (7, 900.0), (20, 1.0), (1, 3.0), (64, 20.0), (2, 2.0 ** -20), (30, 1.0)]):
        k, v = rows(70 + i, n, scale)
        dev.pack(k, v, at, to_dev_i32(table))
        cache.put_rows(table, at, k, v)
        at += n
        dev.same(cache, f"after {at} rows")
    for a, b in zip(dev.unpack(at, to_dev_i32(table)), cache.rows(table, at)):
        np.testing.assert_array_equal(a.astype(np.float64), b)


@pytest.mark.parametrize("code", [R.E4M3, R.INT8])
def test_every_fp16_value_and_every_exponent(code):
    """All finite fp16 bit patterns, 2048 at a time as one block and head, sorted (small exponents) and shuffled
    (exponents set by the largest); infinities and NaN in blocks of their own."""
    bits = np.arange(65536, dtype=np.uint16)
    finite = bits[(bits & 0x7C00) != 0x7C00].view(np.float16)
    order = np.argsort(np.abs(finite.astype(np.float64)), kind="stable")
    shuffled = np.random.default_rng(1).permutation(finite)
    x = np.concatenate([finite[order], shuffled])  # 62 blocks' worth of [16][128], twice over heads
    k = x.reshape(-1, 2, 16, 128).transpose(0, 2, 1, 3).reshape(-1, 2, 128).copy()
    v = k[::-1].copy()
    special = np.zeros((32, 2, 128), np.float16)
    special[3, 0, 5], special[4, 0, 6], special[5, 1, 7], special[6, 1, 8] = np.inf, -np.inf, np.nan, 2.0
    special[20, 0] = np.nan
    k, v = np.concatenate([k, special]), np.concatenate([v, special])
    n = len(k)
    log(f"case: every fp16 value, code={code}, {n} rows")
    cache = R.Cache(n // 16, code)
    dev = Device(cache)
    dev.pack(k, v, 0, None)
    cache.put_rows(np.arange(n // 16), 0, k, v)
    if code == R.E4M3:  # NaN is any of its codes
        nan = lambda a: np.where((a & 0x7F) == 0x7F, 0x7F, a)  # noqa: E731
        import torch
        torch.cuda.synchronize()
        for name in ("key", "value"):
            np.testing.assert_array_equal(nan(getattr(dev, name).cpu().numpy()), nan(getattr(cache, name)))
        np.testing.assert_array_equal(dev.exponents.cpu().numpy(), cache.exponents)
    else:
        dev.same(cache, "every value")
    for a, b in zip(dev.unpack(n, None), cache.rows(np.arange(n // 16), n)):
        np.testing.assert_array_equal(a.astype(np.float64), np.where(np.isnan(b), b, np.clip(b, -65504, 65504)))


def test_bad_blocks_are_skipped_and_read_as_zero():
    log("case: block ids outside the planes")
    cache = R.Cache(6, R.INT8, fill=0x11)
    dev = Device(cache)
    table = np.array([2, -1, 6, 4], np.int32)
    k, v = rows(5, 50)
    dev.pack(k, v, 0, to_dev_i32(table))
    cache.put(2, 0, k[:16], v[:16])
    cache.put(4, 0, k[48:], v[48:])
    dev.same(cache, "bad ids")
    got = dev.unpack(50, to_dev_i32(table))
    for a in got:
        assert not a[16:48].any() and a[:16].any() and a[48:].any()


def test_rows_at_odd_addresses_and_on_another_stream():
    import torch
    log("case: rows 2-byte aligned, on a side stream")
    for offset in (1, 3):
        cache = R.Cache(4, R.E4M3)
        dev = Device(cache)
        k, v = rows(9, 37)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            keep = dev.pack(k, v, 0, None, stream=side, offset=offset)
        side.synchronize()
        cache.put_rows(np.arange(4), 0, k, v)
        dev.same(cache, "odd rows")
        for a, b in zip(dev.unpack(37, None, offset), cache.rows(np.arange(4), 37)):
            np.testing.assert_array_equal(a.astype(np.float64), b)
        del keep


def test_an_append_replayed_from_a_graph():
    """Rows appended behind ten others and read back, captured; each replay starts from the ten rows again."""
    import torch
    log("case: moves from a graph")
    cache = R.Cache(3, R.E4M3)
    dev = Device(cache)
    k, v = rows(21, 40)
    k[10:] *= 8  # the exponents of the first block grow
    table = to_dev_i32(np.array([2, 0, 1], np.int32))
    start = R.Cache(3, R.E4M3)
    start.put_rows(np.array([2, 0, 1]), 0, k[:10], v[:10])
    first = [torch.from_numpy(getattr(start, n).copy()).cuda() for n in ("key", "value", "exponents")]
    dk, dv = torch.from_numpy(k[10:].copy()).cuda(), torch.from_numpy(v[10:].copy()).cuda()
    back = [torch.zeros(40, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2)]

    def step(stream):
        pvlc.kv_pack_q8(dk, dv, 30, dev.key, dev.value, dev.exponents, 3, R.E4M3, table, first_token=10, stream=stream)
        pvlc.kv_unpack_q8(dev.key, dev.value, dev.exponents, 40, back[0], back[1], 3, R.E4M3, table, stream=stream)

    start.put_rows(np.array([2, 0, 1]), 10, k[10:], v[10:])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
    for i in range(4):
        for d, f in zip((dev.key, dev.value, dev.exponents), first):
            d.copy_(f)
        for b in back:
            b.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        dev.same(start, f"replay {i}")
        for a, b in zip(back, start.rows(np.array([2, 0, 1]), 40)):
            np.testing.assert_array_equal(a.cpu().numpy().astype(np.float64), b)


def test_moves_beyond_32_bits_of_offset():
    import torch
    blocks = (1 << 20) + 40
    log(f"case: moves in planes of {blocks} blocks")
    planes = [torch.full((blocks * 4096,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(2)]
    exponents = torch.full((blocks * 4,), 100, dtype=torch.uint8, device="cuda")
    ids = np.array([blocks - 1, 3, blocks - 30], np.int32)
    k, v = rows(22, 41)
    dk, dv, table = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), to_dev_i32(ids)
    pvlc.kv_pack_q8(dk, dv, 41, planes[0], planes[1], exponents, blocks, R.INT8, table)
    back = [torch.zeros(41, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    pvlc.kv_unpack_q8(planes[0], planes[1], exponents, 41, back[0], back[1], blocks, R.INT8, table)
    want = R.Cache(3, R.INT8)
    want.put_rows(np.arange(3), 0, k, v)
    torch.cuda.synchronize()
    for a, b in zip(back, want.rows(np.arange(3), 41)):
        np.testing.assert_array_equal(a.cpu().numpy().astype(np.float64), b)
    for p in planes:
        p = p.view(blocks, 4096)
        p[torch.from_numpy(ids).long().cuda()] = 0x5A
        assert bool((p[:8] == 0x5A).all()) and bool((p[-64:] == 0x5A).all())
    exponents.view(blocks, 4)[torch.from_numpy(ids).long().cuda()] = 100
    assert bool((exponents == 100).all())
