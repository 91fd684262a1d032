"""CPU: the 4-bit cache format as the oracle states it, and the arguments that the new entry
points refuse on the host (nothing here reaches a GPU)."""

import numpy as np
import pytest
import torch

import pa_oracle
from pa_b200 import _lib, ops


def test_scale_bytes_are_fp16_patterns_and_products_are_exact():
    s = pa_oracle.fp4_scale_values()
    assert s[0] == 0 and s[8] == 2.0 ** -14 and s[1] == 2.0 ** -17 and s[0xE2] == 10240
    assert np.isnan(s[0xFF])
    prod = s[:0xE3, None] * pa_oracle.FP4_VALUES[None]
    assert np.array_equal(prod.astype(np.float16).astype(np.float64), prod)
    t = torch.from_numpy(prod)
    assert torch.equal(t.to(torch.bfloat16).double(), t)
    assert prod.max() == 61440


def test_quantiser_picks_the_nearest_of_all_values():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 128)) * np.exp(rng.normal(0, 3, (64, 1)))).astype(np.float16)
    codes, scales = pa_oracle.quantize_fp4(x)
    v = pa_oracle.dequantize_fp4(codes, scales).reshape(64, 8, 16)
    xb = x.astype(np.float64).reshape(64, 8, 16)
    s = pa_oracle.fp4_scale_values()[scales][..., None]
    every = np.concatenate([-pa_oracle.FP4_VALUES, pa_oracle.FP4_VALUES])
    best = np.abs(xb[..., None] - (every * s[..., None])).min(-1)
    assert np.array_equal(np.abs(xb - v), best)
    # The scale is the nearest representable to amax / 6.
    t = np.abs(xb).max(-1) / 6
    grid = pa_oracle.fp4_scale_values()[:0xE3]
    assert np.array_equal(np.abs(grid[scales] - t), np.abs(grid[None, None] - t[..., None]).min(-1))


def test_ties_go_to_the_even_code_and_large_values_saturate():
    x = np.zeros((1, 128))
    x[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5]
    codes, scales = pa_oracle.quantize_fp4(x)
    assert scales[0, 0] == 15 << 3  # 1.0
    assert codes[0, :9].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 14]
    codes, scales = pa_oracle.quantize_fp4(np.full((1, 128), 65504.0))
    assert (scales == 0xE2).all() and (codes == 7).all()


def test_put_and_values_round_trip():
    rng = np.random.default_rng(2)
    for is_v in (False, True):
        cache = np.zeros((5, 2, 2, 1152), np.uint8)
        rows = rng.standard_normal((40, 2, 128))
        slots = rng.permutation(5 * 32)[:40]
        pa_oracle.fp4_put(cache, is_v, rows, slots, 32)
        held = pa_oracle.fp4_values(cache, is_v)
        want = pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(rows))
        for i, s in enumerate(slots):
            assert np.array_equal(held[s // 32, :, s % 32], want[i])


def test_tables_oracle_hands_out_every_block_once():
    free = list(range(20))
    table = np.full((3, 8), -1)
    slots, pos, starts, lens = pa_oracle.extend_tables(table, [0, 0, 0], [17, 0, 33], free, 16)
    assert len(set(slots)) == 50 and starts == [0, 17, 17, 50] and lens == [17, 0, 33]
    assert len(free) == 15 and pos[16] == 16 and pos[17] == 0
    lens = pa_oracle.release_blocks(table, lens, [1, 0, 0], free, 16)
    assert lens == [0, 0, 33] and sorted(free + table[2, :3].tolist()) == list(range(20))


def test_fp4_cache_shape():
    k, v = ops.fp4_cache(7, 3, 32, device="cpu")
    assert tuple(k.shape) == tuple(v.shape) == (7, 3, 2, 1152) and k.dtype == torch.uint8
    assert ops._check_fp4_caches(k, v, 32) == (7, 3)
    for bs in (0, 8, 24, 256):
        with pytest.raises(RuntimeError):
            ops.fp4_cache(1, 1, bs, device="cpu")
    for bad in (k[..., :1024], k.float(), k.view(7, 3, 1, 2304), k[:6]):
        with pytest.raises(RuntimeError):
            ops._check_fp4_caches(bad, v, 32)
        with pytest.raises(RuntimeError):
            ops._check_fp4_caches(k, bad, 32)
    with pytest.raises(RuntimeError):
        ops._check_fp4_caches(k, v, 16)


def test_ops_refuse_cpu_tensors():
    k, v = ops.fp4_cache(4, 2, device="cpu")
    rows = torch.zeros(3, 2, 128, dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(8, 128)
    w = torch.ones(128, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        ops.quantize_into_cache_fp4(rows, rows, k, v, slots)
    with pytest.raises(RuntimeError):
        ops.read_from_cache_fp4(k, v, slots)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(rows, rows, w, w, slots, table)
    with pytest.raises(RuntimeError):
        ops.norm_rope_into_cache(rows, rows, rows, w, w, slots, table, k, v, slots)
    i = torch.zeros(3, dtype=torch.int32)
    bt = torch.zeros(3, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.release_blocks(bt, i, i, i, i[:1])
    with pytest.raises(RuntimeError):
        ops.extend_block_tables(bt, i, i, i, i[:1], 4, max_tokens=4)


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


P = 1 << 20  # a 16-byte aligned address that no call below reaches


def test_c_entry_points_refuse_bad_arguments(lib):
    INV, UNS, F16 = _lib.PA_ERR_INVALID_ARG, _lib.PA_ERR_UNSUPPORTED, _lib.PA_DTYPE_F16

    def write(k=P, dt=F16, stride=256, n=4, kvh=2, d=128, nb=4, bs=16, kc=P):
        return lib.pa_quantize_into_cache_fp4(k, P, dt, stride, P, n, kvh, d, kc, P, nb, bs, None,
                                              None)
    assert write(dt=9) == UNS and write(d=64) == UNS and write(stride=128) == INV
    assert write(k=P + 8) == INV and write(stride=260) == INV and write(kc=P + 4) == INV
    assert write(bs=8) == INV and write(bs=0) == INV and write(nb=0) == INV and write(k=None) == INV
    assert write(n=-1) == INV and write(n=0) == _lib.PA_OK

    def read(out=P, dt=F16, bs=16, d=128, n=4):
        return lib.pa_read_from_cache_fp4(out, P, dt, P, P, P, n, 2, d, 4, bs, None, None)
    assert read(dt=_lib.PA_DTYPE_I8) == UNS and read(bs=24) == INV and read(d=96) == UNS
    assert read(out=P + 2) == INV and read(n=0) == _lib.PA_OK

    def rope(q=P, qs=1024, ks=256, dt=F16, table_len=8, rot=128, n=4, h=8, kvh=2, d=128, eps=1e-6,
             ko=P, pos=P):
        return lib.pa_qk_norm_rope(P, 1024, ko, 256, q, qs, P, ks, dt, P, P, eps, pos, P,
                                   table_len, rot, 0, n, h, kvh, d, None, None)
    assert rope(dt=7) == UNS and rope(d=64) == UNS and rope(rot=24) == UNS and rope(rot=144) == UNS
    assert rope(rot=0) == UNS and rope(table_len=0) == INV and rope(h=-1) == INV
    assert rope(q=None) == INV and rope(q=P + 4) == INV and rope(qs=1000) == INV
    assert rope(qs=1028) == INV and rope(ko=None) == INV and rope(pos=None) == INV
    assert rope(eps=float("nan")) == INV and rope(eps=-1.0) == INV and rope(h=0, kvh=0) == INV
    assert rope(n=0) == _lib.PA_OK

    def into(cd=_lib.PA_DTYPE_FP4E2M1, bs=16, slots=P, ks=P, nb=4):
        return lib.pa_norm_rope_into_cache(P, 1024, P, 1024, P, 256, P, 256, F16, P, P, 1e-6, P,
                                           P, 8, 128, 0, slots, 4, 8, 2, 128, cd, P, P, ks, P, nb,
                                           bs, None, None)
    assert into(cd=_lib.PA_DTYPE_F32) == UNS and into(bs=8) == INV and into(slots=None) == INV
    assert into(cd=_lib.PA_DTYPE_I8, ks=None) == INV and into(nb=0) == INV

    def release(table=P, count=P, pool=8, bs=16, mb=4, s=2):
        return lib.pa_release_blocks(table, P, P, P, count, P, P, s, mb, bs, pool, None, None)
    assert release(table=None) == INV and release(count=None) == INV and release(pool=-1) == INV
    assert release(bs=0) == INV and release(mb=0) == INV and release(s=-1) == INV
    assert release(mb=1 << 20, bs=1 << 12) == UNS

    def extend(slots=P, start=P, nb=4, tok=8, bs=16):
        return lib.pa_extend_block_tables(P, P, P, P, P, P, P, slots, P, start, 2, 4, bs, 8, nb, tok,
                                          None, None)
    assert extend(slots=None) == INV and extend(start=None) == INV and extend(nb=0) == INV
    assert extend(tok=-1) == INV and extend(nb=1 << 30) == UNS


def test_fp4_decode_entry_points_refuse_bad_arguments(lib):
    INV, UNS = _lib.PA_ERR_INVALID_ARG, _lib.PA_ERR_UNSUPPORTED

    def dec(fn, q=P, kc=P, H=8, KVH=2, D=128, NB=4, bs=16, ws=1 << 30):
        return fn(P, q, kc, P, P, P, 1, H, KVH, D, NB, bs, 2, 0.1, P, ws, None)
    for fn in (lib.pa_decode_fp4, lib.pa_splitk_fp4):
        assert dec(fn, D=64) == UNS and dec(fn, H=7) == INV and dec(fn, bs=8) == INV
        assert dec(fn, kc=P + 8) == INV and dec(fn, q=None) == INV
        assert dec(fn, NB=1 << 26, KVH=4) == UNS
    # The new token's rows are read in 16-byte units.
    rc = lib.pa_decode_step(_lib.PA_DTYPE_FP4E2M1, P, P, P + 8, P, _lib.PA_DTYPE_F16, 256, P, P,
                            None, None, None, None, P, P, 1, 8, 2, 128, 4, 16, 2, 0.1, 0, 1, P,
                            1 << 30, None)
    assert rc == INV and b"16-byte" in lib.pa_last_error()
    for bit, word in ((_lib.PA_ERR_FREE_BLOCKS, b"free"), (_lib.PA_ERR_TOKENS, b"max_tokens"),
                      (_lib.PA_ERR_POSITION, b"position")):
        assert word in lib.pa_status_string(bit)


def test_paged_cache_variant():
    from pa_b200.paged_cache import PagedKVCache
    c = PagedKVCache(3, 2, 128, 50, 16, variant="fp4", device="cpu")
    assert tuple(c.k_cache.shape) == tuple(c.v_cache.shape) == (3, 4, 2, 1, 1152)
    assert c.kv_bytes() == 3 * 64 * 2 * 2 * 72 and not c.is_int8
    assert c.kv_bytes_for_len(17) == 3 * 32 * 2 * 2 * 72
    with pytest.raises(AssertionError):
        PagedKVCache(1, 2, 64, 50, 16, variant="fp4", device="cpu")
    with pytest.raises(AssertionError):
        PagedKVCache(1, 2, 128, 50, 16, variant="int4", device="cpu")


def test_decodes_refuse_an_empty_block_size(lib):
    for fn in (lib.pa_decode_fp4, lib.pa_splitk_fp4, lib.pa_decode_f16):
        for bs in (0, -16):
            assert fn(P, P, P, P, P, P, 1, 8, 2, 128, 4, bs, 2, 0.1, P, 1 << 30,
                      None) == _lib.PA_ERR_INVALID_ARG


@pytest.mark.parametrize("n", [1, 4, 32, 33, 200])
def test_lengths_are_checked_alike_through_a_list_and_numpy(n):
    good = torch.full((n,), 7, dtype=torch.int32)
    for shape in ((n,), (n, 1)):
        ops._check_lengths(good, 7, good.view(shape))
        for bad in (0, 8, -1):
            x = good.clone()
            x[n // 2] = bad
            with pytest.raises(RuntimeError):
                ops._check_lengths(good, 7, x.view(shape))
