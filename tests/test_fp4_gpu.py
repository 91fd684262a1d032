"""GPU: the 4-bit K/V cache. Writes are compared value for value with the oracle's quantiser,
decodes with attention in 64 bits over the held values.

Tolerance of a decode (fp16 out): the output's own rounding, half a step, is 2^-11 of its value
(2^-25 where fp16 is subnormal). The scores are fp32 dot products of 128 exact products summed in the tensor
cores: with eight steps of 16 products, each within 2^-22 of the running sum of magnitudes, a
score is off by at most 2^-18 of Q = scale * sum |q k|, plus 2^-22 of |score| <= Q for the scale
and exponent arithmetic. A weight is then off by a factor 1 + e, e = 2^-17 Q + 2^-20 (ex2's and
the two-part fp16 weight's own errors, 2^-21 each at most), the normalised output by 2 e max|v|,
and sums over n tokens by n / 16 more steps of 2^-22 relative to max|v|."""


import numpy as np
import pytest
import torch

import pa_oracle
from pa_testlib import scale_for, to_cuda

pytestmark = pytest.mark.gpu


def _ops():
    from pa_b200 import ops
    return ops


def _rows(rng, n, kvh, dt):
    x = rng.standard_normal((n, kvh, 128)) * np.exp(0.5 * rng.standard_normal((n, kvh, 1)))
    x[..., 5] *= 20
    t = torch.from_numpy(x.astype(np.float32)).to(dt)
    return t, t.double().numpy()


def _held(cache, is_v):
    return pa_oracle.fp4_values(cache.cpu().numpy(), is_v)


def _want(rows, cache, is_v, slots, bs):
    ref = np.zeros(tuple(cache.shape), np.uint8)
    pa_oracle.fp4_put(ref, is_v, rows, slots, bs)
    return pa_oracle.fp4_values(ref, is_v)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs", [16, 32, 128])
@pytest.mark.parametrize("n,kvh", [(1, 1), (3, 2), (257, 4), (40, 3)])
def test_write_and_read_back(dt, bs, n, kvh):
    rng = np.random.default_rng(n + bs)
    nb = n // bs + 3
    k, kd = _rows(rng, n, kvh, dt)
    v, vd = _rows(rng, n, kvh, dt)
    slots = rng.permutation(nb * bs)[:n].astype(np.int32)
    slots[n // 2] = -1 if n > 1 else slots[n // 2]
    kc, vc = _ops().fp4_cache(nb, kvh, bs)
    sl = torch.from_numpy(slots).cuda()
    _ops().quantize_into_cache_fp4(k.cuda(), v.cuda(), kc, vc, sl, bs)
    for rows, cache, is_v in ((kd, kc, False), (vd, vc, True)):
        assert np.array_equal(_held(cache, is_v), _want(rows, cache, is_v, slots, bs))
    for out_dt in (torch.float16, torch.bfloat16, torch.float32):
        mark = tuple(torch.full((n, kvh, 128), 7.0, dtype=out_dt, device="cuda") for _ in "kv")
        got = _ops().read_from_cache_fp4(kc, vc, sl, bs, out=mark)
        for g, rows in zip(got, (kd, vd)):
            want = pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(rows))
            want[slots < 0] = 7.0  # rows without a slot keep what they held
            assert np.array_equal(g.double().cpu().numpy(), want)
    _ops().check_status(kc.device)


def test_write_of_edge_rows():
    """Zero, tiny, huge and non-finite blocks, and values on the borders between codes."""
    rows = np.zeros((12, 1, 128))
    rows[1, 0, :16] = 6e-8                       # below half a scale step: zeros
    rows[2, 0, :16] = 3.1e-5                     # a subnormal scale
    rows[3] = 65504.0                            # above 6 * 10240
    rows[4, 0, 3] = np.inf
    rows[5, 0, 20] = np.nan
    rows[6, 0, 100] = -np.inf
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    for i, s in enumerate([1.0, 1.125, 0.875, 2.0 ** -14, 3 * 2.0 ** -17]):
        x = np.concatenate([[6.0], borders, -borders, [0.1]]) * s
        rows[7 + i, 0] = np.tile(x, 8)
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        t = torch.from_numpy(rows.astype(np.float32)).to(dt)
        kc, vc = _ops().fp4_cache(1, 1)
        sl = torch.arange(12, dtype=torch.int32, device="cuda")
        _ops().quantize_into_cache_fp4(t.cuda(), t.cuda(), kc, vc, sl)
        want = pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(t.double().numpy()))
        for cache, is_v in ((kc, False), (vc, True)):
            assert np.array_equal(_held(cache, is_v)[0, :, :12].transpose(1, 0, 2), want,
                                  equal_nan=True)
        k, _ = _ops().read_from_cache_fp4(kc, vc, sl, dtype=dt)
        assert np.array_equal(k.double().cpu().numpy(), want, equal_nan=True)


def test_every_fp16_value_beside_every_leading_scale():
    """All finite fp16 magnitudes as x, in blocks whose scale is set by a fixed largest value."""
    vals = np.arange(0, 0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)
    for amax in (6.0, 7.1, 0.37, 900.0, 4e-4):
        x = vals[vals <= amax]
        x = np.concatenate([x, np.zeros(-len(x) % (15 * 8))]).reshape(-1, 8, 15)
        rows = np.concatenate([np.full(x.shape[:2] + (1,), np.float16(amax)), x], -1)
        rows = rows.reshape(-1, 1, 128)
        n = rows.shape[0]
        t = torch.from_numpy(rows).half().cuda()
        kc, vc = _ops().fp4_cache(n // 16 + 1, 1)
        sl = torch.arange(n, dtype=torch.int32, device="cuda")
        _ops().quantize_into_cache_fp4(t, t, kc, vc, sl)
        k, v = _ops().read_from_cache_fp4(kc, vc, sl)
        want = pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(t.double().cpu().numpy()))
        assert np.array_equal(k.double().cpu().numpy(), want)
        assert torch.equal(k, v)


def test_write_of_strided_rows_and_slots_outside_the_cache():
    rng = np.random.default_rng(5)
    qkv = torch.from_numpy(rng.standard_normal((9, 20, 128)).astype(np.float32)).half().cuda()
    k, v = qkv[:, 12:16], qkv[:, 16:]
    kc, vc = _ops().fp4_cache(3, 4)
    slots = np.array([0, 17, 48, -1, 47, 5, 1 << 20, 33, 20], np.int32)
    sl = torch.from_numpy(slots).cuda()
    _ops().quantize_into_cache_fp4(k, v, kc, vc, sl)
    with pytest.raises(RuntimeError, match="slot"):
        _ops().check_status(kc.device)
    inside = np.where(slots < 48, slots, -1)
    for t, cache, is_v in ((k, kc, False), (v, vc, True)):
        rows = t.double().cpu().numpy()
        assert np.array_equal(_held(cache, is_v), _want(rows, cache, is_v, inside, 16))
    out = tuple(torch.full((9, 4, 128), 3.0, dtype=torch.float16, device="cuda") for _ in "kv")
    _ops().read_from_cache_fp4(kc, vc, sl, out=out)
    assert _ops().read_status(kc.device) == 256  # PA_ERR_SLOT
    assert bool((out[0][[2, 3, 6]] == 3.0).all()) and not bool((out[0][0] == 3.0).all())


def test_refusals():
    ops = _ops()
    kc, vc = ops.fp4_cache(4, 2)
    rows = torch.zeros(3, 2, 128, dtype=torch.float16, device="cuda")
    sl = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (rows[:, :1].contiguous(), rows.double(), rows.transpose(0, 1), rows[..., :64]):
        with pytest.raises(RuntimeError):
            ops.quantize_into_cache_fp4(bad, bad, kc, vc, sl)
    for s in (sl.long(), sl[:2], sl.cpu(), torch.zeros(6, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(RuntimeError):
            ops.quantize_into_cache_fp4(rows, rows, kc, vc, s)
    with pytest.raises(RuntimeError):
        ops.quantize_into_cache_fp4(rows, rows, kc, vc, sl, 32)
    with pytest.raises(RuntimeError):
        ops.read_from_cache_fp4(kc, vc, sl, dtype=torch.float64)
    with pytest.raises(RuntimeError):
        ops.read_from_cache_fp4(kc, vc, sl, out=(rows, rows[:2]))
    q = torch.zeros(1, 4, 128, dtype=torch.float16, device="cuda")
    bt = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    scales = torch.zeros(4, 2, 16, device="cuda")
    for kw in (dict(k_scales=scales, v_scales=scales), dict(kv_kind="f16"), dict(kv_kind="i8"),
               dict(block_size=32)):
        with pytest.raises(RuntimeError):
            ops.decode(torch.empty_like(q), q, kc, vc, bt, one, 0.1, **kw)
    with pytest.raises(RuntimeError):
        ops.decode(torch.empty_like(q), q, kc, vc.view(torch.int8), bt, one, 0.1)
    with pytest.raises(RuntimeError, match=">= 1"):
        ops.decode(torch.empty_like(q), q, kc, vc, bt, one * 0, 0.1)


# ---- decode ------------------------------------------------------------------------------
def _case(seed, lens, H, KVH, bs=16, pad=0, dt=torch.float16, extra=1):
    """A cache written by the oracle; slots past each context hold the byte `pad`."""
    rng = np.random.default_rng(seed)
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + extra
    perm = rng.permutation(nb).astype(np.int32)
    bt = np.zeros((len(lens), max(need) + 1), np.int32)
    caches = [np.full((nb, KVH, bs // 16, 1152), pad, np.uint8) for _ in "kv"]
    at = 0
    for b, n in enumerate(lens):
        bt[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        t = np.arange(n)
        slots = bt[b, t // bs] * bs + t % bs
        for cache, is_v in zip(caches, (False, True)):
            pa_oracle.fp4_put(cache, is_v, _rows(rng, n, KVH, torch.float16)[1], slots, bs)
    q = torch.from_numpy(rng.standard_normal((len(lens), H, 128)).astype(np.float32)).to(dt)
    return dict(q=q, kc=caches[0], vc=caches[1], bt=bt, lens=np.array(lens, np.int32), bs=bs)


def _gpu(c):
    return [c["q"].cuda()] + to_cuda(c["kc"], c["vc"], c["bt"], c["lens"])


def _close(out, c, kc=None, vc=None, lens=None):
    lens = c["lens"] if lens is None else lens
    ref, qk, vmax = pa_oracle.fp4_decode(c["q"].double().numpy(), c["kc"] if kc is None else kc,
                                         c["vc"] if vc is None else vc, c["bt"], lens,
                                         scale_for())
    half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8 + 2.0 ** -11}[out.dtype]
    e = 2 * (2.0 ** -17 * qk + 2.0 ** -20) + np.asarray(lens) / 16 * 2.0 ** -22
    tol = half * np.abs(ref) + 2.0 ** -25 + (e * vmax)[:, None, None]
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= tol).all(), float((err - tol).max())


SHAPES = [([1], 8, 8), ([1, 15, 16, 17, 33], 12, 2), ([512, 513, 511], 8, 1), ([700, 4096], 12, 2),
          ([300, 64, 1999], 32, 2), ([90, 250], 20, 1), ([2000, 1], 64, 8), ([5] * 40, 28, 4)]


@pytest.mark.parametrize("splitk", [False, True])
@pytest.mark.parametrize("lens,H,KVH", SHAPES)
def test_decode(lens, H, KVH, splitk):
    c = _case(len(lens) + H, lens, H, KVH)
    q, kc, vc, bt, cl = _gpu(c)
    out = torch.full_like(q, float("nan"))
    _ops().decode(out, q, kc, vc, bt, cl, scale_for(), splitk=splitk)
    _close(out, c)
    again = torch.empty_like(q)
    _ops().DecodePlan(again, q, kc, vc, bt, cl, scale_for(), splitk=splitk).run()
    assert torch.equal(out, again)
    _ops().check_status(q.device)


@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize("H,KVH", [(12, 2), (32, 2)])
def test_decode_block_sizes_with_nan_bytes_past_the_context(bs, H, KVH):
    # 0xFF: NaN scales (and codes of -6) in every slot that no token was written to.
    c = _case(bs, [1, bs - 1, bs, bs + 1, 3 * bs + 17, 700], H, KVH, bs=bs, pad=0xFF)
    q, kc, vc, bt, cl = _gpu(c)
    for splitk in (False, True):
        out = torch.full_like(q, float("nan"))
        _ops().decode(out, q, kc, vc, bt, cl, scale_for(), bs, splitk=splitk)
        _close(out, c)
    _ops().check_status(q.device)


@pytest.mark.parametrize("splitk", [False, True])
def test_decode_bf16(splitk):
    c = _case(9, [1, 40, 1500], 28, 4, dt=torch.bfloat16)
    q, kc, vc, bt, cl = _gpu(c)
    out = torch.empty_like(q)
    _ops().decode_bf16(out, q, kc, vc, bt, cl, scale_for(), splitk=splitk)
    _close(out, c)


def test_partials_merge_to_the_decode():
    c = _case(10, [700, 33, 1], 12, 2)
    q, kc, vc, bt, cl = _gpu(c)
    first = torch.minimum(cl, torch.tensor(320, device="cuda", dtype=torch.int32))
    parts = [_ops().decode_partial(q, kc, vc, bt, first, scale_for()),
             _ops().decode_partial(q, kc, vc, bt[:, 20:].contiguous(), cl - first, scale_for())]
    out = torch.empty_like(q)
    _ops().merge_partials(out, torch.stack(parts), 12, 2)
    _close(out, c)
    _ops().check_status(q.device)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("H,KVH,bs", [(12, 2, 16), (28, 4, 32), (40, 2, 16), (32, 2, 128)])
def test_decode_step(dt, fused, H, KVH, bs):
    lens = [1, 16, 17, 300, 129]
    c = _case(11, lens, H, KVH, bs=bs, pad=0xFF)
    rng = np.random.default_rng(3)
    k, kd = _rows(rng, 5, KVH, dt)
    v, vd = _rows(rng, 5, KVH, dt)
    last = c["lens"] - 1
    slots = c["bt"][np.arange(5), last // bs] * bs + last % bs
    for cache, rows, is_v in ((c["kc"], kd, False), (c["vc"], vd, True)):
        pa_oracle.fp4_put(cache, is_v, np.full_like(rows, 99.0), slots, bs)  # what was there
    q, kc, vc, bt, cl = _gpu(c)
    for cache, rows, is_v in ((c["kc"], kd, False), (c["vc"], vd, True)):
        pa_oracle.fp4_put(cache, is_v, rows, slots, bs)
    out = torch.empty_like(q)
    _ops().decode_step(out, q, k.cuda(), v.cuda(), kc, vc, bt, cl, scale_for(), bs, fused=fused)
    _close(out, c)
    for mine, ref, is_v in ((kc, c["kc"], False), (vc, c["vc"], True)):
        assert np.array_equal(_held(mine, is_v), pa_oracle.fp4_values(ref, is_v), equal_nan=True)
    _ops().check_status(q.device)


def test_bad_block_ids_and_lengths_are_flagged():
    c = _case(12, [200, 40], 12, 2)
    q, kc, vc, bt, cl = _gpu(c)
    bad = bt.clone()
    bad[0, 3] = 10 ** 6
    out = torch.empty_like(q)
    _ops().decode(out, q, kc, vc, bad, cl, scale_for())
    assert _ops().read_status(q.device) & 64
    long = cl.clone()
    long[1] = 10 ** 6
    _ops().decode(out, q, kc, vc, bt, long, scale_for(), validate=False)
    assert _ops().read_status(q.device) & 32
    zero = cl * 0
    _ops().decode(out, q, kc, vc, bt, zero, scale_for(), validate=False)
    assert _ops().read_status(q.device) & 16
    assert bool((out == 0).all())
    _ops().decode(out, q, kc, vc, bt, cl, scale_for())
    _close(out, c)


def test_decode_on_another_stream_and_in_a_graph():
    c = _case(13, [900, 33, 1200], 28, 4)
    q, kc, vc, bt, cl = _gpu(c)
    want = torch.empty_like(q)
    _ops().decode(want, q, kc, vc, bt, cl, scale_for())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(q)
    with torch.cuda.stream(s):
        _ops().decode(out, q, kc, vc, bt, cl, scale_for())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            _ops().decode(out, q, kc, vc, bt, cl, scale_for(), validate=False)
    s.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_offsets_past_32_bits():
    """A cache of 2.4 GB a side whose last blocks are the ones in use."""
    nb, bs = 1 << 20, 32
    kc, vc = (torch.empty(nb, 1, 2, 1152, dtype=torch.uint8, device="cuda") for _ in "kv")
    rng = np.random.default_rng(14)
    n = 100
    bt = np.array([[nb - 1, nb - 3, nb - 2, nb - 7]], np.int32)
    t = np.arange(n)
    slots = (bt[0, t // bs] * bs + t % bs).astype(np.int32)
    k, kd = _rows(rng, n, 1, torch.float16)
    v, vd = _rows(rng, n, 1, torch.float16)
    sl = torch.from_numpy(slots).cuda()
    _ops().quantize_into_cache_fp4(k.cuda(), v.cuda(), kc, vc, sl, bs)
    got, _ = _ops().read_from_cache_fp4(kc, vc, sl, bs)
    assert np.array_equal(got.double().cpu().numpy(),
                          pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(kd)))
    c = dict(q=torch.from_numpy(rng.standard_normal((1, 8, 128)).astype(np.float16)), bs=bs)
    small = [np.zeros((4, 1, 2, 1152), np.uint8) for _ in "kv"]
    at = np.arange(n)
    for cache, rows, is_v in ((small[0], kd, False), (small[1], vd, True)):
        pa_oracle.fp4_put(cache, is_v, rows, at, bs)
    c.update(kc=small[0], vc=small[1], bt=np.arange(4, dtype=np.int32)[None],
             lens=np.array([n], np.int32))
    q, bt_, cl = to_cuda(c["q"].numpy(), bt, c["lens"])
    out = torch.empty_like(q)
    _ops().decode(out, q, kc, vc, bt_, cl, scale_for(), bs)
    _close(out, c)


def test_more_sequences_than_one_launch_holds():
    lens = [1 + (i * 7) % 40 for i in range(1100)]
    c = _case(15, lens, 8, 2)
    q, kc, vc, bt, cl = _gpu(c)
    out = torch.empty_like(q)
    _ops().decode(out, q, kc, vc, bt, cl, scale_for())
    _close(out, c)


def test_c_abi_needs_a_large_enough_workspace():
    from pa_b200 import _lib
    L = _lib.lib()
    need = L.pa_decode_workspace_bytes(2, 8, 2, 128, 4, 16, _lib.PA_DTYPE_FP4E2M1, 0)
    assert need > 0
    c = _case(16, [20, 30], 8, 2)
    q, kc, vc, bt, cl = _gpu(c)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    p = [t.data_ptr() for t in (q, kc, vc, bt, cl)]
    rc = L.pa_decode_fp4(p[0], *p, 2, 8, 2, 128, kc.shape[0], 16, bt.shape[1], 0.1, ws.data_ptr(),
                         need - 1 if bt.shape[1] == 4 else 1024, None)
    assert rc == _lib.PA_ERR_WORKSPACE


def test_long_ranges_take_many_batches_of_block_ids():
    """Each warp's range is longer than a batch of 32 block ids and ends inside one; the shared
    memory the ids pass through holds another launch's leavings. The single pass must agree with
    the split-K pair and flag nothing."""
    g = torch.Generator(device="cuda").manual_seed(17)
    S, H, KVH, n = 24, 8, 2, 32768 - 7
    nb = S * 2048 + 1
    kc, vc = _ops().fp4_cache(nb, KVH)
    for c in (kc, vc):
        c[..., :1024] = torch.randint(0, 256, c[..., :1024].shape, generator=g, device="cuda",
                                      dtype=torch.uint8)
        c[..., 1024:] = torch.randint(96, 128, c[..., 1024:].shape, generator=g, device="cuda",
                                      dtype=torch.uint8)
    bt = torch.randperm(nb, generator=g, device="cuda")[:S * 2048].int().view(S, 2048)
    lens = torch.tensor([n - 977 * b for b in range(S)], dtype=torch.int32, device="cuda")
    q = torch.randn(S, H, 128, generator=g, device="cuda").half()
    outs = []
    for splitk in (False, True, False):
        junk = torch.full((1 << 20,), -1.0, device="cuda").softmax(0)  # another kernel's traces
        out = torch.empty_like(q)
        _ops().decode(out, q, kc, vc, bt, lens, scale_for(), splitk=splitk)
        outs.append(out)
        del junk
    _ops().check_status(q.device)
    assert torch.equal(outs[0], outs[2])
    # One sequence against 64 bits; the two forms against each other within both roundings.
    b = 3
    c = dict(q=q[b:b + 1].cpu(), bt=np.arange(2048, dtype=np.int32)[None],
             kc=kc[bt[b].long()].cpu().numpy(), vc=vc[bt[b].long()].cpu().numpy(),
             lens=lens[b:b + 1].cpu().numpy())
    for out in outs[:2]:
        _close(out[b:b + 1], c)
    assert float((outs[0].float() - outs[1].float()).abs().max()) <= 2.0 ** -9


def test_bf16_values_outside_the_fp16_range_are_flagged():
    c = _case(18, [40, 90], 12, 2, dt=torch.bfloat16)
    q, kc, vc, bt, cl = _gpu(c)
    out = torch.empty_like(q)
    _ops().decode_bf16(out, q, kc, vc, bt, cl, scale_for())
    _ops().check_status(q.device)
    q[1, 5, 77] = 1e6
    _ops().decode_bf16(out, q, kc, vc, bt, cl, scale_for())
    assert _ops().read_status(q.device) == 512  # PA_ERR_Q_RANGE


def test_paged_cache_loop():
    """PagedKVCache("fp4") over two layers: a prompt, then tokens appended and decoded."""
    from pa_b200.paged_cache import PagedKVCache
    rng = np.random.default_rng(19)
    cache = PagedKVCache(2, 2, 128, 60, 16, variant="fp4")
    held = [[np.zeros((0, 2, 128))] * 2 for _ in range(2)]
    for step in range(6):
        n = 37 if step == 0 else 1
        for layer in range(2):
            k, kd = _rows(rng, n, 2, torch.float16)
            v, vd = _rows(rng, n, 2, torch.float16)
            held[layer] = [np.concatenate([h, x]) for h, x in zip(held[layer], (kd, vd))]
            L = 37 + step
            q = torch.from_numpy(rng.standard_normal((1, 12, 128)).astype(np.float16))
            if step == 0:
                cache.prefill(layer, k.cuda(), v.cuda())
                continue
            if step % 2:
                out = cache.append_and_decode(layer, k[0].cuda(), v[0].cuda(), q.cuda(), scale_for())
            else:
                assert cache.decode_append(layer, k[0].cuda(), v[0].cuda()) == L
                out = torch.empty(1, 12, 128, dtype=torch.float16, device="cuda")
                _ops().decode(out, q.cuda(), cache.k_cache[layer], cache.v_cache[layer],
                              cache.block_table, cache.context_lens(layer), scale_for())
            caches = [np.zeros((4, 2, 1, 1152), np.uint8) for _ in "kv"]
            for c, rows, is_v in zip(caches, held[layer], (False, True)):
                pa_oracle.fp4_put(c, is_v, rows, np.arange(L), 16)
            _close(out, dict(q=q, kc=caches[0], vc=caches[1], lens=np.array([L]),
                             bt=np.arange(4)[None]))
    _ops().check_status(cache.k_cache.device)


@pytest.mark.parametrize("scale", [-0.11, 0.0, 1e-38, 1.0, 3.0])
@pytest.mark.parametrize("H,KVH", [(12, 2), (8, 4), (32, 2)])
def test_scales_of_either_sign(scale, H, KVH):
    """A negative scale is a positive one over -q, for the 64-bit form as well."""
    c = _case(20, [1, 30, 1700], H, KVH, pad=0xFF)
    q, kc, vc, bt, cl = _gpu(c)
    sign = -1.0 if scale < 0 else 1.0
    ref, qk, vmax = pa_oracle.fp4_decode(sign * c["q"].double().numpy(), c["kc"], c["vc"], c["bt"],
                                         c["lens"], abs(scale))
    e = 2 * (2.0 ** -17 * qk + 2.0 ** -20) + c["lens"] / 16 * 2.0 ** -22
    tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + (e * vmax)[:, None, None]
    for splitk in (False, True):
        out = torch.full_like(q, float("nan"))
        _ops().decode(out, q, kc, vc, bt, cl, scale, splitk=splitk)
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()


def test_one_token_of_any_strides():
    """A single token's strides between tokens (and one head's between heads) do not matter."""
    rng = np.random.default_rng(21)
    qkv = torch.from_numpy(rng.standard_normal((1, 8, 128)).astype(np.float16)).cuda()
    for kvh in (2, 1):
        k, v = qkv[:, 4:4 + kvh], torch.empty(1, kvh, 128, dtype=torch.float16, device="cuda")
        v.copy_(qkv[:, 6:6 + kvh])
        k = k.as_strided(k.shape, (k.stride(0), 1024 if kvh == 1 else 128, 1), k.storage_offset())
        kc, vc = _ops().fp4_cache(1, kvh)
        sl = torch.tensor([5], dtype=torch.int32, device="cuda")
        _ops().quantize_into_cache_fp4(k, v, kc, vc, sl)
        for cache, rows, is_v in ((kc, k, False), (vc, v, True)):
            want = _want(rows.double().cpu().numpy(), cache, is_v, [5], 16)
            assert np.array_equal(_held(cache, is_v), want)


def test_partials_of_empty_contexts_merge():
    """A rank without tokens of a sequence gives an empty partial."""
    c = _case(22, [40, 7, 900], 28, 4)
    q, kc, vc, bt, cl = _gpu(c)
    part = _ops().decode_partial(q, kc, vc, bt, cl, scale_for())
    gone = torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda") * 0
    empty = _ops().decode_partial(q, kc, vc, bt, gone, scale_for())
    out = torch.empty_like(q)
    _ops().merge_partials(out, torch.stack([empty, part, empty]), 28, 4)
    _close(out, c)
    _ops().check_status(q.device)


def test_two_batches_on_two_streams():
    cs = [_case(23 + i, [3000, 1, 77 + 900 * i], 12, 2) for i in range(2)]
    ts = [_gpu(c) for c in cs]
    want = []
    for q, kc, vc, bt, cl in ts:
        want.append(torch.empty_like(q))
        _ops().decode(want[-1], q, kc, vc, bt, cl, scale_for())
    outs = [torch.empty_like(t[0]) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, (q, kc, vc, bt, cl), c in zip(streams, outs, ts, cs):
            with torch.cuda.stream(s):
                _ops().decode(o, q, kc, vc, bt, cl, scale_for(),
                              host_context_lens=torch.from_numpy(c["lens"]))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    _ops().check_status(outs[0].device)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,H,KVH", [([5, 40], 8, 4), ([3000, 70], 12, 2), ([33000], 8, 1),
                                        ([2000, 9], 32, 2), ([9000], 32, 2)])
def test_nan_rows_reach_their_heads_and_no_others(lens, H, KVH, dt):
    """A NaN block in K makes every head of its kv head NaN, one in V the block's 16 values of
    them, whichever way the pieces are merged; a NaN behind the context does nothing."""
    c = _case(30, lens, H, KVH, dt=dt, pad=0xFF)
    q, kc, vc, bt, cl = _gpu(c)
    G, last = H // KVH, c["lens"][0] - 1
    blk, off = int(c["bt"][0, last // 16]), int(last % 16)
    run = _ops().decode if dt == torch.float16 else _ops().decode_bf16
    for splitk in (False, True):
        clean = torch.empty_like(q)
        run(clean, q, kc, vc, bt, cl, scale_for(), splitk=splitk)
        assert bool(torch.isfinite(clean).all())
        for is_v in (False, True):
            k2, v2 = kc.clone(), vc.clone()
            if is_v:
                v2[blk, 0, 0, 1024 + 3 * 16 + off] = 0xFF
            else:
                k2[blk, 0, 0, 1024 + off * 8 + 3] = 0xFF
            out = torch.empty_like(q)
            run(out, q, k2, v2, bt, cl, scale_for(), splitk=splitk)
            want = torch.zeros(len(lens), H, 128, dtype=torch.bool, device="cuda")
            want[0, :G, 48:64] = True
            if not is_v:
                want[0, :G] = True
            assert torch.equal(torch.isnan(out), want)
            assert torch.equal(out[~want], clean[~want])
    _ops().check_status(q.device)


@pytest.mark.parametrize("H,KVH", [(12, 2), (32, 2), (4, 1), (20, 1)])
@pytest.mark.parametrize("lens", [[16] * 200, [17] * 150, [33] * 64, [20000], [6000, 1, 6000],
                                  [250, 2000, 31, 500] * 8, [1] * 30 + [9000] + [1] * 30])
def test_merges_inside_and_across_ctas(lens, H, KVH):
    """Segments within one warp, one CTA, neighbouring CTAs and up to all of them; the same bits in
    every run; partials of the same launch shape merge to the same rows."""
    c = _case(40 + len(lens), lens, H, KVH)
    q, kc, vc, bt, cl = _gpu(c)
    out = torch.full_like(q, float("nan"))
    _ops().decode(out, q, kc, vc, bt, cl, scale_for())
    _close(out, c)
    for _ in range(3):
        again = torch.full_like(q, float("nan"))
        _ops().decode(again, q, kc, vc, bt, cl, scale_for())
        assert torch.equal(out, again)
    part = _ops().decode_partial(q, kc, vc, bt, cl, scale_for())
    merged = torch.full_like(q, float("nan"))
    _ops().merge_partials(merged, part[None], H, KVH)
    _close(merged, c)
    _ops().check_status(q.device)


def test_empty_calls():
    """No tokens, no sequences: nothing is launched or refused."""
    ops = _ops()
    kc, vc = ops.fp4_cache(2, 2)
    half, i32 = dict(dtype=torch.float16, device="cuda"), dict(dtype=torch.int32, device="cuda")
    rows, none = torch.zeros(0, 2, 128, **half), torch.zeros(0, **i32)
    ops.quantize_into_cache_fp4(rows, rows, kc, vc, none)
    k, v = ops.read_from_cache_fp4(kc, vc, none)
    assert k.shape == v.shape == (0, 2, 128)
    q, bt = torch.zeros(0, 4, 128, **half), torch.zeros(0, 3, **i32)
    out = torch.empty_like(q)
    ops.decode(out, q, kc, vc, bt, none, 0.1)
    ops.decode_bf16(out.bfloat16(), q.bfloat16(), kc, vc, bt, none, 0.1)
    ops.decode_step(out, q, rows, rows, kc, vc, bt, none, 0.1)
    ops.decode_partial(q, kc, vc, bt, none, 0.1)
    table = ops.rope_table(4)
    q2, k2 = ops.qk_norm_rope(q, rows, None, None, none, table)
    assert q2.shape == q.shape and k2.shape == rows.shape
    ops.norm_rope_into_cache(q, rows, rows, None, None, none, table, kc, vc, none)
    free, count = torch.arange(2, **i32), torch.full((1,), 2, **i32)
    lens, n = ops.release_blocks(bt, none, none, free, count)
    assert lens.numel() == 0 and n.item() == 2
    slots, pos, start, lens, n = ops.extend_block_tables(bt, none, none, free, count, 2,
                                                         max_tokens=0)
    assert slots.numel() == pos.numel() == lens.numel() == 0
    assert start.tolist() == [0] and n.item() == 2
    slots, pos, *_ = ops.extend_block_tables(bt, none, none, free, count, 2, max_tokens=3)
    assert slots.tolist() == pos.tolist() == [-1] * 3
    assert bool((kc == 0).all()) and bool((vc == 0).all())
    ops.check_status(kc.device)
