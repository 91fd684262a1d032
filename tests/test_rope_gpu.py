"""GPU: RMS norm of q and k heads with the position rotation, against the formula in 64 bits, and
its form that writes K and V into the cache, bit for bit against the separate calls.

Tolerance: the sum of 128 squares in fp32 (eight fused steps and four shuffle adds) is within
12 * 2^-24 of its value, the mean, root and reciprocal add four roundings: 1/rms is within 2^-21
relative. x * inv * w adds two, the rotation's product and fused add two more on terms of at
most |a| + |b|: the fp32 result is within 2^-20 of the pair's magnitude |y_a| + |y_b|. The output's
rounding adds half a step of its type."""

import numpy as np
import pytest
import torch

import pa_oracle

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _ops():
    from pa_b200 import ops
    return ops


def _inputs(seed, n, H, KVH, dt, rot=128, far=5000, norm=True):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n, H + 2 * KVH, 128, generator=g).to(dt).cuda()
    w = [(1 + 0.2 * torch.randn(128, generator=g)).to(dt).cuda() if norm else None for _ in "qk"]
    pos = torch.randint(0, far, (n,), generator=g).int().cuda()
    return (qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:], *w, pos,
            _ops().rope_table(far, rot))


def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _close(out, x, w, pos, table, eps, interleaved):
    ref = pa_oracle.norm_rope(_np(x), _np(w), pos.cpu().numpy(), _np(table), eps, interleaved)
    turned = np.zeros_like(ref)  # |y_a| + |y_b| before the turn, for the pair's two values
    y = pa_oracle.norm_rope(_np(x), _np(w), pos.cpu().numpy() * 0,
                            np.concatenate([np.ones((1, table.shape[1] // 2)),
                                            np.zeros((1, table.shape[1] // 2))], 1), eps,
                            interleaved)
    rot = table.shape[1]
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    turned[...] = np.abs(y)
    turned[..., a] = turned[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    tol = HALF[out.dtype] * (np.abs(ref) + 2.0 ** -20 * turned) + 2.0 ** -20 * turned
    if out.dtype == torch.float16:
        tol += 2.0 ** -25
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,H,KVH,rot", [(1, 1, 1, 128), (3, 12, 2, 64), (65, 28, 4, 128),
                                         (257, 8, 8, 96), (700, 32, 8, 16), (2, 5, 3, 128)])
def test_norm_rope(dt, interleaved, n, H, KVH, rot):
    q, k, _, qw, kw, pos, table = _inputs(n + H, n, H, KVH, dt, rot)
    qo, ko = _ops().qk_norm_rope(q, k, qw, kw, pos, table, eps=1e-5, interleaved=interleaved)
    _close(qo, q, qw, pos, table, 1e-5, interleaved)
    _close(ko, k, kw, pos, table, 1e-5, interleaved)
    _ops().check_status(q.device)


def test_one_side_without_norm_and_no_k_heads():
    q, k, _, qw, _, pos, table = _inputs(3, 17, 6, 2, torch.float16)
    qo, ko = _ops().qk_norm_rope(q, k, qw, None, pos, table)
    _close(qo, q, qw, pos, table, 1e-6, False)
    _close(ko, k, None, pos, table, 1e-6, False)
    qo, ko = _ops().qk_norm_rope(q, k[:, :0], qw, None, pos, table)
    _close(qo, q, qw, pos, table, 1e-6, False)
    assert ko.shape == (17, 0, 128)
    e = q[:0]
    qo, ko = _ops().qk_norm_rope(e, k[:0], qw, None, pos[:0], table)
    assert qo.shape == (0, 6, 128)


def test_in_place_and_padding_and_positions_outside_the_table():
    q, k, _, qw, kw, pos, table = _inputs(4, 40, 12, 2, torch.bfloat16, far=64)
    want_q, want_k = _ops().qk_norm_rope(q, k, qw, kw, pos, table)
    pos2 = pos.clone()
    pos2[[0, 7, 39]] = -1
    pos2[5] = 64
    q0, k0 = q.clone(), k.clone()
    qo, ko = _ops().qk_norm_rope(q, k, qw, kw, pos2, table, q_out=q, k_out=k)
    assert _ops().read_status(q.device) == 4096  # PA_ERR_POSITION
    assert qo.data_ptr() == q.data_ptr()
    kept = torch.zeros(40, dtype=torch.bool, device="cuda")
    kept[[0, 5, 7, 39]] = True
    for got, want, was in ((q, want_q, q0), (k, want_k, k0)):
        assert torch.equal(got[~kept], want[~kept]) and torch.equal(got[kept], was[kept])


def test_zero_rows_and_nan_rows():
    q, k, _, qw, kw, pos, table = _inputs(5, 4, 2, 1, torch.float16)
    q = q.contiguous()
    q[0] = 0
    q[1, 0, 3] = float("nan")
    qo, _ = _ops().qk_norm_rope(q, k, qw, kw, pos, table)
    assert bool((qo[0] == 0).all()) and bool(qo[1, 0].isnan().all())
    assert not bool(qo[1, 1].isnan().any())


CACHES = ["f16", "i8", "f8", "f4"]


def _cache(kind, nb, KVH, bs):
    if kind == "f4":
        return _ops().fp4_cache(nb, KVH, bs), {}
    dt = {"f16": torch.float16, "i8": torch.int8, "f8": torch.float8_e4m3fn}[kind]
    kc = torch.zeros(nb, KVH, 16, bs, 8, device="cuda").to(dt)
    vc = torch.zeros(nb, KVH, 128, bs, device="cuda").to(dt)
    kw = {} if kind == "f16" else dict(k_scales=torch.zeros(nb, KVH, bs, device="cuda"),
                                       v_scales=torch.zeros(nb, KVH, bs, device="cuda"))
    return (kc, vc), kw


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,H,KVH,bs", [(1, 4, 1, 16), (33, 12, 2, 32), (300, 28, 4, 16),
                                        (7, 3, 3, 128)])
def test_into_cache_equals_the_separate_calls(kind, dt, n, H, KVH, bs):
    q, k, v, qw, kw, pos, table = _inputs(n + KVH, n, H, KVH, dt, rot=64 if n == 33 else 128)
    nb = n // bs + 2
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(n))[:n].int().cuda()
    if n > 2:
        slots[1] = -1
        pos[2] = -1
    ops = _ops()
    (kc, vc), sc = _cache(kind, nb, KVH, bs)
    qo = torch.full((n, H, 128), 5.0, dtype=dt, device="cuda")
    ops.norm_rope_into_cache(q, k, v, qw, kw, pos, table, kc, vc, slots, bs, q_out=qo, **sc)
    (kc2, vc2), sc2 = _cache(kind, nb, KVH, bs)
    qo2 = torch.full((n, H, 128), 5.0, dtype=dt, device="cuda")
    ko2 = torch.zeros(n, KVH, 128, dtype=dt, device="cuda")
    ops.qk_norm_rope(q, k, qw, kw, pos, table, q_out=qo2, k_out=ko2)
    vv = torch.empty_like(ko2).copy_(v)  # canonical strides for one token too
    slots2 = torch.where(pos < 0, torch.full_like(slots, -1), slots)
    if kind == "f4":
        ops.quantize_into_cache_fp4(ko2, vv, kc2, vc2, slots2, bs)
    elif kind == "f16":
        ops.write_into_cache(ko2, vv, kc2, vc2, slots2, bs)
    else:
        ops.quantize_into_cache(ko2, vv, kc2, vc2, sc2["k_scales"], sc2["v_scales"], slots2, bs)
    assert torch.equal(qo, qo2)
    for a, b in ((kc, kc2), (vc, vc2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for name in sc:
        assert torch.equal(sc[name], sc2[name])
    ops.check_status(q.device)


def test_into_cache_flags_slots_outside_the_cache():
    q, k, v, qw, kw, pos, table = _inputs(8, 3, 4, 2, torch.float16)
    kc, vc = _ops().fp4_cache(2, 2)
    slots = torch.tensor([0, 32, 31], dtype=torch.int32, device="cuda")
    qo = _ops().norm_rope_into_cache(q, k, v, qw, kw, pos, table, kc, vc, slots)
    assert _ops().read_status(q.device) == 256
    _close(qo, q, qw, pos, table, 1e-6, False)
    got, _ = _ops().read_from_cache_fp4(kc, vc, torch.tensor([31], dtype=torch.int32,
                                                             device="cuda"))
    assert bool((got != 0).any())


def test_refusals():
    ops = _ops()
    q, k, v, qw, kw, pos, table = _inputs(9, 4, 4, 2, torch.float16)
    kc, vc = ops.fp4_cache(2, 2)
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    bad = [dict(k=k.float()), dict(k=k[:3]), dict(qw=qw.float()), dict(qw=qw[:64]),
           dict(pos=pos.long()), dict(pos=pos[:2]), dict(table=table.half()),
           dict(table=table[:, :24].contiguous()), dict(table=table[:0]), dict(q=q[..., :64]),
           dict(q=q.transpose(0, 1)), dict(table=table.t())]
    for b in bad:
        a = dict(q=q, k=k, qw=qw, kw=kw, pos=pos, table=table)
        a.update(b)
        with pytest.raises(RuntimeError):
            ops.qk_norm_rope(*a.values())
        with pytest.raises(RuntimeError):
            ops.norm_rope_into_cache(a["q"], a["k"], v, a["qw"], a["kw"], a["pos"], a["table"], kc,
                                     vc, slots)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(q, k, qw, kw, pos, table, eps=-1.0)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(q, k, qw, kw, pos, table, q_out=torch.empty_like(q[:, :3]))
    for b in (dict(v=v[:, :1]), dict(slots=slots[:2]), dict(kc=kc[:, :1]), dict(bs=32),
              dict(kc=kc.float()), dict(sc=torch.zeros(2, 2, 16, device="cuda"))):
        a = dict(v=v, slots=slots, kc=kc, bs=16, sc=None)
        a.update(b)
        with pytest.raises(RuntimeError):
            ops.norm_rope_into_cache(q, k, a["v"], qw, kw, pos, table, a["kc"], vc, a["slots"],
                                     a["bs"], k_scales=a["sc"], v_scales=a["sc"])


def test_rope_table_keeps_far_angles():
    t = _ops().rope_table(200001, 64, base=1e6).double().cpu().numpy()
    i = np.arange(32)
    ang = 200000 * 1e6 ** (-2 * i / 64)
    assert np.abs(t[200000, :32] - np.cos(ang)).max() <= 2.0 ** -24
    assert np.abs(t[200000, 32:] - np.sin(ang)).max() <= 2.0 ** -24
