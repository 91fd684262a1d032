"""GPU: norm and rotation at the sizes where a half-warp takes four heads (from sixteen warps an SM
on), with head counts that leave part of the last warp empty: in place, and into every cache."""

import pytest
import torch

from test_rope_gpu import _cache, _close, _inputs

pytestmark = pytest.mark.gpu

SIZES = [(800, 28, 4), (1200, 13, 3), (2400, 1, 1), (500, 32, 8)]


def _ops():
    from pa_b200 import ops
    return ops


def _four_heads(n, H, KVH, rows_of_kv):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return n * (-(-H // 8) + rows_of_kv * -(-KVH // 8)) >= 16 * sms


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [128, 96, 16])
@pytest.mark.parametrize("n,H,KVH", SIZES)
def test_in_place(dt, interleaved, rot, n, H, KVH):
    """q and k are views of one projection; the outputs replace them and nothing else."""
    n = max(n, 2400 // (-(-H // 8) + 1))
    assert _four_heads(n, H, KVH, 1)
    q, k, v, qw, kw, pos, table = _inputs(n, n, H, KVH, dt, rot)
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    pos[::7] = -1
    kw_ = dict(eps=1e-5, interleaved=interleaved)
    want = _ops().qk_norm_rope(q, k, qw, kw, pos, table, q_out=q0.clone(), k_out=k0.clone(), **kw_)
    _ops().qk_norm_rope(q, k, qw, kw, pos, table, q_out=q, k_out=k, **kw_)
    assert torch.equal(v, v0)
    on = pos >= 0
    for got, w, was, weight in ((q, want[0], q0, qw), (k, want[1], k0, kw)):
        assert torch.equal(got, w) and torch.equal(got[~on], was[~on])
        _close(got[on], was[on], weight, pos[on], table, 1e-5, interleaved)
    _ops().check_status(q.device)


@pytest.mark.parametrize("kind", ["f16", "i8", "f8", "f4"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,H,KVH,bs,rot,interleaved", [
    (850, 28, 4, 16, 128, False), (900, 13, 3, 32, 64, False), (1300, 12, 2, 128, 128, True),
    (1300, 13, 3, 16, 48, True), (700, 40, 8, 16, 16, True), (1000, 9, 9, 64, 96, False),
    (5, 4, 2, 16, 128, True), (33, 5, 3, 32, 16, True), (9, 3, 1, 16, 48, True)])
def test_into_cache_equals_the_separate_calls(kind, dt, n, H, KVH, bs, rot, interleaved):
    assert n < 100 or _four_heads(n, H, KVH, 2)
    q, k, v, qw, kw, pos, table = _inputs(n + KVH, n, H, KVH, dt, rot)
    ops, nb = _ops(), n // bs + 2
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(n)).int().cuda()
    t = torch.arange(n, device="cuda")
    slots = perm[t // bs] * bs + (t % bs).int()  # a prompt through shuffled blocks
    slots[1], pos[2] = -1, -1
    args = dict(eps=1e-5, interleaved=interleaved)
    (kc, vc), sc = _cache(kind, nb, KVH, bs)
    (kc2, vc2), sc2 = _cache(kind, nb, KVH, bs)
    qo = torch.full((n, H, 128), 5.0, dtype=dt, device="cuda")
    qo2, ko2 = qo.clone(), torch.zeros(n, KVH, 128, dtype=dt, device="cuda")
    ops.norm_rope_into_cache(q, k, v, qw, kw, pos, table, kc, vc, slots, bs, q_out=qo, **sc,
                             **args)
    ops.qk_norm_rope(q, k, qw, kw, pos, table, q_out=qo2, k_out=ko2, **args)
    on = pos >= 0
    _close(qo[on], q[on], qw, pos[on], table, 1e-5, interleaved)
    _close(ko2[on], k[on], kw, pos[on], table, 1e-5, interleaved)
    slots2 = torch.where(on, slots, torch.full_like(slots, -1))
    v2 = torch.empty_like(ko2).copy_(v)
    if kind == "f4":
        ops.quantize_into_cache_fp4(ko2, v2, kc2, vc2, slots2, bs)
    elif kind == "f16":
        ops.write_into_cache(ko2, v2, kc2, vc2, slots2, bs)
    else:
        ops.quantize_into_cache(ko2, v2, kc2, vc2, sc2["k_scales"], sc2["v_scales"], slots2, bs)
    assert torch.equal(qo, qo2)
    for a, b in ((kc, kc2), (vc, vc2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for name in sc:
        assert torch.equal(sc[name], sc2[name])
    ops.check_status(q.device)
