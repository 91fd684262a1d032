"""GPU: norm and rotation of rows with infinities and NaN: they reach the values that the formula
says and no others, and rows in a cache are those of the separate calls."""

import numpy as np
import pytest
import torch

import pa_oracle
from test_rope_gpu import _cache, _close, _inputs, _np

pytestmark = pytest.mark.gpu


def _ops():
    from pa_b200 import ops
    return ops


def _odd_rows(t, rot):
    """An infinity or a NaN in the rows 0 .. 5 of head 0: turned, not turned, and both."""
    past = [i for i in (rot, rot + 1, rot + 5, 127) if i < 128]
    inf, nan = float("inf"), float("nan")
    t = t.clone()
    for n, (at, what) in enumerate([([0], inf), ([rot - 1], nan), (past[:1], inf), (past[-1:], nan),
                                    ([3] + past[1:3], -inf), (past, inf)]):
        t[n, 0, at] = what
    return t


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rot", [16, 64, 112, 128])
@pytest.mark.parametrize("n,H,KVH", [(9, 4, 2), (1200, 13, 3)])
def test_infinities_and_nan(dt, interleaved, norm, rot, n, H, KVH):
    q, k, _, qw, kw, pos, table = _inputs(rot + n, n, H, KVH, dt, rot, norm=norm)
    q, k = _odd_rows(q, rot), _odd_rows(k, rot)
    for got, x, w in zip(_ops().qk_norm_rope(q, k, qw, kw, pos, table, interleaved=interleaved),
                         (q, k), (qw, kw)):
        with np.errstate(invalid="ignore"):
            ref = pa_oracle.norm_rope(_np(x), _np(w), _np(pos).astype(int), _np(table), 1e-6,
                                      interleaved)
        mine = _np(got)
        assert np.array_equal(np.isnan(mine), np.isnan(ref))
        assert np.array_equal(np.isposinf(mine), np.isposinf(ref))
        assert np.array_equal(np.isneginf(mine), np.isneginf(ref))
        ok = torch.arange(6, n, device="cuda")
        _close(got[ok], x[ok], w, pos[ok], table, 1e-6, interleaved)
        # Of a row with an infinity and no norm, the others hold what they would without it.
        if not norm and rot < 128:
            assert torch.equal(got[2, 0, :rot], _ops().qk_norm_rope(
                x[2:3].nan_to_num(posinf=1.0), x[2:3, :0], w, w, pos[2:3], table,
                interleaved=interleaved)[0][0, 0, :rot])


@pytest.mark.parametrize("kind", ["f16", "i8", "f8", "f4"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [7, 1500])
def test_infinities_and_nan_into_caches(kind, dt, n):
    """Bit for bit the separate calls' caches, where those define the bits: a NaN's payload in a
    16-bit cache and the codes beside a NaN scale are anything."""
    H, KVH, bs, rot = 8, 2, 16, 64
    q, k, v, qw, kw, pos, table = _inputs(n, n, H, KVH, dt, rot)
    k, v = _odd_rows(k, rot), _odd_rows(v, rot)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    ops, nb = _ops(), n // bs + 1
    (kc, vc), sc = _cache(kind, nb, KVH, bs)
    ops.norm_rope_into_cache(q, k, v, qw, None, pos, table, kc, vc, slots, bs, **sc)
    (kc2, vc2), sc2 = _cache(kind, nb, KVH, bs)
    _, k2 = ops.qk_norm_rope(q, k, qw, None, pos, table)
    v2 = v.contiguous()
    if kind == "f4":
        ops.quantize_into_cache_fp4(k2, v2, kc2, vc2, slots, bs)
        for a, b in zip(ops.read_from_cache_fp4(kc, vc, slots, bs),
                        ops.read_from_cache_fp4(kc2, vc2, slots, bs)):
            assert np.array_equal(_np(a), _np(b), equal_nan=True)
    elif kind == "f16":
        ops.write_into_cache(k2, v2, kc2, vc2, slots, bs)
        for a, b in ((kc, kc2), (vc, vc2)):
            assert np.array_equal(_np(a), _np(b), equal_nan=True)
    else:
        ops.quantize_into_cache(k2, v2, kc2, vc2, sc2["k_scales"], sc2["v_scales"], slots, bs)
        for a, b in ((kc, kc2), (vc, vc2)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for name in sc:
            assert np.array_equal(_np(sc[name]), _np(sc2[name]), equal_nan=True)
    ops.check_status(q.device)
