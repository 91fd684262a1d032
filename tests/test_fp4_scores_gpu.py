"""GPU: the 4-bit decode where scores are so large that fp32 leaves them no bits below 1. What the
softmax is then is known in two cases whatever the rounding: K rows that are all alike have equal
scores, so the output is the mean of V; a row far above the others takes all the weight.

Tolerance: the weights of equal scores are equal, so the output is off by the sums' rounding,
n / 16 steps of 2^-22 of max |v|, the two-part weights' 2^-20, and the output's own half step."""

import numpy as np
import pytest
import torch

import pa_oracle
from pa_testlib import scale_for

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _ops():
    from pa_b200 import ops
    return ops


def _run(n, H, KVH, dt, mag, k_of, q_sign=1.0, scale=None):
    """Decode of two sequences of n tokens each; K rows hold k_of(token) everywhere."""
    ops = _ops()
    g = torch.Generator().manual_seed(n + H)
    blocks = -(-n // 16)
    kc, vc = ops.fp4_cache(2 * blocks, KVH)
    bt = torch.arange(2 * blocks, dtype=torch.int32, device="cuda").view(2, blocks)
    t = torch.arange(n)
    k = k_of(t).half()[:, None, None].expand(n, KVH, 128).contiguous().cuda()
    v = torch.randn(n, KVH, 128, generator=g).half().cuda()
    for b in range(2):
        slots = (bt[b].cpu()[t // 16] * 16 + t % 16).int().cuda()
        ops.quantize_into_cache_fp4(k, v, kc, vc, slots)
    q = torch.full((2, H, 128), q_sign * mag).to(dt).cuda()
    lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    run = ops.decode if dt == torch.float16 else ops.decode_bf16
    run(out, q, kc, vc, bt, lens, scale_for() if scale is None else scale)
    ops.check_status(q.device)
    held = pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(v.double().cpu().numpy()))
    return out.double().cpu().numpy(), np.repeat(held, H // KVH, 1)  # [n, H, 128]


SHAPES = [(5, 8, 4), (40, 12, 2), (333, 32, 2), (5000, 12, 2), (700, 20, 1)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,H,KVH", SHAPES)
@pytest.mark.parametrize("mag,k,sign", [(60000.0, 61440.0, 1), (60000.0, 61440.0, -1),
                                        (9984.0, 6144.0, 1), (3000.0, 6144.0, -1),
                                        (1000.0, 960.0, 1), (0.5, 0.75, 1)])
def test_equal_scores_average(dt, n, H, KVH, mag, k, sign):
    out, v = _run(n, H, KVH, dt, mag, lambda t: torch.full(t.shape, k), sign)
    ref, vmax = v.mean(0), np.abs(v).max()
    tol = HALF[dt] * np.abs(ref) + 2.0 ** -25 + (n / 16 * 2.0 ** -22 + 2.0 ** -20) * vmax
    assert (np.abs(out - ref[None]) <= tol).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,H,KVH", SHAPES)
@pytest.mark.parametrize("mag,k", [(60000.0, 30720.0), (9984.0, 12288.0), (1000.0, 960.0)])
@pytest.mark.parametrize("at", [0.0, 0.5, 1.0])
def test_the_largest_score_takes_all(dt, n, H, KVH, mag, k, at):
    """Its row is twice the others, whose scores are thousands below."""
    t0 = int(at * (n - 1))
    out, v = _run(n, H, KVH, dt, mag, lambda t: torch.where(t == t0, 2 * k, k))
    tol = HALF[dt] * np.abs(v[t0]) + 2.0 ** -25 + 2.0 ** -20 * np.abs(v).max()
    assert (np.abs(out - v[t0][None]) <= tol).all()


@pytest.mark.parametrize("n,H,KVH", SHAPES)
@pytest.mark.parametrize("step", [1.0, 16.0, 2048.0])
def test_rising_scores_stay_between_the_values(n, H, KVH, step):
    """Scores that rise from token to token move the maximum all along the range."""
    out, v = _run(n, H, KVH, torch.float16, 60000.0,
                  lambda t: (step * t).clamp(max=61440.0), scale=1.0)
    lo, hi = v.min(0)[None], v.max(0)[None]
    tol = 2.0 ** -11 * np.abs(v).max() + 2.0 ** -20 * np.abs(v).max()
    assert (out >= lo - tol).all() and (out <= hi + tol).all()
