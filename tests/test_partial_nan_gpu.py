"""GPU: a NaN that a decode's partials hold reaches the merged rows."""

import numpy as np
import pytest
import torch

from pa_testlib import scale_for
from test_fp4_gpu import _case, _gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,H,KVH", [([5, 40], 8, 4), ([3000, 70], 12, 2), ([2000, 9], 32, 2),
                                        ([700, 30], 20, 1)])
@pytest.mark.parametrize("is_v", [False, True])
def test_nan_block_reaches_the_merged_rows(lens, H, KVH, is_v):
    """Two ranges of each context, the NaN block in the second: as in the decode of the whole, K's
    makes every head of its kv head NaN and V's the block's 16 values of them, and no other."""
    from pa_b200 import ops
    c = _case(50, lens, H, KVH, pad=0xFF)
    q, kc, vc, bt, cl = _gpu(c)
    G, last = H // KVH, c["lens"][0] - 1
    blk, off = int(c["bt"][0, last // 16]), int(last % 16)
    cut = 1 if lens[0] > 16 else 0  # blocks of the first range
    first = torch.clamp(cl, max=16 * cut)

    def merged():
        parts = [ops.decode_partial(q, kc, vc, bt, first, scale_for()),
                 ops.decode_partial(q, kc, vc, bt[:, cut:].contiguous(), cl - first,
                                    scale_for())]
        out = torch.zeros_like(q)
        ops.merge_partials(out, torch.stack(parts), H, KVH)
        return out

    clean = merged()
    assert bool(torch.isfinite(clean).all())
    (vc if is_v else kc)[blk, 0, 0, 1024 + (3 * 16 + off if is_v else off * 8 + 3)] = 0xFF
    out = merged()
    want = torch.zeros(len(lens), H, 128, dtype=torch.bool, device="cuda")
    want[0, :G, 48:64] = True
    if not is_v:
        want[0, :G] = True
    assert torch.equal(torch.isnan(out), want)
    assert torch.equal(out[~want], clean[~want])
    ops.check_status(q.device)


@pytest.mark.parametrize("H,KVH", [(8, 2), (32, 2)])
def test_nan_of_an_fp16_caches_partial(H, KVH):
    from pa_b200 import ops
    g = torch.Generator().manual_seed(1)
    kc = torch.randn(8, KVH, 16, 16, 8, generator=g).half().cuda()
    vc = torch.randn(8, KVH, 128, 16, generator=g).half().cuda()
    kc[3, 1, 2, 4, 5] = float("nan")
    q = torch.randn(1, H, 128, generator=g).half().cuda()
    bt = torch.from_numpy(np.arange(8, dtype=np.int32))[None].cuda()
    one = torch.tensor([128], dtype=torch.int32, device="cuda")
    part = ops.decode_partial(q, kc, vc, bt, one, scale_for())
    out = torch.zeros_like(q)
    ops.merge_partials(out, part[None], H, KVH)
    G = H // KVH
    assert bool(out[0, G:].isnan().all()) and not bool(out[0, :G].isnan().any())
    ops.check_status(q.device)
