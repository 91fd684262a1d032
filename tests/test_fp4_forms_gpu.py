"""GPU: the 4-bit decode's entry points against each other: workspaces of exactly the size asked
for, splitk (which is the same kernel), bf16 activations at bf16's own rounding, steps of more
sequences than a launch holds, and the calls that serve an empty side."""

import numpy as np
import pytest
import torch

import pa_oracle
from pa_testlib import scale_for
from test_fp4_gpu import SHAPES, _case, _gpu, _rows

pytestmark = pytest.mark.gpu


def _ops():
    from pa_b200 import ops
    return ops


@pytest.mark.parametrize("lens,H,KVH", [([700, 4096], 12, 2), ([2000, 90], 32, 2), ([300], 20, 1)])
@pytest.mark.parametrize("form", ["decode", "splitk", "bf16"])
def test_workspace_of_the_size_asked_for(lens, H, KVH, form):
    from pa_b200 import _lib
    L, bf = _lib.lib(), form == "bf16"
    c = _case(60 + H, lens, H, KVH, dt=torch.bfloat16 if bf else torch.float16)
    q, kc, vc, bt, cl = _gpu(c)
    sizes = (len(lens), H, KVH, 128, bt.shape[1], 16, _lib.PA_DTYPE_FP4E2M1, int(form == "splitk"))
    need = (L.pa_decode_bf16q_workspace_bytes if bf else L.pa_decode_workspace_bytes)(*sizes)
    guard = 4096
    ws = torch.zeros(need + guard, dtype=torch.uint8, device="cuda")
    ws[need:] = 0xA5
    out = torch.full_like(q, float("nan"))
    stream = torch.cuda.current_stream().cuda_stream

    def call(nbytes):
        args = [t.data_ptr() for t in (out, q, kc, vc)]
        tail = [bt.data_ptr(), cl.data_ptr(), len(lens), H, KVH, 128, kc.shape[0], 16, bt.shape[1]]
        if bf:
            return L.pa_decode_bf16q(*args, None, None, *tail, _lib.PA_DTYPE_FP4E2M1, 0,
                                     scale_for(), ws.data_ptr(), nbytes, stream)
        fn = L.pa_splitk_fp4 if form == "splitk" else L.pa_decode_fp4
        return fn(*args, *tail, scale_for(), ws.data_ptr(), nbytes, stream)

    assert call(need - 1) == _lib.PA_ERR_WORKSPACE
    assert call(need) == _lib.PA_OK
    want = torch.empty_like(q)
    (_ops().decode_bf16 if bf else _ops().decode)(want, q, kc, vc, bt, cl, scale_for())
    assert torch.equal(out, want)
    assert bool((ws[need:] == 0xA5).all())


@pytest.mark.parametrize("lens,H,KVH", SHAPES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_splitk_is_the_same_kernel_and_bf16_rounds_once(lens, H, KVH, dt):
    """The tolerance of test_fp4_gpu.py, with bf16 outputs rounded from fp32: 2^-8 of the value."""
    c = _case(70 + H, lens, H, KVH, dt=dt)
    q, kc, vc, bt, cl = _gpu(c)
    run = _ops().decode if dt == torch.float16 else _ops().decode_bf16
    outs = []
    for splitk in (False, True):
        outs.append(torch.full_like(q, float("nan")))
        run(outs[-1], q, kc, vc, bt, cl, scale_for(), splitk=splitk)
    assert torch.equal(*outs)
    ref, qk, vmax = pa_oracle.fp4_decode(c["q"].double().numpy(), c["kc"], c["vc"], c["bt"], lens,
                                         scale_for())
    e = 2 * (2.0 ** -17 * qk + 2.0 ** -20) + np.asarray(lens) / 16 * 2.0 ** -22
    tol = 2.0 ** (-11 if dt == torch.float16 else -8) * np.abs(ref) + 2.0 ** -25 + (
        e * vmax)[:, None, None]
    assert (np.abs(outs[0].double().cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("KVH,H", [(2, 8), (1, 16)])
def test_steps_of_more_sequences_than_a_launch_holds(KVH, H):
    """1100 sequences, the new rows views of one projection: the fused and the separate write."""
    lens = [1 + (i * 7) % 40 for i in range(1100)]
    c = _case(80, lens, H, KVH, pad=0xFF)
    rows = torch.cat([_rows(np.random.default_rng(i), 1100, KVH, torch.float16)[0]
                      for i in range(3)], 1).cuda()
    k, v = rows[:, KVH:2 * KVH], rows[:, 2 * KVH:]
    got = []
    for fused in (True, False):
        q, kc, vc, bt, cl = _gpu(c)
        out = torch.full_like(q, float("nan"))
        _ops().decode_step(out, q, k, v, kc, vc, bt, cl, scale_for(), fused=fused)
        got.append((out, kc, vc))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    last = c["lens"] - 1
    slots = c["bt"][np.arange(1100), last // 16] * 16 + last % 16
    for name, r, is_v in (("kc", k, False), ("vc", v, True)):
        pa_oracle.fp4_put(c[name], is_v, r.double().cpu().numpy(), slots, 16)
    ref, qk, vmax = pa_oracle.fp4_decode(c["q"].double().numpy(), c["kc"], c["vc"], c["bt"],
                                         c["lens"], scale_for())
    e = 2 * (2.0 ** -17 * qk + 2.0 ** -20) + np.asarray(lens) / 16 * 2.0 ** -22
    tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + (e * vmax)[:, None, None]
    assert (np.abs(got[0][0].double().cpu().numpy() - ref) <= tol).all()
    _ops().check_status(out.device)


def test_a_captured_step_of_few_sequences():
    """The fused write inside a graph: lengths, rows and q change between replays."""
    H, KVH = 12, 2
    c = _case(81, [33, 700, 16], H, KVH, pad=0xFF)
    q, kc, vc, bt, cl = _gpu(c)
    kc2, vc2 = kc.clone(), vc.clone()
    k, v = (torch.zeros(3, KVH, 128, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    out, out2 = torch.empty_like(q), torch.empty_like(q)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def step(o, a, b):
        _ops().decode_step(o, q, k, v, a, b, bt, cl, scale_for(), validate=False)

    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step(out, kc, vc)
        with torch.cuda.graph(g, stream=s):
            step(out, kc, vc)
    torch.cuda.synchronize()
    step(out2, kc2, vc2)
    gen = torch.Generator().manual_seed(3)
    for i in range(5):
        cl.sub_(1)  # the table has no room for more tokens
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        step(out2, kc2, vc2)
        assert torch.equal(out, out2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
    _ops().check_status(q.device)


def test_no_q_heads():
    """K and V alone into the cache, and a position outside the table that only K's rows can flag."""
    ops = _ops()
    g = torch.Generator().manual_seed(4)
    kv = torch.randn(20, 4, 128, generator=g).half().cuda()
    pos = torch.arange(20, dtype=torch.int32, device="cuda")
    table = ops.rope_table(32)
    slots = pos + 3
    kc, vc = ops.fp4_cache(2, 2)
    none = kv[:, :0]
    q = ops.norm_rope_into_cache(none, kv[:, :2], kv[:, 2:], None, None, pos, table, kc, vc, slots)
    assert q.shape == (20, 0, 128)
    _, want = ops.qk_norm_rope(none, kv[:, :2], None, None, pos, table)
    kc2, vc2 = ops.fp4_cache(2, 2)
    ops.quantize_into_cache_fp4(want, kv[:, 2:].contiguous(), kc2, vc2, slots)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    ops.check_status(kv.device)
    ops.norm_rope_into_cache(none, kv[:, :2], kv[:, 2:], None, None, pos + 13, table, kc, vc, slots)
    assert ops.read_status(kv.device) == 4096  # PA_ERR_POSITION


def test_new_lengths_that_pass_32_bits_together():
    """Blocks of 2^29 tokens: each sequence fits its table, the sum passes 2^31."""
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    slots, pos, start, lens, count = _ops().extend_block_tables(
        table, i(*[0] * 6), i(*[1 << 29] * 6), i(0, 1, 2, 3), i(4), 4, 1 << 29, max_tokens=64)
    assert _ops().read_status(table.device) == 1024 | 2048
    assert lens.tolist() == [0] * 6 and count.item() == 4 and bool((table == 0).all())
    assert bool((slots == -1).all()) and bool((pos == -1).all()) and bool((start == 0).all())
    slots, pos, start, lens, count = _ops().extend_block_tables(
        table, i(*[(1 << 29) - 1] * 3 + [0] * 3), i(2, 1, 0, 0, 0, 0), i(0, 1, 2, 3), i(4), 4,
        1 << 29, max_tokens=4)
    assert pos.tolist() == [(1 << 29) - 1, 1 << 29, (1 << 29) - 1, -1]
    assert slots.tolist() == [(1 << 29) - 1, 3 << 29, (1 << 29) - 1, -1]
    _ops().check_status(table.device)


@pytest.mark.parametrize("S", [1500, 2049])
def test_in_place_lengths_of_more_sequences_than_threads(S):
    """The lengths and the count are replaced by the call that reads them, over several chunks."""
    ops = _ops()
    rng = np.random.default_rng(S)
    bs, MB, NB = 16, 4, 4 * S
    stack = [int(x) for x in rng.permutation(NB)]
    ref, ref_lens = np.zeros((S, MB), int), [0] * S
    dev = dict(dtype=torch.int32, device="cuda")
    table, lens = torch.zeros(S, MB, **dev), torch.zeros(S, **dev)
    free, count = torch.tensor(stack, **dev), torch.tensor([NB], **dev)
    for _ in range(4):
        new = rng.integers(0, np.minimum(20, MB * bs - np.array(ref_lens)) + 1)
        want = pa_oracle.extend_tables(ref, ref_lens, new, stack, bs)
        T = len(want[0]) + 5
        slots, pos, start, _, _ = ops.extend_block_tables(
            table, lens, torch.tensor(new, **dev), free, count, NB, bs, max_tokens=T,
            context_lens_out=lens, free_count_out=count)
        assert slots.tolist() == want[0] + [-1] * 5 and pos.tolist() == want[1] + [-1] * 5
        assert start.tolist() == want[2] and lens.tolist() == want[3]
        done = (rng.random(S) < 0.3).astype(np.int32)
        ref_lens = pa_oracle.release_blocks(ref, want[3], done, stack, bs)
        ops.release_blocks(table, lens, torch.tensor(done, **dev), free, count, bs,
                           context_lens_out=lens, free_count_out=count)
        assert lens.tolist() == ref_lens and count.tolist() == [len(stack)]
        assert free[:len(stack)].tolist() == stack
    ops.check_status(table.device)


@pytest.mark.parametrize("kind", ["f16", "i8", "f8"])
def test_norm_into_caches_of_other_block_sizes(kind):
    """The page layouts take any block size in their writes; so does the fused form."""
    from test_rope_gpu import _cache, _inputs
    ops, n, bs, KVH = _ops(), 50, 24, 3
    q, k, v, qw, kw, pos, table = _inputs(90, n, 6, KVH, torch.float16, 64)
    slots = torch.randperm(96, generator=torch.Generator().manual_seed(5))[:n].int().cuda()
    (kc, vc), sc = _cache(kind, 4, KVH, bs)
    (kc2, vc2), sc2 = _cache(kind, 4, KVH, bs)
    ops.norm_rope_into_cache(q, k, v, qw, kw, pos, table, kc, vc, slots, bs, **sc)
    _, k2 = ops.qk_norm_rope(q, k, qw, kw, pos, table)
    if kind == "f16":
        ops.write_into_cache(k2, v.contiguous(), kc2, vc2, slots, bs)
    else:
        ops.quantize_into_cache(k2, v.contiguous(), kc2, vc2, sc2["k_scales"], sc2["v_scales"],
                                slots, bs)
    for a, b in ((kc, kc2), (vc, vc2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for name in sc:
        assert torch.equal(sc[name], sc2[name])
    ops.check_status(q.device)
