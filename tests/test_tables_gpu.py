"""GPU: block tables, slot maps and positions built from the requests' lengths, against a plain
Python allocator, and a serving step of the calls together."""

import numpy as np
import pytest
import torch

import pa_oracle
from pa_testlib import scale_for

pytestmark = pytest.mark.gpu


def _ops():
    from pa_b200 import ops
    return ops


def _i(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Batch:
    """The same state on both sides: tensors, and lists for the oracle."""

    def __init__(self, S, MB, bs, NB, seed=0):
        self.rng = np.random.default_rng(seed)
        self.S, self.MB, self.bs, self.NB = S, MB, bs, NB
        self.stack = [int(x) for x in self.rng.permutation(NB)]
        self.ref = np.full((S, MB), -7)
        self.ref_lens = [0] * S
        self.table, self.lens = _i(self.ref), _i(self.ref_lens)
        self.free, self.count = _i(self.stack + [-1] * 3), _i([NB])

    def extend(self, new, max_tokens):
        want = pa_oracle.extend_tables(self.ref, self.ref_lens, new, self.stack, self.bs)
        self.ref_lens = want[3]
        slots, pos, start, self.lens, self.count = _ops().extend_block_tables(
            self.table, self.lens, _i(new), self.free, self.count, self.NB, self.bs,
            max_tokens=max_tokens)
        n = len(want[0])
        pad = [-1] * (max_tokens - n)
        assert slots.tolist() == want[0] + pad and pos.tolist() == want[1] + pad
        assert start.tolist() == want[2]
        self.same()
        return slots, pos, start

    def release(self, finished):
        self.ref_lens = pa_oracle.release_blocks(self.ref, self.ref_lens, finished, self.stack,
                                                 self.bs)
        self.lens, self.count = _ops().release_blocks(self.table, self.lens, _i(finished),
                                                      self.free, self.count, self.bs)
        self.same()

    def same(self):
        assert self.lens.tolist() == self.ref_lens
        assert self.count.tolist() == [len(self.stack)]
        assert self.free[:len(self.stack)].tolist() == self.stack
        assert np.array_equal(self.table.cpu().numpy(), self.ref)
        _ops().check_status(self.table.device)


@pytest.mark.parametrize("S,MB,bs", [(1, 4, 16), (3, 10, 16), (70, 12, 32), (1100, 6, 16),
                                     (2500, 3, 1), (5, 300, 128)])
def test_a_life_of_extends_and_releases(S, MB, bs):
    b = Batch(S, MB, bs, S * MB + 2, seed=S)
    cap = MB * bs
    for step in range(6):
        room = cap - np.array(b.ref_lens)
        new = b.rng.integers(0, np.minimum(room, 1 + cap // 3) + 1)
        new[b.rng.random(S) < 0.3] = 0
        b.extend(new, int(new.sum()) + int(b.rng.integers(0, 50)))
        b.release((b.rng.random(S) < 0.25).astype(np.int32))
    b.extend([0] * S, 0)  # nothing to do
    b.release([1] * S)
    assert b.ref_lens == [0] * S


def test_large_prompts_span_the_ctas():
    b = Batch(3, 8000, 16, 24001, seed=1)
    b.extend([70000, 1, 50001], 120002)
    b.extend([1, 57999, 0], 58000)
    b.release([1, 0, 1])


def test_refused_calls_change_nothing():
    b = Batch(4, 4, 16, 9, seed=2)
    b.extend([20, 3, 0, 40], 63)  # 2 + 1 + 3 blocks; 3 left
    before = [t.clone() for t in (b.table, b.lens, b.free, b.count)]

    def refused(bit, new, max_tokens=200, lens=None, count=None):
        slots, pos, start, lens2, count2 = _ops().extend_block_tables(
            b.table, b.lens if lens is None else lens, _i(new), b.free,
            b.count if count is None else count, b.NB, b.bs, max_tokens=max_tokens)
        assert _ops().read_status(b.table.device) == bit
        assert bool((slots == -1).all()) and bool((pos == -1).all())
        assert bool((start == 0).all())
        assert torch.equal(lens2, b.lens if lens is None else lens)
        assert torch.equal(count2, b.count if count is None else count)
        for t, was in zip((b.table, b.lens, b.free, b.count), before):
            assert torch.equal(t, was)

    refused(1024, [0, 0, 64, 0])            # four blocks wanted, three free
    refused(32, [45, 0, 0, 0])              # past the table
    refused(32, [0, 0, -1, 0])
    refused(32, [0, 0, 0, 0], lens=_i([20, 3, -5, 40]))
    refused(2048, [1, 1, 1, 0], max_tokens=2)
    refused(1024, [1, 0, 0, 0], count=_i([-3]))
    refused(1024, [1, 0, 0, 0], count=_i([10 ** 6]))
    for flags, lens, bit in (([0, 1, 0, 0], [20, 65, 0, 40], 32), ([0, 0, 1, 0], [20, 3, -1, 40], 32)):
        l2, c2 = _ops().release_blocks(b.table, _i(lens), _i(flags), b.free, b.count, b.bs)
        assert _ops().read_status(b.table.device) == bit
        assert l2.tolist() == lens and torch.equal(c2, b.count)
        assert torch.equal(b.free, before[2])
    full = _i([11])  # no room to push two blocks into twelve
    l2, c2 = _ops().release_blocks(b.table, b.lens, _i([1, 0, 0, 0]), b.free, full, b.bs)
    assert _ops().read_status(b.table.device) == 1024
    assert torch.equal(l2, b.lens) and torch.equal(c2, full) and torch.equal(b.free, before[2])
    b.extend([1, 0, 48, 0], 49)             # and a call that fits goes through afterwards


def test_bad_free_ids_are_flagged():
    table, lens = _i(np.zeros((2, 4))), _i([0, 0])
    free, count = _i([3, 99, -4, 2]), _i([4])
    slots, pos, _, _, _ = _ops().extend_block_tables(table, lens, _i([16, 33]), free, count, 8, 16,
                                                     max_tokens=50)
    assert _ops().read_status(table.device) == 64
    assert slots[:16].tolist() == list(range(32, 48)) and bool((slots[16:48] == -1).all())
    assert slots[48].item() == 48 and slots[49].item() == -1 and pos[48].item() == 32


def test_in_place_in_a_graph():
    """A captured step whose state stays on the device: in-place lengths and count."""
    S, MB, bs, NB = 9, 8, 16, 80
    rng = np.random.default_rng(4)
    stack = [int(x) for x in rng.permutation(NB)]
    ref, ref_lens = np.zeros((S, MB), int), [0] * S
    table, lens, free, count = _i(ref), _i(ref_lens), _i(stack), _i([NB])
    new, done = _i([0] * S), _i([0] * S)
    slots, pos, start = _i([-1] * 64), _i([-1] * 64), _i([0] * (S + 1))

    def step():
        _ops().release_blocks(table, lens, done, free, count, bs, context_lens_out=lens,
                              free_count_out=count)
        _ops().extend_block_tables(table, lens, new, free, count, NB, bs, max_tokens=64,
                                   slot_mapping=slots, positions=pos, query_start=start,
                                   context_lens_out=lens, free_count_out=count)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    torch.cuda.synchronize()
    for i in range(8):
        add = rng.integers(0, 8, S)
        fin = (rng.random(S) < 0.3).astype(np.int32)
        new.copy_(_i(add))
        done.copy_(_i(fin))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ref_lens = pa_oracle.release_blocks(ref, ref_lens, fin, stack, bs)
        want = pa_oracle.extend_tables(ref, ref_lens, add, stack, bs)
        ref_lens = want[3]
        n = len(want[0])
        assert slots[:n].tolist() == want[0] and bool((slots[n:] == -1).all())
        assert pos[:n].tolist() == want[1] and start.tolist() == want[2]
        assert lens.tolist() == ref_lens and count.tolist() == [len(stack)]
    _ops().check_status(table.device)


def test_refusals():
    ops = _ops()
    bt, i, one = _i(np.zeros((3, 4))), _i([0] * 3), _i([0])
    bad = [dict(bt=bt.long()), dict(bt=bt[:, ::2]), dict(lens=i[:2]), dict(lens=i.cpu()),
           dict(per=i.float()), dict(free=i[::2]), dict(count=i), dict(bs=0)]
    for x in bad:
        a = dict(bt=bt, lens=i, per=i, free=i, count=one, bs=16)
        a.update(x)
        with pytest.raises(RuntimeError):
            ops.release_blocks(*a.values())
        with pytest.raises(RuntimeError):
            ops.extend_block_tables(a["bt"], a["lens"], a["per"], a["free"], a["count"], 4, a["bs"],
                                    max_tokens=4)
    with pytest.raises(RuntimeError):
        ops.extend_block_tables(bt, i, i, i, one, 4, max_tokens=-1)
    with pytest.raises(RuntimeError):
        ops.extend_block_tables(bt, i, i, i, one, 4, max_tokens=4, slot_mapping=i)
    with pytest.raises(RuntimeError):
        ops.extend_block_tables(bt, i, i, i, one, 0, max_tokens=4)
    with pytest.raises(RuntimeError):
        ops.release_blocks(bt, i, i, i, one, context_lens_out=one)


def test_serving_steps_through_all_the_calls():
    """Three requests from prompt to a few generated tokens, one replaced on the way: tables,
    norm and rotation into the 4-bit cache, decode. The cache's contents are checked against the
    oracle's rows, the attention against 64 bits over the held values (the tolerance of
    test_fp4_gpu.py)."""
    ops = _ops()
    S, H, KVH, bs, MB, NB = 3, 12, 2, 16, 8, 20
    g = torch.Generator().manual_seed(5)
    qw, kw = ((1 + 0.1 * torch.randn(128, generator=g)).half().cuda() for _ in "qk")
    rope = ops.rope_table(256)
    kc, vc = ops.fp4_cache(NB, KVH, bs)
    table, lens = _i(np.zeros((S, MB))), _i([0] * S)
    free, count = _i(np.random.default_rng(6).permutation(NB)), _i([NB])
    held = [[np.zeros((0, KVH, 128))] * 2 for _ in range(S)]  # K and V rows of each request
    plan = [([37, 5, 16], [0, 0, 0]), ([1, 1, 1], [0, 0, 0]), ([1, 30, 1], [0, 1, 0]),
            ([1, 1, 1], [0, 0, 0])]
    for new, done in plan:
        T = sum(new) + 3
        lens, count = ops.release_blocks(table, lens, _i(done), free, count, bs)
        slots, pos, start, lens, count = ops.extend_block_tables(
            table, lens, _i(new), free, count, NB, bs, max_tokens=T)
        qkv = torch.randn(T, H + 2 * KVH, 128, generator=g).half().cuda()
        q = torch.full((T, H, 128), 9.0, dtype=torch.float16, device="cuda")
        ops.norm_rope_into_cache(qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:], qw, kw, pos,
                                 rope, kc, vc, slots, bs, q_out=q)
        assert bool((q[-3:] == 9.0).all())  # the padding's rows are left alone
        st = start.tolist()
        last = q[[st[b + 1] - 1 for b in range(S)]].contiguous()
        out = torch.empty_like(last)
        ops.decode(out, last, kc, vc, table, lens, scale_for(), bs)
        ops.check_status(out.device)
        # K rows as the unfused call gives them (rounded to fp16), quantised by the oracle.
        _, k2 = ops.qk_norm_rope(qkv[:, :H], qkv[:, H:H + KVH], qw, kw, pos, rope)
        kcn, vcn, bt = kc.cpu().numpy(), vc.cpu().numpy(), table.cpu().numpy()
        for b in range(S):
            if done[b]:
                held[b] = [np.zeros((0, KVH, 128))] * 2
            rows = (k2[st[b]:st[b + 1]], qkv[st[b]:st[b + 1], H + KVH:])
            held[b] = [np.concatenate([h, pa_oracle.dequantize_fp4(*pa_oracle.quantize_fp4(
                r.double().cpu().numpy()))]) for h, r in zip(held[b], rows)]
            n = lens[b].item()
            assert n == held[b][0].shape[0]
            for cache, is_v in ((kcn, False), (vcn, True)):
                v = pa_oracle.fp4_values(cache[bt[b, :-(-n // bs)]], is_v)
                v = v.transpose(0, 2, 1, 3).reshape(-1, KVH, 128)[:n]
                assert np.array_equal(v, held[b][int(is_v)])
        ref, qk, vmax = pa_oracle.fp4_decode(last.double().cpu().numpy(), kcn, vcn, bt,
                                             lens.cpu().numpy(), scale_for())
        e = 2 * (2.0 ** -17 * qk + 2.0 ** -20) + lens.cpu().numpy() / 16 * 2.0 ** -22
        tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + (e * vmax)[:, None, None]
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()


def test_a_captured_step_equals_the_eager_calls():
    """One graph of release, extend, norm and rotation into the cache and decode, replayed with
    new lengths and rows, against the same calls made one by one: every byte alike."""
    ops = _ops()
    S, H, KVH, bs, MB, NB, T = 5, 12, 2, 16, 8, 34, 24
    rope = ops.rope_table(256)
    rng = np.random.default_rng(8)
    perm = rng.permutation(NB)

    def state():
        kc, vc = ops.fp4_cache(NB, KVH, bs)
        z = torch.zeros
        return dict(kc=kc, vc=vc, table=_i(np.zeros((S, MB))), lens=_i([0] * S), free=_i(perm),
                    count=_i([NB]), new=_i([0] * S), done=_i([0] * S), slots=_i([-1] * T),
                    pos=_i([-1] * T), start=_i([0] * (S + 1)),
                    qkv=z(T, H + 2 * KVH, 128, dtype=torch.float16, device="cuda"),
                    q=z(T, H, 128, dtype=torch.float16, device="cuda"),
                    out=z(S, H, 128, dtype=torch.float16, device="cuda"))

    def step(s):
        ops.release_blocks(s["table"], s["lens"], s["done"], s["free"], s["count"], bs,
                           context_lens_out=s["lens"], free_count_out=s["count"])
        ops.extend_block_tables(s["table"], s["lens"], s["new"], s["free"], s["count"], NB, bs,
                                max_tokens=T, slot_mapping=s["slots"], positions=s["pos"],
                                query_start=s["start"], context_lens_out=s["lens"],
                                free_count_out=s["count"])
        x = s["qkv"]
        ops.norm_rope_into_cache(x[:, :H], x[:, H:H + KVH], x[:, H + KVH:], None, None, s["pos"],
                                 rope, s["kc"], s["vc"], s["slots"], bs, q_out=s["q"])
        last = s["q"].index_select(0, (s["start"][1:] - 1).clamp(min=0))
        ops.decode(s["out"], last, s["kc"], s["vc"], s["table"], s["lens"], scale_for(), bs,
                   validate=False)

    a, b = state(), state()
    for s in (a, b):
        s["new"].fill_(1)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step(a)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step(a)
    torch.cuda.synchronize()
    step(b)
    for i in range(10):
        # Every sequence gets a token at least; some leave and come back with a prompt.
        done = (rng.random(S) < 0.3).astype(np.int32)
        add = np.where(done, rng.integers(1, 5, S), 1)
        x = torch.from_numpy(rng.standard_normal((T, H + 2 * KVH, 128)).astype(np.float16)).cuda()
        for s in (a, b):
            s["new"].copy_(_i(add))
            s["done"].copy_(_i(done))
            s["qkv"].copy_(x)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        step(b)
        torch.cuda.synchronize()
        for name in a:
            assert torch.equal(a[name], b[name]), (i, name)
    ops.check_status(a["out"].device)
