"""Operators of one serving step over a 4-bit K/V cache: what each computes in plain torch, the
cases that stand for its use, and the same passes through the library's own calls.

  plan    block tables, slot maps and positions of a step from the requests' lengths
  rope    RMS norm of every q and k head and the position rotation, in one pass
  fused   the same, with K and V going straight into the 4-bit cache
  write   K/V rows into the 4-bit cache, and rows read back from it
  step    one decode step over the 4-bit cache: the new tokens' rows written, then attention
  decode  attention of single tokens over the 4-bit cache

The 4-bit cache. Codes are e2m1 (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3,
4, 6), sixteen neighbouring head_dim values share a scale of five exponent and three mantissa
bits (bias 15, no sign; byte << 7 is the scale's fp16 pattern), and value = e2m1 * scale. Every
16 tokens of one block and kv head are one 1152-byte group, in a uint8 tensor
[num_blocks, kv_heads, block_size / 16, 1152]: 16 rows of 64 code bytes (byte j of a token holds
head_dim 2j in its low half and 2j + 1 in its high half), then the scales, [token][8] in the K
cache and [8][token] in the V cache.
Quantisation: scale = the nearest representable to amax / 6 (ties to even, at most 10240, so that
6 * scale is an fp16 number), code = the nearest e2m1 to x / scale (ties to the even code,
magnitudes above 6 become 6); a zero scale has zero codes.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

D = 128
GROUP = 16          # tokens of a cache group
GROUP_BYTES = 1152  # 16 x (64 code bytes + 8 scale bytes)
BYTES_PER_ROW = 72  # K or V of one token and kv head

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # The next token of 256 running requests: launch latency.
        dict(name="plan_decode_256", kind="plan", seqs=256, low=16, high=8192, new_low=1,
             new_high=1, idle=0.0, block_size=16, max_blocks=544, max_tokens=256),
        # Prompts admitted beside running requests, some requests leaving.
        dict(name="plan_admit_64", kind="plan", seqs=64, low=16, high=4096, new_low=16,
             new_high=8192, idle=0.6, block_size=16, max_blocks=1024, max_tokens=65536),
        # q and k of one decode step, 64 requests.
        dict(name="rope_step_64", kind="rope", tokens=64, heads=32, kv_heads=8, dtype="bf16",
             rot=128, interleaved=False, norm=True),
        # q and k of a batch of prompts.
        dict(name="rope_prompts_16384", kind="rope", tokens=16384, heads=32, kv_heads=8,
             dtype="bf16", rot=128, interleaved=False, norm=True),
        # An odd token count, neighbouring pairs rotated, half of the head rotated.
        dict(name="rope_partial_4099", kind="rope", tokens=4099, heads=28, kv_heads=4,
             dtype="fp16", rot=64, interleaved=True, norm=True),
        # One prompt chunk: q rotated, K and V quantised into the cache, read back for the
        # chunk's own attention.
        dict(name="fused_chunk_2048", kind="fused", tokens=2048, heads=28, kv_heads=4,
             dtype="bf16", rot=128, interleaved=False, block_size=16, runs=True),
        # New rows of 256 requests at scattered slots.
        dict(name="write_rows_256", kind="write", tokens=256, kv_heads=4, dtype="bf16",
             block_size=16, runs=False),
        # The prompts of 64 requests of 8192 tokens, and all their rows read back.
        dict(name="write_prompts_64x8192", kind="write", tokens=64 * 8192, kv_heads=2,
             dtype="fp16", block_size=16, runs=True),
        # A step of four short requests: latency.
        dict(name="step_4_short", kind="step", seqs=4, heads=12, kv_heads=2, low=64, high=512,
             shape="uniform", dtype="fp16", block_size=16, splitk=False),
        # 64 requests at 8192 tokens.
        dict(name="decode_64x8192", kind="decode", seqs=64, heads=12, kv_heads=2, low=8192,
             high=8192, shape="uniform", dtype="fp16", block_size=16, splitk=False),
        # A ragged serving batch with a long tail of lengths, bf16 activations.
        dict(name="decode_ragged_256", kind="decode", seqs=256, heads=28, kv_heads=4, low=16,
             high=16384, shape="lognormal", dtype="bf16", block_size=16, splitk=False),
        # Few requests, very long contexts.
        dict(name="decode_long_8", kind="decode", seqs=8, heads=64, kv_heads=8, low=65536,
             high=131072, shape="uniform", dtype="fp16", block_size=16, splitk=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "fused", "write", "step", "decode", "decode"])
    bs = rng.choice([16, 16, 32, 64, 128])
    if kind == "plan":
        seqs = _log(rng, 1, 512)
        high = _log(rng, 16, 8192)
        new_high = rng.choice([1, 1, _log(rng, 2, 8192)])
        return dict(kind=kind, seqs=seqs, low=rng.choice([0, 1, min(high, 16)]), high=high,
                    new_low=rng.choice([0, 1]), new_high=new_high,
                    idle=round(rng.uniform(0, 0.8), 2), block_size=bs,
                    max_blocks=(high + new_high) // bs + 1 + rng.randrange(32),
                    max_tokens=_log(rng, max(seqs, min(1024, seqs * new_high) // 2),
                                    max(1024, seqs * new_high // 3)))
    heads, kv_heads = rng.choice([(12, 2), (28, 4), (32, 8), (64, 8), (8, 8), (8, 1), (32, 2),
                                  (20, 1)])
    if kind == "rope":
        return dict(kind=kind, tokens=_log(rng, 1, 16384 * 40 // (heads + kv_heads) // 2),
                    heads=heads, kv_heads=kv_heads, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    rot=rng.choice([128, 128, 64, 96, 32]),
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.85)
    if kind == "fused":
        return dict(kind=kind, tokens=_log(rng, 1, 8192 // kv_heads), heads=heads,
                    kv_heads=kv_heads, dtype=rng.choice(["fp16", "bf16"]),
                    rot=rng.choice([128, 128, 64]), interleaved=rng.random() < 0.3,
                    block_size=bs, runs=rng.random() < 0.6)
    if kind == "write":
        return dict(kind=kind, tokens=_log(rng, 1, 1048576 // kv_heads), kv_heads=kv_heads,
                    dtype=rng.choice(["fp16", "bf16"]), block_size=bs,
                    runs=rng.random() < 0.7)
    shape = rng.choice(["uniform", "lognormal"])
    seqs = _log(rng, 1, 256)
    high = _log(rng, 16, max(16, min(131072, 8 * 131072 * 8 // (2 * seqs * kv_heads))))
    return dict(kind=kind, seqs=seqs, heads=heads, kv_heads=kv_heads,
                low=rng.choice([1, max(1, high // 2), high]), high=high, shape=shape,
                dtype="fp16" if kind == "step" else rng.choice(["fp16", "bf16"]), block_size=bs,
                splitk=rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case, rng, n):
    lo, hi = case["low"], case["high"]
    if case.get("shape") == "lognormal":
        return np.clip(np.exp(rng.normal(math.log(max(1, hi // 8)), 1.0, n)), lo, hi).astype(
            np.int32)
    return rng.integers(lo, hi + 1, n).astype(np.int32)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _kv_values(g, rows):
    """K or V rows as a model gives them: each row with its own magnitude, and one channel in
    a hundred 20 times larger."""
    x = _randn(g, *rows, D)
    x *= torch.exp(0.5 * _randn(g, *rows, 1))
    x[..., 37] *= 20.0
    return x


def _rope_table(positions, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    ang = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _caches(g, blocks, kv_heads, bs):
    """Filled K and V caches, made a part at a time."""
    out = []
    for is_v in (False, True):
        c = torch.empty(blocks, kv_heads, bs // GROUP, GROUP_BYTES, dtype=torch.uint8,
                        device="cuda")
        flat = c.view(-1, GROUP_BYTES)
        for i in range(0, flat.shape[0], 1 << 16):
            part = flat[i:i + (1 << 16)]
            codes, scales = _quantise(_kv_values(g, (part.shape[0], GROUP)))
            part[:, :1024] = codes.view(-1, 1024)
            part[:, 1024:] = (scales.transpose(1, 2) if is_v else scales).reshape(-1, 128)
        out.append(c)
    return out


def _tables(rng, blocks, lens, bs, width):
    """Block tables of shuffled blocks, and the blocks that are left."""
    row, col = np.nonzero(np.arange(width) < ((lens + bs - 1) // bs)[:, None])
    perm = rng.permutation(blocks).astype(np.int32)
    bt = np.zeros((len(lens), width), np.int32)
    bt[row, col] = perm[:len(row)]
    return bt, perm[len(row):]


def _slots(rng, tokens, bs, runs):
    """`runs`: whole prompts through shuffled blocks; else every token anywhere."""
    blocks = (tokens + bs - 1) // bs + 3
    if runs:
        t = np.arange(tokens)
        return blocks, (rng.permutation(blocks)[t // bs] * bs + t % bs).astype(np.int32)
    return blocks, rng.permutation(blocks * bs)[:tokens].astype(np.int32)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    kind, bs = case["kind"], case.get("block_size", 16)
    s = dict(case=case, bs=bs)
    if kind == "plan":
        n = case["seqs"]
        lens = _lengths(case, rng, n)
        new = np.exp(rng.uniform(math.log(max(1, case["new_low"])),
                                 math.log(case["new_high"] + 0.999), n)).astype(np.int32)
        new = np.clip(new, case["new_low"], case["new_high"])
        what = rng.random(n)
        done = what < case["idle"] / 4                       # requests that leave
        start = (what >= case["idle"] / 4) & (what < case["idle"])  # requests that come
        if case["idle"] > 0:  # the others go on by a token
            new = np.where(start, new, 1)
        lens = np.where(start, 0, lens).astype(np.int32)
        new = np.where(done, 0, new).astype(np.int32)
        # The step's token budget: later requests get what is left of it.
        before = np.cumsum(new.astype(np.int64)) - new
        new = np.minimum(new, np.clip(case["max_tokens"] - before, 0, None)).astype(np.int32)
        blocks = n * case["max_blocks"] + 1
        table, left = _tables(rng, blocks, lens, bs, case["max_blocks"])
        free = np.zeros(blocks, np.int32)
        free[:len(left)] = left
        s.update(blocks=blocks, table=_cuda(table), lens=_cuda(lens), new=_cuda(new),
                 done=_cuda(done.astype(np.int32)), free=_cuda(free),
                 count=_cuda(np.array([len(left)], np.int32)),
                 max_tokens=case["max_tokens"])
        return s
    dt = DTYPES[case["dtype"]]
    if kind in ("rope", "fused"):
        n, H, KVH = case["tokens"], case["heads"], case["kv_heads"]
        far = 32768
        qkv = _randn(g, n, H + 2 * KVH, D).to(dt)  # one projection's output; q, k, v are views
        s.update(q=qkv[:, :H], k=qkv[:, H:H + KVH], v=qkv[:, H + KVH:],
                 qw=(1 + 0.1 * _randn(g, D)).to(dt), kw=(1 + 0.1 * _randn(g, D)).to(dt),
                 pos=_cuda(rng.integers(0, far, n).astype(np.int32)),
                 table=_rope_table(far, case["rot"]), eps=1e-6)
        if not case.get("norm", True):
            s.update(qw=None, kw=None)
        if kind == "rope":
            return s
        blocks, slots = _slots(rng, n, bs, case["runs"])
    elif kind == "write":
        n, KVH = case["tokens"], case["kv_heads"]
        s.update(k=_kv_values(g, (n, KVH)).to(dt), v=_kv_values(g, (n, KVH)).to(dt))
        blocks, slots = _slots(rng, n, bs, case["runs"])
    if kind in ("fused", "write"):
        s.update(slots=_cuda(slots))
        s["kc"], s["vc"] = (torch.zeros(blocks, KVH, bs // GROUP, GROUP_BYTES, dtype=torch.uint8,
                                        device="cuda") for _ in range(2))
        return s
    H, KVH = case["heads"], case["kv_heads"]
    lens = _lengths(case, rng, case["seqs"])
    need = (lens + bs - 1) // bs
    blocks = int(need.sum()) + 1
    bt, _ = _tables(rng, blocks, lens, bs, int(need.max()))
    s["kc"], s["vc"] = _caches(g, blocks, KVH, bs)
    s.update(q=_randn(g, case["seqs"], H, D).to(dt), bt=_cuda(bt), lens=_cuda(lens),
             host_lens=torch.from_numpy(lens), scale=1.0 / math.sqrt(D))
    if kind == "step":
        last = lens.astype(np.int64) - 1
        s.update(k=_kv_values(g, (case["seqs"], KVH)).to(dt),
                 v=_kv_values(g, (case["seqs"], KVH)).to(dt),
                 slots=_cuda((bt[np.arange(len(lens)), last // bs] * bs + last % bs).astype(
                     np.int32)))
    return s


# ---------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------
def _e2m1():
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    return torch.cat([v, -v])


def _scale_value(b):
    """uint8 scale bytes as fp32: the byte, seven places up, is an fp16 pattern."""
    return (b.to(torch.int16) << 7).view(torch.float16).float()


def _quantise(x):
    """Code bytes [..., 64] and scale bytes [..., 8] of rows x [..., 128] (fp32)."""
    x = x.reshape(*x.shape[:-1], 8, 16)
    t = x.abs().amax(-1).double() / 6
    # t = m * 2^e, m in [0.5, 1): four significant bits are steps of 2^(e-4); below 2^-14 the
    # steps stay 2^-17.
    e = torch.where(t > 0, torch.frexp(t)[1], -13).clamp(min=-13)
    byte = torch.round(t / torch.exp2((e - 4).double())) + 8 * (e + 13)
    byte = byte.clamp(max=(28 << 3) + 2)  # 10240 = 1.25 * 2^13
    scales = byte.to(torch.uint8)
    s = _scale_value(scales).double()[..., None]
    y = torch.where(s > 0, x.abs().double() / s, torch.zeros_like(s))
    # Codes by how many of the borders between neighbours y has passed; a border itself goes to
    # the even code of the two.
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75).to(torch.uint8) + (y > 1.25).to(torch.uint8) +
            (y >= 1.75).to(torch.uint8) + (y > 2.5).to(torch.uint8) + (y >= 3.5).to(torch.uint8) +
            (y > 5).to(torch.uint8))
    code = (code | ((x < 0) & (s > 0)).to(torch.uint8) << 3).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def _values(codes, scales):
    """fp32 rows [..., 128] of code bytes [..., 64] and scale bytes [..., 8]."""
    pair = torch.arange(256, device="cuda")
    lut = torch.stack([_e2m1()[pair & 15], _e2m1()[pair >> 4]], 1)
    x = lut.index_select(0, codes.reshape(-1).int()).view(*codes.shape[:-1], 8, 16)
    return x.mul_(_scale_value(scales)[..., None]).flatten(-2)


def _parts(cache, is_v):
    """Views of a cache's code bytes [..., 16 tokens, 64] and scale bytes [..., 16 tokens, 8]."""
    lead = cache.shape[:-1]
    codes = cache[..., :1024].unflatten(-1, (16, 64))
    scales = cache[..., 1024:].unflatten(-1, (8, 16) if is_v else (16, 8))
    assert codes.shape[:-2] == lead
    return codes, scales.transpose(-1, -2) if is_v else scales


def _put(cache, is_v, rows, slots, bs):
    codes, scales = _parts(cache, is_v)
    c, sc = _quantise(rows.float())
    blk, grp, t = slots // bs, slots % bs // GROUP, slots % GROUP
    codes[blk, :, grp, t] = c
    scales[blk, :, grp, t] = sc


def _get(cache, is_v, slots, bs, dt):
    codes, scales = _parts(cache, is_v)
    blk, grp, t = slots // bs, slots % bs // GROUP, slots % GROUP
    return _values(codes[blk, :, grp, t], scales[blk, :, grp, t]).to(dt)


def _norm_rope(x, w, pos, table, eps, interleaved):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()
    half = table.shape[1] // 2
    cs = table[pos.long()]
    c, sn = cs[:, None, :half], cs[:, None, half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _attend(q, kc, vc, bt, lens, scale):
    """softmax(scale q k) v over each sequence's pages, padded to the longest."""
    B, H, _ = q.shape
    KVH = kc.shape[1]

    def rows(cache, is_v):
        page = cache[bt.long()].transpose(1, 2)          # [B, KVH, pages, groups, bytes]
        codes, scales = _parts(page, is_v)
        return _values(codes.reshape(B, KVH, -1, 64), scales.reshape(B, KVH, -1, 8))

    k = rows(kc, False)
    x = torch.matmul(q.float().view(B, KVH, H // KVH, D), k.transpose(-1, -2)) * scale
    del k
    past = torch.arange(x.shape[-1], device="cuda") >= lens[:, None]
    x = x.masked_fill(past[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    v = rows(vc, True)
    return torch.matmul(x, v).view(B, H, D)


def _plan(s):
    bs, table, free = s["bs"], s["table"], s["free"]
    lens, new, done = s["lens"].long(), s["new"].long(), s["done"].bool()
    n, width = table.shape
    F = s["count"].long()
    dump = free.shape[0]
    # Blocks of the requests that leave go on top of the free stack, in sequence order.
    back = torch.where(done, (lens + bs - 1) // bs, torch.zeros_like(lens))
    at = F + torch.cumsum(back, 0) - back
    j = torch.arange(width, device="cuda")
    to = torch.where(j < back[:, None], at[:, None] + j, torch.full_like(at[:, None], dump))
    padded = torch.cat([free, free.new_zeros(1)])
    padded.scatter_(0, to.flatten(), table.flatten())
    free.copy_(padded[:-1])
    F = F + back.sum()
    lens = torch.where(done, torch.zeros_like(lens), lens)
    # New blocks from the top of the stack, in sequence order.
    had = (lens + bs - 1) // bs
    need = (lens + new + bs - 1) // bs - had
    first = torch.cumsum(need, 0) - need
    ends = torch.cumsum(new, 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    tok = torch.arange(s["max_tokens"], device="cuda")
    live = tok < ends[-1]
    seq = torch.searchsorted(ends, tok, right=True).clamp(max=n - 1)
    pos = torch.where(live, lens[seq] + tok - starts[seq], torch.zeros_like(tok))
    col = pos // bs
    fresh = live & (col >= had[seq])
    popped = free[(F - 1 - first[seq] - (col - had[seq])).clamp(0, dump - 1)]
    blk = torch.where(fresh, popped, table[seq, col])
    flat = torch.cat([table.flatten(), table.new_zeros(1)])
    flat.scatter_(0, torch.where(fresh, seq * width + col, torch.full_like(tok, n * width)), blk)
    table.copy_(flat[:-1].view(n, width))
    minus = torch.full_like(tok, -1)
    return dict(slots=torch.where(live, blk * bs + pos % bs, minus).int(),
                positions=torch.where(live, pos, minus).int(), query_start=starts.int(),
                lens=(lens + new).int(), count=(F - need.sum()).int(), table=table, free=free)


def _run_plain(s):
    case, kind, bs = s["case"], s["case"]["kind"], s["bs"]
    if kind == "plan":
        return _plan(s)
    if kind in ("rope", "fused"):
        dt, il = s["q"].dtype, case["interleaved"]
        q = _norm_rope(s["q"], s["qw"], s["pos"], s["table"], s["eps"], il).to(dt)
        k = _norm_rope(s["k"], s["kw"], s["pos"], s["table"], s["eps"], il).to(dt)
        if kind == "rope":
            return dict(q=q, k=k)
    if kind in ("fused", "write", "step"):
        k = k if kind == "fused" else s["k"]
        slots = s["slots"].long()
        _put(s["kc"], False, k, slots, bs)
        _put(s["vc"], True, s["v"], slots, bs)
        out = dict(k=_get(s["kc"], False, slots, bs, k.dtype),
                   v=_get(s["vc"], True, slots, bs, k.dtype))
        if kind == "write":
            return out
        if kind == "fused":
            return dict(out, q=q)
    o = _attend(s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["scale"]).to(s["q"].dtype)
    return dict(out, out=o) if kind == "step" else dict(out=o)


# ---------------------------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------------------------
def _ops():
    here = os.path.join(os.getcwd(), "cuda-pa-int8_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from pa_b200 import ops
    return ops


def _run_own(s):
    ops = _ops()
    case, kind, bs = s["case"], s["case"]["kind"], s["bs"]
    if kind == "plan":
        lens, count = ops.release_blocks(s["table"], s["lens"], s["done"], s["free"], s["count"],
                                         bs)
        slots, positions, starts, lens, count = ops.extend_block_tables(
            s["table"], lens, s["new"], s["free"], count, s["blocks"], bs,
            max_tokens=s["max_tokens"])
        return dict(slots=slots, positions=positions, query_start=starts, lens=lens, count=count,
                    table=s["table"], free=s["free"])
    if kind == "rope":
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["pos"], s["table"],
                                eps=s["eps"], interleaved=case["interleaved"])
        return dict(q=q, k=k)
    if kind == "fused":
        q = ops.norm_rope_into_cache(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["pos"],
                                     s["table"], s["kc"], s["vc"], s["slots"], bs, eps=s["eps"],
                                     interleaved=case["interleaved"])
        k, v = ops.read_from_cache_fp4(s["kc"], s["vc"], s["slots"], bs, dtype=q.dtype)
        return dict(q=q, k=k, v=v)
    if kind == "write":
        ops.quantize_into_cache_fp4(s["k"], s["v"], s["kc"], s["vc"], s["slots"], bs)
        k, v = ops.read_from_cache_fp4(s["kc"], s["vc"], s["slots"], bs, dtype=s["k"].dtype)
        return dict(k=k, v=v)
    out = torch.empty_like(s["q"])
    if kind == "step":
        ops.decode_step(out, s["q"], s["k"], s["v"], s["kc"], s["vc"], s["bt"], s["lens"],
                        s["scale"], bs, splitk=case["splitk"], host_context_lens=s["host_lens"])
        k, v = ops.read_from_cache_fp4(s["kc"], s["vc"], s["slots"], bs, dtype=out.dtype)
        return dict(out=out, k=k, v=v)
    if out.dtype == torch.bfloat16:
        ops.decode_bf16(out, s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["scale"], bs,
                        splitk=case["splitk"], validate=False)
    else:
        ops.decode(out, s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["scale"], bs,
                   splitk=case["splitk"], host_context_lens=s["host_lens"])
    return dict(out=out)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    kind, bs = case["kind"], case.get("block_size", 16)
    if kind == "plan":
        n = case["seqs"]
        mean = (case["new_low"] + case["new_high"]) / 2 if case["idle"] == 0 else (
            0.75 * case["idle"] * (case["new_high"] - case["new_low"]) /
            math.log(max(1.01, case["new_high"] / max(1, case["new_low"]))) + 1 - case["idle"])
        tokens = min(case["max_tokens"], n * max(1.0, mean))
        # Per token a slot and a position; per new block its id read and written; per sequence
        # two lengths and a flag read, a length and a start written.
        return dict(bytes=8 * tokens + 8 * tokens / bs + 20 * n, flops=10 * tokens)
    size = 4 if case["dtype"] == "fp32" else 2
    if kind in ("rope", "fused"):
        n, H, KVH, rot = case["tokens"], case["heads"], case["kv_heads"], case["rot"]
        rows = n * (H + KVH)
        b = 2 * rows * D * size + n * 4 + n * rot * 4 + 2 * D * size
        f = rows * (5 * D + 3 * rot)
        if kind == "rope":
            return dict(bytes=b, flops=f)
        # K and V as 72-byte rows instead of K rows, V read, and both read back.
        b += n * 4 + n * KVH * (D * size - D * size + 2 * BYTES_PER_ROW)
        return dict(bytes=b + n * KVH * 2 * (BYTES_PER_ROW + D * size),
                    flops=f + n * KVH * 2 * 4 * D)
    if kind == "write":
        rows = case["tokens"] * case["kv_heads"]
        return dict(bytes=case["tokens"] * 4 + rows * 4 * (BYTES_PER_ROW + D * size),
                    flops=rows * 2 * 6 * D)
    H, KVH, n = case["heads"], case["kv_heads"], case["seqs"]
    if case["shape"] == "lognormal":
        mid, hi = max(1, case["high"] // 8), case["high"]
        z = np.linspace(-4, 4, 4001)
        w = np.exp(-z * z / 2)
        mean = float((np.clip(mid * np.exp(z), case["low"], hi) * w).sum() / w.sum())
    else:
        mean = (case["low"] + case["high"]) / 2
    tokens = n * mean
    b = tokens * KVH * 2 * BYTES_PER_ROW + 2 * n * H * D * size + tokens / bs * 4 + 4 * n
    if kind == "step":
        b += n * KVH * 2 * (2 * BYTES_PER_ROW + 2 * D * size)
    return dict(bytes=b, flops=4 * tokens * H * D)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _x_scales():
    b = np.arange(0, (28 << 3) + 3)
    e, m = b >> 3, b & 7
    return torch.from_numpy(np.where(e == 0, m * 2.0 ** -17, (8 + m) * 2.0 ** (e - 18.0))).cuda()


def _x_nearest(t, grid):
    """Index of the nearest of `grid` (ascending) to each of t; a tie goes to the even index."""
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.searchsorted(mid, t, right=False), torch.searchsorted(mid, t, right=True)
    return torch.where((lo != hi) & (lo % 2 != 0), hi, lo)


def _x_quantised(x):
    """The values that rows x [..., 128] (fp64) are held as."""
    grid = _x_scales()
    mags = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    x = x.unflatten(-1, (8, 16))
    s = grid[_x_nearest((x.abs().amax(-1) / 6).contiguous(), grid)][..., None]
    y = torch.where(s > 0, x.abs() / s, 0.0)
    return (mags[_x_nearest(y.contiguous(), mags)] * s * torch.sign(x)).flatten(-2)


def _x_held(cache, is_v):
    """The values a cache holds, fp64 [blocks, kv_heads, block_size, 128]."""
    n, h, g, _ = cache.shape
    b = cache.view(n, h, g, GROUP_BYTES).long()
    nib = torch.stack([b[..., :1024] % 16, b[..., :1024] // 16], -1).view(n, h, g, 16, 128)
    mags = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    val = mags[nib % 8] * (1 - 2 * (nib // 8)).double()
    sc = b[..., 1024:].view(n, h, g, 8, 16).transpose(-1, -2) if is_v else (
        b[..., 1024:].view(n, h, g, 16, 8))
    e, m = sc // 8, (sc % 8).double()
    sv = torch.where(e == 0, m * 2.0 ** -17, (8 + m) * torch.exp2(e.double() - 18))
    return (val.view(n, h, g, 16, 8, 16) * sv[..., None]).reshape(n, h, g * 16, 128)


def _x_turned(x, w, pos, table, eps, interleaved):
    x = x.double()
    if w is not None:
        x = w.double() * x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + eps)
    rot = table.shape[1]
    i = torch.arange(rot // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    z = torch.complex(x[..., a], x[..., b]) * torch.complex(
        table[pos.long(), :rot // 2].double(), table[pos.long(), rot // 2:].double())[:, None]
    y = x.clone()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":  # whole numbers
        return None
    s = prepare(case, seed)
    bs = s["bs"]
    if kind in ("rope", "fused"):
        q, k = (_x_turned(s[n], s[n + "w"], s["pos"], s["table"], s["eps"], case["interleaved"])
                for n in "qk")
        if kind == "rope":
            return dict(q=q, k=k)
        # K is rounded to the activations' type before it is quantised.
        return dict(q=q, k=_x_quantised(k.to(s["q"].dtype).double()),
                    v=_x_quantised(s["v"].double()))
    out = {}
    if kind in ("write", "step"):
        out = dict(k=torch.empty(s["k"].shape, dtype=torch.float64, device="cuda"))
        out["v"] = torch.empty_like(out["k"])
        for n in "kv":
            for i in range(0, s[n].shape[0], 1 << 16):
                out[n][i:i + (1 << 16)] = _x_quantised(s[n][i:i + (1 << 16)].double())
        if kind == "write":
            return out
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    KVH = case["kv_heads"]
    for i, n in enumerate(s["host_lens"].tolist()):
        page = s["bt"][i, :(n + bs - 1) // bs].long()
        k = _x_held(s["kc"][page], False).transpose(0, 1).reshape(KVH, -1, D)[:, :n]
        v = _x_held(s["vc"][page], True).transpose(0, 1).reshape(KVH, -1, D)[:, :n]
        if kind == "step":  # the last token is the new one
            k, v = k.clone(), v.clone()
            k[:, n - 1], v[:, n - 1] = out["k"][i], out["v"][i]
        q = s["q"][i].double().view(KVH, -1, D)
        p = torch.softmax(q @ k.transpose(1, 2) * s["scale"], -1)
        o[i] = (p @ v).view(-1, D)
    return dict(out, out=o)
