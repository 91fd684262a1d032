"""Torch-facing wrappers of the C ABI.

Each op checks its arguments with the error conditions of the reference launchers
(kernels/paged_attention_v4_splitk.cu:197-205, kernels/paged_attention_v6_splitk_int8.cu:
201-221 and siblings) and raises RuntimeError like their TORCH_CHECKs, then calls the
library on the current CUDA stream of the tensors' device. Temporaries of the decodes (split
partials, arrival counters, their status word) live in a per-(device, stream) workspace that is
zero-filled once when allocated and kept for later calls; the other kernels set the library's own
status word of the device.
"""

import ctypes

import torch

from . import _lib

HEAD_DIM = 128
X = 8

_DTYPE_CODE = {
    torch.float16: _lib.PA_DTYPE_F16,
    torch.bfloat16: _lib.PA_DTYPE_BF16,
    torch.float32: _lib.PA_DTYPE_F32,
}

_workspaces = {}
_outgrown = []      # (key, workspace) replaced inside a capture, where its status cannot be carried
_status_words = {}  # device index -> address of the library's status word there


def _ptr(t):
    return t.data_ptr() if t is not None else None


# The current stream's handle without building a Stream object, which costs 2 us a call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def workspace(device, nbytes):
    """The zero-initialised workspace of (device, current stream), grown to nbytes.

    Growing replaces the buffer, and a CUDA graph keeps the address it captured: run the
    largest shape once on a stream before capturing graphs on it, so no later call on that
    stream replaces the buffer a graph uses. The status word moves along with a grown
    workspace, so bits that were set and not read yet stay."""
    stream = _stream(device)
    key = (device.index, stream)
    ws = _workspaces.get(key)
    nbytes = max(int(nbytes), 256)
    if ws is None or ws.numel() < nbytes:
        old = ws
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        if old is not None:
            if torch.cuda.is_current_stream_capturing():
                _outgrown.append((key, old))  # a captured copy would run again in every replay
            else:
                ws[:4].copy_(old[:4])
        _workspaces[key] = ws
    return ws


def _status_word(device):
    """Address of the library's own status word on `device`, the current one: for the kernels that
    use nothing else of a workspace. It never moves, so graphs may hold it."""
    p = _status_words.get(device.index)
    if p is None:
        out = ctypes.c_void_p()
        _lib.check(_lib.lib().pa_device_status(ctypes.byref(out)), "pa_device_status")
        p = _status_words[device.index] = out.value
    return p


def read_status(device=None):
    """OR of this device's status words (the library's own and those of its workspaces), which are
    then cleared. Waits for all work on the device first. Bits are the PA_ERR_* codes of
    include/pa_b200.h. A workspace that reports an error also gets its arrival counters zeroed,
    since a kernel that stopped part-way can leave some of them set."""
    if device is None or device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    status = 0
    L = _lib.lib()
    with _Guard(device):
        # A graph runs on another stream than the one it was captured on, whose key its
        # workspace has.
        torch.cuda.synchronize(device)

        def read(address, stream):
            out = ctypes.c_int(0)
            _lib.check(L.pa_read_status(address, ctypes.byref(out), stream), "pa_read_status")
            return out.value

        word = _status_words.get(device.index)
        if word is not None:
            status |= read(word, _stream(device))
        for (idx, stream), ws in list(_workspaces.items()) + _outgrown:
            if idx != device.index:
                continue
            bits = read(ws.data_ptr(), stream)
            if bits:
                _lib.check(L.pa_reset_workspace(ws.data_ptr(), ws.numel(), stream),
                           "pa_reset_workspace")
                torch.cuda.synchronize(device)
            status |= bits
    return status


def check_status(device=None):
    """Raise RuntimeError if a kernel on `device` recorded an error since the last check."""
    status = read_status(device)
    if status:
        raise RuntimeError("paged-attention kernel reported: " +
                           _lib.lib().pa_status_string(status).decode() + f" (status {status})")


class _Guard:
    """Make `device` current for the duration of a call (no-op when it already is)."""

    def __init__(self, device):
        self.device = device
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.device.index:
            self.prev = cur
            torch.cuda.set_device(self.device)
        return self

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


def _require(cond, msg):
    if not cond:
        raise RuntimeError(msg)


_FP8 = getattr(torch, "float8_e4m3fn", None)
FP4_GROUP_TOKENS = 16    # tokens of a group of the 4-bit cache
FP4_GROUP_BYTES = 1152   # its codes (16 x 64 bytes) and scales (16 x 8)


def _kv_kind(k_cache, k_scales):
    """'f4' for a 4-bit cache (uint8), 'f8' for an fp8 e4m3 cache, 'i8' for int8 (or whenever
    scales are given), else 'f16'."""
    if k_cache.dtype == torch.uint8:
        return "f4"
    if _FP8 is not None and k_cache.dtype == _FP8:
        return "f8"
    return "i8" if (k_scales is not None or k_cache.dtype == torch.int8) else "f16"


_KV_CODE = {"f16": _lib.PA_DTYPE_F16, "i8": _lib.PA_DTYPE_I8, "f8": _lib.PA_DTYPE_FP8E4M3,
            "f4": _lib.PA_DTYPE_FP4E2M1}


def _check_lengths(context_lens, capacity, host_context_lens=None):
    """The reference's context_lens >= 1 check (and this library's upper bound). It reads
    host_context_lens, a CPU copy of the lengths, when the caller has one (no
    synchronisation); otherwise one device-to-host copy of context_lens, which synchronises
    the current stream."""
    if host_context_lens is not None:
        _require(host_context_lens.device.type == "cpu" and
                 host_context_lens.numel() == context_lens.numel(),
                 "host_context_lens must be a CPU tensor with one length per sequence")
        cl = host_context_lens
    else:
        cl = context_lens.cpu()
    if cl.numel() == 0:
        return
    if cl.dim() == 1 and cl.numel() <= 32:  # for 4 lengths 1.2 us; numpy's reductions 3.4
        v = cl.tolist()
        low, high = min(v), max(v)
    else:
        a = cl.numpy()  # a view: numpy's reductions cost less per call than torch's on the CPU
        low, high = int(a.min()), int(a.max())
    _require(low >= 1, "context_lens must be >= 1 (empty sequences unsupported)")
    _require(high <= capacity, "context_lens exceeds max_blocks_per_seq * block_size")


def _check_fp4_caches(k_cache, v_cache, block_size):
    """(num_blocks, kv_heads) of 4-bit caches [num_blocks, kv_heads, block_size/16, 1152]."""
    shape = k_cache.shape
    if not (k_cache.dtype == torch.uint8 and v_cache.dtype == torch.uint8 and
            v_cache.shape == shape and len(shape) == 4 and shape[3] == FP4_GROUP_BYTES and
            shape[2] * FP4_GROUP_TOKENS == block_size):
        raise RuntimeError(
            f"a 4-bit cache is uint8 [num_blocks, kv_heads, block_size/16, {FP4_GROUP_BYTES}], K "
            f"and V alike; got {k_cache.dtype} {tuple(shape)} and {v_cache.dtype} "
            f"{tuple(v_cache.shape)} for block_size {block_size}")
    return shape[0], shape[1]


def _check_decode_args_fp4(out, q, k_cache, v_cache, block_table, context_lens, block_size,
                           k_scales, v_scales, act_dtype):
    """_check_decode_args over a 4-bit cache."""
    dev, shape = q.device, q.shape
    if not (q.is_cuda and q.dtype == act_dtype and len(shape) == 3 and shape[2] == HEAD_DIM and
            q.is_contiguous()):
        raise RuntimeError(f"q must be contiguous {act_dtype} [num_seqs, num_heads, {HEAD_DIM}] on "
                           "CUDA")
    if out is not None and not (out.dtype == act_dtype and out.device == dev and
                                out.shape == shape and out.is_contiguous()):
        raise RuntimeError("out must have the type and shape of q and be contiguous")
    if block_size <= 0 or 128 % block_size != 0:
        raise RuntimeError("block_size must divide TILE (multiple of 16)")
    NB, KVH = _check_fp4_caches(k_cache, v_cache, block_size)
    _check_on(dev, k_cache, v_cache)
    if k_scales is not None or v_scales is not None:
        raise RuntimeError("a 4-bit cache holds its own scales")
    B, H, D = shape
    if KVH == 0 or H % KVH != 0:
        raise RuntimeError("num_heads must be a multiple of num_kv_heads")
    if not (block_table.dtype == torch.int32 and block_table.device == dev and
            block_table.dim() == 2 and block_table.shape[0] == B and block_table.is_contiguous()):
        raise RuntimeError("block_table must be contiguous int32 [num_seqs, max_blocks_per_seq] on "
                           "q's device")
    if not (context_lens.dtype == torch.int32 and context_lens.device == dev and
            context_lens.dim() == 1 and context_lens.shape[0] == B and
            context_lens.is_contiguous()):
        raise RuntimeError("context_lens must be contiguous int32 [num_seqs] on q's device")
    return B, H, KVH, D, NB


def _check_decode_args(out, q, k_cache, v_cache, block_table, context_lens, block_size,
                       kind, k_scales, v_scales, act_dtype=torch.float16):
    if kind == "f4":
        return _check_decode_args_fp4(out, q, k_cache, v_cache, block_table, context_lens,
                                      block_size, k_scales, v_scales, act_dtype)
    scaled = kind != "f16"  # one-byte cache with per-token scales (int8 or fp8)
    _require(q.is_cuda and (out is None or out.is_cuda), "tensors must be on CUDA")
    act_name = "fp16" if act_dtype == torch.float16 else "bf16"
    _require(q.dtype == act_dtype, f"q must be {act_name}")
    if kind == "f8":
        _require(k_cache.dtype == _FP8, "k_cache must be float8_e4m3fn")
        _require(v_cache.dtype == _FP8, "v_cache must be float8_e4m3fn")
    if kind == "i8":
        _require(k_cache.dtype == torch.int8, "k_cache must be int8")
        _require(v_cache.dtype == torch.int8, "v_cache must be int8")
    if scaled:
        _require(k_scales is not None and k_scales.dtype == torch.float32,
                 "k_scales must be fp32")
        _require(v_scales is not None and v_scales.dtype == torch.float32,
                 "v_scales must be fp32")
    else:
        _require(k_cache.dtype == torch.float16, "k_cache must be fp16")
        _require(v_cache.dtype == torch.float16, "v_cache must be fp16")
    _require(block_table.dtype == torch.int32, "block_table must be int32")
    _require(context_lens.dtype == torch.int32, "context_lens must be int32")
    dev = q.device
    tensors = [q, k_cache, v_cache, block_table, context_lens]
    if out is not None:
        tensors.append(out)
    if scaled:
        tensors += [k_scales, v_scales]
    for t in tensors:
        _require(t.device == dev, "all tensors must be on the same CUDA device")
        _require(t.is_contiguous(), "all tensors must be contiguous")
    _require(q.dim() == 3, "q must be [num_seqs, num_heads, head_dim]")
    B, H, D = q.shape
    if out is not None:
        _require(tuple(out.shape) == (B, H, D) and out.dtype == act_dtype,
                 f"out must be {act_name} with the shape of q")
    _require(k_cache.dim() == 5,
             "k_cache must be [num_blocks, kv_heads, head_dim/x, block_size, x]")
    NB, KVH, DX, BS, x = k_cache.shape
    if scaled:
        _require(x == 8, "int8 K cache requires x == 8")
    _require(x == X, "K cache requires x == 8")
    _require(D == HEAD_DIM, f"head_dim {D} unsupported (this build: {HEAD_DIM})")
    _require(DX * x == D, "k_cache head_dim/x does not match q")
    _require(block_size % 16 == 0 and 128 % block_size == 0,
             "block_size must divide TILE (multiple of 16)")
    _require(BS == block_size, f"k_cache block dimension {BS} != block_size {block_size}")
    _require(tuple(v_cache.shape) == (NB, KVH, D, block_size),
             "v_cache must be [num_blocks, kv_heads, head_dim, block_size]")
    if scaled:
        _require(tuple(k_scales.shape) == (NB, KVH, block_size) and
                 tuple(v_scales.shape) == (NB, KVH, block_size),
                 "scales must be [num_blocks, kv_heads, block_size]")
    _require(KVH > 0 and H % KVH == 0, "num_heads must be a multiple of num_kv_heads")
    _require(block_table.dim() == 2 and block_table.shape[0] == B,
             "block_table must be [num_seqs, max_blocks_per_seq]")
    _require(context_lens.dim() == 1 and context_lens.shape[0] == B,
             "context_lens must be [num_seqs]")
    return B, H, KVH, D, NB


def decode(out, q, k_cache, v_cache, block_table, context_lens, scale, block_size=16, *,
           k_scales=None, v_scales=None, splitk=False, validate=True, kv_kind=None,
           host_context_lens=None):
    """Paged decode attention into `out` (fp16 [num_seqs, num_heads, head_dim]).

    The cache type follows the tensors: fp16; int8 or float8_e4m3fn, each with per-token fp32
    k_scales/v_scales (an int8 cache is assumed whenever scales are given); uint8 for a 4-bit
    cache (fp4_cache), which holds its own scales. splitk selects the partition + LSE-reduce
    kernel pair (512-token splits); otherwise, and always over a 4-bit cache, the single-pass
    kernel with the fused combine runs. validate=False skips the one host sync that checks
    context_lens (the kernels still flag bad lengths in the status word).
    kv_kind ('f16', 'i8', 'f8' or 'f4') pins the cache type instead of inferring it from the
    tensors, so a cache of another type is rejected (the reference-named ops use this).
    host_context_lens, a CPU tensor holding the same lengths (for instance the pinned copy the
    lengths were uploaded from), moves that check to the host: the call then does not
    synchronise.
    """
    kind = kv_kind or _kv_kind(k_cache, k_scales)
    B, H, KVH, D, NB = _check_decode_args(out, q, k_cache, v_cache, block_table, context_lens,
                                          block_size, kind, k_scales, v_scales)
    if B == 0:
        return out
    L = _lib.lib()
    max_blocks = block_table.shape[1]
    with _Guard(q.device):
        kv = _KV_CODE[kind]
        need = L.pa_decode_workspace_bytes(B, H, KVH, D, max_blocks, block_size, kv,
                                           1 if splitk else 0)
        _require(need > 0, "unsupported decode shape: " + _lib.last_error())
        ws = workspace(q.device, need)
        stream = _stream(q.device)
        if kind in ("i8", "f8"):
            if kind == "f8":
                fn = L.pa_splitk_fp8 if splitk else L.pa_decode_fp8
            else:
                fn = L.pa_splitk_i8 if splitk else L.pa_decode_i8
            args = (out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                    k_scales.data_ptr(), v_scales.data_ptr(), block_table.data_ptr(),
                    context_lens.data_ptr(), B, H, KVH, D, NB, block_size, max_blocks,
                    float(scale), ws.data_ptr(), ws.numel(), stream)
        else:
            if kind == "f4":
                fn = L.pa_splitk_fp4 if splitk else L.pa_decode_fp4
            else:
                fn = L.pa_splitk_f16 if splitk else L.pa_decode_f16
            args = (out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                    block_table.data_ptr(), context_lens.data_ptr(), B, H, KVH, D, NB,
                    block_size, max_blocks, float(scale), ws.data_ptr(), ws.numel(), stream)
        # The one host sync (if any) comes last, so the launch follows it with no Python work
        # between.
        if validate:
            _check_lengths(context_lens, max_blocks * block_size, host_context_lens)
        _lib.check(fn(*args), "paged decode")
    return out


class DecodePlan:
    """decode() for a serving loop: the argument checks run once, at construction.

    Construction takes the same arguments as decode() and validates them the same way; it
    resolves the entry point, the launch sizes and the cache pointers. run() launches the
    decode on the current stream, with the tensors given at construction or, per call, other
    out / q / block_table / context_lens tensors of the same shape, dtype and device (checked
    cheaply; anything else raises RuntimeError). The cache tensors stay those of construction.
    Results are identical to decode()'s. host_context_lens / validate behave as in decode().
    """

    def __init__(self, out, q, k_cache, v_cache, block_table, context_lens, scale, block_size=16,
                 *, k_scales=None, v_scales=None, splitk=False):
        kind = _kv_kind(k_cache, k_scales)
        B, H, KVH, D, NB = _check_decode_args(out, q, k_cache, v_cache, block_table,
                                              context_lens, block_size, kind, k_scales,
                                              v_scales)
        L = _lib.lib()
        self.max_blocks = block_table.shape[1]
        kv = _KV_CODE[kind]
        self.need = L.pa_decode_workspace_bytes(B, H, KVH, D, self.max_blocks, block_size, kv,
                                                1 if splitk else 0)
        _require(B == 0 or self.need > 0, "unsupported decode shape: " + _lib.last_error())
        if kind == "f8":
            self.fn = L.pa_splitk_fp8 if splitk else L.pa_decode_fp8
        elif kind == "i8":
            self.fn = L.pa_splitk_i8 if splitk else L.pa_decode_i8
        elif kind == "f4":
            self.fn = L.pa_splitk_fp4 if splitk else L.pa_decode_fp4
        else:
            self.fn = L.pa_splitk_f16 if splitk else L.pa_decode_f16
        self.scaled = kind in ("i8", "f8")
        self.device = q.device
        self.sizes = (B, H, KVH, D, NB, block_size, self.max_blocks, float(scale))
        self.caches = ((k_cache.data_ptr(), v_cache.data_ptr()) +
                       ((k_scales.data_ptr(), v_scales.data_ptr()) if self.scaled else ()))
        self._keep = (k_cache, v_cache, k_scales, v_scales)  # the cache tensors stay alive
        self.capacity = self.max_blocks * block_size
        self.tensors = [out, q, block_table, context_lens]
        self.specs = [(tuple(t.shape), t.dtype) for t in self.tensors]

    def _match(self, i, t):
        if t is None:
            return self.tensors[i]
        shape, dtype = self.specs[i]
        _require(t.dtype == dtype and tuple(t.shape) == shape and t.device == self.device and
                 t.is_contiguous(),
                 "DecodePlan.run: tensors must match the plan's shapes, dtypes and device")
        return t

    def run(self, out=None, q=None, block_table=None, context_lens=None, *,
            host_context_lens=None, validate=True):
        out, q = self._match(0, out), self._match(1, q)
        block_table, context_lens = self._match(2, block_table), self._match(3, context_lens)
        B, H, KVH, D, NB, bs, mb, scale = self.sizes
        if B == 0:
            return out
        with _Guard(self.device):
            ws = workspace(self.device, self.need)
            ptrs = (out.data_ptr(), q.data_ptr()) + self.caches[:2]
            if self.scaled:
                ptrs += self.caches[2:]
            args = ptrs + (block_table.data_ptr(), context_lens.data_ptr(), B, H, KVH, D, NB,
                           bs, mb, scale, ws.data_ptr(), ws.numel(), _stream(self.device))
            if validate:
                _check_lengths(context_lens, self.capacity, host_context_lens)
            _lib.check(self.fn(*args), "paged decode")
        return out


def decode_step(out, q, new_k, new_v, k_cache, v_cache, block_table, context_lens, scale,
                block_size=16, *, k_scales=None, v_scales=None, k_scale=None, v_scale=None,
                splitk=False, fused=None, validate=True, host_context_lens=None):
    """One decode step: append every sequence's new token to the cache, then decode.

    context_lens already counts the new token: new_k / new_v [num_seqs, kv_heads, head_dim]
    (fp16, bf16 or fp32 rows) go to position context_lens[b] - 1 of sequence b through
    block_table, written like quantize_into_cache (int8 cache, per-token scales or the
    per-tensor k_scale / v_scale), its FP8 and 4-bit counterparts or write_into_cache (fp16
    cache); then the decode of decode() runs over the whole context. This is the bridge's
    PagedKVCache.decode_append + split-K op (benchmarks/int8_bridge/paged_cache.py:132-156,
    qwen_paged_attn.py:61-73) for a whole batch in one call. With fused=True (and at most 16 q
    heads per kv head) the decode kernel writes each token itself just before reading its
    page, so a step is one launch (two with splitk); fused=False runs the write as its own
    kernel first. Both give bit-identical caches and outputs. The default (fused=None) fuses
    small batches (at most 64 sequence x kv-head rows), where the saved launch dominates, and
    writes larger ones first: on a B200 the separate write measured 0.4 % faster at 128 rows
    and 2 % faster at 1024 rows, because the fused write lengthens the warps that carry it.
    Over a 4-bit cache a fused step also checks every page for the new token, which costs more
    than a launch where sequences are few and long: 12/2 heads, fused and separate, 1 x 512
    tokens 12.9 and 13.3 us, 1 x 32768 18.0 and 20.1, 4 x 32768 26.1 and 23.2; 64/8 heads, 8 x
    512 14.4 and 14.4, 8 x 98304 202 and 174. Pass fused=False there.

    With validate=False the call does no host synchronisation and allocates nothing once the
    stream's workspace exists, so after one call on a stream it can be captured in a CUDA
    graph (the kernels still flag bad lengths in the status word). host_context_lens (a CPU
    copy of the lengths) checks them on the host without synchronising, as in decode().
    """
    kind = _kv_kind(k_cache, k_scales)
    B, H, KVH, D, NB = _check_decode_args(out, q, k_cache, v_cache, block_table, context_lens,
                                          block_size, kind, k_scales, v_scales)
    _check_rows(new_k, new_v)
    if fused is None:
        fused = B * KVH <= 64
    _require(tuple(new_k.shape) == (B, KVH, D), "new_k/new_v must be [num_seqs, kv_heads, "
             "head_dim]")
    _require(new_k.device == q.device, "new_k/new_v must be on q's device")
    if k_scale is not None or v_scale is not None:
        _require(kind == "i8" and k_scale is not None and v_scale is not None,
                 "per-tensor scales need an int8 cache and both of k_scale and v_scale")
        for t in (k_scale, v_scale):
            _require(t.dtype == torch.float32 and t.numel() == 1 and t.device == q.device,
                     "fixed scales must be one fp32 element on q's device")
    if B == 0:
        return out
    L = _lib.lib()
    max_blocks = block_table.shape[1]
    with _Guard(q.device):
        kv = _KV_CODE[kind]
        need = L.pa_decode_workspace_bytes(B, H, KVH, D, max_blocks, block_size, kv,
                                           1 if splitk else 0)
        _require(need > 0, "unsupported decode shape: " + _lib.last_error())
        ws = workspace(q.device, need)
        args = (kv, out.data_ptr(), q.data_ptr(), new_k.data_ptr(), new_v.data_ptr(),
                _DTYPE_CODE[new_k.dtype], new_k.stride(0), k_cache.data_ptr(),
                v_cache.data_ptr(), _ptr(k_scales), _ptr(v_scales), _ptr(k_scale),
                _ptr(v_scale), block_table.data_ptr(), context_lens.data_ptr(), B, H, KVH, D, NB,
                block_size, max_blocks, float(scale), 1 if splitk else 0, 1 if fused else 0,
                ws.data_ptr(), ws.numel(), _stream(q.device))
        if validate:
            _check_lengths(context_lens, max_blocks * block_size, host_context_lens)
        _lib.check(L.pa_decode_step(*args), "paged decode step")
    return out


def decode_bf16(out, q, k_cache, v_cache, block_table, context_lens, scale, block_size=16, *,
                k_scales=None, v_scales=None, splitk=False, validate=True):
    """decode() with bf16 activations: q and out are bf16, the cache fp16, per-token INT8,
    per-token FP8 (e4m3) or 4-bit.

    q is converted to fp16 on the device (exact for magnitudes in the fp16 normal range; larger
    values saturate and set the PA_ERR_Q_RANGE status bit), the fp16 decode runs, and its output
    is rounded to bf16. Over a 4-bit cache the decode kernel does both itself: its fp32 result is
    rounded once, to bf16.
    """
    kind = _kv_kind(k_cache, k_scales)
    int8 = kind in ("i8", "f8")
    B, H, KVH, D, NB = _check_decode_args(out, q, k_cache, v_cache, block_table, context_lens,
                                          block_size, kind, k_scales, v_scales,
                                          act_dtype=torch.bfloat16)
    if B == 0:
        return out
    L = _lib.lib()
    max_blocks = block_table.shape[1]
    with _Guard(q.device):
        kv = _KV_CODE[kind]
        need = L.pa_decode_bf16q_workspace_bytes(B, H, KVH, D, max_blocks, block_size, kv,
                                                 1 if splitk else 0)
        _require(need > 0, "unsupported decode shape: " + _lib.last_error())
        ws = workspace(q.device, need)
        if validate:
            _check_lengths(context_lens, max_blocks * block_size)
        rc = L.pa_decode_bf16q(out.data_ptr(), q.data_ptr(), k_cache.data_ptr(),
                               v_cache.data_ptr(), _ptr(k_scales) if int8 else None,
                               _ptr(v_scales) if int8 else None, block_table.data_ptr(),
                               context_lens.data_ptr(), B, H, KVH, D, NB, block_size, max_blocks,
                               kv, 1 if splitk else 0, float(scale), ws.data_ptr(), ws.numel(),
                               _stream(q.device))
        _lib.check(rc, "paged decode (bf16 q)")
    return out


def partial_floats(num_heads, num_kv_heads, head_dim=HEAD_DIM):
    return _lib.lib().pa_partial_floats(num_heads, num_kv_heads, head_dim)


def decode_partial(q, k_cache, v_cache, block_table, context_lens, scale, block_size=16, *,
                   k_scales=None, v_scales=None, partials=None):
    """Un-normalised per-(sequence, kv-head) partials (O, m, l) for this device's token
    ranges: fp32 [num_seqs, num_kv_heads * slot]. Sequences with context 0 give empty
    partials. Used to split one sequence's context across GPUs."""
    kind = _kv_kind(k_cache, k_scales)
    B, H, KVH, D, NB = _check_decode_args(None, q, k_cache, v_cache, block_table, context_lens,
                                          block_size, kind, k_scales, v_scales)
    per = partial_floats(H, KVH, D) * KVH  # floats per sequence: kv_heads x head tiles x slot
    if partials is None:
        partials = torch.empty(B, per, dtype=torch.float32, device=q.device)
    _require(partials.dtype == torch.float32 and partials.is_contiguous() and
             partials.numel() == B * per, "partials must be fp32 [num_seqs, per_seq_floats]")
    if B == 0:
        return partials
    L = _lib.lib()
    max_blocks = block_table.shape[1]
    with _Guard(q.device):
        kv = _KV_CODE[kind]
        need = L.pa_decode_workspace_bytes(B, H, KVH, D, max_blocks, block_size, kv, 0)
        _require(need > 0, "unsupported decode shape: " + _lib.last_error())
        ws = workspace(q.device, need)
        rc = L.pa_decode_partial(kv, partials.data_ptr(), q.data_ptr(), k_cache.data_ptr(),
                                 v_cache.data_ptr(), _ptr(k_scales), _ptr(v_scales),
                                 block_table.data_ptr(), context_lens.data_ptr(), B, H, KVH, D,
                                 NB, block_size, max_blocks, float(scale), ws.data_ptr(),
                                 ws.numel(), _stream(q.device))
        _lib.check(rc, "partial decode")
    return partials


def merge_partials(out, partials, num_heads, num_kv_heads):
    """LSE-merge partials gathered from several GPUs, fp32 [num_parts, num_seqs, ...], into
    out fp16 [num_seqs, num_heads, head_dim]."""
    _require(out.is_cuda and partials.is_cuda, "tensors must be on CUDA")
    _require(partials.dtype == torch.float32 and partials.is_contiguous(),
             "partials must be contiguous fp32")
    P, B = partials.shape[0], partials.shape[1]
    _require(tuple(out.shape) == (B, num_heads, HEAD_DIM) and out.dtype == torch.float16,
             "out must be fp16 [num_seqs, num_heads, head_dim]")
    per = partial_floats(num_heads, num_kv_heads, HEAD_DIM) * num_kv_heads
    _require(per > 0 and partials.numel() == P * B * per,
             "partials must be fp32 [num_parts, num_seqs, per_seq_floats]")
    _require(partials.device == out.device, "partials and out must be on the same device")
    with _Guard(out.device):
        status = _status_word(out.device)
        rc = _lib.lib().pa_merge_partials(out.data_ptr(), partials.data_ptr(), P, B, num_heads,
                                          num_kv_heads, HEAD_DIM, status,
                                          _stream(out.device))
        _lib.check(rc, "merge partials")
    return out


# ---------------------------------------------------------------------------------------
# Cache writes
# ---------------------------------------------------------------------------------------
def _check_cache_layout(k_cache, v_cache, num_kv_heads, head_dim, block_size, k_scales=None,
                        v_scales=None):
    """The paged layout the write kernels address, given the rows' kv-head count and head_dim:
    K [num_blocks, kv_heads, head_dim/8, block_size, 8], V [num_blocks, kv_heads, head_dim,
    block_size], scales [num_blocks, kv_heads, block_size] (tests/paged_decode_attn.py:76-81,
    156-164). The kernels take only num_blocks and block_size, so any other shape would be
    written out of bounds; it is rejected here. Returns num_blocks."""
    _require(k_cache.dim() == 5,
             "k_cache must be [num_blocks, kv_heads, head_dim/x, block_size, x]")
    NB = k_cache.shape[0]
    _require(head_dim % X == 0 and tuple(k_cache.shape) == (NB, num_kv_heads, head_dim // X,
                                                             block_size, X),
             f"k_cache must be [num_blocks, {num_kv_heads}, {head_dim // X}, {block_size}, {X}] "
             f"for these rows; got {tuple(k_cache.shape)}")
    _require(tuple(v_cache.shape) == (NB, num_kv_heads, head_dim, block_size),
             f"v_cache must be [{NB}, {num_kv_heads}, {head_dim}, {block_size}]; "
             f"got {tuple(v_cache.shape)}")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if t is not None:
            _require(tuple(t.shape) == (NB, num_kv_heads, block_size),
                     f"{name} must be [{NB}, {num_kv_heads}, {block_size}]; got {tuple(t.shape)}")
    return NB


def _check_rows(key, value):
    _require(key.is_cuda and value.is_cuda, "tensors must be on CUDA")
    _require(key.dtype in _DTYPE_CODE and value.dtype == key.dtype,
             "key/value must both be fp16, bf16 or fp32")
    _require(key.dim() == 3 and key.shape == value.shape,
             "key/value must be [num_tokens, num_kv_heads, head_dim]")
    _require(key.stride(2) == 1 and key.stride(1) == key.shape[2] and
             value.stride() == key.stride(), "key/value rows must be contiguous")


def quantize_into_cache(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping,
                        block_size=16, *, k_scale=None, v_scale=None):
    """Per-token symmetric INT8 write of key/value [num_tokens, kv_heads, head_dim] into the
    paged cache at slot_mapping (int32, block*block_size+offset; negative = skip).

    Values and scales are bit-identical to quantize_per_token
    (tests/paged_decode_attn.py:106-112). With k_scale/v_scale (one fp32 device scalar each)
    the given per-tensor scale is used instead, as PagedKVCache.decode_append does in
    per-tensor mode (benchmarks/int8_bridge/paged_cache.py:142-145).
    """
    _check_rows(key, value)
    fp8 = _FP8 is not None and k_cache.dtype == _FP8
    if fp8:
        _require(v_cache.dtype == _FP8, "v_cache must be float8_e4m3fn like k_cache")
        _require(k_scale is None and v_scale is None,
                 "the fp8 cache write has per-token scales only")
    else:
        _require(k_cache.dtype == torch.int8 and v_cache.dtype == torch.int8,
                 "cache must be int8")
    _require(k_scales.dtype == torch.float32 and v_scales.dtype == torch.float32,
             "scales must be fp32")
    _require(slot_mapping.dtype == torch.int32 and slot_mapping.is_cuda,
             "slot_mapping must be int32 on CUDA")
    N, KVH, D = key.shape
    _require(slot_mapping.numel() == N, "slot_mapping must have one entry per token")
    _check_cache_layout(k_cache, v_cache, KVH, D, block_size, k_scales, v_scales)
    for t in (k_cache, v_cache, k_scales, v_scales, slot_mapping):
        _require(t.is_contiguous() and t.device == key.device,
                 "cache tensors must be contiguous and on the key's device")
    for t in (k_scale, v_scale):
        if t is not None:
            _require(t.dtype == torch.float32 and t.numel() == 1 and t.device == key.device,
                     "fixed scales must be one fp32 element on the key's device")
    with _Guard(key.device):
        status = _status_word(key.device)
        if fp8:
            rc = _lib.lib().pa_quantize_into_cache_fp8(
                key.data_ptr(), value.data_ptr(), _DTYPE_CODE[key.dtype], key.stride(0),
                slot_mapping.data_ptr(), N, KVH, D, k_cache.data_ptr(), v_cache.data_ptr(),
                k_scales.data_ptr(), v_scales.data_ptr(), k_cache.shape[0], block_size,
                status, _stream(key.device))
            _lib.check(rc, "quantize_into_cache (fp8)")
            return
        rc = _lib.lib().pa_quantize_into_cache(
            key.data_ptr(), value.data_ptr(), _DTYPE_CODE[key.dtype], key.stride(0),
            slot_mapping.data_ptr(), N, KVH, D, k_cache.data_ptr(), v_cache.data_ptr(),
            k_scales.data_ptr(), v_scales.data_ptr(), k_cache.shape[0], block_size,
            _ptr(k_scale), _ptr(v_scale), status, _stream(key.device))
        _lib.check(rc, "quantize_into_cache")


def write_into_cache(key, value, k_cache, v_cache, slot_mapping, block_size=16):
    """FP16 copy of key/value [num_tokens, kv_heads, head_dim] into an fp16 paged cache."""
    _check_rows(key, value)
    _require(k_cache.dtype == torch.float16 and v_cache.dtype == torch.float16,
             "cache must be fp16")
    _require(slot_mapping.dtype == torch.int32 and slot_mapping.is_cuda,
             "slot_mapping must be int32 on CUDA")
    N, KVH, D = key.shape
    _require(slot_mapping.numel() == N, "slot_mapping must have one entry per token")
    _check_cache_layout(k_cache, v_cache, KVH, D, block_size)
    for t in (k_cache, v_cache, slot_mapping):
        _require(t.is_contiguous() and t.device == key.device,
                 "cache tensors must be contiguous and on the key's device")
    with _Guard(key.device):
        status = _status_word(key.device)
        rc = _lib.lib().pa_write_into_cache_f16(
            key.data_ptr(), value.data_ptr(), _DTYPE_CODE[key.dtype], key.stride(0),
            slot_mapping.data_ptr(), N, KVH, D, k_cache.data_ptr(), v_cache.data_ptr(),
            k_cache.shape[0], block_size, status, _stream(key.device))
        _lib.check(rc, "write_into_cache")


def prefill_into_cache(k, v, k_cache, v_cache, block_table, context_lens, block_size=16, *,
                       k_scales=None, v_scales=None, k_scale=None, v_scale=None):
    """Bulk write of contiguous per-sequence K/V [num_seqs, max_len, kv_heads, head_dim] into
    the blocks listed by block_table (a warp per 16-token group of one page, K or V, its rows
    loaded into registers together; 16-byte stores into the page layout). INT8
    caches are quantised per token (or with k_scale/v_scale); FP16 caches get a copy.
    Tokens past a sequence's context inside its last block are written as zeros."""
    _require(k.is_cuda and v.is_cuda, "tensors must be on CUDA")
    _require(k.dtype in _DTYPE_CODE and v.dtype == k.dtype, "k/v must be fp16, bf16 or fp32")
    _require(k.dim() == 4 and k.shape == v.shape and k.is_contiguous() and v.is_contiguous(),
             "k/v must be contiguous [num_seqs, max_len, kv_heads, head_dim]")
    S, Lmax, KVH, D = k.shape
    int8 = k_cache.dtype == torch.int8
    _require(int8 or k_cache.dtype == torch.float16, "cache must be int8 or fp16")
    _require(block_table.dtype == torch.int32 and context_lens.dtype == torch.int32,
             "block_table and context_lens must be int32")
    _require(block_table.dim() == 2 and block_table.shape[0] == S and context_lens.numel() == S,
             "block_table must be [num_seqs, max_blocks] and context_lens [num_seqs]")
    tensors = [k_cache, v_cache, block_table, context_lens]
    if int8:
        _require(k_scales is not None and v_scales is not None, "int8 cache needs scales")
        tensors += [k_scales, v_scales]
    _check_cache_layout(k_cache, v_cache, KVH, D, block_size, k_scales if int8 else None,
                        v_scales if int8 else None)
    for t in tensors:
        _require(t.is_contiguous() and t.device == k.device,
                 "cache tensors must be contiguous and on k's device")
    with _Guard(k.device):
        status = _status_word(k.device)
        rc = _lib.lib().pa_prefill_into_cache(
            k.data_ptr(), v.data_ptr(), _DTYPE_CODE[k.dtype], S, Lmax, KVH, D,
            block_table.data_ptr(), context_lens.data_ptr(), block_table.shape[1],
            _lib.PA_DTYPE_I8 if int8 else _lib.PA_DTYPE_F16, k_cache.data_ptr(),
            v_cache.data_ptr(), _ptr(k_scales), _ptr(v_scales), k_cache.shape[0], block_size,
            _ptr(k_scale), _ptr(v_scale), status, _stream(k.device))
        _lib.check(rc, "prefill_into_cache")


def fp4_cache(num_blocks, num_kv_heads, block_size=16, device="cuda"):
    """A zeroed 4-bit K/V cache: (k_cache, v_cache), each uint8 [num_blocks, num_kv_heads,
    block_size/16, 1152]. The layout is include/pa_b200.h's; 72 bytes hold K or V of one token
    and kv head (4.5 bits a value), against 132 in an int8 cache and 256 in an fp16 one."""
    _require(block_size > 0 and block_size % FP4_GROUP_TOKENS == 0 and 128 % block_size == 0,
             "block_size must divide TILE (multiple of 16)")
    return tuple(torch.zeros(num_blocks, num_kv_heads, block_size // FP4_GROUP_TOKENS,
                             FP4_GROUP_BYTES, dtype=torch.uint8, device=device)
                 for _ in range(2))


# The checks of the calls below are written out as single conditions: they run once per launch of
# kernels that take a few microseconds.
def _check_slots(slot_mapping, num_tokens, device):
    if not (slot_mapping.dtype == torch.int32 and slot_mapping.device == device and
            slot_mapping.numel() == num_tokens and slot_mapping.is_contiguous()):
        raise RuntimeError("slot_mapping must be contiguous int32 with one entry per token, on the "
                           "rows' CUDA device")


def _check_on(device, *tensors):
    for t in tensors:
        if t is not None and not (t.device == device and t.is_contiguous()):
            raise RuntimeError("cache tensors must be contiguous and on the rows' device")


def quantize_into_cache_fp4(key, value, k_cache, v_cache, slot_mapping, block_size=16):
    """Write key/value [num_tokens, kv_heads, 128] (fp16, bf16 or fp32) into a 4-bit cache
    (fp4_cache) at slot_mapping (int32, block*block_size+offset; negative = skip).

    Sixteen neighbouring values share a scale: the nearest representable to amax / 6, ties to
    even; a value becomes the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even
    code. A block holding a NaN or an infinity reads back as NaN. Two tokens with the same slot
    in one call leave a mixture of their blocks there."""
    dev, dt = key.device, key.dtype
    if not (key.is_cuda and dt in _DTYPE_CODE and value.dtype == dt and value.device == dev):
        raise RuntimeError("key/value must both be fp16, bf16 or fp32, on one CUDA device")
    shape, stride, vstride = key.shape, key.stride(), value.stride()
    if not (len(shape) == 3 and value.shape == shape and shape[2] == HEAD_DIM):
        raise RuntimeError("key/value must be [num_tokens, num_kv_heads, 128]")
    N, KVH, D = shape
    if not (stride[2] == 1 == vstride[2] and
            (KVH == 1 or stride[1] == D == vstride[1]) and
            (N == 1 or stride[0] == vstride[0])):
        raise RuntimeError("key/value rows must be contiguous per token, with one token stride")
    _check_slots(slot_mapping, N, dev)
    NB, kvh = _check_fp4_caches(k_cache, v_cache, block_size)
    if kvh != KVH:
        raise RuntimeError(f"the cache has {kvh} kv heads, the rows {KVH}")
    _check_on(dev, k_cache, v_cache)
    with _Guard(dev):
        rc = _lib.lib().pa_quantize_into_cache_fp4(
            key.data_ptr(), value.data_ptr(), _DTYPE_CODE[dt],
            stride[0] if N > 1 else KVH * D, slot_mapping.data_ptr(), N, KVH, D,
            k_cache.data_ptr(), v_cache.data_ptr(), NB,
            block_size, _status_word(dev), _stream(dev))
        _lib.check(rc, "quantize_into_cache (fp4)")


def read_from_cache_fp4(k_cache, v_cache, slot_mapping, block_size=16, *, dtype=torch.float16,
                        out=None):
    """Rows read back from a 4-bit cache: (key, value) [num_tokens, kv_heads, 128] of the tokens
    at slot_mapping, for instance a cached prefix for the attention of a prompt's next chunk.
    Held values are exact in fp16, bf16 and fp32. Rows of negative slots are not written: they
    keep what `out`, a pair of tensors to write into, held, and are undefined without it."""
    dev = k_cache.device
    if not k_cache.is_cuda:
        raise RuntimeError("tensors must be on CUDA")
    NB, KVH = _check_fp4_caches(k_cache, v_cache, block_size)
    N = slot_mapping.numel()
    _check_slots(slot_mapping, N, dev)
    _check_on(dev, k_cache, v_cache)
    if out is None:
        if dtype not in _DTYPE_CODE:
            raise RuntimeError("dtype must be fp16, bf16 or fp32")
        key = torch.empty((N, KVH, HEAD_DIM), dtype=dtype, device=dev)
        value = torch.empty_like(key)
    else:
        key, value = out
        for t in (key, value):
            if not (t.dtype in _DTYPE_CODE and t.dtype == key.dtype and t.device == dev and
                    tuple(t.shape) == (N, KVH, HEAD_DIM) and t.is_contiguous()):
                raise RuntimeError(f"out must be two contiguous [{N}, {KVH}, {HEAD_DIM}] tensors "
                                   "of one type on the cache's device")
    with _Guard(dev):
        rc = _lib.lib().pa_read_from_cache_fp4(
            key.data_ptr(), value.data_ptr(), _DTYPE_CODE[key.dtype], k_cache.data_ptr(),
            v_cache.data_ptr(), slot_mapping.data_ptr(), N, KVH, HEAD_DIM, NB, block_size,
            _status_word(dev), _stream(dev))
        _lib.check(rc, "read_from_cache (fp4)")
    return key, value


# ---------------------------------------------------------------------------------------
# Norm and position rotation
# ---------------------------------------------------------------------------------------
def rope_table(num_positions, rot_dim=HEAD_DIM, base=10000.0, device="cuda"):
    """Rotation table [num_positions, rot_dim] fp32: cos(p * base^(-2i/rot_dim)) for i <
    rot_dim/2, then the sines. Angles are formed in 64 bits (far positions lose them in 32)."""
    _require(rot_dim > 0 and rot_dim % 2 == 0, "rot_dim must be even: values turn in pairs")
    inv = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) /
                          rot_dim)
    ang = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _head_rows(name, t, tokens, heads, dtype, device):
    """Number of heads and token stride of rows [tokens, heads, 128], contiguous per token."""
    shape, stride = t.shape, t.stride()
    if not (len(shape) == 3 and shape[0] == tokens and shape[2] == HEAD_DIM and
            (heads is None or shape[1] == heads) and t.dtype == dtype and t.device == device):
        raise RuntimeError(f"{name} must be [{tokens}, {heads or 'heads'}, {HEAD_DIM}] of q's type "
                           f"on q's device; got {t.dtype} {tuple(shape)} on {t.device}")
    H = shape[1]
    row = H * HEAD_DIM
    if row == 0 or tokens == 0:
        return H, row
    if not (stride[2] == 1 and (H == 1 or stride[1] == HEAD_DIM) and
            (tokens == 1 or stride[0] >= row)):
        raise RuntimeError(f"{name} rows must be contiguous per token")
    return H, stride[0] if tokens > 1 else row


def _check_norm_rope(q, k, q_weight, k_weight, positions, table, eps):
    dev, dt = q.device, q.dtype
    if not (q.is_cuda and dt in _DTYPE_CODE and q.dim() == 3):
        raise RuntimeError("q must be fp16, bf16 or fp32 [num_tokens, num_heads, 128] on CUDA")
    N = q.shape[0]
    H, qs = _head_rows("q", q, N, None, dt, dev)
    KVH, ks = _head_rows("k", k, N, None, dt, dev)
    for w in (q_weight, k_weight):
        if w is not None and not (w.dtype == dt and w.device == dev and w.dim() == 1 and
                                  w.numel() == HEAD_DIM and w.is_contiguous()):
            raise RuntimeError(f"weights must be [{HEAD_DIM}] of q's type, on q's device")
    if not (positions.dtype == torch.int32 and positions.device == dev and
            positions.numel() == N and positions.is_contiguous()):
        raise RuntimeError("positions must be int32, one per token, on q's device")
    size = table.shape
    if not (table.dtype == torch.float32 and table.device == dev and len(size) == 2 and
            size[0] > 0 and table.is_contiguous()):
        raise RuntimeError("table must be fp32 [positions, rot_dim] on q's device")
    if not (0 < size[1] <= HEAD_DIM and size[1] % 16 == 0):
        raise RuntimeError("rot_dim must be a multiple of 16 up to 128")
    if not eps >= 0:
        raise RuntimeError("eps must be >= 0")
    return N, H, qs, KVH, ks


def qk_norm_rope(q, k, q_weight, k_weight, positions, table, *, eps=1e-6, interleaved=False,
                 q_out=None, k_out=None):
    """RMS norm of every q and k head and the position rotation, in one launch.

    q [num_tokens, heads, 128] and k [num_tokens, kv_heads, 128] (fp16, bf16 or fp32; views into
    one projection are fine, each token's rows contiguous); weights [128] of the same type, or
    None for no norm; positions int32 [num_tokens]; table [positions, rot_dim] fp32 as rope_table
    makes it: the first rot_dim values of a head turn, value i with i + rot_dim/2, or 2i with
    2i + 1 when interleaved. fp32 arithmetic, rounded once. Rows of tokens with a negative
    position (extend_block_tables' padding) are not written: they keep what q_out and k_out held,
    and are undefined where those are not given. q_out may be q and k_out k. Returns
    (q_out, k_out)."""
    N, H, qs, KVH, ks = _check_norm_rope(q, k, q_weight, k_weight, positions, table, eps)
    dev, dt = q.device, q.dtype
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        qos = H * HEAD_DIM
    else:
        _, qos = _head_rows("q_out", q_out, N, H, dt, dev)
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        kos = KVH * HEAD_DIM
    else:
        _, kos = _head_rows("k_out", k_out, N, KVH, dt, dev)
    with _Guard(dev):
        rc = _lib.lib().pa_qk_norm_rope(
            q_out.data_ptr(), qos, k_out.data_ptr(), kos, q.data_ptr(), qs, k.data_ptr(), ks,
            _DTYPE_CODE[dt], _ptr(q_weight), _ptr(k_weight), eps, positions.data_ptr(),
            table.data_ptr(), table.shape[0], table.shape[1], 1 if interleaved else 0, N, H, KVH,
            HEAD_DIM, _status_word(dev), _stream(dev))
        _lib.check(rc, "qk_norm_rope")
    return q_out, k_out


def norm_rope_into_cache(q, k, v, q_weight, k_weight, positions, table, k_cache, v_cache,
                         slot_mapping, block_size=16, *, eps=1e-6, interleaved=False,
                         q_out=None, k_scales=None, v_scales=None):
    """qk_norm_rope with the new K and the V rows going straight into the paged cache at
    slot_mapping, in one launch: bit for bit what qk_norm_rope followed by the cache's write
    (write_into_cache, quantize_into_cache with per-token scales, or quantize_into_cache_fp4)
    gives. The cache is fp16, int8 or float8_e4m3fn (with k_scales and v_scales), or 4-bit (with
    rot_dim a multiple of 32 unless interleaved). A negative slot writes nothing to the cache, a
    negative position skips the token; slots of one call have to differ. Returns q_out
    [num_tokens, heads, 128]; it may be q. It saves a launch and is the faster form for up to
    about a thousand tokens; for long prompts the separate calls are (16384 tokens, 32/8 heads, bf16,
    in slot order: 4-bit 100 us against 77, fp16 179 against 91, int8 214 against 92)."""
    N, H, qs, KVH, ks = _check_norm_rope(q, k, q_weight, k_weight, positions, table, eps)
    dev, dt = q.device, q.dtype
    _, vs = _head_rows("v", v, N, KVH, dt, dev)
    _check_slots(slot_mapping, N, dev)
    kind = _kv_kind(k_cache, k_scales)
    if kind == "f4":
        NB, kvh = _check_fp4_caches(k_cache, v_cache, block_size)
        if kvh != KVH:
            raise RuntimeError(f"the cache has {kvh} kv heads, the rows {KVH}")
        if not (k_scales is None and v_scales is None):
            raise RuntimeError("a 4-bit cache holds its own scales")
    else:
        want = {"f16": torch.float16, "i8": torch.int8, "f8": _FP8}[kind]
        _require(k_cache.dtype == want and v_cache.dtype == want,
                 "cache must be fp16, int8, float8_e4m3fn or 4-bit, K and V alike")
        if kind != "f16":
            _require(k_scales is not None and v_scales is not None and
                     k_scales.dtype == torch.float32 and v_scales.dtype == torch.float32,
                     "scales must be fp32")
        NB = _check_cache_layout(k_cache, v_cache, KVH, HEAD_DIM, block_size, k_scales, v_scales)
    _check_on(dev, k_cache, v_cache, k_scales, v_scales)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        qos = H * HEAD_DIM
    else:
        _, qos = _head_rows("q_out", q_out, N, H, dt, dev)
    with _Guard(dev):
        rc = _lib.lib().pa_norm_rope_into_cache(
            q_out.data_ptr(), qos, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
            _DTYPE_CODE[dt], _ptr(q_weight), _ptr(k_weight), eps, positions.data_ptr(),
            table.data_ptr(), table.shape[0], table.shape[1], 1 if interleaved else 0,
            slot_mapping.data_ptr(), N, H, KVH, HEAD_DIM, _KV_CODE[kind], k_cache.data_ptr(),
            v_cache.data_ptr(), _ptr(k_scales), _ptr(v_scales), NB, block_size,
            _status_word(dev), _stream(dev))
        _lib.check(rc, "norm_rope_into_cache")
    return q_out


# ---------------------------------------------------------------------------------------
# Block tables of a step
# ---------------------------------------------------------------------------------------
def _check_int(device, *rows):
    """rows: (name, tensor, entries or None): contiguous int32 vectors on the device."""
    for name, t, n in rows:
        if not (t.dtype == torch.int32 and t.device == device and t.dim() == 1 and
                (n is None or t.numel() == n) and t.is_contiguous()):
            raise RuntimeError(f"{name} must be a contiguous int32 vector"
                               + (f" of {n}" if n is not None else "")
                               + " on block_table's device")


def _check_tables(block_table, context_lens, per_seq, free_blocks, free_count, block_size):
    dev, shape = block_table.device, block_table.shape
    if not (block_table.is_cuda and len(shape) == 2 and block_table.dtype == torch.int32 and
            block_table.is_contiguous()):
        raise RuntimeError("block_table must be contiguous int32 [num_seqs, max_blocks_per_seq] on "
                           "CUDA")
    if not (shape[1] > 0 and block_size > 0):
        raise RuntimeError("max_blocks_per_seq and block_size must be > 0")
    S = shape[0]
    _check_int(dev, ("context_lens", context_lens, S), ("the per-sequence values", per_seq, S),
               ("free_blocks", free_blocks, None), ("free_count", free_count, 1))
    return S, shape[1], dev


def release_blocks(block_table, context_lens, finished, free_blocks, free_count, block_size=16,
                   *, context_lens_out=None, free_count_out=None):
    """Push the blocks of finished sequences (finished[b] != 0, int32) onto the free stack.

    free_blocks (int32 buffer) holds the free block ids in [0, free_count[0]); blocks go on top in
    sequence order, by block index. Returns (context_lens, free_count): new tensors, or the given
    ones, which may be the inputs. Finished sequences get length 0. A call that does not fit
    (a length past the table, no room in the buffer) changes nothing and sets a status bit
    (check_status)."""
    S, max_blocks, dev = _check_tables(block_table, context_lens, finished, free_blocks,
                                       free_count, block_size)
    lens, count = context_lens_out, free_count_out
    if lens is None:
        lens = torch.empty_like(context_lens)
    else:
        _check_int(dev, ("context_lens_out", lens, S))
    if count is None:
        count = torch.empty_like(free_count)
    else:
        _check_int(dev, ("free_count_out", count, 1))
    with _Guard(dev):
        status = _status_word(dev)
        rc = _lib.lib().pa_release_blocks(
            block_table.data_ptr(), context_lens.data_ptr(), finished.data_ptr(),
            free_blocks.data_ptr(), free_count.data_ptr(), lens.data_ptr(), count.data_ptr(), S,
            max_blocks, block_size, free_blocks.numel(), status, _stream(dev))
        _lib.check(rc, "release_blocks")
    return lens, count


def extend_block_tables(block_table, context_lens, new_lens, free_blocks, free_count, num_blocks,
                        block_size=16, *, max_tokens, slot_mapping=None, positions=None,
                        query_start=None, context_lens_out=None, free_count_out=None):
    """Grow sequence b by new_lens[b] tokens (int32, >= 0): pop the blocks it needs from the free
    stack (see release_blocks) into its row of block_table, and lay out the step's packed batch.

    Returns (slot_mapping, positions, query_start, context_lens, free_count): for token i of the
    batch, sequences in order, its cache slot and its position, -1 in both past the last token
    (both int32 [max_tokens], what the cache writes and qk_norm_rope take); sequence b's tokens
    are [query_start[b], query_start[b + 1]). context_lens counts the new tokens, as the decodes
    expect. Nothing is read on the host, so the call can be captured in a CUDA graph. A call that
    does not fit (lengths past the table, more than max_tokens tokens, too few free blocks)
    changes nothing, gives slots and positions of -1 and query_start of 0, and sets a status bit
    (check_status)."""
    S, max_blocks, dev = _check_tables(block_table, context_lens, new_lens, free_blocks,
                                       free_count, block_size)
    max_tokens = int(max_tokens)
    if max_tokens < 0:
        raise RuntimeError("max_tokens must be >= 0")
    outs = [slot_mapping, positions, query_start, context_lens_out, free_count_out]
    sizes = [max_tokens, max_tokens, S + 1, S, 1]
    if all(t is None for t in outs):  # one allocation, split
        outs = torch.split_with_sizes(
            torch.empty(2 * max_tokens + 2 * S + 2, dtype=torch.int32, device=dev), sizes)
    else:
        names = ("slot_mapping", "positions", "query_start", "context_lens_out", "free_count_out")
        for i, n in enumerate(sizes):
            if outs[i] is None:
                outs[i] = torch.empty(n, dtype=torch.int32, device=dev)
            _check_int(dev, (names[i], outs[i], n))
    slot_mapping, positions, query_start, lens, count = outs
    with _Guard(dev):
        status = _status_word(dev)
        rc = _lib.lib().pa_extend_block_tables(
            block_table.data_ptr(), context_lens.data_ptr(), new_lens.data_ptr(),
            free_blocks.data_ptr(), free_count.data_ptr(), lens.data_ptr(), count.data_ptr(),
            slot_mapping.data_ptr(), positions.data_ptr(), query_start.data_ptr(), S, max_blocks,
            block_size, free_blocks.numel(), num_blocks, max_tokens, status, _stream(dev))
        _lib.check(rc, "extend_block_tables")
    return slot_mapping, positions, query_start, lens, count


def absmax_scale(x, semantics=_lib.PA_SCALE_CLAMP_THEN_DIVIDE):
    """Per-tensor INT8 scale of x as a 0-d fp32 device tensor.

    CLAMP_THEN_DIVIDE matches quantize_per_tensor (tests/paged_decode_attn.py:118-119);
    DIVIDE_THEN_CLAMP matches PagedKVCache.prefill's per-tensor scale
    (benchmarks/int8_bridge/paged_cache.py:101-102)."""
    _require(x.is_cuda and x.dtype in _DTYPE_CODE and x.is_contiguous(),
             "x must be a contiguous fp16/bf16/fp32 CUDA tensor")
    out = torch.empty((), dtype=torch.float32, device=x.device)
    with _Guard(x.device):
        scratch = torch.empty(1, dtype=torch.int32, device=x.device)
        rc = _lib.lib().pa_absmax_scale(x.data_ptr(), _DTYPE_CODE[x.dtype], x.numel(),
                                        out.data_ptr(), semantics, scratch.data_ptr(),
                                        _stream(x.device))
        _lib.check(rc, "absmax_scale")
    return out
