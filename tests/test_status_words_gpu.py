"""GPU: error bits stay until they are read -- while a stream's workspace grows, between the
replays of a graph, and whichever stream, graph or name of the device they come by. No call here
faults: each refusal is found by the kernels' own checks of lengths, blocks and slots."""

import pytest
import torch

from pa_testlib import fp16_case, scale_for, to_cuda

pytestmark = pytest.mark.gpu

FREE_BLOCKS, SLOT, BLOCK_ID = 1024, 256, 64


def _ops():
    from pa_b200 import ops
    return ops


def _i(*a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _tables():
    """A table call that wants two blocks of a stack that holds as many as its last entry says."""
    return [_i(0, 0, 0)[None], _i(0), _i(20), _i(3, 4, 5), _i(1)]


def _extend(t):
    return _ops().extend_block_tables(*t, 8, 16, max_tokens=32)


def _decode_fp4():
    kc, vc = _ops().fp4_cache(4, 1)
    q = torch.ones(1, 8, 128, dtype=torch.float16, device="cuda")
    _ops().decode(torch.empty_like(q), q, kc, vc, _i(0)[None], _i(5), scale_for())


def test_a_refusal_before_a_streams_first_decode():
    t = _tables()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        _extend(t)
        _decode_fp4()
    assert _ops().read_status(t[0].device) == FREE_BLOCKS
    assert _ops().read_status(t[0].device) == 0


def test_a_decodes_error_before_a_larger_decode():
    """Sixteen heads a kv head take twice the partials of eight."""
    small, large = fp16_case(1, 1, 8, 1, [40]), fp16_case(2, 2, 32, 2, [2000, 30])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for c in (small, large):
            q, kc, vc, bt, cl = to_cuda(c["q"], c["k_cache"], c["v_cache"], c["block_table"],
                                        c["context_lens"])
            if c is small:
                bt[0, 1] = 10 ** 6
            _ops().decode(torch.empty_like(q), q, kc, vc, bt, cl, scale_for())
    assert _ops().read_status(q.device) == BLOCK_ID


@pytest.mark.parametrize("first", [True, False])
def test_a_graphs_refusal_before_its_next_replay(first):
    """first: no call of this process has been made on the capturing stream; then neither the
    capture's own work nor a later growth of the stream's workspace may touch the bit."""
    t = _tables()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        if not first:
            _extend(t)
            s.synchronize()
            _ops().read_status(t[0].device)
        with torch.cuda.graph(g, stream=s):
            keep = _extend(t)
    g.replay()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        _decode_fp4()
    t[4].fill_(3)  # three free blocks: the second replay fits
    g.replay()
    torch.cuda.synchronize()
    assert keep[0][:20].tolist() == [80 + i for i in range(16)] + [64 + i for i in range(4)]
    assert _ops().read_status(t[0].device) == FREE_BLOCKS


def test_a_replay_on_a_busy_stream_is_waited_for():
    t = _tables()
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            keep = _extend(t)
    with torch.cuda.stream(other):
        torch.cuda._sleep(20_000_000)  # about 10 ms
        g.replay()
    assert _ops().read_status(t[0].device) == FREE_BLOCKS
    del keep


def test_a_device_without_an_index():
    t = _tables()
    _extend(t)
    assert _ops().read_status(torch.device("cuda")) == FREE_BLOCKS
    _extend(t)
    with pytest.raises(RuntimeError, match="free-block"):
        _ops().check_status(torch.device("cuda"))


def test_every_call_without_a_workspace_reports():
    """Slots outside the cache, by each of the calls that take a slot map."""
    ops = _ops()
    rows = torch.ones(1, 2, 128, dtype=torch.float16, device="cuda")
    bad = _i(64)
    kc, vc = ops.fp4_cache(4, 2)
    k16 = torch.zeros(4, 2, 16, 16, 8, dtype=torch.float16, device="cuda")
    v16 = torch.zeros(4, 2, 128, 16, dtype=torch.float16, device="cuda")
    sc = torch.zeros(2, 4, 2, 16, device="cuda")
    table = ops.rope_table(4)
    for call in (lambda: ops.quantize_into_cache_fp4(rows, rows, kc, vc, bad),
                 lambda: ops.read_from_cache_fp4(kc, vc, bad),
                 lambda: ops.write_into_cache(rows, rows, k16, v16, bad),
                 lambda: ops.quantize_into_cache(rows, rows, k16.to(torch.int8),
                                                 v16.to(torch.int8), *sc, bad),
                 lambda: ops.norm_rope_into_cache(rows, rows, rows, None, None, _i(0), table, kc,
                                                  vc, bad)):
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            call()
            _decode_fp4()
        assert ops.read_status(rows.device) == SLOT


def test_capture_may_be_the_first_call_of_a_process(tmp_path):
    """The status word's address is looked up inside the capture."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    repo = os.path.dirname(here)
    paths = [here] + [os.path.join(repo, d) for d in ("cuda-pa-int8_b200", "oracle")]
    script = tmp_path / "first.py"
    script.write_text(f"""
import sys
sys.path[:0] = {paths!r}
import torch
from test_status_words_gpu import FREE_BLOCKS, _extend, _ops, _tables
t = _tables()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    keep = _extend(t)
for _ in range(2):
    g.replay()
    assert _ops().read_status(t[0].device) == FREE_BLOCKS
print("first ok")
""")
    res = subprocess.run([sys.executable, str(script)], capture_output=True, text=True,
                         timeout=300)
    assert res.returncode == 0 and "first ok" in res.stdout, res.stdout + res.stderr
