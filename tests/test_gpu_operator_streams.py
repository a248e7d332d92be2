"""The three operators on a stream that is not the current one (tensors that the
caller drops after the call are not handed out again before it has run), and as
the first call of a process inside a capture."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HQ, HKV, HD, N = 8, 2, 128, 3


@pytest.fixture(scope="module")
def hx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hxinfer_b200 import kv
    kv.load()
    kv.device_status(clear=True)
    return kv


def rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").half()


def cases(hx, g):
    """name -> (call on tensors that it gets as copies, those tensors)"""
    from hxinfer_b200 import w4
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = hx.KVCache(1, HKV, HD, N + 1, 256)
    cache.pool().zero_()
    cache.reserve(N, 100)
    cache.write(0, N, 0, rand(g, 100, HKV, HD), rand(g, 100, HKV, HD))
    for i in range(N):
        cache.share(i, N, 100)
        cache.reserve(i, 120)
    codes, scales = w4.w4_quantize(rand(g, 256, 512) * 0.05, 64)

    def linear(stream, x, bias, codes, scales):
        w = w4.W4Weight(codes, scales, stream=stream)
        return w4.w4_linear(x, w, bias=bias, stream=stream)

    def append(stream, q, k, v, sid, pos, qw, kw):
        out = cache.norm_rope_append(0, q, k, v, sid, pos, HQ, q_weight=qw, k_weight=kw, stream=stream)
        return torch.cat([out.flatten(), cache.pool().flatten()]) if stream is None else (out, cache.pool())

    def shared(stream, q, sid, length):
        return cache.decode_shared(0, q, sid, length, HQ, prefix_seq=N, prefix_len=100, stream=stream)

    seqs = torch.arange(N, **i32)
    return {
        "linear": (linear, [rand(g, 1, 512), rand(g, 256), codes, scales]),
        "append": (append, [rand(g, N, HQ * HD), rand(g, N, HKV * HD), rand(g, N, HKV * HD), seqs,
                            torch.full((N,), 110, **i32), rand(g, HD), rand(g, HD)]),
        "shared": (shared, [rand(g, N, HQ * HD), seqs, torch.full((N,), 100, **i32)]),
    }


@pytest.mark.parametrize("name", ["linear", "append", "shared"])
def test_dropped_tensors_are_not_reused_early(hx, name):
    g = torch.Generator(device="cuda").manual_seed(3)
    call, args = cases(hx, g)[name]
    want = call(None, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    sizes = [(t.shape, t.dtype) for t in args]
    for _ in range(3):
        copies = [t.clone() for t in args]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # about 10 ms: the call runs well after what follows
        got = call(side, *copies)
        del copies
        # whatever the allocator gives to the current stream now is overwritten
        # at once, with values that are valid but other
        junk = [torch.zeros(shape, dtype=dtype, device="cuda") for shape, dtype in sizes for _ in range(4)]
        torch.cuda.current_stream().synchronize()
        side.synchronize()
        del junk
        if isinstance(got, tuple):
            got = torch.cat([t.flatten() for t in got])
        assert torch.equal(got, want)
    hx.device_status()


@pytest.mark.parametrize("n,call", [
    (1, "cache.norm_rope_append(0, q, k, k, sid, pos, 8, table=table)"),
    (9, "cache.norm_rope_append(0, q.float(), k.float(), k.float(), sid, pos, 8)"),
    (1, "cache.decode_shared(0, q, sid, pos, 8, prefix_seq=n, prefix_len=100)"),
    (9, "cache.decode_shared(0, qh, sid, pos, 32, prefix_seq=n, prefix_len=100)"),
])
def test_first_call_of_a_process_inside_a_capture(n, call):
    """Nothing that a call sets up on its first use breaks a capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = f"""
import torch
from hxinfer_b200 import kv
n = {n}
g = torch.Generator(device="cuda").manual_seed(3)
rand = lambda *s: torch.randn(s, generator=g, device="cuda").half()
cache = kv.KVCache(1, 2, 128, n + 1, 256)
cache.reserve(n, 100)
cache.write(0, n, 0, rand(100, 2, 128), rand(100, 2, 128))
for i in range(n):
    cache.share(i, n, 100)
    cache.reserve(i, 200)
ang = torch.arange(256, device="cuda")[:, None] * torch.rand(64, generator=g, device="cuda")
table = kv.RopeTable.from_values(ang.cos(), ang.sin())
q, qh, k = rand(n, 1024), rand(n, 4096), rand(n, 256)
sid, pos = torch.arange(n, dtype=torch.int32, device="cuda"), torch.full((n,), 100, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = {call}
graph.replay()
torch.cuda.synchronize()
kv.device_status()
assert torch.equal(y, {call}) and bool(y.isfinite().all())
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
