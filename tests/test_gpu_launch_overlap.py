"""HX_KV_OVERLAP_LAUNCH: decode attention reads positions below the newest one
before the kernel just before it has finished, so that kernel must not let it
in before everything behind it has.

A graph of
    many positions appended -> one call between -> decode attention
on a cache with overlapped launches gives, over many replays with new inputs,
the bits that plain stream order gives.  The call between is each of the
library's that may stand there; it is small, so that the decode finds room on
the GPU beside it.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HQ, HKV, HD, HIDDEN = 8, 2, 128, 512
CHUNK = 6000      # positions appended: several rounds of the append's CTAs
REPLAYS = 25


@pytest.fixture(scope="module")
def hx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hxinfer_b200 import kv
    kv.load()
    kv.device_status(clear=True)
    return kv


def rand(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).half()


def w4_between(n):
    def make(hx, cache, g, s):
        from hxinfer_b200 import w4
        w = w4.W4Weight.quantize(rand(g, 640, HIDDEN, scale=0.05), 64)
        x = rand(g, n, HIDDEN)
        out = torch.empty((n, 640), dtype=torch.float16, device="cuda")
        return lambda: w4.w4_linear(x, w, out=out)
    return make


def newest(g, s, n):
    """n tokens at the newest position and behind it, of which one is real."""
    sid = torch.full((n,), 1, dtype=torch.int32, device="cuda")
    sid[0] = 0
    return sid, s["newest"] - torch.arange(n, dtype=torch.int32, device="cuda")


def append_between(hx, cache, g, s):
    k, v = rand(g, 1, HKV * HD), rand(g, 1, HKV * HD)
    return lambda: cache.rope_append(0, k, v, s["one"], s["newest"])


def norm_between(hx, cache, g, s):
    k, v = rand(g, 1, HKV * HD), rand(g, 1, HKV * HD)
    return lambda: cache.norm_rope_append(0, None, k, v, s["one"], s["newest"])


def qkv_between(n):
    def make(hx, cache, g, s):
        wq, wk, wv = (rand(g, h * HD, HIDDEN, scale=0.05) for h in (HQ, HKV, HKV))
        x, (sid, pos) = rand(g, n, HIDDEN), newest(g, s, n)
        q_out = torch.empty((n, HQ * HD), dtype=torch.float16, device="cuda")
        return lambda: cache.qkv_rope_append(0, x, wq, wk, wv, sid, pos, HQ, q_out=q_out)
    return make


def decode_between(hx, cache, g, s):
    """Decode of another layer."""
    q, out = rand(g, 1, HQ * HD), torch.empty((1, HQ * HD), dtype=torch.float16, device="cuda")
    ws = torch.zeros(cache.workspace_bytes(1, HQ), dtype=torch.uint8, device="cuda")
    length = torch.full((1,), 70, dtype=torch.int32, device="cuda")
    return lambda: cache.decode(1, q, s["one"], length, HQ, out=out, workspace=ws)


def append_decode_between(hx, cache, g, s):
    """One-launch step of another layer."""
    q, k, v = rand(g, 1, HQ * HD), rand(g, 1, HKV * HD), rand(g, 1, HKV * HD)
    out = torch.empty((1, HQ * HD), dtype=torch.float16, device="cuda")
    ws = torch.zeros(cache.workspace_bytes(1, HQ), dtype=torch.uint8, device="cuda")
    length = torch.full((1,), 70, dtype=torch.int32, device="cuda")
    return lambda: cache.append_decode(1, q, k, v, s["one"], length, HQ, out=out, workspace=ws)


def shared_between(hx, cache, g, s):
    """Shared-prefix decode of another layer."""
    q, out = rand(g, 1, HQ * HD), torch.empty((1, HQ * HD), dtype=torch.float16, device="cuda")
    ws = torch.zeros(cache.shared_workspace_bytes(1, HQ, 64), dtype=torch.uint8, device="cuda")
    length = torch.full((1,), 70, dtype=torch.int32, device="cuda")
    return lambda: cache.decode_shared(1, q, s["one"], length, HQ, prefix_seq=0, prefix_len=64, out=out, workspace=ws)


BETWEEN = {"w4_1": w4_between(1), "w4_2": w4_between(2), "w4_5": w4_between(5), "w4_40": w4_between(40),
           "append": append_between, "norm_append": norm_between, "qkv_1": qkv_between(1), "qkv_2": qkv_between(2),
           "qkv_8": qkv_between(8), "decode": decode_between,
           "append_decode": append_decode_between, "shared": shared_between}


def run(hx, between, overlap):
    """The decode outputs of every replay."""
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = hx.KVCache(2, HKV, HD, 2, CHUNK + 1, overlap=overlap)
    for seq in range(2):
        cache.reserve(seq, CHUNK + 1)
    cache.pool().zero_()
    qkv = rand(g, CHUNK, (HQ + 2 * HKV) * HD)
    _, k, v = qkv.split([HQ * HD, HKV * HD, HKV * HD], 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    s = dict(sid=torch.zeros(CHUNK, **i32), pos=torch.arange(CHUNK, **i32), one=torch.zeros(1, **i32),
             newest=torch.full((1,), CHUNK, **i32), length=torch.full((1,), CHUNK + 1, **i32))
    q, out = rand(g, 1, HQ * HD), torch.empty((1, HQ * HD), dtype=torch.float16, device="cuda")
    ws = torch.zeros(cache.workspace_bytes(1, HQ), dtype=torch.uint8, device="cuda")
    call = between(hx, cache, g, s)

    def step():
        cache.norm_rope_append(0, None, k, v, s["sid"], s["pos"])
        call()
        cache.decode(0, q, s["one"], s["length"], HQ, out=out, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    outs = []
    for _ in range(REPLAYS):
        qkv.copy_(rand(g, *qkv.shape))
        graph.replay()
        outs.append(out.clone())
    torch.cuda.synchronize()
    hx.device_status()
    return torch.stack(outs)


@pytest.mark.parametrize("name", BETWEEN)
def test_decode_sees_what_lies_two_kernels_back(hx, name):
    got = run(hx, BETWEEN[name], True)
    assert bool(got.isfinite().all())
    assert torch.equal(got, run(hx, BETWEEN[name], False))
