"""Which tensors the added operators mark as used on a stream of the caller's
(torch's caching allocator hands a dropped tensor's memory out again otherwise),
read off the calls with stand-ins for the library and the tensors: no GPU."""
import pytest

torch = pytest.importorskip("torch")
from hxinfer_b200 import kv, w4  # noqa: E402


class Fake:
    """A tensor's shape and type, which notes the streams that it is used on."""

    def __init__(self, *shape, dtype=torch.float16):
        self.shape, self.dtype, self.device, self.used = shape, dtype, "cuda", []

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096

    def element_size(self):
        return 2

    def record_stream(self, s):
        self.used.append(s)


class Stream:
    cuda_stream = 1


@pytest.fixture
def library(monkeypatch):
    class Lib:
        def __getattr__(self, name):
            return lambda *a: 0
    for m in (kv, w4):
        monkeypatch.setattr(m, "load", Lib)
    cache = kv.KVCache.__new__(kv.KVCache)
    cache.num_kv_heads, cache.head_dim, cache.handle = 2, 128, 1
    return cache


def run(call, tensors, stream):
    call(stream)
    for name, t in tensors.items():
        assert t.used == ([stream] if stream else []), name


@pytest.mark.parametrize("stream", [None, Stream()])
def test_every_tensor_of_a_call_is_marked(library, monkeypatch, stream):
    monkeypatch.setattr(kv, "_raw_stream", lambda s=None: 0)
    monkeypatch.setattr(w4, "_raw_stream", lambda s=None: 0)
    i32 = dict(dtype=torch.int32)
    t = dict(q=Fake(3, 1024), k=Fake(3, 256), v=Fake(3, 256), sid=Fake(3, **i32), pos=Fake(3, **i32),
             qw=Fake(128), kw=Fake(128), q_out=Fake(3, 1024))
    run(lambda s: library.norm_rope_append(0, t["q"], t["k"], t["v"], t["sid"], t["pos"], 8, q_weight=t["qw"],
                                           k_weight=t["kw"], q_out=t["q_out"], stream=s), t, stream)
    u = dict(q=Fake(3, 1024), sid=Fake(3, **i32), length=Fake(3, **i32), out=Fake(3, 1024), ws=Fake(64))
    run(lambda s: library.decode_shared(0, u["q"], u["sid"], u["length"], 8, prefix_seq=0, prefix_len=5,
                                        out=u["out"], workspace=u["ws"], stream=s), u, stream)
    w = w4.W4Weight.__new__(w4.W4Weight)
    x = dict(x=Fake(1, 256), packed=Fake(64), bias=Fake(16), out=Fake(1, 16))
    w.in_features, w.out_features, w.group, w.has_zeros, w.packed = 256, 16, 64, False, x["packed"]
    run(lambda s: w4.w4_linear(x["x"], w, bias=x["bias"], out=x["out"], stream=s), x, stream)
