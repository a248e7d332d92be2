"""The attention layers of a decode step, as a model would run them: q/k/v
projection from 4-bit weights into packed rows, norm + rotation + append,
attention of a batch that shares a prompt, 4-bit output projection.  Every
operator is checked in 64 bits on the inputs that it got, with the bounds of its
own tests; the whole step runs eagerly and as a replayed graph.
"""
import pytest

torch = pytest.importorskip("torch")
import test_gpu_norm_append as norm  # noqa: E402
import test_gpu_shared_decode as shared  # noqa: E402
import test_gpu_w4 as lin  # noqa: E402

pytestmark = pytest.mark.gpu

LAYERS, HIDDEN, HQ, HKV, HD, GROUP = 2, 512, 8, 2, 128, 64
SEQS, PROMPT, STEPS, EPS = 5, 150, 4, 1e-6
WIDTH = (HQ + 2 * HKV) * HD


@pytest.fixture(scope="module")
def hx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hxinfer_b200 import kv
    kv.load()
    kv.device_status(clear=True)
    return kv


class Layers:
    def __init__(self, hx, g):
        from hxinfer_b200 import w4
        self.hx, self.w4 = hx, w4
        rand = lambda *s, scale=1.0: (torch.randn(s, generator=g, device="cuda") * scale).half()
        self.qkv, self.out, self.dense, self.norms = [], [], [], []
        for _ in range(LAYERS):
            for into, o, k in ((self.qkv, WIDTH, HIDDEN), (self.out, HIDDEN, HQ * HD)):
                codes, scales = w4.w4_quantize(rand(o, k, scale=k ** -0.5), GROUP)
                into.append((w4.W4Weight(codes, scales),
                             (codes.double() - 8) * scales.double().repeat_interleave(GROUP, 1)))
            self.norms.append(((1 + rand(HD, scale=0.1)).half(), (1 + rand(HD, scale=0.1)).half()))
        pos = torch.arange(PROMPT + STEPS, dtype=torch.float64, device="cuda")
        ang = pos[:, None] * 1e4 ** (-torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.table = hx.RopeTable.from_values(self.cos, self.sin)
        self.cache = hx.KVCache(LAYERS, HKV, HD, SEQS + 1, PROMPT + STEPS)

    def append(self, la, qkv, sid, pos, q_out=None):
        q, k, v = qkv.split([HQ * HD, HKV * HD, HKV * HD], 1)
        return self.cache.norm_rope_append(la, q, k, v, sid, pos, HQ, q_weight=self.norms[la][0],
                                           k_weight=self.norms[la][1], eps=EPS, table=self.table, q_out=q_out)

    def prompt(self, x):
        """The shared prompt into sequence SEQS, then shared with the others."""
        self.cache.reserve(SEQS, PROMPT)
        sid = torch.full((PROMPT,), SEQS, dtype=torch.int32, device="cuda")
        pos = torch.arange(PROMPT, dtype=torch.int32, device="cuda")
        for la in range(LAYERS):
            qkv = self.w4.w4_linear(x, self.qkv[la][0])
            q = self.append(la, qkv, sid, pos)
            attn = self.cache.prefill(la, q, SEQS, 0, HQ)
            x = x + self.w4.w4_linear(attn, self.out[la][0])
        for i in range(SEQS):
            self.cache.share(i, SEQS, PROMPT)
            self.cache.reserve(i, PROMPT + STEPS)

    def step(self, x, sid, pos, lengths, ws, keep):
        for la in range(LAYERS):
            qkv = self.w4.w4_linear(x, self.qkv[la][0], out=keep[la]["qkv"])
            q = self.append(la, qkv, sid, pos, keep[la]["q"])
            attn = self.cache.decode_shared(la, q, sid, lengths, HQ, prefix_seq=SEQS, prefix_len=PROMPT,
                                            out=keep[la]["attn"], workspace=ws)
            y = self.w4.w4_linear(attn, self.out[la][0], out=keep[la]["y"])
            keep[la]["x"].copy_(x)
            x = torch.add(x, y, out=keep[la]["next"])
        return x

    def check_step(self, keep, pos, lengths):
        cs = (self.cos[pos.long()], self.sin[pos.long()])
        for la in range(LAYERS):
            t = keep[la]
            lin.check(t["qkv"], t["x"], self.qkv[la][1], None, GROUP)
            q, k, v = t["qkv"].split([HQ * HD, HKV * HD, HKV * HD], 1)
            y, bound = norm.formula(q, self.norms[la][0], EPS, cs, HD)
            norm.check(t["q"].view(SEQS, HQ, HD), y, bound, "q")
            y, bound = norm.formula(k, self.norms[la][1], EPS, cs, HD)
            b = shared.Batch.__new__(shared.Batch)
            b.hkv, b.hd, b.lengths, b.k, b.v = HKV, HD, lengths.tolist(), [], []
            for i in range(SEQS):
                kk, vv = self.cache.read(la, i, 0, b.lengths[i])
                norm.check(kk[-1:], y[i:i + 1], bound[i:i + 1], "k")
                assert torch.equal(vv[-1].flatten(), v[i])
                b.k.append(kk)
                b.v.append(vv)
            b.check(t["attn"], t["q"], HQ, HD ** -0.5)
            lin.check(t["y"], t["attn"], self.out[la][1], None, GROUP)
        self.hx.device_status()


@pytest.mark.parametrize("graph", [False, True])
def test_decode_steps_behind_a_shared_prompt(hx, graph):
    g = torch.Generator(device="cuda").manual_seed(21)
    m = Layers(hx, g)
    rand = lambda n: torch.randn((n, HIDDEN), generator=g, device="cuda").half()
    m.prompt(rand(PROMPT))
    hx.device_status()
    empty = lambda w: torch.empty((SEQS, w), dtype=torch.float16, device="cuda")
    keep = [dict(x=empty(HIDDEN), qkv=empty(WIDTH), q=empty(HQ * HD), attn=empty(HQ * HD), y=empty(HIDDEN),
                 next=empty(HIDDEN)) for _ in range(LAYERS)]
    ws = torch.zeros(m.cache.shared_workspace_bytes(SEQS, HQ, PROMPT), dtype=torch.uint8, device="cuda")
    sid = torch.arange(SEQS, dtype=torch.int32, device="cuda")
    pos = torch.zeros(SEQS, dtype=torch.int32, device="cuda")
    lengths = torch.zeros_like(pos)
    x = rand(SEQS)
    run = lambda: m.step(x, sid, pos, lengths, ws, keep)
    if graph:
        pos.fill_(PROMPT)
        lengths.fill_(PROMPT + 1)
        run()  # warm-up outside the capture
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            run()
        run = captured.replay
    before = [[t.clone() for t in m.cache.read(la, SEQS, 0, PROMPT)] for la in range(LAYERS)]
    for step in range(STEPS):
        x.copy_(rand(SEQS))
        pos.fill_(PROMPT + step)
        lengths.fill_(PROMPT + step + 1)
        run()
        torch.cuda.synchronize()
        m.check_step(keep, pos, lengths)
    for la in range(LAYERS):  # the shared prompt is as it was
        for a, b in zip(before[la], m.cache.read(la, SEQS, 0, PROMPT)):
            assert torch.equal(a, b)


def test_one_sequence_steps_like_plain_decode(hx):
    """A single sequence and token through the same operators and through
    hx_decode_attention: the same attention within both bounds."""
    g = torch.Generator(device="cuda").manual_seed(22)
    m = Layers(hx, g)
    m.prompt(torch.randn((PROMPT, HIDDEN), generator=g, device="cuda").half())
    x = torch.randn((1, HIDDEN), generator=g, device="cuda").half()
    sid = torch.tensor([3], dtype=torch.int32, device="cuda")
    pos = torch.full_like(sid, PROMPT)
    qkv = m.w4.w4_linear(x, m.qkv[0][0])
    q = m.append(0, qkv, sid, pos)
    b = shared.Batch.__new__(shared.Batch)
    b.hkv, b.hd, b.lengths = HKV, HD, [PROMPT + 1]
    k, v = m.cache.read(0, 3, 0, PROMPT + 1)
    b.k, b.v = [k], [v]
    for out in (m.cache.decode(0, q, sid, pos + 1, HQ),
                m.cache.decode_shared(0, q, sid, pos + 1, HQ, prefix_seq=SEQS, prefix_len=PROMPT)):
        b.check(out, q, HQ, HD ** -0.5)
    hx.device_status()


def test_calls_on_two_streams_at_once(hx):
    """The three operators on two streams side by side, on caches, weights and
    workspaces of their own, give what they give one after the other."""
    from hxinfer_b200 import w4
    g = torch.Generator(device="cuda").manual_seed(77)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").half()
    sides = []
    for n in (3, 40):
        codes, scales = w4.w4_quantize(rand(1000, 512) * 0.05, 64)
        cache = hx.KVCache(1, HKV, HD, n + 1, 700)
        cache.reserve(n, 600)
        cache.write(0, n, 0, rand(600, HKV, HD), rand(600, HKV, HD))
        for i in range(n):
            cache.share(i, n, 600)
            cache.reserve(i, 650)
        sides.append(dict(
            n=n, w=w4.W4Weight(codes, scales), cache=cache, x=rand(n, 512), rows=rand(n, WIDTH),
            sid=torch.arange(n, dtype=torch.int32, device="cuda"),
            pos=torch.full((n,), 600, dtype=torch.int32, device="cuda"),
            len=torch.full((n,), 601, dtype=torch.int32, device="cuda"), stream=torch.cuda.Stream()))

    def run(side, stream=None):
        q, k, v = side["rows"].split([HQ * HD, HKV * HD, HKV * HD], 1)
        outs = []
        for _ in range(6):
            y = w4.w4_linear(side["x"], side["w"], stream=stream)
            r = side["cache"].norm_rope_append(0, q, k, v, side["sid"], side["pos"], HQ, stream=stream)
            a = side["cache"].decode_shared(0, r, side["sid"], side["len"], HQ, prefix_seq=side["n"],
                                            prefix_len=600, stream=stream)
            outs.append((y, r, a))
        return outs

    want = [run(s) for s in sides]
    torch.cuda.synchronize()
    got = [run(s, s["stream"]) for s in sides]
    torch.cuda.synchronize()
    hx.device_status()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert all(torch.equal(i, j) for i, j in zip(x, y))
