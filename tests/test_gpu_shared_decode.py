"""Sequences that share a prefix: hx_kv_share and hx_decode_attention_shared.

Tolerance of an attention output against 64 bits, for a row with probabilities
p_j (sum 1) and L keys:
  * a score is a sum of hd products, off by (hd + 2) 2^-24 scale sum|q k| =: e_j,
    and the power of two by 2^-21, so a probability by 2 max e + 2^-20 relative
    (its own and the sum's share of it);
  * probabilities enter the second product in fp16: half a step, 2^-11 of a
    normal one, and 2^-25 of the row's largest for a subnormal one;
  * the fp32 sums over the keys add (L + 64) 2^-24;
all of sum p_j |v_j| (the subnormal part of sum |v_j|), then the store half a
step of the stored type.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hxinfer_b200 import kv
    kv.load()
    kv.device_status(clear=True)
    return kv


class Batch:
    """A cache whose sequences 0..n-1 begin with `prefix` positions of sequence
    n, and the K/V they hold, as [positions, hkv, hd] per sequence.  Everything
    that no sequence wrote is NaN."""

    def __init__(self, hx, suffixes, prefix, hkv, hd=128, layers=1, seed=1, q_scale=1.0, spare=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.hx, self.prefix, self.hkv, self.hd = g, hx, prefix, hkv, hd
        n = len(suffixes)
        cap = prefix + max(suffixes) + spare
        need = (prefix + 63) // 64 + sum(2 + s // 64 for s in suffixes)
        self.cache = hx.KVCache(layers, hkv, hd, n + 1, cap, need)
        self.cache.pool().fill_(float("nan"))
        self.layer = layers - 1
        self.k, self.v, self.lengths = [], [], [prefix + s for s in suffixes]
        rand = lambda m: torch.randn((m, hkv, hd), generator=g, device="cuda").half()
        pk, pv = rand(prefix), rand(prefix)
        self.cache.reserve(n, prefix)
        if prefix:
            self.cache.write(self.layer, n, 0, pk, pv)
        for i, s in enumerate(suffixes):
            self.cache.share(i, n, prefix)
            self.cache.reserve(i, prefix + s)
            sk, sv = rand(s), rand(s)
            if s:
                self.cache.write(self.layer, i, prefix, sk, sv)
            self.k.append(torch.cat((pk, sk)))
            self.v.append(torch.cat((pv, sv)))
        self.seq_ids = torch.arange(n, dtype=torch.int32, device="cuda")
        self.len_dev = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")

    def q(self, hq, scale=1.0):
        n = len(self.lengths)
        return (torch.randn((n, hq * self.hd), generator=self.g, device="cuda") * scale).half()

    def check(self, out, q, hq, scale, rows=None):
        group = hq // self.hkv
        out, q = out.view(-1, hq, self.hd), q.view(-1, hq, self.hd)
        fi = torch.finfo(out.dtype)
        for i in range(len(self.lengths)) if rows is None else rows:
            if self.lengths[i] == 0:
                assert bool((out[i] == 0).all())
                continue
            k = self.k[i].double().repeat_interleave(group, 1)
            v = self.v[i].double().repeat_interleave(group, 1)
            qi = q[i].double()
            p = torch.softmax(torch.einsum("hd,lhd->hl", qi, k) * scale, -1)
            want = torch.einsum("hl,lhd->hd", p, v)
            e = (self.hd + 2) * 2.0 ** -24 * scale * torch.einsum("hd,lhd->hl", qi.abs(), k.abs()).amax(-1)
            mass = torch.einsum("hl,lhd->hd", p, v.abs())
            L = k.shape[0]
            bound = (2 * e[:, None] + 2.0 ** -20 + 2.0 ** -11 + (L + 64) * 2.0 ** -24) * mass \
                + 2.0 ** -25 * p.amax(-1)[:, None] * v.abs().sum(0)
            lim = bound + fi.eps / 2 * torch.clamp(want.abs() + bound, min=fi.smallest_normal)
            err = (out[i].double() - want).abs()
            assert bool((err <= lim).all()), f"row {i}: off by {(err - lim).max().item():.3e} past the bound"


def run(b, q, hq, scale=None, **kw):
    out = b.cache.decode_shared(b.layer, q, b.seq_ids, b.len_dev, hq, prefix_seq=len(b.lengths),
                                prefix_len=b.prefix, scale=scale, **kw)
    b.hx.device_status()
    return out


# ------------------------------------------------------------------ sharing blocks

def test_share_counts_blocks(hx):
    cache = hx.KVCache(1, 2, 64, 4, 640, 12)
    free = lambda: cache.info()["free_blocks"]
    cache.reserve(0, 200)                       # 4 blocks
    assert free() == 8
    cache.share(1, 0, 200)                      # 3 shared, 1 copied
    assert free() == 7
    cache.share(2, 1, 192)                      # 3 shared, none copied
    assert free() == 7
    cache.share(3, 0, 0)                        # nothing
    cache.reserve(3, 1)
    assert free() == 6
    cache.reserve(2, 300)                       # 2 more of its own
    assert free() == 4
    cache.release(0)                            # its 4th block alone comes back
    assert free() == 5
    cache.release(1)
    assert free() == 6
    cache.release(2)
    assert free() == 11
    cache.release(3)
    assert free() == 12
    cache.reserve(0, 640)
    cache.release(0)
    assert free() == 12


def test_share_refusals(hx):
    cache = hx.KVCache(1, 1, 64, 3, 256, 3)
    cache.reserve(0, 100)
    for seq, src, n, status in ((0, 0, 1, 1), (3, 0, 1, 1), (1, 3, 1, 1), (-1, 0, 1, 1), (1, -1, 1, 1),
                                (1, 0, -1, 2), (1, 0, 129, 2), (1, 0, 257, 2), (1, 2, 1, 2)):
        with pytest.raises(hx._lib.HXError) as e:
            cache.share(seq, src, n)
        assert e.value.status == status, (seq, src, n)
    cache.reserve(1, 1)
    with pytest.raises(hx._lib.HXError):
        cache.share(1, 0, 64)                   # holds a block
    with pytest.raises(hx._lib.HXError) as e:
        cache.share(2, 0, 65)                   # needs a block for one position
    assert e.value.status == 2
    cache.share(2, 0, 64)
    k = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    for seq in (0, 2):
        with pytest.raises(hx._lib.HXError):
            cache.write(0, seq, 63, k, k)
        with pytest.raises(hx._lib.HXError):
            cache.restore(seq, 10, torch.zeros(4096, dtype=torch.uint8, device="cuda"))
    cache.write(0, 0, 64, k, k)                 # its own block
    cache.release(2)
    cache.write(0, 0, 63, k, k)                 # no longer shared
    kt = torch.zeros(64 * 64, dtype=torch.float16, device="cuda")
    wrapped = hx.KVCache.wrap(kt, kt.clone(), 1, 64, 64)
    with pytest.raises(hx._lib.HXError):
        wrapped.share(0, 0, 1)


@pytest.mark.parametrize("hd", [10, 128])
@pytest.mark.parametrize("prefix", [1, 63, 64, 130])
def test_shared_positions_read_like_copies(hx, hd, prefix):
    """Every layer reads the prefix from both; what either appends behind it is
    not seen by the other; K2 over a sharing sequence equals K2 over a copy."""
    layers, hkv = 3, 2
    g = torch.Generator(device="cuda").manual_seed(prefix)
    rand = lambda n: torch.randn((n, hkv, hd), generator=g, device="cuda").half()
    cache = hx.KVCache(layers, hkv, hd, 3, 256)
    cache.reserve(0, prefix)
    cache.reserve(2, prefix + 20)
    for la in range(layers):
        k, v = rand(prefix), rand(prefix)
        cache.write(la, 0, 0, k, v)
        cache.write(la, 2, 0, k, v)
    cache.share(1, 0, prefix)
    cache.reserve(0, prefix + 20)
    cache.reserve(1, prefix + 20)
    for la in range(layers):
        a, b = (rand(20), rand(20)), (rand(20), rand(20))
        cache.write(la, 0, prefix, *a) if prefix % 64 == 0 or prefix > 64 else None
        cache.write(la, 1, prefix, *b)
        cache.write(la, 2, prefix, *b)
        for x, y in zip(cache.read(la, 1, 0, prefix + 20), cache.read(la, 2, 0, prefix + 20)):
            assert torch.equal(x, y)
        for x, y in zip(cache.read(la, 0, 0, prefix), cache.read(la, 2, 0, prefix)):
            assert torch.equal(x, y)
        q = torch.randn((1, 4 * hd), generator=g, device="cuda").half()
        one = torch.tensor([1], dtype=torch.int32, device="cuda")
        ln = one * (prefix + 20)
        assert torch.equal(cache.decode(la, q, one, ln, 4), cache.decode(la, q, one * 2, ln, 4))
    hx.device_status()


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("hd", [128, 64, 80, 256])
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 127, 128, 129, 300])
def test_prefix_and_suffix_lengths(hx, hd, prefix):
    """Prefixes that end inside, at and behind blocks and 128-key tiles;
    suffixes of 0 (the prefix alone), 1, and across block ends."""
    b = Batch(hx, [1, 0 if prefix else 2, 63, 64, 65, 200, 129], prefix, 2, hd)
    q = b.q(6)
    b.check(run(b, q, 6), q, 6, 1 / math.sqrt(hd))


@pytest.mark.parametrize("hkv,group", [(1, 1), (2, 2), (1, 3), (4, 4), (2, 5), (4, 7), (8, 1), (2, 8),
                                       (1, 9), (1, 16), (1, 17), (1, 40), (1, 128), (1, 130)])
@pytest.mark.parametrize("n", [1, 3, 37])
def test_head_layouts(hx, hkv, group, n):
    b = Batch(hx, [(37 * i) % 150 + 1 for i in range(n)], 333, hkv, seed=group, layers=2)
    q = b.q(hkv * group, 2.0)
    b.check(run(b, q, hkv * group, out_dtype=torch.float32), q, hkv * group, 128 ** -0.5)


@pytest.mark.parametrize("n,hkv,group", [(129, 2, 4), (300, 1, 8), (300, 4, 1), (1000, 1, 2)])
def test_many_rows(hx, n, hkv, group):
    """More sequences than a lane keeps step counts of; several row tiles."""
    b = Batch(hx, [(53 * i) % 97 for i in range(n)], 200, hkv, seed=n)
    q = b.q(hkv * group)
    b.check(run(b, q, hkv * group), q, hkv * group, 128 ** -0.5)


def test_one_long_prefix(hx):
    b = Batch(hx, [5, 900, 1], 20000, 2, seed=4)
    q = b.q(8, 3.0)
    b.check(run(b, q, 8), q, 8, 128 ** -0.5)


def test_long_suffixes_and_short_prefix(hx):
    b = Batch(hx, [7000, 1, 64, 3, 2048, 4097], 70, 4, seed=5)
    q = b.q(28)
    b.check(run(b, q, 28, scale=0.05), q, 28, 0.05)


def test_many_sequences(hx):
    """More rows than one launch's tiles, ragged over three orders of length."""
    b = Batch(hx, [(i * i * 7) % 500 for i in range(300)], 1000, 2, seed=6)
    q = b.q(8)
    b.check(run(b, q, 8), q, 8, 128 ** -0.5, rows=range(0, 300, 13))


def test_growing_scores(hx):
    """Scores that rise along the prefix at a different pace in every row, so
    running maxima move apart, and a suffix far above or below them."""
    b = Batch(hx, [40, 40, 40, 40, 40], 900, 1, seed=7)
    n, hq, pre = 5, 7, 900
    u = torch.nn.functional.normalize(torch.randn(128, generator=b.g, device="cuda"), dim=0)
    ramp = torch.linspace(-30, 30, pre, device="cuda")
    pk = (ramp[:, None, None] * u).half()
    b.cache.release(n)
    for i in range(n):
        b.cache.release(i)
    b.cache.reserve(n, pre)
    b.cache.write(0, n, 0, pk, b.v[0][:pre].contiguous())
    for i in range(n):
        b.cache.share(i, n, pre)
        b.cache.reserve(i, pre + 40)
        sk = (u * (60.0 if i % 2 else -60.0)).half().expand(40, 1, 128).contiguous()
        b.cache.write(0, i, pre, sk, b.v[i][pre:].contiguous())
        b.k[i] = torch.cat((pk, sk))
    q = (u * torch.linspace(-20, 20, n * hq, device="cuda")[:, None]).half().view(n, hq * 128)
    b.check(run(b, q, hq, scale=0.3), q, hq, 0.3)


def test_same_result_as_decode(hx):
    """Within rounding of hx_decode_attention over the same blocks, and the
    same bits when called twice."""
    b = Batch(hx, [10, 80, 200, 64], 512, 4, seed=8)
    q = b.q(32)
    one = run(b, q, 32)
    assert torch.equal(one, run(b, q, 32))
    plain = b.cache.decode(0, q, b.seq_ids, b.len_dev, 32)
    b.check(plain, q, 32, 128 ** -0.5)
    b.check(one, q, 32, 128 ** -0.5)


def test_wrapped_cache(hx):
    """A caller's own K and V tensors, whose capacity is no multiple of a block:
    its one sequence, several times with different lengths."""
    g = torch.Generator(device="cuda").manual_seed(16)
    hkv, cap = 3, 700
    k, v = (torch.randn((hkv, cap, 128), generator=g, device="cuda").half() for _ in range(2))
    b = Batch.__new__(Batch)
    b.cache, b.hx, b.layer, b.hkv, b.hd, b.prefix = hx.KVCache.wrap(k, v, hkv, 128, cap), hx, 0, hkv, 128, 450
    b.lengths = [700, 451, 450, 513]
    b.k, b.v = ([t.transpose(0, 1)[:n].contiguous() for n in b.lengths] for t in (k, v))
    b.len_dev = torch.tensor(b.lengths, dtype=torch.int32, device="cuda")
    b.seq_ids = torch.zeros_like(b.len_dev)
    q = torch.randn((4, 6 * 128), generator=g, device="cuda").half()
    out = b.cache.decode_shared(0, q, b.seq_ids, b.len_dev, 6, prefix_seq=0, prefix_len=450)
    hx.device_status()
    b.check(out, q, 6, 128 ** -0.5)


def test_prefix_of_a_member_and_repeated_sequences(hx):
    """prefix_seq may be in the batch; a sequence may appear twice, in any order."""
    b = Batch(hx, [3, 70, 20], 100, 2, seed=9)
    q = b.q(4)
    order = [2, 0, 2, 1]
    sid = torch.tensor(order, dtype=torch.int32, device="cuda")
    ql = q[[2, 0, 0, 1]].contiguous()
    out = b.cache.decode_shared(0, ql, sid, b.len_dev[order].contiguous(), 4, prefix_seq=1, prefix_len=100)
    hx.device_status()
    for row, i in enumerate(order):
        b2 = Batch.__new__(Batch)
        b2.__dict__.update(b.__dict__)
        b2.k, b2.v, b2.lengths = [b.k[i]], [b.v[i]], [b.lengths[i]]
        b2.check(out[row:row + 1], ql[row:row + 1], 4, 128 ** -0.5)


@pytest.mark.parametrize("hd", [128, 64])
def test_padding_empty_and_bad_rows(hx, hd):
    """Padding keeps its output and an empty row is zeros, both unrecorded; a
    bad row is zeros, recorded, and the others are right."""
    b = Batch(hx, [10, 30, 50, 70], 90, 2, hd, seed=10)
    q = b.q(4)
    q[1] = float("nan")  # nothing of a padding row is used
    n = 4

    def call(sid, ln):
        out = torch.full((n, 4 * hd), 11.0, dtype=torch.float16, device="cuda")
        b.cache.decode_shared(0, q, torch.tensor(sid, dtype=torch.int32, device="cuda"),
                              torch.tensor(ln, dtype=torch.int32, device="cuda"), 4, prefix_seq=4,
                              prefix_len=90, out=out)
        return out

    out = call([0, -1, 2, 3], [100, 120, 0, 160])
    hx.device_status()
    assert bool((out[1] == 11).all()) and bool((out[2] == 0).all())
    b.check(out, q, 4, hd ** -0.5, rows=[0, 3])
    out = call([-1, -1, -1, -1], [100, 120, 140, 160])
    hx.device_status()
    assert bool((out == 11).all())
    for sid, ln in ((2, 89), (2, -1), (2, 1 << 30), (5, 140), (-2, 140), (1 << 30, 140)):
        out = call([0, -1, sid, 3], [100, 120, ln, 160])
        with pytest.raises(hx._lib.HXError) as e:
            hx.device_status()
        assert e.value.status == 2, (sid, ln)
        assert bool((out[2] == 0).all()) and bool((out[1] == 11).all())
        b.check(out, q, 4, hd ** -0.5, rows=[0, 3])


def test_unmapped_suffix_is_recorded(hx):
    """A length inside the capacity whose blocks were never reserved."""
    b = Batch(hx, [10, 30], 90, 2, seed=11, spare=300)
    q = b.q(4)
    b.cache.decode_shared(0, q, b.seq_ids, torch.tensor([100, 400], dtype=torch.int32, device="cuda"), 4,
                          prefix_seq=2, prefix_len=90)
    with pytest.raises(hx._lib.HXError) as e:
        hx.device_status()
    assert e.value.status == 2
    b.check(run(b, q, 4), q, 4, 128 ** -0.5)  # the next call is unharmed


def test_values_of_the_type_s_range(hx):
    """Keys at the type's lowest and highest values, and infinite values in a
    row's own suffix reach that row alone."""
    b = Batch(hx, [20, 20, 20], 200, 1, seed=12)
    q = b.q(2)
    clean = run(b, q, 2)
    k = torch.zeros((1, 1, 128), dtype=torch.float16, device="cuda")
    v = torch.full((1, 1, 128), float("inf"), dtype=torch.float16, device="cuda")
    b.cache.write(0, 1, 210, k, v)
    out = run(b, q, 2)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert bool((out[1] == float("inf")).all())
    low = torch.full((1, 1, 128), torch.finfo(torch.float16).min, dtype=torch.float16, device="cuda")
    b.cache.write(0, 2, 205, low, low)
    b.k[2][205], b.v[2][205] = low[0], low[0]
    b.check(run(b, q.abs(), 2), q.abs(), 2, 128 ** -0.5, rows=[0, 2])


def test_two_graphs_share_a_workspace(hx):
    """Two captured calls of different shapes over one workspace, replayed in
    turn on a side stream with changing lengths."""
    a, b = Batch(hx, [5, 64, 300], 256, 2, seed=13, spare=64), Batch(hx, [9] * 40, 700, 1, seed=14)
    qa, qb = a.q(8), b.q(5)
    need = max(a.cache.shared_workspace_bytes(3, 8, 256), b.cache.shared_workspace_bytes(40, 5, 700))
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    oa, ob = torch.empty_like(qa), torch.empty_like(qb)
    side, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for x, q, o, hq in ((a, qa, oa, 8), (b, qb, ob, 5)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            x.cache.decode_shared(0, q, x.seq_ids, x.len_dev, hq, prefix_seq=len(x.lengths),
                                  prefix_len=x.prefix, out=o, workspace=ws, stream=side)
        graphs.append(gr)
    for step in range(3):
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        hx.device_status()
        a.check(oa, qa, 8, 128 ** -0.5)
        b.check(ob, qb, 5, 128 ** -0.5)
        oa.zero_(), ob.zero_()
        a.lengths = [n - 1 for n in a.lengths]  # the rows drop their newest position
        a.len_dev -= 1
        a.k, a.v = [k[:-1] for k in a.k], [v[:-1] for v in a.v]


def test_refusals(hx):
    b = Batch(hx, [10, 20], 100, 2, seed=15)
    q = b.q(4)
    ok = dict(layer=0, q=q, seq_ids=b.seq_ids, lengths=b.len_dev, num_q_heads=4, prefix_seq=2, prefix_len=100)

    def call(**kw):
        b.cache.decode_shared(**{**ok, **kw})

    ws = torch.empty(b.cache.shared_workspace_bytes(2, 4, 100), dtype=torch.uint8, device="cuda")
    for kw in (dict(layer=1), dict(layer=-1), dict(num_q_heads=3, q=q[:, :384].contiguous()),
               dict(prefix_seq=3), dict(prefix_seq=-1), dict(prefix_len=-1), dict(prefix_len=1 << 20),
               dict(prefix_seq=0, prefix_len=b.cache.max_tokens_per_seq + 1), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(workspace=ws[:ws.numel() - 1]),
               dict(out=torch.empty(2 * 512 + 4, dtype=torch.float16, device="cuda")[4:].view(2, 512))):
        with pytest.raises(hx._lib.HXError):
            call(**kw)
    for kw in (dict(q=q.cpu()), dict(q=q[:1]), dict(q=q.t().contiguous().t()), dict(lengths=b.len_dev[:1]),
               dict(out=q[:1])):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(q=q.float()), dict(lengths=b.len_dev.long()), dict(out=q.bfloat16())):
        with pytest.raises(TypeError):
            call(**kw)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    call(q=q[:0], seq_ids=none, lengths=none)
    b.check(run(b, q, 4), q, 4, 128 ** -0.5)
