"""hx_norm_rope_append against its formula in 64 bits.

Tolerance, per element y of a head of hd elements, u = 2^-24: the sum of
squares of hd terms is off by at most (hd + 1) u relative, which the root
halves; the mean and eps add u, the reciprocal root 4 u (2 ulp), the two
products with it and the weight 2 u, the rotation's product and difference
1.5 u of |y1| + |y2|:  (hd / 2 + 9) u (|y1| + |y2|), and the store half a step of
the stored type.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def hx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hxinfer_b200 import kv
    kv.load()
    kv.device_status(clear=True)
    return kv


def tables(hx, hd, n):
    pos = torch.arange(n, dtype=torch.float64, device="cuda")
    ang = pos[:, None] * 1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    c, s = ang.cos().float(), ang.sin().float()
    return hx.RopeTable.from_values(c, s), c, s


def formula(x, w, eps, cs, hd):
    """(y, bound before the store) of rows [n, H*hd] in 64 bits; cs: per-token (cos, sin)."""
    x = x.double().reshape(x.shape[0], -1, hd)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    mag = (a.abs() + b.abs()).repeat(1, 1, 2)
    if cs is not None:
        c, s = cs[0].double()[:, None], cs[1].double()[:, None]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return y, (hd / 2 + 9) * U * mag


def check(got, want, bound, what):
    eps, tiny = torch.finfo(got.dtype).eps, torch.finfo(got.dtype).smallest_normal
    lim = bound + eps / 2 * torch.clamp(want.abs() + bound, min=tiny)
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), f"{what}: off by {(err - lim).max().item():.3e} past the bound"


def make(g, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("hd,hq,hkv", [(2, 1, 1), (16, 4, 2), (64, 12, 4), (80, 10, 5), (96, 8, 8),
                                       (100, 6, 2), (128, 28, 4), (128, 32, 8), (192, 6, 1),
                                       (250, 3, 3), (256, 16, 2)])
@pytest.mark.parametrize("form", ["packed", "separate", "odd"])
def test_matches_the_formula(hx, dt, hd, hq, hkv, form):
    """Packed rows, rows of their own and rows off the 16-byte grid; fp16 and
    fp32 q_out; untouched cache positions stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(hd + hq)
    seqs = [0, 1, 0, 2, 1, 0, 2]
    poss = [0, 63, 64, 65, 1, 190, 127]
    n, eps = len(seqs), 1e-5
    width = (hq + 2 * hkv) * hd
    if form == "odd":
        store = make(g, (n, width + 3), dt, 3.0)
        q, k, v = store[:, 1:width + 1].split([hq * hd, hkv * hd, hkv * hd], 1)
    else:
        q, k, v = make(g, (n, width), dt, 3.0).split([hq * hd, hkv * hd, hkv * hd], 1)
        if form == "separate":
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    wq, wk = make(g, (hd,), dt), make(g, (hd,), dt)
    table, c, s = tables(hx, hd, 191)
    cache = hx.KVCache(2, hkv, hd, 3, 200)
    for i in range(3):
        cache.reserve(i, 200)
    cache.pool().fill_(7.0)
    sid = torch.tensor(seqs, dtype=torch.int32, device="cuda")
    pos = torch.tensor(poss, dtype=torch.int32, device="cuda")
    q_out = torch.empty((n, hq * hd), device="cuda",
                        dtype=torch.float32 if form == "separate" else torch.float16)
    cache.norm_rope_append(1, q, k, v, sid, pos, hq, q_weight=wq, k_weight=wk, eps=eps, table=table,
                           q_out=q_out)
    hx.device_status()
    cs = (c[pos.long()], s[pos.long()])
    y, bound = formula(q, wq, eps, cs, hd)
    check(q_out.view(n, hq, hd), y, bound, "q")
    y, bound = formula(k, wk, eps, cs, hd)
    written = torch.zeros((3, 200), dtype=torch.bool)
    rows = [cache.read(1, i, 0, 200) for i in range(3)]
    for t, (sq, ps) in enumerate(zip(seqs, poss)):
        check(rows[sq][0][ps], y[t], bound[t], f"k of token {t}")
        assert torch.equal(rows[sq][1][ps], v[t].reshape(hkv, hd).half())
        written[sq, ps] = True
    for sq in range(3):
        rest = ~written[sq].cuda()
        assert bool((rows[sq][0][rest] == 7).all()) and bool((rows[sq][1][rest] == 7).all())
    assert bool((cache.pool()[0] == 7).all())  # the other layer


@pytest.mark.parametrize("weights,rope", [(False, True), (True, False), (False, False)])
def test_without_weights_or_table(hx, weights, rope):
    g = torch.Generator(device="cuda").manual_seed(5)
    hd, hq, hkv, n = 128, 8, 2, 5
    q, k, v = (make(g, (n, h * hd), torch.float16) for h in (hq, hkv, hkv))
    w = make(g, (hd,), torch.float16) if weights else None
    table, c, s = tables(hx, hd, 64)
    cache = hx.KVCache(1, hkv, hd, 1, 64)
    cache.reserve(0, 64)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    out = cache.norm_rope_append(0, q, k, v, torch.zeros_like(pos), pos, hq, q_weight=w, k_weight=w,
                                 eps=1e-6, table=table if rope else None)
    hx.device_status()
    cs = (c[:n], s[:n]) if rope else None
    y, bound = formula(q, w, 1e-6, cs, hd)
    check(out.view(n, hq, hd), y, bound, "q")
    y, bound = formula(k, w, 1e-6, cs, hd)
    check(cache.read(0, 0, 0, n)[0], y, bound, "k")


def test_long_prompt_into_wrapped_tensors_and_in_place_q(hx):
    """3001 tokens of one sequence in a wrapped cache, q rotated in place; and
    k and v alone give the same cache."""
    g = torch.Generator(device="cuda").manual_seed(6)
    hd, hq, hkv, n, start = 128, 7, 7, 3001, 40
    q, k, v = (make(g, (n, h * hd), torch.float16) for h in (hq, hkv, hkv))
    table, c, s = tables(hx, hd, start + n)
    pos = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
    sid = torch.zeros_like(pos)
    want, bound = formula(q, None, 1e-6, (c[start:], s[start:]), hd)
    kv = []
    for with_q in (True, False):
        kt, vt = (torch.zeros((hkv, start + n, hd), dtype=torch.float16, device="cuda") for _ in range(2))
        cache = hx.KVCache.wrap(kt, vt, hkv, hd, start + n)
        out = cache.norm_rope_append(0, q if with_q else None, k, v, sid, pos, hq, table=table,
                                     q_out=q if with_q else None)
        hx.device_status()
        kv.append((kt, vt))
        assert (out is q) if with_q else out is None
    check(q.view(n, hq, hd), want, bound, "q in place")
    assert torch.equal(kv[0][0], kv[1][0]) and torch.equal(kv[0][1], kv[1][1])
    assert torch.equal(kv[0][1][:, start:], v.view(n, hkv, hd).transpose(0, 1))


def test_more_tokens_than_a_grid_has_rows(hx):
    """70,001 tokens, one in seven of them padding, over 35 sequences."""
    g = torch.Generator(device="cuda").manual_seed(9)
    hd, hq, hkv, n, each = 64, 2, 1, 70001, 2001
    q, k, v = (make(g, (n, h * hd), torch.float16) for h in (hq, hkv, hkv))
    cache = hx.KVCache(1, hkv, hd, 35, each)
    for i in range(35):
        cache.reserve(i, each)
    token = torch.arange(n, device="cuda")
    sid, pos = (token // each).int(), (token % each).int()
    pad = token % 7 == 3
    out = torch.full((n, hq * hd), 9.0, dtype=torch.float16, device="cuda")
    cache.norm_rope_append(0, q, k, v, torch.where(pad, -1, sid).int(), pos, hq, q_out=out)
    hx.device_status()
    assert bool((out[pad] == 9).all())
    y, bound = formula(q, None, 1e-6, None, hd)
    check(out.view(n, hq, hd)[~pad], y[~pad], bound[~pad], "q")
    y, bound = formula(k, None, 1e-6, None, hd)
    for i in (0, 17, 34):
        rows = slice(i * each, min(n, (i + 1) * each))
        kept = ~pad[rows]
        kr, vr = cache.read(0, i, 0, rows.stop - rows.start)
        check(kr[kept], y[rows][kept], bound[rows][kept], "k")
        assert torch.equal(vr.flatten(1)[kept], v[rows][kept])
        assert bool((kr[~kept] == 0).all()) and bool((vr[~kept] == 0).all())


def test_special_values(hx):
    """A row of zeros stays zero (eps keeps the root above 0), the largest fp16
    values normalise without overflow, and a NaN stays in its head."""
    hd, hq, hkv = 128, 2, 1
    q = torch.zeros((3, hq * hd), dtype=torch.float16, device="cuda")
    q[1] = 65504
    q[2, 3] = float("nan")
    q[2, hd:] = 1
    k = torch.ones((3, hd), dtype=torch.float16, device="cuda")
    cache = hx.KVCache(1, hkv, hd, 1, 64)
    cache.reserve(0, 64)
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    out = cache.norm_rope_append(0, q, k, k, torch.zeros_like(pos), pos, hq, eps=1e-6)
    hx.device_status()
    assert bool((out[0] == 0).all()) and bool((out[1] == 1).all())
    assert bool(out[2, :hd].isnan().all()) and bool((out[2, hd:] == 1).all())


def test_padding_rows_and_bad_rows(hx):
    """seq_ids -1 is skipped without a record; unknown sequences, positions
    outside the cache, the table or the mapped blocks are recorded and not
    written.  Rows that are left out keep what q_out and the cache held."""
    hd, hq, hkv = 64, 4, 2
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (make(g, (3, h * hd), torch.float16) for h in (hq, hkv, hkv))
    table, _, _ = tables(hx, hd, 100)
    cache = hx.KVCache(1, hkv, hd, 2, 256)
    cache.reserve(0, 64)
    pool = cache.pool()

    def run(sid, pos):
        pool.fill_(3.0)
        out = torch.full((3, hq * hd), 9.0, dtype=torch.float16, device="cuda")
        cache.norm_rope_append(0, q, k, v, torch.tensor(sid, dtype=torch.int32, device="cuda"),
                               torch.tensor(pos, dtype=torch.int32, device="cuda"), hq, table=table,
                               q_out=out)
        return out

    out = run([0, -1, 0], [4, 5, 6])
    hx.device_status()
    assert bool((out[1] == 9).all()) and not bool((out[0] == 9).any())
    kr, vr = cache.read(0, 0, 0, 64)
    assert bool((kr[5] == 3).all()) and bool((vr[5] == 3).all()) and torch.equal(vr[6].flatten(), v[2])
    for sid, pos in ((2, 5), (-2, 5), (0, -1), (0, 256), (0, 100), (1, 0), (0, 64)):
        out = run([0, sid, 0], [4, pos, 6])
        with pytest.raises(Exception) as e:
            hx.device_status()
        assert e.value.status == 2, (sid, pos)
        assert bool((out[1] == 9).all())
        kr, vr = cache.read(0, 0, 0, 64)
        kept = torch.ones(64, dtype=torch.bool, device="cuda")
        kept[[4, 6]] = False
        assert bool((kr[kept] == 3).all()) and bool((vr[kept] == 3).all())
        assert torch.equal(vr[6].flatten(), v[2])


def test_captured_on_another_stream(hx):
    """Captured in a graph on a side stream and replayed on new inputs."""
    hd, hq, hkv, n = 128, 8, 4, 6
    g = torch.Generator(device="cuda").manual_seed(8)
    qkv = make(g, (n, (hq + 2 * hkv) * hd), torch.float16)
    q, k, v = qkv.split([hq * hd, hkv * hd, hkv * hd], 1)
    cache = hx.KVCache(1, hkv, hd, n, 64, overlap=True)
    for i in range(n):
        cache.reserve(i, 64)
    sid = torch.arange(n, dtype=torch.int32, device="cuda")
    pos = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    out = torch.empty((n, hq * hd), dtype=torch.float16, device="cuda")
    table, c, s = tables(hx, hd, 64)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        cache.norm_rope_append(0, q, k, v, sid, pos, hq, table=table, q_out=out, stream=side)
    for step in range(3):
        qkv.copy_(make(g, qkv.shape, torch.float16))
        pos.fill_(3 + step)
        graph.replay()
        torch.cuda.synchronize()
        y, bound = formula(q, None, 1e-6, (c[pos.long()], s[pos.long()]), hd)
        check(out.view(n, hq, hd), y, bound, "q")
    hx.device_status()


def test_refusals(hx):
    hd, hq, hkv = 64, 4, 2
    cache = hx.KVCache(1, hkv, hd, 2, 64)
    z = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt, device="cuda")
    q, k, sid = z(3, hq * hd), z(3, hkv * hd), z(3, dt=torch.int32)
    ok = dict(q=q, k=k, v=k, seq_ids=sid, positions=sid, num_q_heads=hq)

    def call(layer=0, **kw):
        cache.norm_rope_append(layer, **{**ok, **kw})

    for bad in (dict(layer=1), dict(layer=-1), dict(num_q_heads=3, q=z(3, 3 * hd)), dict(eps=-1.0),
                dict(eps=float("nan")), dict(table=tables(hx, 32, 4)[0])):
        with pytest.raises(RuntimeError):
            call(**bad)
    for bad in (dict(q=z(2, hq * hd)), dict(q=z(hq * hd, 3).t()), dict(k=z(1, hkv * hd).expand(3, -1)),
                dict(positions=z(2, dt=torch.int32)), dict(q_weight=z(hd + 1)),
                dict(k=k.cpu()), dict(q_out=z(2, hq * hd)), dict(q=None, q_out=q)):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(k=k.float()), dict(q=q.bfloat16()), dict(seq_ids=sid.long()),
                dict(q_weight=z(hd).float())):
        with pytest.raises(TypeError):
            call(**bad)
    none = z(0, dt=torch.int32)
    cache.norm_rope_append(0, z(0, hq * hd), z(0, hkv * hd), z(0, hkv * hd), none, none, hq)
    hx.device_status()
