"""4-bit weights: layout, quantisation and hx_w4_linear against 64 bits.

Tolerance: the codes minus their zero point and the fp16 x are exact, so only
the fp32 sums round.  A sum of K products is off by at most (K + 2) 2^-24 of
the sum of their magnitudes, the scale, the eight partial sums and the bias
add 12 2^-24 of it, and the store half a step of the stored type.  For one or
two tokens x itself is rounded to 23-bit fixed point first: its step is
2^(floor(log2 m) - 21) for m the group's largest |x|, so each x is off by at
most half of that, 2^-22 m, and y by 2^-22 sum_g m_g sum_(k in g) |w|.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def w4():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hxinfer_b200 import kv, w4
    kv.load()
    return w4


def weight(g, o, k, group, zeros):
    codes = torch.randint(0, 16, (o, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((o, k // group), generator=g, device="cuda") * 0.02).half()
    z = torch.randint(0, 16, (o, k // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    zf = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    return codes, scales, z, (codes.double() - zf) * scales.double().repeat_interleave(group, 1)


def check(got, x, dense, bias, group):
    want = x.double() @ dense.T
    mag = x.double().abs() @ dense.abs().T
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    bound = (dense.shape[1] + 14) * 2.0 ** -24 * mag
    if x.shape[0] <= 2:
        m = x.double().abs().view(x.shape[0], -1, group).amax(-1)
        bound = bound + 2.0 ** -22 * m @ dense.abs().view(dense.shape[0], -1, group).sum(-1).T
    fi = torch.finfo(got.dtype)
    lim = bound + fi.eps / 2 * torch.clamp(want.abs() + bound, min=fi.smallest_normal)
    err = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= lim).all()), f"off by {(err - lim).max().item():.3e} past the bound"


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,o,k", [(1, 1, 128), (1, 16, 256), (2, 17, 384), (7, 33, 128), (8, 64, 1024),
                                   (9, 100, 640), (16, 48, 2048), (17, 31, 896), (32, 16, 128),
                                   (33, 20, 256), (70, 47, 512), (3, 515, 4096), (1, 130, 8192), (2, 2400, 1024),
                                   (1, 5000, 640), (24, 77, 256), (5, 4800, 384), (14, 9500, 256)])
def test_matches_64_bits(w4, group, zeros, n, o, k):
    g = torch.Generator(device="cuda").manual_seed(n * o + k)
    codes, scales, z, dense = weight(g, o, k, group, zeros)
    x = torch.randn((n, k), generator=g, device="cuda").half()
    bias = torch.randn(o, generator=g, device="cuda").half() if n % 2 else None
    w = w4.W4Weight(codes, scales, z)
    out = torch.full((n + 1, o), 5.0, dtype=torch.float16, device="cuda")
    assert w4.w4_linear(x, w, bias=bias, out=out[:n]).data_ptr() == out.data_ptr()
    check(out[:n], x, dense, bias, group)
    assert bool((out[n] == 5).all())  # rows behind the last token
    check(w4.w4_linear(x, w, bias=bias, out_dtype=torch.float32), x, dense, bias, group)


@pytest.mark.parametrize("k", [32, 96, 160, 224, 288])
def test_inputs_that_end_inside_a_unit(w4, k):
    """Groups of 32 whose inputs are no multiple of the kernel's 128."""
    g = torch.Generator(device="cuda").manual_seed(k)
    codes, scales, z, dense = weight(g, 40, k, 32, True)
    x = torch.randn((5, k), generator=g, device="cuda").half()
    check(w4.w4_linear(x, w4.W4Weight(codes, scales, z), out_dtype=torch.float32), x, dense, None, 32)


@pytest.mark.parametrize("n", [1, 2])
def test_groups_of_unlike_size(w4, n):
    """Inputs over fp16's whole range, group by group: zeros, subnormals, the
    largest values, one large input among small ones; exact where x has few bits."""
    g = torch.Generator(device="cuda").manual_seed(n)
    codes, scales, z, dense = weight(g, 50, 640, 64, True)
    x = torch.randn((n, 640), generator=g, device="cuda")
    size = torch.tensor([0.0, 2.0 ** -24, 1e-6, 1e-3, 1.0, 1.0, 100.0, 9000.0, 1.0, 0.0], device="cuda")
    x = (x * size.repeat_interleave(64)).half()
    x[:, 300] = 60000.0
    w = w4.W4Weight(codes, scales, z)
    check(w4.w4_linear(x, w, out_dtype=torch.float32), x, dense, None, 64)
    whole = torch.randint(-2000, 2001, (n, 640), generator=g, device="cuda").half()
    ones = w4.W4Weight(codes, torch.ones_like(scales), z)
    exact = whole.double() @ (codes.double() - z.double().repeat_interleave(64, 1)).T
    assert torch.equal(w4.w4_linear(whole, ones, out_dtype=torch.float32).double(), exact)


@pytest.mark.parametrize("n", [1, 2])
def test_special_values_in_one_or_two_tokens(w4, n):
    g = torch.Generator(device="cuda").manual_seed(4)
    codes, scales, z, dense = weight(g, 24, 256, 64, False)
    w = w4.W4Weight(codes, scales, z)
    for value in (float("inf"), float("-inf"), float("nan")):
        x = torch.randn((n, 256), generator=g, device="cuda").half()
        clean = w4.w4_linear(x, w)
        x[0, 70] = value
        got = w4.w4_linear(x, w)
        assert not bool(got[0].isfinite().any()) and torch.equal(got[1:], clean[1:])


def test_many_inputs(w4):
    """More inputs than the one-token kernel keeps in shared memory."""
    g = torch.Generator(device="cuda").manual_seed(5)
    codes, scales, z, dense = weight(g, 20, 40960, 128, False)
    for n in (1, 2, 3):
        x = torch.randn((n, 40960), generator=g, device="cuda").half()
        check(w4.w4_linear(x, w4.W4Weight(codes, scales, z), out_dtype=torch.float32), x, dense, None, 128)


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("n,o,k", [(33, 129, 128), (34, 1, 1152), (64, 100, 4096), (65, 4099, 384), (40, 19000, 256),
                                   (63, 38000, 640), (127, 9472, 1024), (128, 15000, 896), (300, 7111, 512),
                                   (1000, 2049, 256), (150, 260, 2176)])
def test_many_tokens(w4, n, o, k, group, zeros):
    """Past 32 tokens: one tile shared by up to eight CTAs, several tiles of a
    CTA, outputs and tokens that end inside a tile."""
    g = torch.Generator(device="cuda").manual_seed(n + o + k)
    codes, scales, z, dense = weight(g, o, k, group, zeros)
    x = torch.randn((n, k), generator=g, device="cuda").half()
    bias = torch.randn(o, generator=g, device="cuda").half() if n % 2 else None
    w = w4.W4Weight(codes, scales, z)
    out = torch.full((n + 1, o), 5.0, dtype=torch.float16, device="cuda")
    w4.w4_linear(x, w, bias=bias, out=out[:n])
    check(out[:n], x, dense, bias, group)
    assert bool((out[n] == 5).all())
    y = w4.w4_linear(x, w, bias=bias, out_dtype=torch.float32)
    check(y, x, dense, bias, group)
    assert torch.equal(y, w4.w4_linear(x, w, bias=bias, out_dtype=torch.float32))  # sums in a fixed order


@pytest.mark.parametrize("n", [33, 64, 128])
@pytest.mark.parametrize("k", [32, 96, 160, 288])
def test_many_tokens_with_inputs_that_end_inside_a_unit(w4, n, k):
    g = torch.Generator(device="cuda").manual_seed(k + n)
    codes, scales, z, dense = weight(g, 150, k, 32, True)
    x = torch.randn((n, k), generator=g, device="cuda").half()
    check(w4.w4_linear(x, w4.W4Weight(codes, scales, z), out_dtype=torch.float32), x, dense, None, 32)


def test_a_token_of_infinities_and_nan_stays_alone(w4):
    g = torch.Generator(device="cuda").manual_seed(44)
    codes, scales, z, dense = weight(g, 300, 512, 64, True)
    w = w4.W4Weight(codes, scales, z)
    for n in (2, 7, 20, 40, 130):
        x = torch.randn((n, 512), generator=g, device="cuda").half()
        x[1, 5], x[1, 300] = float("inf"), float("nan")
        y = w4.w4_linear(x, w, out_dtype=torch.float32)
        keep = torch.arange(n, device="cuda") != 1
        assert bool(torch.isnan(y[1]).all())
        want = x[keep].double() @ dense.T
        lim = 530 * 2.0 ** -24 * (x[keep].double().abs() @ dense.abs().T)
        if n == 2:
            m = x[keep].double().abs().view(1, -1, 64).amax(-1)
            lim = lim + 2.0 ** -22 * m @ dense.abs().view(300, -1, 64).sum(-1).T
        assert bool(((y[keep].double() - want).abs() <= lim + 2.0 ** -24 * want.abs()).all())


def test_many_tokens_replayed_as_a_graph(w4):
    """Three products in a row, each reading the one before, as programmatic
    dependents; then the same graph on other inputs."""
    g = torch.Generator(device="cuda").manual_seed(45)
    ws = []
    for o, k in ((512, 256), (1024, 512), (256, 1024)):
        codes, scales, z, _ = weight(g, o, k, 128, True)
        ws.append(w4.W4Weight(codes, scales, z))
    x = torch.randn((50, 256), generator=g, device="cuda").half()

    def run():
        y = x
        for w in ws:
            y = w4.w4_linear(y, w)
        return y

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for seed in (1, 2):
        x.copy_(torch.randn((50, 256), generator=g, device="cuda").half() * 0.1 * seed)
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, run())


@pytest.mark.parametrize("n,o,k,group", [(1, 152064, 256, 64), (2, 152064, 256, 64), (2, 37888, 3584, 128),
                                         (1, 70001, 1152, 32), (1, 5, 16384, 128)])
def test_wide_weights(w4, n, o, k, group):
    """A vocabulary's worth of outputs (more tiles than one round of CTAs keeps
    sums of), and few outputs of many inputs."""
    g = torch.Generator(device="cuda").manual_seed(o)
    codes, scales, z, dense = weight(g, o, k, group, True)
    x = torch.randn((n, k), generator=g, device="cuda").half()
    check(w4.w4_linear(x, w4.W4Weight(codes, scales, z), out_dtype=torch.float32), x, dense, None, group)


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("k", [128, 384, 1024, 1152, 2432, 8064])
def test_pairs_of_warps_that_share_inputs(w4, n, k):
    """Tiles enough that two warps take the same units of x, which they put
    into fixed point together: units of a way from one (the second warp has
    none) to eight; the same bits every time."""
    g = torch.Generator(device="cuda").manual_seed(k + n)
    codes, scales, z, dense = weight(g, 14300, k, 128, True)
    w = w4.W4Weight(codes, scales, z)
    x = torch.randn((n, k), generator=g, device="cuda").half()
    y = w4.w4_linear(x, w, out_dtype=torch.float32)
    check(y, x, dense, None, 128)
    for _ in range(20):
        assert torch.equal(y, w4.w4_linear(x, w, out_dtype=torch.float32))


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("ratio", [1e3, 3e4, 6e5])
def test_a_large_input_under_a_zero_weight(w4, n, ratio):
    """One input far above its group that every weight takes times zero: the
    others keep their bits.  x is off by half a unit at most, 2^-30 of the
    largest.  Signed digits d_j of f in base 256 have sum |d_j| 256^j <= 3.1 |f|:
    those below the top one, j, add up to 0.51 256^j at most and |f| is 0.49 256^j
    at least.  So the sums round by (K + 14) 2^-24 of 3.1 sum |w x|, x as it is
    held; what a group sums up are exact integers."""
    g = torch.Generator(device="cuda").manual_seed(int(ratio) + n)
    codes, scales, z, _ = weight(g, 200, 512, 128, True)
    zw = z.repeat_interleave(128, 1)
    codes[:, ::128] = zw[:, ::128]
    dense = (codes.double() - zw.double()) * scales.double().repeat_interleave(128, 1)
    x = (torch.randn((n, 512), generator=g, device="cuda") * 6e4 / ratio).half()
    x[:, ::128] = 6e4
    y = w4.w4_linear(x, w4.W4Weight(codes, scales, z), out_dtype=torch.float32)
    want = x.double() @ dense.T
    unit = 2.0 ** -30 * 6e4 * dense.abs().sum(-1)
    lim = unit + (512 + 14) * 2.0 ** -24 * 3.1 * (x.double().abs() @ dense.abs().T + unit)
    err = (y.double() - want).abs()
    assert bool((err <= lim).all()), f"off by {(err - lim).max().item():.3e} past the bound"
    assert bool((lim <= 2e-3 * (x.double().abs() @ dense.abs().T)).all())  # the bound says something


def test_every_code_and_zero_point_is_exact(w4):
    """x = unit vectors and scale 1 read every weight back exactly."""
    codes = torch.arange(16, dtype=torch.uint8, device="cuda").repeat(16, 8)
    zeros = torch.arange(16, dtype=torch.uint8, device="cuda")[:, None].contiguous()
    w = w4.W4Weight(codes, torch.ones((16, 1), dtype=torch.float16, device="cuda"), zeros)
    got = w4.w4_linear(torch.eye(128, dtype=torch.float16, device="cuda"), w)
    assert torch.equal(got, (codes.half() - zeros.half()).T)


def test_infinities_and_nan_stay_in_their_row(w4):
    g = torch.Generator(device="cuda").manual_seed(3)
    codes, scales, z, dense = weight(g, 24, 256, 64, False)
    x = torch.randn((4, 256), generator=g, device="cuda").half()
    clean = w4.w4_linear(x, w4.W4Weight(codes, scales, z))
    bad = x.clone()
    bad[1, 7], bad[2, 200] = float("inf"), float("nan")
    got = w4.w4_linear(bad, w4.W4Weight(codes, scales, z))
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])
    assert not bool(got[1].isfinite().any())  # inf * 0 is NaN
    assert bool(got[2].isnan().all())


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(w4, group):
    """Codes and scales are those of exact arithmetic: half-way values, a group
    of zeros, one of subnormals, and the largest fp16."""
    g = torch.Generator(device="cuda").manual_seed(group)
    w = torch.randn((37, 512), generator=g, device="cuda").half()
    w[0, :group] = 0
    w[1] = torch.randint(-9, 10, (512,), generator=g, device="cuda").half() * 2.0 ** -24
    w[2] = 65504 * torch.sign(torch.randn(512, generator=g, device="cuda")).half()
    w[3] = torch.randint(-14, 15, (512,), generator=g, device="cuda").half() / 2  # ties at scale 1
    w[3, ::group] = 7
    codes, scales = w4.w4_quantize(w, group)
    wd = w.double().view(37, -1, group)
    s = (wd.abs().amax(-1) / 7).half()
    assert torch.equal(scales, s)
    sd = s.double()[..., None]
    want = torch.where(sd > 0, (wd / sd.clamp(min=1e-30)).round().clamp(-8, 7), torch.zeros_like(wd)) + 8
    assert torch.equal(codes.double().view_as(want), want)
    x = torch.randn((2, 512), generator=g, device="cuda").half()
    dense = ((want - 8) * sd).view(37, 512)
    check(w4.w4_linear(x, w4.W4Weight.quantize(w, group), out_dtype=torch.float32), x, dense, None, group)


def test_captured_on_another_stream(w4):
    g = torch.Generator(device="cuda").manual_seed(11)
    codes, scales, z, dense = weight(g, 96, 512, 128, True)
    w = w4.W4Weight(codes, scales, z)
    x = torch.zeros((3, 512), dtype=torch.float16, device="cuda")
    out = torch.empty((3, 96), dtype=torch.float16, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        w4.w4_linear(x, w, out=out, stream=side)
    for _ in range(2):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        check(out, x, dense, None, 128)


def test_refusals(w4):
    z = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt, device="cuda")
    u8 = torch.uint8
    w = w4.W4Weight(z(16, 256, dt=u8), z(16, 2))
    assert w4.w4_linear(z(0, 256), w).shape == (0, 16)
    for args in ((z(16, 256, dt=u8), z(15, 2)), (z(16, 256, dt=u8), z(16, 3)), (z(256, dt=u8), z(2)),
                 (z(16, 256, dt=u8), z(16, 2), z(16, 1, dt=u8)), (z(256, 16, dt=u8).t(), z(16, 2)),
                 (z(16, 256, dt=u8).cpu(), z(16, 2))):
        with pytest.raises(ValueError):
            w4.W4Weight(*args)
    with pytest.raises(RuntimeError):
        w4.W4Weight(z(16, 256, dt=u8), z(16, 1))  # groups of 256
    for args in ((z(16, 256), z(16, 2)), (z(16, 256, dt=u8), z(16, 2, dt=torch.float32))):
        with pytest.raises(TypeError):
            w4.W4Weight(*args)
    for kw in (dict(x=z(2, 128)), dict(x=z(256)), dict(x=z(256, 2).t()), dict(bias=z(15)),
               dict(out=z(3, 16)), dict(out=z(16, 2).t())):
        with pytest.raises(ValueError):
            w4.w4_linear(**{**dict(x=z(2, 256), weight=w), **kw})
    for kw in (dict(x=z(2, 256).float()), dict(out=z(2, 16).bfloat16()), dict(bias=z(16).float())):
        with pytest.raises(TypeError):
            w4.w4_linear(**{**dict(x=z(2, 256), weight=w), **kw})
    with pytest.raises(RuntimeError):
        w4.w4_linear(z(600).view(-1)[4:516].view(2, 256), w)  # 8-byte aligned
    with pytest.raises(ValueError):
        w4.w4_quantize(z(4, 100), 32)


@pytest.mark.parametrize("n", [1, 2, 5, 30, 40, 130])
def test_a_weight_past_32_bits(w4, n):
    """2.3e9 codes: the last rows against 64 bits."""
    o, k, group = 140001, 16384, 128
    g = torch.Generator(device="cuda").manual_seed(n)
    codes = torch.randint(0, 16, (o, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((o, k // group), generator=g, device="cuda") * 0.02).half()
    x = torch.randn((n, k), generator=g, device="cuda").half()
    y = w4.w4_linear(x, w4.W4Weight(codes, scales), out_dtype=torch.float32)
    last = slice(o - 50, o)
    dense = (codes[last].double() - 8) * scales[last].double().repeat_interleave(group, 1)
    check(y[:, last].contiguous(), x, dense, None, group)


@pytest.mark.parametrize("n", [1, 5, 50])
def test_first_call_of_a_process_inside_a_capture(w4, n):
    """Nothing that a call sets up on its first use breaks a capture (a process of its own)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = f"""
import torch
from hxinfer_b200 import w4
g = torch.Generator(device="cuda").manual_seed(3)
codes, scales = w4.w4_quantize(torch.randn((300, 256), generator=g, device="cuda").half(), 64)
w, x = w4.W4Weight(codes, scales), torch.randn(({n}, 256), generator=g, device="cuda").half()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = w4.w4_linear(x, w)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, w4.w4_linear(x, w)) and bool(y.isfinite().all())
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
