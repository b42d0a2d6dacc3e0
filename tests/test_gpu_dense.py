"""linear / mx8 on the HIP kernels against 64-bit formulas (tests/dense_ref.py), at the sizes and layouts where tiles, splits
and guards can go wrong.

Tolerances, elementwise, from the arithmetic: u = 2^-24 for each of the fp32 additions of a sum (a sum of n terms is off by
at most n u times the sum of the magnitudes), h = half a step of the type (lo: its absolute value below the normal numbers) for each rounding to it; activations are within
3e-6 (1 + |z|) in fp32 of any route taken here and have slopes of at most 1.13."""
import pytest
import torch

from tests import dense_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e} over its bound"


def _ints(g, *s, lo=-4, hi=5):
    return torch.randint(lo, hi, s, generator=g, device="cuda").double()


def _inputs(M, K, N, dt, seed=0, exact=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if exact:   # sums of these are exact in fp32 (and z is never decided by rounding)
        x, w, b, r, dy = _ints(g, M, K), _ints(g, N, K) / 8, _ints(g, N) / 8, _ints(g, M, N), _ints(g, M, N)
    else:
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        x, w, b, r, dy = rn(M, K), rn(N, K) * K ** -0.5, rn(N), rn(M, N), rn(M, N)
    return [t.to(dt) for t in (x, w, b, r, dy)]


def _check_linear(x, w, b, r, dy, act, ckpt=None):
    from latte_amd import functional as LF
    dt = x.dtype
    h, lo = R.EPS[dt], R.LOW[dt]
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = LF.linear(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3], checkpoint=ckpt)
    live = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip("xwbr", leaves) if t is not None], torch.autograd.grad(y, live, dy)))
    X, W, DY = x.double(), w.double(), dy.double()
    K, N, M = X.shape[1], W.shape[0], X.shape[0]
    Z = X @ W.t()
    mag = X.abs() @ W.abs().t()
    if b is not None:
        Z, mag = Z + b.double(), mag + b.double().abs()
    A, D = R.act(Z, act)
    zerr = (K + 1) * U * mag
    Y = A + r.double() if r is not None else A
    tol = 1.13 * zerr + (3e-6 * (1 + Z.abs()) if act in ("gelu", "silu") else 0) + 2 * U * Y.abs()
    _close(y, Y, tol + h * (Y.abs() + tol) + lo, "y")
    # what the backward pass reads: act' off by its own rounding (1/384 on the 8-bit grid) and by z's error times 0.8
    derr = torch.zeros_like(D)
    if act in ("gelu", "silu"):
        derr = 0.8 * zerr + 3e-6 * (1 + Z.abs()) + ((1 / 384 + 1e-6) if ckpt else h * D.abs() + lo)
    DZ = DY * D
    zabs = DZ.abs() + DY.abs() * derr
    dzerr = DY.abs() * derr + h * zabs + lo                # dz is rounded to the type
    Xh = R.mx8(x)[0] if ckpt else X
    dX = DZ @ W
    t = dzerr @ W.abs() + N * U * (zabs @ W.abs())
    _close(grads["x"], dX, t + h * (dX.abs() + t) + lo, "dx")
    dW = DZ.t() @ Xh
    t = dzerr.t() @ Xh.abs() + M * U * (zabs.t() @ Xh.abs())
    _close(grads["w"], dW, t + h * (dW.abs() + t) + lo, "dw")
    if b is not None:
        dB = DZ.sum(0)
        t = dzerr.sum(0) + (M + 2) * U * zabs.sum(0)
        _close(grads["b"], dB, t + h * (dB.abs() + t) + lo, "db")
    if r is not None:
        assert torch.equal(grads["r"], dy)


SIZES = [(1, 1, 1), (1, 64, 64), (2, 33, 17), (5, 128, 96), (16, 1000, 48), (17, 64, 256), (63, 40, 130), (64, 256, 33), (65, 72, 64),
         (130, 65, 129), (257, 96, 32), (300, 512, 20), (1000, 48, 72), (777, 200, 311), (2048, 320, 256), (5000, 32, 256)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_sizes(size, dt):
    M, K, N = size
    x, w, b, r, dy = _inputs(M, K, N, dt)
    _check_linear(x, w, b, r, dy, "none")
    _check_linear(x, w, None, None, dy, "gelu")


@pytest.mark.parametrize("ckpt", [None, "mx8"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", [(3, 40, 24), (200, 96, 50), (1031, 256, 144)], ids=str)
def test_linear_act_and_checkpoint(size, dt, act, ckpt):
    x, w, b, r, dy = _inputs(*size, dt, seed=1, exact=act == "relu")
    _check_linear(x, w, b, r, dy, act, ckpt)
    _check_linear(x, w, b, None, dy, act, ckpt)


@pytest.mark.parametrize("dt", TYPES)
def test_linear_large_tiles(dt):
    """shapes that take the widest tiles in forward and backward, with odd edges"""
    for M, K, N in ((4100, 1032, 3000), (3000, 2056, 4104)):
        x, w, b, r, dy = _inputs(M, K, N, dt, seed=2)
        _check_linear(x, w, b, r, dy, "silu")


@pytest.mark.parametrize("dt", TYPES)
def test_linear_strides(dt):
    """rows with a stride, at any alignment, repeated rows, transposed weights, leading dimensions"""
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(90, 203, generator=g, device="cuda").to(dt)
    wt = torch.randn(70, 44, generator=g, device="cuda").to(dt)
    for x in (big[:, 3:73], big[::2, 1:71], big[:, 133:], big[:1].expand(90, 203)[:, 5:75], big[:, :140:2]):
        w = wt.t()                                     # [44, 70], columns along memory
        r = big[:1, :44].expand(x.shape[0], 44)
        y = LF.linear(x, w, residual=r)
        Y = x.double() @ w.double().t() + r.double()
        tol = 72 * U * (x.double().abs() @ w.double().abs().t() + r.double().abs())
        _close(y, Y, tol + R.EPS[dt] * (Y.abs() + tol) + R.LOW[dt], "y")
    x = big[:60, :180].reshape(3, 20, 180).transpose(0, 1).requires_grad_(True)      # no 2-D view exists
    w = wt.reshape(-1)[:180 * 17].reshape(17, 180).contiguous().requires_grad_(True)
    y = LF.linear(x, w)
    assert y.shape == (20, 3, 17)
    dy = torch.randn(3, 20, 17, generator=g, device="cuda").to(dt).transpose(0, 1)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    want = dy.double().reshape(60, 17) @ w.detach().double()
    tol = 20 * U * (dy.double().abs().reshape(60, 17) @ w.detach().double().abs())
    _close(gx.reshape(60, 180), want, tol + R.EPS[dt] * (want.abs() + tol) + R.LOW[dt], "dx")
    one = LF.linear(big[0, :180], w)
    assert one.shape == (17,) and torch.equal(one, LF.linear(big[:1, :180], w)[0])


@pytest.mark.parametrize("dt", TYPES)
def test_linear_no_rows(dt):
    from latte_amd import functional as LF
    x = torch.zeros(0, 24, device="cuda", dtype=dt, requires_grad=True)
    w = torch.ones(40, 24, device="cuda", dtype=dt, requires_grad=True)
    b = torch.ones(40, device="cuda", dtype=dt, requires_grad=True)
    for ck in (None, "mx8"):
        y = LF.linear(x, w, b, act="gelu", checkpoint=ck)
        assert y.shape == (0, 40)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert gx.shape == (0, 24) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0


def test_linear_non_finite_values_stay_where_they_belong():
    """a NaN or an infinity reaches the outputs of its own row (or, in the weights, its own column) and no others"""
    from latte_amd import functional as LF
    for dt in TYPES:
        for M, K, N in ((40, 70, 50), (300, 136, 160)):
            x, w, b, _, _ = _inputs(M, K, N, dt, seed=4)
            clean = LF.linear(x, w, b, act="relu")
            x2 = x.clone()
            x2[7, 3], x2[M - 1, K - 1] = float("nan"), float("inf")
            y = LF.linear(x2, w, b, act="relu")
            keep = [i for i in range(M) if i not in (7, M - 1)]
            assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[7]).all())
            w2 = w.clone()
            w2[N - 1, 0] = float("nan")
            y = LF.linear(x, w2, b)
            assert bool(torch.isnan(y[:, N - 1]).all()) and not bool(torch.isnan(y[:, :N - 1]).any())


def test_linear_backward_is_reproducible_and_partial():
    """the same bits every time; leaves that need no gradient cost none and change nothing"""
    from latte_amd import functional as LF
    x, w, b, r, dy = _inputs(20000, 64, 96, torch.float32, seed=5)
    def run(need):
        t = [v.clone().requires_grad_(n) for v, n in zip((x, w, b), need)]
        y = LF.linear(*t, act="silu", checkpoint="mx8")
        return torch.autograd.grad(y, [v for v in t if v.requires_grad], dy)
    full = run((True, True, True))
    assert all(torch.equal(a, c) for a, c in zip(full, run((True, True, True))))
    for i in range(3):
        need = [j == i for j in range(3)]
        assert torch.equal(run(need)[0], full[i])


def test_linear_gradients_by_differences():
    """the derivative along a random direction, by central differences of the 64-bit formula at the same point"""
    x, w, b, r, dy = _inputs(37, 29, 23, torch.float32, seed=6)
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(7)
    for act in ("gelu", "silu"):
        t = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
        grads = torch.autograd.grad(LF.linear(t[0], t[1], t[2], act=act, residual=t[3]), t, dy)
        dirs = [torch.randn(v.shape, generator=g, device="cuda").double() for v in (x, w, b, r)]
        def f(e):
            X, W, B, Rr = (v.double() + e * d for v, d in zip((x, w, b, r), dirs))
            return float(((R.act(X @ W.t() + B, act)[0] + Rr) * dy.double()).sum())
        e = 1e-5
        num = (f(e) - f(-e)) / (2 * e)
        ana = sum(float((gr.double() * d).sum()) for gr, d in zip(grads, dirs))
        mag = sum(float((gr.double() * d).abs().sum()) for gr, d in zip(grads, dirs))
        assert abs(num - ana) < 1e-5 * mag, (act, num, ana)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", [(1, 1), (1, 31), (3, 32), (7, 33), (50, 100), (129, 1001), (1, 5000)], ids=str)
def test_mx8_values_and_scales(size, dt):
    """bit for bit what the definition says, over the whole range of the type"""
    from latte_amd import functional as LF
    M, K = size
    g = torch.Generator(device="cuda").manual_seed(8)
    ex = torch.randint(-12, 13, (M, K), generator=g, device="cuda")
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.ldexp(torch.ones(M, K, device="cuda"), ex)).to(dt)
    q = LF.quantize_mx8(x)
    val, sc = R.mx8(x)
    assert torch.equal(q.scales.int(), sc.int()) and torch.equal(q.dequantize().double(), val)
    assert torch.equal(q.dequantize(torch.bfloat16).double(), val)


def test_mx8_borders():
    """ties, the largest and smallest magnitudes of each type, zeros, non-finite elements"""
    from latte_amd import functional as LF
    for dt in TYPES:
        fi = torch.finfo(dt)
        rows = [[0.0] * 4, [fi.max, -fi.max, 1.0, 0.0], [fi.tiny, -fi.tiny, fi.tiny / 2, 0.0], [448.0, 449.0, 17.0, 19.0],
                [float("nan"), 2.0, float("inf"), -3.0], [float("nan")] * 4, [1.0625, 1.1875, 1.75, 0.875], [fi.max / 2, fi.max / 4, 8.0, 1.0]]
        x = torch.zeros(len(rows), 40, dtype=torch.float64)
        x[:, 30:34] = torch.tensor(rows, dtype=torch.float64)      # across the border of two blocks
        x = x.to(dt).cuda()
        q = LF.quantize_mx8(x)
        val, sc = R.mx8(x)
        got = q.dequantize().double()
        assert torch.equal(q.scales.int(), sc.int())
        assert torch.equal(torch.nan_to_num(got, nan=-7.0), torch.nan_to_num(val, nan=-7.0))
        back = q.dequantize(dt).double()
        fin = torch.isfinite(x)
        assert bool(torch.isfinite(back[fin]).all()) and not bool(torch.isfinite(back[~fin]).any())
        big = fin & (x.abs() > fi.tiny * 2 ** 14)
        rel = ((back - x.double()).abs() / x.double().abs())[big]
        assert float(rel.max()) <= 2.0 ** -4


def test_linear_mx8_checkpoint_holds_a_quarter():
    """between forward and backward a checkpointed layer holds 1 + 1/32 bytes an input element and 1 a derivative"""
    from latte_amd import functional as LF
    x = torch.randn(4096, 512, device="cuda", requires_grad=True)
    w = torch.randn(512, 512, device="cuda", requires_grad=True)
    held = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731  (what was asked for, not its blocks)
    before = held()
    y = LF.linear(x, w, act="gelu", checkpoint="mx8")
    assert held() - before == y.numel() * 4 + 4096 * (512 + 16 + 512)
    assert torch.equal(y, LF.linear(x, w, act="gelu"))


def test_linear_in_a_graph_on_another_stream():
    """forward and backward captured together, replayed over new inputs between eager work; two graphs share no workspace"""
    from latte_amd import functional as LF
    x, w, b, r, dy = _inputs(3000, 96, 64, torch.float32, seed=9)
    def step(t, d):
        y = LF.linear(t[0], t[1], t[2], act="silu", residual=t[3], checkpoint="mx8")
        return (y.detach(),) + torch.autograd.grad(y, t, d)
    graphs = []
    for _ in range(2):
        t = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
        d = dy.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(t, d)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(t, d)
        graphs.append((gr, t, d, out))
    for k in range(4):
        wants = []
        for j, (gr, t, d, out) in enumerate(graphs):
            n = _inputs(3000, 96, 64, torch.float32, seed=20 + 2 * k + j)
            with torch.no_grad():
                for dst, src in zip(t + [d], n):
                    dst.copy_(src)
            wants.append([v.clone() for v in step([v.detach().clone().requires_grad_(True) for v in t], d)])
        for gr, *_ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (gr, t, d, out), want in zip(graphs, wants):
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_linear_on_another_stream_matches():
    from latte_amd import functional as LF
    x, w, b, r, dy = _inputs(5000, 128, 96, torch.bfloat16, seed=10)
    want = LF.linear(x, w, b, act="gelu", residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = LF.linear(x, w, b, act="gelu", residual=r)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


ROWS = [(8192, 32, 256), (8200, 128, 96), (9001, 96, 20), (8193, 256, 64), (2048, 64, 64), (2049, 33, 65), (3000, 130, 100), (2500, 256, 128),
        (2100, 100, 256), (20000, 17, 5), (8197, 250, 31), (256, 64, 17), (300, 128, 96), (3001, 96, 10), (40000, 96, 9),
        (1000, 256, 250), (2600, 40, 129)]


@pytest.mark.parametrize("ckpt", [None, "mx8"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", ROWS, ids=str)
def test_linear_long_and_narrow(size, dt, ckpt):
    """the one-pass kernels over many rows, with odd widths and a cut last tile"""
    x, w, b, r, dy = _inputs(*size, dt, seed=11, exact=True)
    _check_linear(x, w, b, r, dy, "relu", ckpt)
    x, w, b, r, dy = _inputs(*size, dt, seed=12)
    _check_linear(x, w, b, None, dy, "silu", ckpt)
    _check_linear(x[:, 1:], w[:, 1:], None, r, dy, "none", ckpt) if size[1] > 1 else None


@pytest.mark.parametrize("ckpt", [None, "mx8"])
@pytest.mark.parametrize("dt", TYPES)
def test_linear_large_odd_sizes(dt, ckpt):
    """lines that are no multiple of 16 bytes, large enough for copies with their lines filled up"""
    for M, K, N in ((2500, 1001, 1003), (2300, 1002, 1100)) if dt is torch.float32 else ((9000, 1001, 1505), (9001, 1000, 1503), (8999, 1003, 1504)):
        x, w, b, r, dy = _inputs(M, K, N, dt, seed=4)
        _check_linear(x, w, b, r, dy, "gelu" if K == 1001 else "none", ckpt)


@pytest.mark.parametrize("dt", TYPES)
def test_linear_large_odd_sizes_layouts_and_values(dt):
    """the same from strided operands, and non-finite values that stay in their rows and columns; each gradient alone has the same bits"""
    from latte_amd import functional as LF
    M, K, N = (2500, 1001, 1003) if dt is torch.float32 else (9000, 1001, 1505)
    x, w, b, r, dy = _inputs(M, K, N, dt, seed=5)
    wide = torch.full((M, K + 6), float("nan"), device="cuda", dtype=dt)
    wide[:, 3:K + 3] = x
    xs, ws, dys = wide[:, 3:K + 3], w.t().contiguous().t(), torch.cat([dy, dy], 1)[:, N:]
    out = []
    for a, c, d in ((x, w, dy), (xs, ws, dys)):
        a, c = a.requires_grad_(True), c.requires_grad_(True)
        y = LF.linear(a, c, b, act="silu")
        both = torch.autograd.grad(y, (a, c), d, retain_graph=True)
        assert torch.equal(both[1], torch.autograd.grad(y, c, d, retain_graph=True)[0])
        assert torch.equal(both[0], torch.autograd.grad(y, a, d)[0])
        out.append((y.detach(), *both))
    assert all(torch.equal(p, q) for p, q in zip(*out))
    x2, dy2 = x.detach().clone(), dy.clone()
    x2[7, K - 1], dy2[11, N - 1] = float("nan"), float("inf")
    x2.requires_grad_(True)
    y = LF.linear(x2, w, b)
    assert torch.isnan(y[7]).all() and torch.isfinite(y).all(1).sum() == M - 1
    gx, gw = torch.autograd.grad(y, (x2, w), dy2)
    assert (~torch.isfinite(gx)).any(1).nonzero().flatten().tolist() == [11]
    assert (~torch.isfinite(gw[:-1])).any(0).nonzero().flatten().tolist() == [K - 1] and not torch.isfinite(gw[-1]).any()


@pytest.mark.parametrize("act", ["none", "silu", "relu"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_linear_long_with_many_odd_columns(dt, act):
    """an odd number of columns, few inputs: dz comes with its lines filled up where there is an act', dy as it is else"""
    x, w, b, r, dy = _inputs(40001, 96, 511, dt, seed=6, exact=act == "relu")
    _check_linear(x, w, b, r, dy, act)
