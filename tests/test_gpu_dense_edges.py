"""linear, rms_norm and mx8 where two rules of theirs meet, at the ends of the types, and as torch's other modes call them.
Tolerances as in test_gpu_dense.py: u = 2^-24 per fp32 addition of a sum, h = half a step per rounding to a type."""
import pytest
import torch

from tests import dense_ref as R
from tests.test_gpu_dense import TYPES, U, _check_linear, _close, _inputs

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("size", [(1024, 262144, 4), (65, 229376, 63), (4096, 262144, 1)], ids=str)
def test_two_terms_of_dz_with_filled_up_rows(size, dt):
    """a small dz over a very wide input: it goes in as two terms, and both come with their rows filled up"""
    x, w, b, _, dy = _inputs(*size, dt, seed=1)
    _check_linear(x, w, b, None, dy, "gelu")


def _mx8(x):
    """(values read back, scale exponents + 127) of quantize_mx8 in 64 bits: the smallest scale that brings the block to 448, cut
    at 240 only where 256 times the scale is infinite in the type"""
    M, K = x.shape
    b = torch.nn.functional.pad(x.double(), (0, (-K) % 32)).view(M, -1, 32)
    m, e = torch.frexp(b.abs().amax(2, keepdim=True))                        # m 2^e, m in [0.5, 1)
    E = torch.where(m > 0, e - 9 + (m > 0.875), torch.full_like(e, -126)).clamp(min=-126)
    s = R.two_to(E)
    lim = torch.where(256 * s > torch.finfo(x.dtype).max, 240.0, 448.0).to(b)
    v = torch.maximum(torch.minimum(b / s, lim), -lim)
    step = R.two_to((torch.frexp(v.abs())[1] - 4).clamp(min=-9))
    return (torch.round(v / step) * step * s).view(M, -1)[:, :K], (E + 127).view(M, -1)


@pytest.mark.parametrize("dt", HALF)
def test_mx8_over_every_value(dt):
    """every finite 16-bit number alone in its block, and beside the largest of the blocks of its binade"""
    from latte_amd import functional as LF
    every = torch.arange(65536, device="cuda").to(torch.int32).to(torch.int16).view(dt)
    every = every[torch.isfinite(every)].view(-1, 1)
    top = torch.ldexp(torch.ones((), device="cuda", dtype=torch.float64), torch.frexp(every.double())[1]) * 1.0   # next power of two
    for x in (every, torch.cat([every, (top * 0.875).to(dt), (top * 0.5).to(dt)], 1)):
        x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
        q = LF.quantize_mx8(x)
        val, sc = _mx8(x)
        assert torch.equal(q.scales.int(), sc.int()) and torch.equal(q.dequantize().double(), val)
        back = q.dequantize(dt).double()
        assert torch.equal(back, val.to(dt).double()) and bool(torch.isfinite(back).all())
        big = x.double().abs() > torch.finfo(dt).tiny * 2 ** 14              # above the scales' lower end
        assert bool(((val - x.double()).abs() <= 2.0 ** -4 * x.double().abs())[big].all())


def test_mx8_checkpoint_of_large_half_values():
    """a layer over fp16 inputs of the last binade: its weight gradient is that of values within 2^-4 of x"""
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(2)
    x = (torch.rand(64, 96, generator=g, device="cuda") * 24000 + 33000).half()
    w = (torch.randn(48, 96, generator=g, device="cuda") * 1e-4).half().requires_grad_(True)
    dy = torch.randint(-2, 3, (64, 48), generator=g, device="cuda").half() / 1024
    gw, = torch.autograd.grad(LF.linear(x, w, checkpoint="mx8"), w, dy)
    held = _mx8(x)[0]
    assert float(((held - x.double()) / x.double()).abs().max()) <= 2.0 ** -4
    want = dy.double().t() @ held
    t = 64 * U * (dy.double().abs().t() @ held.abs())
    _close(gw, want, t + R.EPS[torch.float16] * (want.abs() + t), "dw")


def test_forward_mode_is_refused():
    """a tangent is never dropped without a word, with and without a graph for the backward pass, and not in a backward pass either"""
    from latte_amd import functional as LF
    from torch.autograd import forward_ad as fw
    x, w, g, b = (torch.randn(*s, device="cuda") for s in ((6, 8), (5, 8), (8,), (5,)))
    x8, w8 = LF.quantize_mx8(x), LF.quantize_mx8(w)
    y, n = LF.linear(x, w.clone().requires_grad_(True)), LF.rms_norm(x, g.clone().requires_grad_(True))
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: LF.linear(dual(x), w), lambda: LF.linear(x, dual(w)), lambda: LF.linear(x, w, dual(b)),
                 lambda: LF.linear(x, w, residual=dual(x[:, :5])), lambda: LF.linear(dual(x), w.requires_grad_(True)),
                 lambda: LF.rms_norm(dual(x), g), lambda: LF.rms_norm(x, dual(g)), lambda: LF.rms_norm(x, g, dual(x)),
                 lambda: LF.rms_norm(dual(x), g, out="mx8"), lambda: LF.linear(x8, w8, dual(b.half())),
                 lambda: LF.batch_norm(dual(x), g.requires_grad_(True), g.detach(), checkpoint="mx8"),
                 lambda: y.backward(dual(torch.ones_like(y))), lambda: n.backward(dual(torch.ones_like(n)))]
        for grad in (False, True):
            for call in calls[:10] if not grad else calls:
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        assert fw.unpack_dual(LF.linear(fw.unpack_dual(dual(x)).primal, w.detach())).tangent is None


def test_function_transforms_are_refused():
    from latte_amd import functional as LF
    x, w = torch.randn(6, 8, device="cuda"), torch.randn(8, 8, device="cuda")
    for call in (lambda: torch.func.grad(lambda t: LF.linear(t, w).sum())(x), lambda: torch.func.vmap(lambda t: LF.linear(t, w))(x),
                 lambda: torch.func.jvp(lambda t: LF.rms_norm(t, w[0]), (x,), (x,))):
        with pytest.raises(RuntimeError):
            call()


def test_mx8_scales_at_their_ends():
    """scale bytes 0 and 255 (only a caller's own Mx8 has them) stand for 2^-127 and NaN, read back and in the matrix instruction"""
    from latte_amd import functional as LF
    v = torch.zeros(1, 32, device="cuda")
    v[0, :2] = torch.tensor([1.0, -448.0])
    one = torch.zeros(16, 32, device="cuda")
    one[0, 0] = one[1, 1] = 1
    one = LF.quantize_mx8(one)
    for byte in (0, 1, 127, 245, 255):
        q = LF.Mx8(v.to(torch.float8_e4m3fn), torch.full((1, 1), byte, dtype=torch.uint8, device="cuda"))
        want = v.double() * 2.0 ** (byte - 127) if byte < 255 else torch.full_like(v, float("nan")).double()
        assert torch.equal(torch.nan_to_num(q.dequantize().double(), nan=-7.0), torch.nan_to_num(want, nan=-7.0))
        with torch.no_grad():
            y = LF.linear(q, one)[0, :2].double()
        assert torch.equal(torch.nan_to_num(y, nan=-7.0), torch.nan_to_num(want[0, :2], nan=-7.0))


@pytest.mark.parametrize("dt", HALF)
def test_activation_tails(dt):
    """GELU and SiLU of 16-bit types far below zero keep their relative accuracy: the fp32 value is within 5e-5 of itself there (3.2e-5
    of the tail's polynomial; the exponent's argument, at most 128, is off by 2^-24 of itself twice: 1.1e-5; some last places), and
    is rounded once.  One input, weight 1, no bias: z is x."""
    from latte_amd import functional as LF
    x = -torch.linspace(0, 13, 4001, device="cuda").to(dt).view(-1, 1)
    one = torch.ones(1, 1, device="cuda", dtype=dt)
    for act in ("gelu", "silu"):
        want = R.act(x.double(), act)[0]
        for xi in (x, x[::200]):                     # tiles, few rows
            y, t = LF.linear(xi, one, act=act), R.act(xi.double(), act)[0]
            _close(y, t, (R.EPS[dt] * 1.00005 + 5e-5) * t.abs() + R.LOW[dt], act)
        assert float(want.abs().min()) == 0          # x = 0 among them


@pytest.mark.parametrize("post", [False, True])
def test_bn_residual_gradient_alone(post):
    """the residual's gradient needs no column sums: asked for alone it takes its own memory (none where it is dy itself) and
    comes out as with the others"""
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r, dy = (torch.randn(3000, 96, generator=g, device="cuda") for _ in range(3))
    leaves = [t.requires_grad_(True) for t in (x, torch.ones(96, device="cuda"), torch.zeros(96, device="cuda"), r)]
    y = LF.batch_norm(*leaves[:3], residual=r, relu=True, post_add=post, checkpoint="mx8")
    full = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    made = lambda: torch.cuda.memory_stats()["allocation.all.allocated"]  # noqa: E731
    before = made()
    alone, = torch.autograd.grad(y, r, dy, retain_graph=True)
    count = made() - before
    assert torch.equal(alone, full[3]) and torch.equal(alone, dy if post else dy * (y > 0))
    assert count <= (0 if post else 3)               # the gradient, and two unread vectors that the kernel is handed


def test_capture_over_inputs_that_were_computed_before_it():
    """the gradient of such an input leads back into an eager graph on the default stream: refused; of the others it is captured"""
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(4)
    leaf, w, n, dy, dn = (torch.randn(*s, generator=g, device="cuda") for s in ((64, 32), (48, 32), (32,), (64, 48), (64, 32)))
    leaf.requires_grad_(True)
    h, n, w = leaf * 2, n.requires_grad_(True), w.requires_grad_(True)
    calls = [(lambda: LF.linear(h, w, act="gelu", checkpoint="mx8"), w, dy), (lambda: LF.rms_norm(h, n), n, dn),
             (lambda: LF.batch_norm(h, n, n, checkpoint="mx8"), n, dn)]
    for call, other, d in calls:
        with pytest.raises(RuntimeError, match="can not be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(call(), h, d)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, = torch.autograd.grad(call(), other, d)
        want, = torch.autograd.grad(call(), other, d)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            want = torch.autograd.grad(call(), other, d)[0]


def test_lazily_negated_views():
    """the imaginary part of a conjugate is a view with a minus sign still to be carried out: in every operand it is"""
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(5)

    def neg(*s):
        t = torch.conj(torch.randn(*s, generator=g, device="cuda", dtype=torch.complex64)).imag
        flat = torch._neg_view(torch.randn(*s, generator=g, device="cuda"))
        assert t.is_neg() and flat.is_neg()
        return flat if s[-1] > 1 else t              # a single column has no stride that would ask for a copy
    real = lambda *ts: [t.resolve_neg().clone() for t in ts]  # noqa: E731
    for M, K, N in ((40, 1, 24), (40, 32, 24)):
        x, w, b, r, dy, n, beta, dx = neg(M, K), neg(N, K), neg(N), neg(M, N), neg(M, N), neg(K), neg(K), neg(M, K)
        calls = [(lambda *t: LF.linear(*t[:3], act="silu", residual=t[3]), (x, w, b, r), dy),
                 (lambda *t: LF.rms_norm(*t)[0], (x, n, dx), dx)]
        if K > 1:
            calls.append((lambda *t: LF.batch_norm(*t[:3], residual=t[3], relu=True, checkpoint="mx8"), (x, n, beta, dx), dx))
        for call, args, d in calls:
            out = []
            for ts, dd in ((args, d), (real(*args), *real(d))):
                ts = [t.detach().requires_grad_(True) for t in ts]
                y = call(*ts)
                out.append([y.detach(), *torch.autograd.grad(y, ts, dd)])
            assert all(torch.equal(a, c) for a, c in zip(*out))
        q, p = LF.quantize_mx8(x), LF.quantize_mx8(*real(x))
        assert torch.equal(q.dequantize(), p.dequantize())
        with torch.no_grad():
            assert torch.equal(LF.linear(q, LF.quantize_mx8(w), torch._neg_view(b.resolve_neg().half())), LF.linear(p, LF.quantize_mx8(*real(w)), -b.resolve_neg().half()))
            assert torch.equal(LF.rms_norm(x, n, out="mx8").dequantize(), LF.rms_norm(*real(x, n), out="mx8").dequantize())


@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("size", [(1, 512, 1000), (16, 300, 48), (40, 77, 100), (64, 128, 64), (300, 96, 130), (2048, 320, 256), (2600, 40, 129),
                                  (20000, 64, 24)], ids=str)
def test_sixteen_bit_gradients_keep_what_is_kept(size, dt, act):
    """what the backward pass of a 16-bit layer may lose, and no more: act' is within 1e-5 (its 16-bit grid), dz is rounded once for
    the products, to h^2 of itself where it goes in as two terms (up to 4096 elements, GELU and SiLU), and not at all for db"""
    from latte_amd import functional as LF
    M, K, N = size
    x, w, b, _, dy = _inputs(M, K, N, dt, seed=7)
    h, lo = R.EPS[dt], R.LOW[dt]
    t = [v.clone().requires_grad_(True) for v in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(LF.linear(*t, act=act), t, dy)
    X, W, DY = x.double(), w.double(), dy.double()
    Z = X @ W.t() + b.double()
    zerr = (K + 1) * U * (X.abs() @ W.abs().t() + b.double().abs())
    D = R.act(Z, act)[1]
    derr = torch.zeros_like(D) if act == "none" else 1e-5 + 0.8 * zerr + 3e-6 * (1 + Z.abs())
    DZ = DY * D
    zabs = DZ.abs() + DY.abs() * derr
    summed = DY.abs() * derr + 2 * U * zabs
    dzerr = summed if act == "none" else summed + (h * h if M * N <= 4096 else h) * zabs + lo
    for got, want, e, mag, n in ((gx, DZ @ W, dzerr @ W.abs(), zabs @ W.abs(), 2 * N), (gw, DZ.t() @ X, dzerr.t() @ X.abs(), zabs.t() @ X.abs(), 2 * M),
                                 (gb, DZ.sum(0), summed.sum(0), zabs.sum(0), M + 2)):
        e = e + n * U * mag
        _close(got, want, e + h * (want.abs() + e) + lo, act)


def test_rms_norm_mx8_output_beyond_half():
    """y is computed in fp32 whatever the operands' type: beyond the largest float16 it is held like any other"""
    from latte_amd import functional as LF
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(300, 96, generator=g, device="cuda").half()
    for top in (20000.0, 30000.0, 60000.0):
        w = (torch.rand(96, generator=g, device="cuda") * top + 3000).half()
        q = LF.rms_norm(x, w, eps=2.0 ** -20, out="mx8")
        X = x.double()
        Y = X / torch.sqrt(X.square().mean(1, keepdim=True) + 2.0 ** -20) * w.double()
        scale = R.two_to(q.scales.to(torch.int64) - 127).repeat_interleave(32, 1)
        bound = Y.abs() * 2.0 ** -4 + scale * 2.0 ** -10
        _close(q.dequantize(), Y, bound * (1 + 116 * U), "y8")
        assert bool((Y.abs() > 65504).any())         # x reaches 4 in 28800 draws, w 20000 and more


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M", [8, 300])
def test_infinite_gradients(dt, M):
    """an infinity in dy reaches the gradients as one, by the sign of what it meets, whether dz goes in as one term or two"""
    from latte_amd import functional as LF
    K, N = 40, 16
    x, w, b, _, dy = _inputs(M, K, N, dt, seed=9)
    w[w == 0], x[x == 0] = 1, 1                      # 0 times an infinity would be NaN
    for act in ("silu", "gelu"):
        d = dy.clone()
        d[2, 3], d[5, 7] = float("inf"), float("-inf")
        t = [v.clone().requires_grad_(True) for v in (x, w, b)]
        gx, gw, gb = torch.autograd.grad(LF.linear(*t, act=act), t, d)
        D = R.act(x.double() @ w.double().t() + b.double(), act)[1]
        for i, j, s in ((2, 3, 1.0), (5, 7, -1.0)):
            s = s * float(torch.sign(D[i, j]))
            inf = torch.tensor(float("inf"), device="cuda")
            assert torch.equal(gx[i].float(), s * torch.sign(w[j].float()) * inf) and torch.equal(gw[j].float(), s * torch.sign(x[i].float()) * inf)
            assert float(gb[j]) == s * float("inf")
        assert int((~torch.isfinite(gx)).any(1).sum()) == 2 and int((~torch.isfinite(gw)).any(1).sum()) == 2 and not bool(torch.isnan(gb).any())
