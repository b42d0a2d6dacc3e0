"""The dense operators as a program uses them: refusals on the GPU, long matrices, several streams and threads, the TTA step."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rn(seed, dt, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device="cuda").to(dt) for s in shapes]


def test_refusals():
    from latte_amd import functional as LF
    x, w, b, r = _rn(0, torch.float32, (5, 8), (6, 8), (6,), (5, 6))
    with pytest.raises(TypeError, match="weight"):
        LF.linear(x, w.half())
    with pytest.raises(TypeError, match="bias"):
        LF.linear(x, w, b.bfloat16())
    with pytest.raises(TypeError, match="expected float32"):
        LF.linear(x.double(), w.double())
    with pytest.raises(TypeError, match="operands' type"):
        LF.linear(x, w, dtype=torch.float16)
    for bad in (w[:, :7], w[:0], w[0], torch.zeros(6, 0, device="cuda")):
        with pytest.raises(ValueError):
            LF.linear(x, bad)
    with pytest.raises(ValueError, match="bias"):
        LF.linear(x, w, b[:5])
    with pytest.raises(ValueError, match="residual"):
        LF.linear(x, w, residual=r[:1])
    with pytest.raises(ValueError, match="on cpu"):
        LF.linear(x, w.cpu())
    with pytest.raises(ValueError, match="weight"):
        LF.rms_norm(x, b)
    with pytest.raises(ValueError, match="16384"):
        LF.rms_norm(torch.zeros(2, 16385, device="cuda"), torch.zeros(16385, device="cuda"))
    q = LF.quantize_mx8(x)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        LF.linear(q, LF.quantize_mx8(w), dtype=torch.float32)
    with pytest.raises(ValueError):
        LF.linear(q, LF.quantize_mx8(w[:, :7]))
    with pytest.raises(TypeError):
        LF.quantize_mx8(torch.zeros(3, 4, dtype=torch.int32, device="cuda"))
    bg = b.half().requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        LF.linear(q, LF.quantize_mx8(w), bg)
    with pytest.raises(RuntimeError, match="no gradient"):
        LF.rms_norm(x.requires_grad_(True), torch.ones(8, device="cuda"), out="mx8")
    y = LF.linear(x, w, act="gelu").sum()
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(y, x, create_graph=True)
    with pytest.raises(ValueError, match="more than 1 value"):
        LF.batch_norm(torch.zeros(1, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda"), torch.zeros(8, device="cuda"),
                      checkpoint="mx8")
    with pytest.raises(RuntimeError, match="multiple of 4"):
        LF.batch_norm(torch.zeros(5, 6, device="cuda", requires_grad=True), torch.ones(6, device="cuda"), torch.zeros(6, device="cuda"),
                      checkpoint="mx8")


def test_changed_inputs_are_noticed():
    """a leaf overwritten between forward and backward is refused, not used"""
    from latte_amd import functional as LF
    x, w = _rn(1, torch.float32, (50, 24), (16, 24))
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    y = LF.linear(x, w).sum()
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_rows_past_two_gigabytes():
    """offsets of more than 32 bits: a long matrix of repeated blocks gives repeated results, in every direction"""
    from latte_amd import functional as LF
    block, w, dyb = _rn(2, torch.bfloat16, (1024, 2048), (24, 2048), (1024, 24))
    n = 1100                                              # 1 126 400 x 2048: 4.6 GB
    x, dy = block.repeat(n, 1), dyb.repeat(n, 1)
    y = LF.linear(x, w, act="relu").view(n, 1024, 24)
    assert bool((y == y[:1]).all())
    q = LF.quantize_mx8(x)
    assert bool((q.values.view(torch.uint8).view(n, -1) == q.values.view(torch.uint8).view(n, -1)[:1]).all())
    with torch.no_grad():
        y8 = LF.linear(q, LF.quantize_mx8(w)).view(n, 1024, 24)
    assert bool((y8 == y8[:1]).all())
    del y8, q
    ones = torch.ones(2048, dtype=torch.bfloat16, device="cuda")
    h = LF.rms_norm(x, ones).view(n, 1024, 2048)
    assert bool((h[0] == h[-1]).all()) and bool((h[0] == h[n // 2]).all())
    del h
    xg = x.requires_grad_(True)
    wg = w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(LF.linear(xg, wg), (xg, wg), dy)
    assert bool((gx.view(n, -1) == gx.view(n, -1)[:1]).all())
    want = (dyb.double().t() @ block.double()) * n
    mag = (dyb.double().abs().t() @ block.double().abs()) * n
    # split sums: at most 2^-24 of the magnitudes for each of the ~ rows / splits + splits additions in a chain
    assert bool(((gw.double() - want).abs() <= 2.0 ** -8 * want.abs() + (1126400 / 256 + 2048) * 2.0 ** -24 * mag).all())


def test_streams_and_threads_at_once():
    """calls from several threads on several streams, forward and backward, give what they give alone"""
    from latte_amd import functional as LF
    jobs, want, got = [], [], [None] * 4
    for i, (M, K, N, dt) in enumerate(((9000, 96, 64, torch.float32), (700, 512, 300, torch.bfloat16), (20, 1000, 77, torch.float16),
                                       (4000, 260, 510, torch.float32))):
        jobs.append(_rn(10 + i, dt, (M, K), (N, K), (N,), (M, N), (K,)))

    def work(x, w, b, dy, nw):
        t = [v.clone().requires_grad_(True) for v in (x, w, b, nw)]
        y = LF.linear(LF.rms_norm(t[0], t[3], checkpoint="mx8"), t[1], t[2], act="silu", checkpoint="mx8")
        return (y.detach(),) + torch.autograd.grad(y, t, dy)
    for j in jobs:
        want.append(work(*j))
    torch.cuda.synchronize()

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = work(*jobs[i])
        s.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want, got):
        assert b is not None and all(torch.equal(u, v) for u, v in zip(a, b))


def test_shared_leaves_and_accumulation():
    """one weight in two layers, one input through two branches, gradients accumulated into .grad"""
    from latte_amd import functional as LF
    x, w, dy = _rn(20, torch.float32, (300, 64), (64, 64), (300, 64))
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    y = LF.linear(LF.linear(x, w, act="gelu"), w, residual=x)
    y.backward(dy)
    y2 = LF.linear(LF.linear(x, w, act="gelu"), w, residual=x)
    g1 = [x.grad.clone(), w.grad.clone()]
    y2.backward(dy)
    # fp32 additions of the same addends twice over: exactly double
    assert torch.equal(x.grad, 2 * g1[0]) and torch.equal(w.grad, 2 * g1[1])
    X, W = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    Y = torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(X, W)), W) + X
    Y.backward(dy.double())
    for a, b in ((g1[0], X.grad), (g1[1], W.grad)):
        assert float((a.double() - b).norm() / b.norm()) < 1e-5


def test_modules_and_sparse_tensors():
    from latte_amd import functional as LF
    from latte_amd import sparse_modules as spnn
    from latte_amd.tensor import SparseTensor
    feats, other = _rn(21, torch.float32, (500, 32), (500, 48))
    coords = torch.zeros(500, 4, dtype=torch.int32, device="cuda")
    lin, ref = spnn.Linear(32, 48, act="relu").cuda(), torch.nn.Linear(32, 48).cuda()
    lin.load_state_dict(ref.state_dict())
    out = lin(SparseTensor(feats, coords, 1), residual=SparseTensor(other, coords, 1))
    assert isinstance(out, SparseTensor) and torch.equal(out.feats, LF.linear(feats, lin.weight, lin.bias, act="relu", residual=other))
    norm = spnn.RMSNorm(32).cuda()
    y = norm(SparseTensor(feats, coords, 1))
    assert torch.equal(y.feats, LF.rms_norm(feats, norm.weight))
    y, h = norm(SparseTensor(feats, coords, 1), residual=feats)
    assert torch.equal(h.feats, feats + feats) and torch.equal(y.feats, norm(feats, residual=feats)[0])


def test_tta_step_with_checkpoints():
    """one TTA iteration whose student keeps its BatchNorm inputs in 8 bits: the same losses (the forward pass is the same up
    to the composites' rounding), every norm parameter updated, the teacher on the one-call pass"""
    from latte_amd import synth
    from latte_amd.spvcnn import Net3DSeg
    from latte_amd.tta_step import LatteStep
    from latte_amd.workload import build_batch, hr_cfg_of
    w = synth.workload("tiny")
    losses = []
    for ck in (None, "mx8"):
        torch.manual_seed(5)
        net = Net3DSeg(w["C"], True, "SPVCNN", {"cr": 0.5}).cuda()
        step = LatteStep(net, w["C"], hr_cfg_of(w), activation_checkpoint=ck)
        before = [p.detach().clone() for p in step.params]
        batch = build_batch(w, device="cuda:0")
        losses.append({k: float(v) for k, v in step.step(batch).items()})
        assert all(bool(torch.isfinite(p).all()) for p in step.params)
        assert sum(not torch.equal(a, p) for a, p in zip(before, step.params)) > len(before) * 0.9
        assert step.ema_model.net_3d.stem[1].checkpoint is None
    for k in losses[0]:
        assert abs(losses[0][k] - losses[1][k]) < 1e-3 * (1 + abs(losses[0][k])), (k, losses)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_results_may_be_changed_in_place(dt):
    from latte_amd import functional as F
    g = torch.Generator().manual_seed(9)
    make = lambda *s: torch.randn(*s, generator=g).to(dt).cuda().requires_grad_()  # noqa: E731
    x, w, b, r, rw = make(3, 5, 24), make(16, 24), make(16), make(3, 5, 24), make(24)
    F.linear(x, w, b, act="gelu").mul(2).sum().backward()
    want = [t.grad.clone() for t in (x, w, b)]
    x.grad = w.grad = b.grad = None
    y = F.linear(x, w, b, act="gelu")
    y.mul_(2)
    y.sum().backward()
    assert all(torch.equal(t.grad, v) for t, v in zip((x, w, b), want))
    x.grad = None
    y, _ = F.rms_norm(x, rw, r)
    y.mul(2).sum().backward()
    want = [t.grad.clone() for t in (x, rw, r)]
    x.grad = rw.grad = r.grad = None
    y, h = F.rms_norm(x, rw, r)
    y.mul_(2)
    if dt is not torch.float32:   # beside fp32 the sum is what the backward pass reads
        h.add_(1)
    y.sum().backward()
    assert all(torch.equal(t.grad, v) for t, v in zip((x, rw, r), want))


def test_checkpoints_with_cross_rank_statistics():
    """one rank, a real collective: the statistics go through fp64 sums and come back within an fp32 rounding, so the result
    and its gradients are those of the local path (a few roundings of 2^-24, each on terms no larger than the largest); a
    rank without rows takes part in both collectives"""
    import os
    import socket

    import torch.distributed as dist
    from latte_amd import functional as LF
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    C = 40
    gamma, beta = (t.requires_grad_() for t in _rn(31, torch.float32, (C,), (C,)))

    def run(rows, **kw):
        x, r, dy = _rn(32 + rows, torch.float32, (rows, C), (rows, C), (rows, C))
        leaves = [x.requires_grad_(), gamma, beta, r.requires_grad_()]
        y = LF.batch_norm(x, gamma, beta, residual=r, relu=True, **kw)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    want = run(700, checkpoint="mx8")
    dist.init_process_group("gloo", rank=0, world_size=1, init_method=f"tcp://127.0.0.1:{port}")
    calls, real = [], LF._allreduce_small
    LF._allreduce_small = lambda t, g: (calls.append(t.numel()), real(t, g))[1]
    LF.SYNC_BN_GROUP = dist.group.WORLD
    try:
        got, plain = run(700, checkpoint="mx8"), run(700)
        assert torch.equal(got[0], plain[0]) and calls == [2 * C + 1, 2 * C] * 2
        for a, b in zip(got, want):
            assert (a - b).abs().max() <= 64 * 2.0 ** -24 * b.abs().max()
        for rows in (0, 1):
            calls.clear()
            out = run(rows, checkpoint="mx8")
            assert calls == [2 * C + 1, 2 * C] and out[0].shape == out[1].shape == (rows, C)
            assert all(torch.isfinite(t).all() for t in out)
    finally:
        LF.SYNC_BN_GROUP = None
        LF._allreduce_small = real
        dist.destroy_process_group()


def test_capture_is_refused_while_an_eager_graph_holds_a_leaf():
    from latte_amd import functional as LF
    x, w, g = (t.requires_grad_() for t in _rn(41, torch.float32, (64, 32), (48, 32), (32,)))

    def step():
        return LF.linear(x, w, act="relu", checkpoint="mx8"), LF.rms_norm(x, g), LF.batch_norm(x, g, g, checkpoint="mx8")
    dys = _rn(42, torch.float32, (64, 48), (64, 32), (64, 32))
    want = torch.autograd.grad(step(), [x, w, g], dys)
    held = step()
    for leaf in (lambda: LF.linear(x, w), lambda: LF.rms_norm(x, g), lambda: LF.batch_norm(x, g, g, checkpoint="mx8")):
        graph = torch.cuda.CUDAGraph()
        dead = torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError, match="still holds it"):
            with torch.cuda.graph(graph):
                dead.add_(1)   # a graph of something: the refused call has recorded nothing
                leaf()
        with torch.no_grad():   # no backward pass, nothing to refuse
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                leaf()
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(step(), [x, w, g], dys)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_some_of_the_gradients(dt):
    """a backward pass asked for some inputs of several gives the same bits for them"""
    from itertools import combinations

    from latte_amd import functional as LF
    M, K, N = 700, 96, 40
    x, w, b, r, dy, g, rx, dyx = _rn(51, dt, (M, K), (N, K), (N,), (M, N), (M, N), (K,), (M, K), (M, K))
    leaves = [t.requires_grad_() for t in (x, w, b, r, g, rx)]
    calls = [((x, w, b, r), dy, lambda: LF.linear(x, w, b, act="silu", residual=r)),
             ((x, w, r), dy, lambda: LF.linear(x, w, act="relu", residual=r, checkpoint="mx8")),
             ((x, w), dy, lambda: LF.linear(x, w, b.detach())),
             ((x, g, rx), dyx, lambda: LF.rms_norm(x, g, rx)[0])]
    if dt is torch.float32:
        beta = _rn(52, dt, (K,))[0].requires_grad_()
        calls.append(((x, g, beta, rx), dyx, lambda: LF.batch_norm(x, g, beta, residual=rx, relu=True, checkpoint="mx8")))
    for args, d, call in calls:
        y = call()
        full = torch.autograd.grad(y, args, d, retain_graph=True)
        for n in range(1, len(args)):
            for pick in combinations(range(len(args)), n):
                some = torch.autograd.grad(y, [args[i] for i in pick], d, retain_graph=True)
                assert all(torch.equal(s, full[i]) for s, i in zip(some, pick)), pick
    assert all(t.grad is None for t in leaves)
