"""What the dense operators refuse, and how: no GPU needed (CPU tensors, argument checks, C entry points with bad sizes)."""
import ctypes

import pytest
import torch

from latte_amd import _lib
from latte_amd import functional as LF
from latte_amd import sparse_modules as spnn


def test_no_cpu_fallback():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for f in (lambda: LF.linear(x, w), lambda: LF.rms_norm(x, torch.ones(8)), lambda: LF.quantize_mx8(x),
              lambda: LF.rms_norm(x, torch.ones(8), out="mx8"), lambda: LF.rms_norm(x, torch.ones(8), checkpoint="mx8"),
              lambda: spnn.Linear(8, 6)(x), lambda: spnn.RMSNorm(8)(x),
              lambda: LF.batch_norm(x, torch.ones(8), torch.zeros(8), checkpoint="mx8")):
        with pytest.raises(_lib.LatteHipError):
            f()
    q = LF.Mx8(torch.zeros(4, 8).to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8))
    with pytest.raises(_lib.LatteHipError):
        q.dequantize()
    with pytest.raises(_lib.LatteHipError):
        LF.linear(q, q)


def test_names_are_checked_before_anything_runs():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match="act must be one of"):
        LF.linear(x, w, act="tanh")
    with pytest.raises(ValueError, match="checkpoint"):
        LF.linear(x, w, checkpoint="fp8")
    with pytest.raises(ValueError, match="checkpoint"):
        LF.rms_norm(x, torch.ones(8), checkpoint="fp8")
    with pytest.raises(ValueError, match="out must be"):
        LF.rms_norm(x, torch.ones(8), out="e4m3")
    with pytest.raises(ValueError, match="checkpoint"):
        LF.batch_norm(x, torch.ones(8), torch.zeros(8), checkpoint="e4m3")
    with pytest.raises(ValueError, match="mode"):
        spnn.set_activation_checkpoint(torch.nn.Sequential(), "fp8")
    with pytest.raises(TypeError, match="expected a tensor"):
        LF.linear([1.0], w)


def test_mx8_holder_checks_its_parts():
    v, s = torch.zeros(4, 40).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8)
    assert LF.Mx8(v, s).shape == (4, 40)
    with pytest.raises(TypeError):
        LF.Mx8(torch.zeros(4, 40), s)
    with pytest.raises(TypeError):
        LF.Mx8(v[0], s)
    for bad in (s[:, :1], s[:3], s.int(), torch.zeros(4, 3, dtype=torch.uint8)):
        with pytest.raises(ValueError):
            LF.Mx8(v, bad)
    with pytest.raises(TypeError, match="both Mx8 or neither"):
        LF.linear(LF.Mx8(v, s), torch.zeros(3, 40))


def test_set_activation_checkpoint_reaches_every_layer():
    net = torch.nn.ModuleList([spnn.BatchNorm(8), torch.nn.ModuleList([spnn.Linear(8, 8), spnn.RMSNorm(8)]), torch.nn.Linear(8, 8)])
    assert spnn.set_activation_checkpoint(net, "mx8") is net
    assert [net[0].checkpoint, net[1][0].checkpoint, net[1][1].checkpoint] == ["mx8"] * 3 and not hasattr(net[2], "checkpoint")
    spnn.set_activation_checkpoint(net, None)
    assert net[0].checkpoint is None and "checkpoint" not in net.state_dict()
    assert set(spnn.Linear(8, 4, act="gelu").state_dict()) == {"weight", "bias"} and "gelu" in repr(spnn.Linear(8, 4, act="gelu"))


P = ctypes.c_void_p


def test_c_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    bad = P(256)   # never read: every call below is refused before a launch

    def refused(rc, code, text):
        assert rc == code and text in lib.lt_last_error(), (rc, lib.lt_last_error())
    lin = lambda M=4, K=8, N=8, dt=0, act=0, kind=0, x=bad, y=bad, deriv=None: lib.lt_linear_fwd(  # noqa: E731
        x, K, bad, K, None, None, 0, act, M, K, N, dt, y, deriv, kind, None, 0, None)
    refused(lin(dt=3), -1, b"none of LT_DT_")
    refused(lin(M=-1), -1, b"bad sizes")
    refused(lin(K=0), -1, b"bad sizes")
    refused(lin(N=0), -1, b"bad sizes")
    refused(lin(M=1 << 41), -4, b"too large")
    refused(lin(act=4), -1, b"LT_ACT_")
    refused(lin(act=1, kind=2, deriv=bad), -1, b"does not go with")
    refused(lin(act=2, kind=1, deriv=bad), -1, b"does not go with")
    refused(lin(act=2, kind=3), -1, b"null pointer")
    refused(lin(x=None), -1, b"null pointer")
    assert lin(M=0, x=None, y=None) == 0          # nothing to do
    bwd = lambda M=4, K=8, N=8, dt=0, kind=0, ws=bad, nb=1 << 30, ldx=8, xs=None, dy=bad: lib.lt_linear_bwd(  # noqa: E731
        dy, N, bad, ldx, xs, bad, K, bad, kind, M, K, N, dt, bad, bad, bad, ws, nb, None)
    refused(bwd(kind=4), -1, b"deriv_kind")
    refused(bwd(ws=bad, nb=16), -3, b"workspace too small")
    refused(bwd(xs=bad, ldx=9), -1, b"mx8")
    refused(bwd(dy=None), -1, b"null pointer")
    refused(lib.lt_rms_norm_fwd(bad, 8, None, 0, bad, 1e-6, 4, 16385, 0, None, bad, None, None, None, None, None, None), -4, b"at most 16384")
    refused(lib.lt_rms_norm_fwd(bad, 8, None, 0, bad, 1e-6, 4, 8, 0, None, None, None, None, None, None, None, None), -1, b"null pointer")
    refused(lib.lt_rms_norm_bwd(bad, 8, None, 0, bad, 8, None, 0, None, None, bad, bad, 4, 8, 0, bad, bad, bad, 8, None), -3, b"workspace")
    refused(lib.lt_linear_mx8_fwd(bad, bad, bad, bad, None, None, 0, 0, 4, 8, 8, 0, bad, None, 0, None), -1, b"bfloat16 or float16")
    refused(lib.lt_linear_mx8_fwd(None, bad, bad, bad, None, None, 0, 0, 4, 8, 8, 1, bad, None, 0, None), -1, b"null pointer")
    refused(lib.lt_mx8_quantize(bad, 8, 4, 0, 0, bad, bad, None), -1, b"bad sizes")
    refused(lib.lt_mx8_dequantize(None, bad, 4, 8, 0, bad, None), -1, b"null pointer")
    refused(lib.lt_bn_apply_mx8(bad, bad, bad, bad, bad, 1e-5, None, 3, bad, bad, bad, bad, 4, 8, None), -1, b"needs a residual")
    refused(lib.lt_bn_apply_mx8(bad, bad, bad, bad, bad, 1e-5, None, 1, bad, bad, bad, None, 4, 8, None), -1, b"mask")
    refused(lib.lt_bn_apply_mx8(bad, bad, bad, bad, bad, 1e-5, None, 0, bad, bad, bad, None, 4, 6, None), -1, b"multiple of 4")
    assert lib.lt_linear_workspace_bytes(4, 0, 8, 0) == -1 and lib.lt_linear_bwd_workspace_bytes(4, 8, 8, 9, 0) == -1
    assert lib.lt_linear_mx8_workspace_bytes(-1, 8, 8) == -1 and lib.lt_rms_norm_bwd_workspace_bytes(4, 1 << 20) == -1


@pytest.mark.parametrize("dt", [0, 1, 2])
def test_workspaces_cover_every_plan(dt):
    """sizes are answers without a GPU: non-negative, bounded, and monotone where more rows are more splits' worth"""
    lib = _lib.load()
    for M in (0, 1, 31, 33, 64, 2047, 2048, 8192, 310017, 1 << 22):
        for K, N in ((1, 1), (17, 5), (64, 64), (128, 96), (250, 33), (1024, 4096), (4096, 17)):
            f, b = lib.lt_linear_workspace_bytes(M, K, N, dt), lib.lt_linear_bwd_workspace_bytes(M, K, N, dt, 1)
            assert 0 <= f <= 4 * 256 * max(M, 1) * N + 256 and b >= M * N * (4 if dt == 0 else 2)
            assert b < 20 * (M * (K + N) + 1024 * (K * N + N) + 4096)


def test_sizes_past_any_memory_are_refused():
    """products of the sizes stay within 64 bits: a byte count never wraps round to a small one"""
    lib = _lib.load()
    big = (1 << 31) - 2048
    for M, K, N in ((1 << 40, 1 << 20, 1 << 20), (4, big, big), (1 << 39, 16, 1), (1 << 39, 1, 16)):
        for dt in (0, 1):
            assert lib.lt_linear_workspace_bytes(M, K, N, dt) == -1 and b"too large" in lib.lt_last_error()
            assert lib.lt_linear_bwd_workspace_bytes(M, K, N, dt, 1) == -1
        assert lib.lt_linear_mx8_workspace_bytes(M, K, N) == -1 and b"too large" in lib.lt_last_error()
    assert lib.lt_linear_workspace_bytes(1 << 30, 1024, 1024, 1) >= 0
