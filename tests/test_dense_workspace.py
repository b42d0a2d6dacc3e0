"""What the backward pass of linear writes into its workspace against what lt_linear_bwd_workspace_bytes asks for: no GPU
needed.  Every region's extent is worked out here from the strides that its kernel is handed."""
import pytest

from latte_amd import _lib

UP = 256                                     # regions start at multiples of this


def _up(n, a):
    return (n + a - 1) // a * a


def _written(M, K, N, sz, x_mx8, has_act):
    """bytes up to the end of the last region, without the joins' partial sums, for inputs too wide for the one-pass route"""
    ch = 16 // sz
    k, n = K % ch != 0, N % ch != 0
    as_is, filled = (78, 103) if sz == 4 else (240, 700)
    copied = ((M + N) * K if k else 0) + (M * N if n and not has_act else 0)
    pad = (k or n) and 2e-6 * 2.0 * M * N * K * (1 / as_is - 1 / filled) > 10 + 1e6 * copied * 2 * sz / 3.5e12
    N8, K8 = (_up(N, ch), _up(K, ch)) if pad else (N, K)
    own_dz, two = has_act or N8 != N, has_act and sz == 2 and M * N <= 4096
    end = _up(M * N8 * sz, UP) if own_dz else 0                              # dz
    end += _up(M * N8 * sz, UP) if two else 0                                # what its rounding left
    cg = (N8 + 3) // 4
    tx = 1
    while tx < cg and tx < 64:
        tx *= 2
    gx, ty = (cg + tx - 1) // tx, 256 // tx
    most = 1 if M <= ty * 16 else (M + ty * 4 - 1) // (ty * 4)
    s = max(1, min((2048 + gx - 1) // gx, most))
    rows = max(1, (M + s - 1) // s)
    end += _up((M + rows - 1) // rows * N * 4, UP)                           # column sums of the slabs
    if K8 != K or (x_mx8 and (N > 256 or pad)):
        end += _up(M * K8 * sz, UP)                                          # x, its rows filled up
    if K8 != K:
        end += _up(N * K8 * sz, UP)                                          # W likewise
    return end, pad, two


@pytest.mark.parametrize("dt", [0, 1, 2])
def test_backward_regions_fit_the_workspace(dt):
    """sizes on both sides of every rule: filled-up rows or not, one or two terms of dz, widened x or not"""
    lib, sz = _lib.load(), 4 if dt == 0 else 2
    seen = set()
    rows = (1, 4, 32, 63, 64, 65, 400, 512, 1024, 2049, 4096, 9000)
    for M in rows:
        for N in (1, 4, 5, 8, 9, 63, 64, 129, 255, 256, 257, 1001, 1505):
            for K in (257, 300, 1001, 4096, 229376, 262144, 300001, 360448, 1000003):
                if M * K > 1 << 32:
                    continue
                for x_mx8 in (0, 1):
                    has = lib.lt_linear_bwd_workspace_bytes(M, K, N, dt, x_mx8)
                    for has_act in (False, True):
                        end, pad, two = _written(M, K, N, sz, x_mx8, has_act)
                        assert end <= has, (M, K, N, dt, x_mx8, has_act, end, has)
                        seen.add((bool(pad), two))
    assert seen >= ({(False, False), (True, False)} if dt == 0 else {(a, b) for a in (False, True) for b in (False, True)})
