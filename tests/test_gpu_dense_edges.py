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
