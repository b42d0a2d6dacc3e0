"""Row lengths and widths past 32 bits are refused before anything is allocated or launched, never cut to their low half: no GPU
needed (expanded tensors of one element, handed to the nodes behind latte_amd.dense)."""
import pytest
import torch

from latte_amd import dense

FAR = [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 8, 2 ** 33 + 1]


@pytest.mark.parametrize("n", FAR)
def test_far_extents_are_refused(n):
    nodes = dense._nodes()
    e4m3, byte = torch.zeros(1, 1).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8)
    row, col = torch.zeros(1, 1).expand(1, n), torch.zeros(1, 1).expand(n, 1)
    with pytest.raises(ValueError, match="do not go together"):
        nodes.linear(row, row, None, None, 0, False)
    with pytest.raises(ValueError, match="do not go together"):
        nodes.linear(torch.zeros(1, 1), col, None, None, 0, False)
    with pytest.raises(ValueError, match="quantize_mx8"):
        nodes.quantize_mx8(row)
    with pytest.raises(ValueError, match="dequantize"):
        nodes.dequantize_mx8(e4m3.expand(1, n), byte, torch.float32)
    with pytest.raises(ValueError, match="do not go together"):
        nodes.linear_mx8(e4m3.expand(1, n), byte, e4m3.expand(1, n), byte, None, None, 0, None)
    with pytest.raises(ValueError, match="do not go together"):
        nodes.linear_mx8(e4m3, byte, e4m3.expand(n, 1), byte, None, None, 0, None)
    with pytest.raises(ValueError, match="16384"):
        nodes.rms_norm(row, row[0], None, 1e-6, False)
    with pytest.raises(ValueError, match="batch_norm"):
        nodes.batch_norm_mx8(row, row[0], row[0], None, 1e-5, False, False)
