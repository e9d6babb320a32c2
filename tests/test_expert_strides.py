"""Strides of the matrices' gradients that are refused, without a GPU: matrices that overlap."""
import pytest
import torch

A, B, C, D, G = 4096, 8192, 12288, 16384, 24576  # addresses that no call reads


@pytest.mark.parametrize("row,expert", [(64, 2047), (64, 64), (191, 64), (192, 63), (192, 65), (4096, 63), (63, 4096), (0, 64)])
def test_overlapping_matrices(row, expert):
    """Three matrices of 32 rows of 64 values."""
    import lc_parallel_primitive_amd as lcpp

    at = torch.arange(3)[:, None, None] * expert + torch.arange(32)[:, None] * row + torch.arange(64)
    assert at.unique().numel() < at.numel()
    assert lcpp.lib().lcpp_expert_product_backward(6, A, 32, B, 64, C, 64, 2048, D, None, 0, 6, G, row, expert, 10, 3, 32, 64, None) == -1
    grad = torch.zeros(8192 + 32 * 4096 * 2).as_strided((3, 32, 64), (expert, row, 1))
    x = torch.zeros(10, 64)
    with pytest.raises(ValueError, match="must not overlap"):
        lcpp.device_expert._matrices(grad, "d_grad_weight", True)
    with pytest.raises(ValueError):
        lcpp.DeviceExpertProduct().Backward(torch.zeros(10, 32), x, torch.zeros(3, 32, 64), torch.zeros(4, dtype=torch.int32), None, grad,
                                            stream=0)
