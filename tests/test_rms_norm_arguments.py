"""Arguments of the RMS norm that belong together, checked before anything else: no GPU is needed."""
import pytest
import torch


def test_sum_without_residual():
    """AddForward would write the norm and leave d_sum as it was."""
    import lc_parallel_primitive_amd as lcpp

    x = torch.zeros(4, 32)
    norm = lcpp.DeviceRMSNorm()
    with pytest.raises(ValueError, match="d_residual"):
        norm.AddForward(x, None, x.clone(), x.clone(), stream=0)
    with pytest.raises(ValueError, match="d_sum"):
        norm.AddForward(x, x.clone(), None, x.clone(), stream=0)


def test_scales_without_values():
    """Forward and AddForward would leave d_scales as it was."""
    import lc_parallel_primitive_amd as lcpp

    x, scales = torch.zeros(4, 32), torch.zeros(4, 1)
    norm = lcpp.DeviceRMSNorm()
    with pytest.raises(ValueError, match="d_quant"):
        norm.Forward(x, x.clone(), d_scales=scales, stream=0)
    with pytest.raises(ValueError, match="d_quant"):
        norm.AddForward(x, x, x.clone(), x.clone(), d_scales=scales, stream=0)
