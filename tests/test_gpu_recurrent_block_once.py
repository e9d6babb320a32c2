"""The example's autograd functions give first gradients only: asking for a gradient of a gradient is an error."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT, log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(gpu):
    spec = importlib.util.spec_from_file_location("recurrent_block", os.path.join(ROOT, "examples", "recurrent_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("name", ["Norm", "AddNorm", "Recurrence"])
def test_second_gradients_are_refused(example, name):
    log(f"example: second gradient of {name}")
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, width = 40, 24
    x, r = (torch.randn(rows, width, generator=g, device="cuda").requires_grad_() for _ in range(2))
    w, b = torch.ones(width, device="cuda").requires_grad_(), torch.zeros(width, device="cuda").requires_grad_()
    begin = torch.tensor([0, 25], dtype=torch.int32, device="cuda")
    end = torch.tensor([25, 40], dtype=torch.int32, device="cuda")
    if name == "Norm":
        y = example.Norm.apply(x, w, b)
    elif name == "AddNorm":
        total, normed = example.AddNorm.apply(x, r, w, b, 0.1, 3, 4)
        y = total * 0.5 + normed
    else:
        y = example.Recurrence.apply(r, x, begin, end, 25)
    (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    assert torch.isfinite(dx).all() and bool(dx.any())
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dx * dx).sum().backward()
