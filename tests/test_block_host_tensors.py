"""A tensor that is not on the GPU is refused before its address reaches a kernel, whichever argument it is."""
import pytest
import torch

from conftest import log


def calls(lcpp, device):
    """name -> (method, its tensor arguments by name, the others)"""
    def rows(dtype=torch.float32):
        return torch.zeros(4, 32, dtype=dtype, device=device)

    def vec(n, dtype=torch.float32):
        return torch.zeros(n, dtype=dtype, device=device)

    norm, drop, mix = lcpp.DeviceLayerNorm(), lcpp.DeviceDropout(), lcpp.DeviceGatedRecurrence()
    counter = vec(1, torch.int64)
    stats = dict(d_mean=vec(4), d_rstd=vec(4))
    grads = dict(d_grad_weight=vec(32), d_grad_bias=vec(32))
    temp = torch.zeros(1 << 16, dtype=torch.uint8, device=device)
    offsets = dict(d_begin_offsets=vec(2, torch.int32), d_end_offsets=vec(2, torch.int32))
    seq = dict(d_gate=rows(), d_in=rows())
    states = torch.zeros(2, 32, device=device)
    out = {
        "norm forward": (norm.Forward, dict(d_in=rows(), d_out=rows(), d_weight=vec(32), d_bias=vec(32), **stats), {}),
        "norm add forward": (norm.AddForward, dict(d_in=rows(), d_residual=rows(), d_sum=rows(), d_out=rows(), d_weight=vec(32),
                                                   d_bias=vec(32), d_offset=counter, **stats), {"p": 0.1}),
        "norm backward": (norm.Backward, dict(temp_storage=temp, d_grad_out=rows(), d_in=rows(), d_weight=vec(32),
                                              d_grad_in=rows(), **stats, **grads), {}),
        "norm add backward": (norm.AddBackward, dict(temp_storage=temp, d_grad_out=rows(), d_grad_sum=rows(), d_sum=rows(),
                                                     d_weight=vec(32), d_grad_residual=rows(), d_grad_in=rows(),
                                                     d_offset=counter, **stats, **grads), {"p": 0.1}),
        "dropout": (drop.Forward, dict(d_in=rows(), d_out=rows(), d_residual=rows(), d_offset=counter), {"p": 0.1, "seed": 1}),
        "dropout backward": (drop.Backward, dict(d_grad_out=rows(), d_grad_in=rows(), d_offset=counter), {"p": 0.1, "seed": 1}),
        "recurrence forward": (mix.Forward, dict(temp_storage=temp, d_out=rows(), d_initial=states, d_final=states.clone(),
                                                 d_checkpoints=states.clone(), **seq, **offsets),
                               {"gate": "decay", "max_length": 2}),
        "recurrence backward": (mix.Backward, dict(temp_storage=temp, d_checkpoints=states, d_grad_out=rows(),
                                                   d_grad_gate=rows(), d_grad_in=rows(), d_grad_final=states.clone(),
                                                   d_grad_initial=states.clone(), **seq, **offsets),
                                {"gate": "decay", "max_length": 2}),
        "step": (mix.Step, dict(d_gate=rows()[:2], d_in=rows()[:2], d_state_in=states, d_state_out=states.clone(),
                                d_out=rows()[:2], d_slots=vec(2, torch.int32)), {"gate": "decay"}),
    }
    out["step in place"] = (mix.Step, {**out["step"][1], "d_state_out": None}, {"gate": "decay"})
    # three dimensions, which take another way through the checks
    cube = dict(d_gate=rows()[None], d_in=rows()[None], d_out=rows()[None])
    out["recurrence of three dimensions"] = (mix.Forward, dict(temp_storage=None, **cube), {"gate": "decay"})
    wide = {k: torch.zeros(2, 4, 32, device=device) for k in ("d_in", "d_out")}
    out["norm of three dimensions"] = (norm.Forward, wide, {})
    return out


def invoke(method, tensors, others):
    if "d_state_out" in tensors and tensors["d_state_out"] is None:
        tensors = {**tensors, "d_state_out": tensors["d_state_in"]}
    method(**tensors, **others)


NAMES = ["norm forward", "norm add forward", "norm backward", "norm add backward", "dropout", "dropout backward",
         "recurrence forward", "recurrence backward", "step", "step in place", "recurrence of three dimensions",
         "norm of three dimensions"]


@pytest.mark.parametrize("name", NAMES)
def test_host_tensors(name):
    import lc_parallel_primitive_amd as lcpp

    method, tensors, others = calls(lcpp, "cpu")[name]
    with pytest.raises(ValueError, match="must be on the GPU"):
        invoke(method, tensors, {**others, "stream": 0})


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_one_host_tensor_among_others(gpu, name):
    import lc_parallel_primitive_amd as lcpp

    method, tensors, others = calls(lcpp, "cuda")[name]
    invoke(method, tensors, others)
    torch.cuda.synchronize()
    for k, v in tensors.items():
        if v is None:
            continue
        log(f"{name}: {k} on the host")
        with pytest.raises(ValueError, match="must be on the GPU"):
            invoke(method, {**tensors, k: v.cpu()}, others)
    torch.cuda.synchronize()
