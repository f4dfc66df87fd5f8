"""The MXFP4 products are for inference: a call that would lose a gradient is refused
before it reaches a GPU."""
import pytest
import torch

from lynnreal_omni_amd import mxfp4, mxfp4_gemm


def _layer():
    return mxfp4.Mxfp4Linear(torch.nn.Linear(64, 32).bfloat16())


def test_layer_refuses_inputs_that_require_a_gradient():
    layer = _layer()
    assert not any(p.requires_grad for p in layer.parameters())
    x = torch.zeros(3, 64, dtype=torch.bfloat16, requires_grad=True)
    for value in (x, x[None], x * 2):
        with pytest.raises(RuntimeError, match="gradients are not supported"):
            layer(value)
    for context in (torch.no_grad, torch.inference_mode):
        with context(), pytest.raises(ValueError, match="GPU"):      # as far as the device check
            layer(x)
    with pytest.raises(ValueError, match="GPU"):
        layer(x.detach())


@pytest.mark.parametrize("which", ["residual", "table", "bias"])
def test_epilogue_tensors_that_require_a_gradient(which):
    layer = _layer()
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    codes, scales = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8)
    given = dict(residual=torch.zeros(3, 32, dtype=torch.bfloat16), table=torch.zeros(1, 32, dtype=torch.bfloat16),
                 indices=torch.zeros(3, dtype=torch.int64), gate_slot=0)
    bias = torch.zeros(32, dtype=torch.bfloat16)
    (bias if which == "bias" else given[which]).requires_grad_()
    calls = [lambda: mxfp4_gemm.linear_rows(x, layer.weight_codes, layer.weight_scale, bias, **given),
             lambda: mxfp4_gemm.mxfp4_matmul(codes, layer.weight_codes, scales, layer.weight_scale, bias, **given)]
    for call in calls:
        with pytest.raises(RuntimeError, match="gradients are not supported"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            call()
