"""The bounds that tests/test_gpu_sequence_accuracy.py holds the sequence operators to, tried on the host: the fp32 forms with operands
of three bf16 terms pass them, with two terms -- in all operands, or only where bf16 outputs are formed -- they do not."""
import pytest
import torch

import sequence_forms as F


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", F.DELTA, ids=str)
def test_delta_bounds_tell_two_terms_from_three(shape, dtype):
    args = F.delta_inputs(1, *shape, dtype)
    scale = shape[4] ** -0.5
    (wo, ws), (po, ps) = F.delta_exact(*args, scale), F.delta_fp32(*args, scale)
    o, s = F.delta_fp32(*args, scale, cut=3)
    assert F.held(o.to(dtype), wo, po) <= 1 and F.held(s, ws, ps) <= 1
    o, s = F.delta_fp32(*args, scale, cut=2)
    assert F.held(s, ws, ps) > 1
    if dtype is torch.float32:
        assert F.held(o, wo, po) > 1
    o, _ = F.delta_fp32(*args, scale, out_cut=2)
    assert F.held(o.to(dtype), wo, po) > 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", F.LINEAR, ids=str)
def test_linear_bounds_tell_two_terms_from_three(shape, dtype):
    args = F.linear_inputs(2, *shape, dtype, adapter=4.0)
    want, plain = F.linear_exact(*args), F.linear_fp32(*args)
    assert F.held(F.linear_fp32(*args, cut=3, z_cut=3).to(dtype), want, plain) <= 1
    assert F.held(F.linear_fp32(*args, z_cut=2).to(dtype), want, plain) > 1
    if dtype is torch.float32:
        assert F.held(F.linear_fp32(*args, cut=2), want, plain) > 1
