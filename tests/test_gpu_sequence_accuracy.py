"""The sequence operators on the GPU are as accurate as the same sums in fp32 (tests/sequence_forms.py; that the bounds notice an
operand of 16 bits is tried on the host, tests/test_sequence_accuracy_cpu.py)."""
import pytest

import sequence_forms as F
from test_gpu_sequence import ops  # noqa: F401  (the model object as a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", F.DELTA, ids=str)
def test_delta_rule_is_as_accurate_as_fp32_sums(ops, shape, dtype):  # noqa: F811
    import torch
    args = F.delta_inputs(1, *shape, getattr(torch, dtype))
    scale = shape[4] ** -0.5
    (wo, ws), (po, ps) = F.delta_exact(*args, scale), F.delta_fp32(*args, scale)
    q, k, v, g, beta, state = (t.cuda() for t in args)
    o, s = ops.delta_rule(q, k, v, g, beta, None, state)
    assert F.held(s.cpu(), ws, ps) <= 1
    assert F.held(o.cpu(), wo, po) <= 1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", F.LINEAR, ids=str)
def test_linear_adapted_is_as_accurate_as_fp32_sums(ops, shape, dtype):  # noqa: F811
    import torch
    args = F.linear_inputs(2, *shape, getattr(torch, dtype), adapter=4.0)
    y = ops.linear_adapted(*(t.cuda() for t in args))
    assert F.held(y.cpu(), F.linear_exact(*args), F.linear_fp32(*args)) <= 1
