"""The sequence operators where values overflow or are infinite."""
import math

import pytest

import sequence_forms as F
from test_gpu_sequence import ops  # noqa: F401  (the model object as a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first, second", [(3, 16), (3, 20), (15, 31), (2, 9), (17, 30), (5, 40), (3, 7)], ids=str)
def test_delta_rule_products_of_finite_keys_that_overflow(ops, first, second):  # noqa: F811
    """Two frames with keys of 1e20 along one component, all other keys across it: k . k of the two passes fp32's range.  From the second
    one on, a column whose u does so too is not finite, and what is finite is the definition's value: its sums see the large
    component times zero only, so they are as near as without it (the rule's own tolerance for values up to 5, or the value).  The
    frames before it are what they are without it."""
    import torch
    T, dk, dv = 50, 32, 16
    q, k, v, g, beta, state = F.delta_inputs(7, 1, T, 1, 1, dk, dv, torch.float32)
    q[..., 0] = 0
    k[..., 0] = 0
    state[:] = 0
    q[0, second, 0, 0] = 1.0
    k[0, first] = 0
    k[0, first, 0, 0] = 1e20
    args = [t.cuda() for t in (q, k, v, g, beta)]
    clean, _ = ops.delta_rule(*args, None, state.cuda())
    assert torch.isfinite(clean).all()
    k[0, second] = 0
    k[0, second, 0, 0] = 1e20
    o, s = (t.cpu() for t in ops.delta_rule(q.cuda(), k.cuda(), *args[2:], None, state.cuda()))
    assert torch.equal(o[:, :second], clean.cpu()[:, :second])
    want, _ = F.delta_exact(q, k, v, g, beta, state, dk ** -0.5)
    _, before = F.delta_exact(*(t[:, :second] for t in (q, k, v, g, beta)), state, 1.0)
    u = beta[0, second, 0].double() * (v[0, second, 0].double() - 1e20 * g[0, second, 0].double().exp() * before[0, 0, 0])
    over = u.abs() > torch.finfo(torch.float32).max
    assert not torch.isfinite(o[0, second:, 0][:, over]).any() and not torch.isfinite(s[0, 0][:, over]).any()
    there = torch.isfinite(o)
    tol = 4 * 2.0 ** -24 * math.sqrt(dk + 128) * 3 * want.abs().clamp_min(5.0)
    assert ((o.double() - want).abs() <= tol)[there].all()
