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


LINEARS = [(1, 1, 60, 256, 3, 4), (3, 40, 100, 70, 2, 5), (130, 1, 600, 65, 40, 16), (1, 300, 512, 96, 1, 1), (9, 250, 136, 96, 5, 33), (9, 300, 100, 300, 4, 1), (41, 100, 64, 1060, 5, 8), (4, 1600, 64, 2048, 3, 8),
           (4, 1600, 72, 2050, 3, 8)]


@pytest.mark.parametrize("where", ["x", "weight", "bias", "down", "up", "scale", "x twice"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", LINEARS, ids=str)
def test_linear_adapted_infinite_and_largest_values(ops, shape, dtype, where):  # noqa: F811
    """An infinity, the type's largest number and a NaN give what the sums give in IEEE arithmetic: the 64-bit definition's infinities and
    NaN where it has them, its values elsewhere; an infinite z's share of an output is infinite or NaN as the sum over the adapter's
    components is (scale belongs to z = scale Down x: an infinite one makes the sum over its components infinite or NaN, in front of the
    sum or behind it).  Values beside FLT_MAX may overflow on the way, in z or in the sum: they are let go.  All of the kernel's
    tiles, one launch and two."""
    import torch
    t = getattr(torch, dtype)
    top = float(torch.finfo(t).max)
    for value in (float("inf"), -float("inf"), top, float("nan")):
        linear_with(ops, shape, t, top, value, where)


def linear_with(ops, shape, t, top, bad, where):  # noqa: F811
    import torch
    B, T, K, M, n, r = shape
    args = F.linear_inputs(10, *shape, t)
    x, w, b, down, up, scale, ids = args
    ids[0] = 0
    if where.startswith("x"):
        x[0, T // 2, K // 3] = bad
        if where == "x twice":
            x[B - 1, T - 1, K - 1], x[B - 1, T - 1, 0] = bad, -bad
    else:
        {"weight": w[M // 2], "bias": b[M - 1:], "down": down[0, r // 2], "up": up[0, M // 3], "scale": scale[:1]}[where][-1] = bad
    want = F.linear_exact(*args)
    mag = F.linear_exact(*(s.abs() for s in args[:6]), ids)                # (magnitudes: ids stay)
    y = ops.linear_adapted(*(s.cuda() for s in args)).cpu().double()
    z = torch.stack([(x[i].abs().double() @ down[a].abs().double().t() * abs(float(scale[a]))).amax(-1) if a >= 0 else torch.zeros(T, dtype=torch.double)
                     for i, a in enumerate(ids.tolist())])[..., None]
    way = torch.maximum(mag, z)
    sure = ~(way.isfinite() & (way > top / 2))
    if where == "scale" and math.isinf(bad):
        theirs = (ids == 0)[:, None, None].expand_as(sure)
        assert not y[theirs].isfinite().any()
        sure &= ~theirs
    assert torch.equal(y.isnan()[sure], want.isnan()[sure])
    inf = want.isinf() & sure
    assert torch.equal(y[inf], want[inf]) and not y.isinf()[sure & ~inf].any()
    there = want.isfinite() & sure
    tol = 4 * 2.0 ** -24 * math.sqrt(K + r + 3) * mag + (want.abs() * 2.0 ** -8 if t is torch.bfloat16 else 0)
    assert ((y - want).abs() <= tol)[there].all()


def test_block_of_the_model_with_an_infinite_sample(ops):  # noqa: F811
    """Sequences without an adapter answer an infinite sample beside others with adapters as the block without adapters does."""
    import torch
    from test_gpu_sequence import block_adapters
    dev = {k: tuple(t.cuda() for t in v) for k, v in block_adapters("velocity", 2, 4, 8, 60).items()}
    x = torch.randn(4, 20, 132, generator=torch.Generator().manual_seed(61))
    x[1, 7, 30], x[3, 2, 5] = float("inf"), -float("inf")
    x[3, 9, 0], x[3, 9, 1] = 3.4e38, -3.4e38
    want, _ = ops.rnn_forward("velocity", x.cuda(), [20] * 4)
    got, _ = ops.rnn_forward("velocity", x.cuda(), [20] * 4, None, dev, [0, -1, 1, -1])
    for i in (1, 3):
        assert torch.equal(got[i].isnan(), want[i].isnan()) and float((got[i] - want[i]).nan_to_num().abs().max()) < 1e-4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", LINEARS[:6], ids=str)
def test_linear_adapted_of_nothing_finite(ops, shape, dtype):  # noqa: F811
    import torch
    x, w, b, down, up, scale, ids = (t.cuda() for t in F.linear_inputs(11, *shape, getattr(torch, dtype)))
    assert ops.linear_adapted(torch.full_like(x, float("nan")), w, b, down, up, scale, ids, relu=True).isnan().all()
    signs = torch.where(w[:, :1] < 0, -1.0, 1.0).to(w.dtype) * w.abs()      # every weight of a column has the same sign
    y = ops.linear_adapted(torch.full_like(x, float("inf")), signs, b, down, up, scale, torch.full_like(ids, -1))
    assert torch.equal(y, torch.where(signs[:, 0] < 0, -float("inf"), float("inf")).to(y.dtype).expand_as(y))
