"""The sequence operators (mobileposer_amd/sequence.py: delta_rule, delta_rule_online, linear_adapted) on the GPU against their
definitions in 64 bits.

Tolerances.  One fp32 rounding is off by at most u = 2^-24 of the value; a sum of n products accumulated in fp32 by
lambda sqrt(n) u of the sum of the products' magnitudes, with lambda = 4 for every one of some 10^5 outputs.  The gated delta
rule with |k| = 1, 0 <= beta <= 1 and g <= 0 does not expand a deviation of its state (|I - beta k k^T| <= 1, e^g <= 1), so the
deviations of the chunks of 32 frames add up: each one's sums run over dk, 32 and 32 values (and as many again in the inverse
and in the update), n = dk + 128, relative to the state's largest magnitude.  An output is scale S^T q with |q| = 1 and
scale sqrt(dk) <= 1: no further off than the state.  A bf16 output adds its own rounding, 2^-8 of the value."""
import math

import numpy as np
import pytest

from conftest import npy

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LAMBDA = 4.0
BF16 = 2.0 ** -8


@pytest.fixture(scope="module")
def ops():
    import torch
    from mobileposer_amd import synthetic
    from mobileposer_amd.net import MobilePoserNet
    assert torch.cuda.is_available(), "-m gpu tests need an MI355X"
    n = MobilePoserNet.from_numpy(synthetic.make_weights(0), synthetic.synthetic_smpl(), device="cuda:0")
    yield n
    n.close()


def unit(x):
    return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)


def delta_inputs(seed, B, T, Hk, Hv, dk, dv, dtype, packed=False, same_keys=False):
    import torch
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    q, k, v = unit(rn(B, T, Hk, dk)), unit(rn(B, T, Hk, dk)), rn(B, T, Hv, dv)
    if same_keys:
        k = k[:, :1].expand(B, T, Hk, dk).clone()
    g = -torch.exp(torch.linspace(-4, 1, Hv)) * torch.rand(B, T, Hv, generator=gen)
    beta = torch.sigmoid(2 * rn(B, T, Hv)) if not same_keys else torch.ones(B, T, Hv)
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    if packed:
        row = torch.cat((q.flatten(2), k.flatten(2), v.flatten(2)), -1)
        q, k, v = row[..., :Hk * dk].unflatten(-1, (Hk, dk)), row[..., Hk * dk:2 * Hk * dk].unflatten(-1, (Hk, dk)), row[..., 2 * Hk * dk:].unflatten(-1, (Hv, dv))
    return q, k, v, g.cuda(), beta.cuda(), 0.5 * rn(B, Hv, dk, dv).cuda()


def delta_ref(q, k, v, g, beta, lengths, state, scale):
    """The definition, frame by frame, in 64 bits on the host."""
    import torch
    q, k, v, g, beta = (t.detach().cpu().double() for t in (q, k, v, g, beta))
    B, T, Hv, dv = v.shape
    rep = Hv // q.shape[2]
    S = torch.zeros(B, Hv, q.shape[3], dv, dtype=torch.float64) if state is None else state.cpu().double()
    o = torch.zeros(B, T, Hv, dv, dtype=torch.float64)
    top = S.abs().max()
    for b in range(B):
        s = S[b]
        for t in range(lengths[b]):
            kt, qt = k[b, t].repeat_interleave(rep, 0), q[b, t].repeat_interleave(rep, 0)
            s = s * torch.exp(g[b, t].clamp_min(-1e4))[:, None, None]
            u = beta[b, t][:, None] * (v[b, t] - (s * kt[..., None]).sum(1))
            s = s + kt[..., None] * u[:, None, :]
            o[b, t] = scale * (s * qt[..., None]).sum(1)
            top = torch.maximum(top, s.abs().nan_to_num(0, 0, 0).max())
        S[b] = s
    return o.numpy(), S.numpy(), float(top)


def delta_tol(T, dk, top):
    return LAMBDA * U * math.sqrt(dk + 128) * (-(-T // 32) + 1) * top


def assert_delta(got_o, got_s, want_o, want_s, tol, bf16):
    o, s = npy(got_o.float()).astype(np.float64), npy(got_s).astype(np.float64)
    assert np.array_equal(np.isnan(o), np.isnan(want_o)) and np.array_equal(np.isnan(s), np.isnan(want_s))
    err = np.abs(o - want_o) - (BF16 * np.abs(want_o) if bf16 else 0)
    assert np.nanmax(err, initial=0) <= tol, (np.nanmax(err), tol)
    assert np.nanmax(np.abs(s - want_s), initial=0) <= tol, (np.nanmax(np.abs(s - want_s)), tol)


SHAPES = [  # B, T, Hk, Hv, dk, dv
    (1, 1, 1, 1, 1, 1), (2, 1, 1, 2, 16, 16), (1, 31, 2, 2, 32, 32), (1, 32, 1, 1, 64, 64), (2, 33, 2, 4, 64, 48), (3, 65, 1, 3, 40, 41),
    (1, 130, 2, 2, 128, 128), (2, 97, 1, 2, 96, 130), (1, 70, 1, 1, 256, 33), (1, 64, 1, 1, 200, 64), (2, 50, 3, 6, 7, 5), (1, 300, 1, 1, 129, 16)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_delta_rule(ops, shape, dtype):
    import torch
    B, T, Hk, Hv, dk, dv = shape
    q, k, v, g, beta, s0 = delta_inputs(1, B, T, Hk, Hv, dk, dv, getattr(torch, dtype))
    lens = [max(0, T - 17 * b) for b in range(B)]
    for state in (None, s0):
        o, s = ops.delta_rule(q, k, v, g, beta, lens, state)
        wo, ws, top = delta_ref(q, k, v, g, beta, lens, state, dk ** -0.5)
        assert o.dtype == q.dtype and s.dtype == torch.float32
        assert_delta(o, s, wo, ws, delta_tol(T, dk, max(top, float(v.abs().max()))), dtype == "bfloat16")
        for b in range(B):
            assert not npy(o[b, lens[b]:].float()).any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 512, 1, 1, 64, 64), (2, 1000, 1, 2, 64, 40), (1, 1400, 1, 1, 128, 130), (1, 530, 1, 1, 200, 20), (2, 4500, 16, 32, 64, 40), (1, 2100, 8, 16, 100, 128), (3, 777, 1, 1, 7, 5), (1, 3000, 1, 1, 72, 33)], ids=str)
def test_delta_rule_long_sequences_on_few_heads(ops, shape, dtype):
    """Long enough, and few enough, to be run as segments side by side; ragged: a sequence that ends inside a segment, at a border
    between two, in the first one, and an empty one."""
    import torch
    B, T, Hk, Hv, dk, dv = shape
    q, k, v, g, beta, s0 = delta_inputs(14, B, T, Hk, Hv, dk, dv, getattr(torch, dtype))
    for lens in ([T] * B, [T - 300] + [T - 33, 0][:B - 1], [128] + [T - 1, 1][:B - 1]):
        for state in (None, s0):
            o, s = ops.delta_rule(q, k, v, g, beta, lens, state)
            wo, ws, top = delta_ref(q, k, v, g, beta, lens, state, dk ** -0.5)
            assert_delta(o, s, wo, ws, delta_tol(T, dk, max(top, float(v.float().abs().max()))), dtype == "bfloat16")


@pytest.mark.parametrize("where", ["k", "v", "g", "state"])
def test_delta_rule_non_finite_values_in_segments(ops, where):
    import torch
    T, dk, dv, t0 = 900, 32, 20, 333
    q, k, v, g, beta, s0 = delta_inputs(15, 1, T, 1, 1, dk, dv, torch.float32)
    clean = ops.delta_rule(q, k, v, g, beta, None, s0)
    {"k": k[0, t0, 0], "v": v[0, t0, 0], "g": g[0, t0], "state": s0[0, 0, 3]}[where][0 if where == "g" else 7] = float("nan")
    o, s = ops.delta_rule(q, k, v, g, beta, None, s0)
    hit = torch.zeros(1, T, 1, dv, dtype=torch.bool, device="cuda")
    if where in ("v", "state"):
        hit[:, t0 if where == "v" else 0:, :, 7] = True
    else:
        hit[:, t0:] = True
    assert torch.equal(torch.isnan(o), hit)
    assert torch.equal(torch.isnan(s), hit[0, -1, 0].expand(1, 1, dk, dv))
    assert torch.equal(o[~hit], clean[0][~hit])


def test_delta_rule_lengths_strides_and_garbage_behind_the_end(ops):
    import torch
    B, T, Hk, Hv, dk, dv = 4, 80, 2, 4, 72, 40
    q, k, v, g, beta, s0 = delta_inputs(2, B, T, Hk, Hv, dk, dv, torch.float32, packed=True)
    lens = [80, 0, 1, 45]
    for b, n in enumerate(lens):                 # what lies behind a sequence's end is never read into the result
        for t in (q, k, v, g, beta):
            t[b, n:] = float("nan") if b % 2 else float("inf")
    want = delta_ref(q, k, v, g, beta, lens, s0, 0.3)
    tol = delta_tol(T, dk, max(want[2], 5.0))
    o, s = ops.delta_rule(q, k, v, g, beta, lens, s0, scale=0.3)
    assert_delta(o, s, want[0], want[1], tol, False)
    assert torch.equal(s[1], s0[1])
    # lengths on the device (values are clamped to 0..T), int64 too; a transposed, padded layout of every input
    dl = torch.tensor([81, -3, 1, 45], device="cuda", dtype=torch.int32)
    wide = [torch.full((T, B, *t.shape[2:-1], t.shape[-1] + 3), float("nan"), device="cuda") for t in (q, k, v)]
    qq, kk, vv = (w[..., :t.shape[-1]].transpose(0, 1).copy_(t) for w, t in zip(wide, (q, k, v)))
    gg, bb = (t.permute(2, 1, 0).contiguous().permute(2, 1, 0) for t in (g, beta))
    for l in (dl, dl.long()):
        o2, s2 = ops.delta_rule(qq, kk, vv, gg, bb, l, s0, scale=0.3)
        assert torch.equal(o, o2) and torch.equal(s, s2)
    # a last dimension that is not contiguous is copied
    o3, s3 = ops.delta_rule(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, g, beta, lens, s0, scale=0.3)
    assert torch.equal(o, o3) and torch.equal(s, s3)


def test_delta_rule_resets_equal_keys_and_zero_beta(ops):
    """g that clears the state inside a chunk (-1e4, -inf, -3e38), keys that are all the same (I + A far from the identity), beta = 0."""
    import torch
    q, k, v, g, beta, s0 = delta_inputs(3, 2, 100, 1, 3, 64, 32, torch.float32, same_keys=True)
    g[0, 5, 0] = -1e4
    g[0, 40, 1] = -float("inf")
    g[1, 41, 2] = -3e38
    g[1, 42, 2] = -float("inf")
    g[0, 50:70] = 0.0
    beta[1, 10:30] = 0.0
    o, s = ops.delta_rule(q, k, v, g, beta, [100, 100], s0)
    wo, ws, top = delta_ref(q, k, v, g, beta, [100, 100], s0, 64 ** -0.5)
    assert_delta(o, s, wo, ws, delta_tol(100, 64, max(top, 5.0)), False)


@pytest.mark.parametrize("where", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_delta_rule_non_finite_values_stay_behind(ops, where, value):
    """A value that is not finite reaches its own and later frames of its (sequence, head) only; in v and in the state its own
    column only."""
    import torch
    B, T, H, dk, dv, t0 = 2, 75, 2, 32, 20, 41
    q, k, v, g, beta, s0 = delta_inputs(4, B, T, H, H, dk, dv, torch.float32)
    clean = ops.delta_rule(q, k, v, g, beta, None, s0)
    {"q": q[1, t0, 0], "k": k[1, t0, 0], "v": v[1, t0, 0], "g": g[1, t0], "beta": beta[1, t0], "state": s0[1, 0, 3]}[where][0 if where in ("g", "beta") else 7] = value
    o, s = ops.delta_rule(q, k, v, g, beta, None, s0)
    hit = torch.zeros(B, T, H, dv, dtype=torch.bool)
    if where == "q":
        hit[1, t0, 0] = True
    elif where == "v":
        hit[1, t0:, 0, 7] = True
    elif where == "state":
        hit[1, :, 0, 7] = True
    else:
        hit[1, t0:, 0] = True
    hit = hit.cuda()
    assert torch.equal(o[~hit], clean[0][~hit])
    if where in ("g", "beta") and value == float("inf"):
        assert not torch.isfinite(o[1, t0 + 1:, 0]).any()
    else:
        assert not torch.isfinite(o[hit]).any()
    assert torch.equal(s[0], clean[1][0]) and torch.equal(s[1, 1], clean[1][1, 1])


def test_delta_rule_in_pieces_equals_whole_and_state_in_place(ops):
    """A sequence cut at any frame, the state carried: the same within the sum of the pieces' tolerances (other chunk borders); the
    state buffer may be the one it came from; two calls give the same bits."""
    import torch
    T, dk = 150, 64
    q, k, v, g, beta, s0 = delta_inputs(5, 2, T, 2, 2, dk, 64, torch.float32)
    o, s = ops.delta_rule(q, k, v, g, beta, None, s0)
    again = ops.delta_rule(q, k, v, g, beta, None, s0)
    assert torch.equal(o, again[0]) and torch.equal(s, again[1])
    for cut in (1, 32, 77):
        o1, s1 = ops.delta_rule(q[:, :cut], k[:, :cut], v[:, :cut], g[:, :cut], beta[:, :cut], None, s0)
        o2, s2 = ops.delta_rule(q[:, cut:], k[:, cut:], v[:, cut:], g[:, cut:], beta[:, cut:], None, s1)
        tol = 2 * delta_tol(T + 64, dk, max(float(s0.abs().max()), float(v.abs().max())) * 2)
        assert float((torch.cat((o1, o2), 1) - o).abs().max()) <= tol and float((s2 - s).abs().max()) <= tol


def test_delta_rule_empty(ops):
    import torch
    q, k, v, g, beta, s0 = delta_inputs(6, 2, 4, 1, 1, 16, 16, torch.float32)
    o, s = ops.delta_rule(q[:, :0], k[:, :0], v[:, :0], g[:, :0], beta[:, :0], None, s0)
    assert o.shape == (2, 0, 1, 16) and torch.equal(s, s0)
    o, s = ops.delta_rule(q[:0], k[:0], v[:0], g[:0], beta[:0])
    assert o.shape[0] == 0 and s.shape[0] == 0
    o, s = ops.delta_rule(q, k, v, g, beta, [0, 0], None)
    assert not o.any() and not s.any()


# ---------------------------------------------------------------- ticks
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 1, 2, 16, 16), (5, 2, 4, 64, 64), (4, 1, 1, 128, 128), (3, 3, 3, 96, 41), (2, 1, 2, 256, 36), (2, 1, 1, 256, 41), (2, 1, 1, 129, 50), (3, 1, 2, 128, 63), (2, 1, 1, 128, 129),
                                   (2, 1, 1, 33, 260), (70, 2, 2, 20, 12)], ids=str)
def test_delta_rule_online(ops, shape, dtype):
    import torch
    S, Hk, Hv, dk, dv = shape
    q, k, v, g, beta, _ = delta_inputs(7, S, 3, Hk, Hv, dk, dv, getattr(torch, dtype), packed=True)
    n = S + 3
    gen = torch.Generator().manual_seed(8)
    state = torch.randn(n, Hv, dk, dv, generator=gen).cuda()
    slots = torch.randperm(n, generator=gen)[:S].to(torch.int32).cuda()
    start = state.clone()
    idle = torch.ones(n, dtype=torch.bool, device="cuda")
    idle[slots.long()] = False
    outs = [ops.delta_rule_online(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], state, slots) for t in range(3)]
    wo, ws, top = delta_ref(q, k, v, g, beta, [3] * S, start[slots.long()], dk ** -0.5)
    # (three frames: each one's sums run over dk values)
    assert_delta(torch.stack(outs, 1), state[slots.long()], wo, ws, 3 * delta_tol(1, dk, max(top, float(v.abs().max()))), dtype == "bfloat16")
    assert torch.equal(state[idle], start[idle])


def test_delta_rule_online_slots_that_are_absent_negative_or_taken(ops):
    import torch
    S, H, dk, dv = 6, 2, 32, 24
    q, k, v, g, beta, _ = delta_inputs(9, S, 1, H, H, dk, dv, torch.float32)
    q, k, v, g, beta = (t[:, 0] for t in (q, k, v, g, beta))
    state = torch.randn(4, H, dk, dv, device="cuda")
    one = state.clone()
    slots = torch.tensor([2, -1, 4, 2, 0, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    o = ops.delta_rule_online(q, k, v, g, beta, state, slots)
    keep = [0, 4]
    ok = ops.delta_rule_online(q[keep], k[keep], v[keep], g[keep], beta[keep], one, [2, 0])
    assert torch.equal(state, one) and torch.equal(o[keep], ok)
    assert not o[1].any() and torch.isnan(o[[2, 3, 5]]).all()
    far = ops.delta_rule_online(q, k, v, g, beta, state, torch.tensor([2 ** 32, 0, 1, 2, 3, -2 ** 40], device="cuda"))
    assert torch.isnan(far[0]).all() and not far[5].any() and torch.isfinite(far[1:5]).all()


def test_a_tick_equals_the_sequence_of_one_frame(ops):
    import torch
    q, k, v, g, beta, s0 = delta_inputs(10, 3, 1, 2, 4, 64, 40, torch.float32)
    o, s = ops.delta_rule(q, k, v, g, beta, None, s0)
    state = s0.clone()
    o1 = ops.delta_rule_online(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state)
    tol = 2 * delta_tol(1, 64, max(float(s.abs().max()), float(v.abs().max())))
    assert float((o[:, 0] - o1).abs().max()) <= tol and float((s - state).abs().max()) <= tol


# ---------------------------------------------------------------- linear layer with adapters
def linear_inputs(seed, B, T, K, M, n, r, dtype):
    import torch
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    x, w, b = rn(B, T, K), rn(M, K) / math.sqrt(K), rn(M)
    down, up, scale = rn(n, r, K) / math.sqrt(K), rn(n, M, r), torch.rand(n, generator=gen) + 0.5
    ids = torch.randint(-1, n, (B,), generator=gen).to(torch.int32)
    return [t.to(dtype).cuda() for t in (x, w, b, down, up)] + [scale.cuda(), ids.cuda()]


def linear_ref(x, w, b, down, up, scale, ids, relu):
    """-> the definition in 64 bits and, elementwise, the sum of the magnitudes that an fp32 sum is off by a share of."""
    x, w, down, up = (npy(t.float()).astype(np.float64) for t in (x, w, down, up))
    b = np.zeros(w.shape[0]) if b is None else npy(b.float()).astype(np.float64)
    s = np.ones(down.shape[0]) if scale is None else npy(scale).astype(np.float64)
    y, mag = x @ w.T + b, np.abs(x) @ np.abs(w).T + np.abs(b)
    for i, a in enumerate(npy(ids).tolist()):
        if a >= 0:
            y[i] += s[a] * ((x[i] @ down[a].T) @ up[a].T)
            mag[i] += s[a] * ((np.abs(x[i]) @ np.abs(down[a]).T) @ np.abs(up[a]).T)
    return (np.where(y < 0, 0, y) if relu else y), mag


def assert_linear(y, want, mag, K, r, bf16):
    err = np.abs(npy(y.float()).astype(np.float64) - want) - (BF16 * np.abs(want) if bf16 else 0)
    tol = LAMBDA * U * math.sqrt(K + r + 3) * mag
    assert (err <= tol).all(), (float((err / tol).max()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1), (1, 1, 60, 256, 3, 8), (5, 1, 132, 96, 2, 4), (130, 1, 64, 65, 40, 16), (3, 40, 100, 70, 2, 5), (2, 129, 256, 300, 4, 32),
                                   (7, 125, 72, 2, 3, 64), (2, 64, 33, 31, 1, 128), (1, 300, 512, 96, 2, 8), (9, 17, 130, 257, 5, 33),
                                   (130, 1, 600, 65, 40, 16), (300, 2, 64, 40, 5, 8), (3, 40, 600, 70, 2, 5), (280, 45, 200, 70, 3, 9), (100, 129, 96, 33, 3, 64), (4, 2100, 70, 200, 3, 20),
                                   (2, 4100, 33, 150, 2, 40)], ids=str)
def test_linear_adapted(ops, shape, dtype):
    import torch
    B, T, K, M, n, r = shape
    x, w, b, down, up, scale, ids = linear_inputs(11, B, T, K, M, n, r, getattr(torch, dtype))
    for relu in (False, True):
        y = ops.linear_adapted(x, w, b, down, up, scale, ids, relu=relu)
        assert y.shape == (B, T, M) and y.dtype == x.dtype
        assert_linear(y, *linear_ref(x, w, b, down, up, scale, ids, relu), K, r, dtype == "bfloat16")
    y = ops.linear_adapted(x, w, None, down, up, None, ids.long())
    assert_linear(y, *linear_ref(x, w, None, down, up, None, ids, False), K, r, dtype == "bfloat16")
    if T == 1:
        assert torch.equal(ops.linear_adapted(x[:, 0], w, None, down, up, None, ids), y[:, 0])


@pytest.mark.parametrize("shape", [(3, 2043, 128, 2050, 2, 20), (5, 1250, 192, 2048, 3, 32), (6200, 1, 64, 2048, 4, 8), (2, 3100, 72, 2048, 2, 4), (1, 6200, 64, 2100, 1, 33)], ids=str)
def test_linear_adapted_many_rows_to_many_columns(ops, shape):
    """The large tiles: rows that are whole cache lines go to LDS directly, others through registers; both ends ragged; a view whose
    rows start in the middle of a line."""
    import torch
    B, T, K, M, n, r = shape
    x, w, b, down, up, scale, ids = linear_inputs(13, B, T, K, M, n, r, torch.bfloat16)
    want = linear_ref(x, w, b, down, up, scale, ids, True)
    assert_linear(ops.linear_adapted(x, w, b, down, up, scale, ids, relu=True), *want, K, r, True)
    wide = torch.full((B, T, K + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
    for at in (8, 4, 1):
        wide[..., at:at + K] = x
        assert_linear(ops.linear_adapted(wide[..., at:at + K], w, b, down, up, scale, ids, relu=True), *want, K, r, True)


def test_linear_adapted_strides_ids_and_non_finite_values(ops):
    import torch
    B, T, K, M, n, r = 4, 37, 48, 80, 3, 8
    x, w, b, down, up, scale, _ = linear_inputs(12, B, T, K, M, n, r, torch.float32)
    y = ops.linear_adapted(x, w, b, down, up, scale, [2, -1, 0, -5])
    pad = torch.full((T, B, K + 5), float("nan"), device="cuda")
    xs = pad[..., :K].transpose(0, 1).copy_(x)
    assert torch.equal(ops.linear_adapted(xs, w, b, down, up, scale, [2, -1, 0, -1]), y)
    assert torch.equal(ops.linear_adapted(x.transpose(1, 2).contiguous().transpose(1, 2), w.t().contiguous().t(), b, down, up, scale, [2, -1, 0, -1]), y)
    # an adapter that is not there: that sequence's rows only
    z = ops.linear_adapted(x, w, b, down, up, scale, torch.tensor([2, 3, 0, 2 ** 31 - 1], device="cuda", dtype=torch.int32), relu=True)
    assert torch.isnan(z[[1, 3]]).all() and torch.equal(z[[0, 2]], torch.relu(y[[0, 2]]))
    # an adapter with NaN that nobody uses, and a row of NaN: ReLU keeps it, its neighbours do not see it
    down[1], up[1], scale[1] = float("nan"), float("inf"), float("nan")
    x[2, 20, 3] = float("nan")
    z = ops.linear_adapted(x, w, b, down, up, scale, [2, -1, 0, -1], relu=True)
    assert torch.isnan(z[2, 20]).all()
    z[2, 20], y[2, 20] = 0, 0
    assert torch.equal(z, torch.relu(y))
    assert ops.linear_adapted(x[:0], w, b, down, up, scale, []).shape == (0, T, M)
    assert ops.linear_adapted(x[:, :0], w, b, down, up, scale, [0] * B).shape == (B, 0, M)


# ---------------------------------------------------------------- together
class Block:
    """A personalised recurrent block: projections with an adapter per sequence, the gated delta rule, an output projection."""

    def __init__(self, ops, K, Hk, Hv, dk, dv, n, r, dtype, seed=20):
        import torch
        gen = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=gen)
        self.ops, self.dims = ops, (Hk, Hv, dk, dv)
        M = 2 * Hk * dk + Hv * dv + 2 * Hv
        t = lambda x: x.to(dtype).cuda()
        self.w1, self.b1, self.d1, self.u1 = t(rn(M, K) / math.sqrt(K)), t(rn(M) * 0.1), t(rn(n, r, K) / math.sqrt(K)), t(rn(n, M, r) * 0.3)
        self.w2, self.d2, self.u2 = t(rn(K, Hv * dv) / math.sqrt(Hv * dv)), t(rn(n, r, Hv * dv) / math.sqrt(Hv * dv)), t(rn(n, K, r) * 0.3)
        self.scale = torch.full((n,), 0.5).cuda()

    def split(self, p):
        import torch
        Hk, Hv, dk, dv = self.dims
        a, b, c = Hk * dk, 2 * Hk * dk, 2 * Hk * dk + Hv * dv
        q, k, v = unit(p[..., :a].unflatten(-1, (Hk, dk))), unit(p[..., a:b].unflatten(-1, (Hk, dk))), p[..., b:c].unflatten(-1, (Hv, dv))
        return q, k, v, -torch.nn.functional.softplus(p[..., c:c + Hv].float()), torch.sigmoid(p[..., c + Hv:].float())

    def sequence(self, x, ids, lengths, state):
        o, state = self.ops.delta_rule(*self.split(self.ops.linear_adapted(x, self.w1, self.b1, self.d1, self.u1, self.scale, ids)), lengths, state)
        return self.ops.linear_adapted(o.flatten(-2), self.w2, None, self.d2, self.u2, self.scale, ids), state

    def tick(self, x, ids, state, slots):
        o = self.ops.delta_rule_online(*self.split(self.ops.linear_adapted(x, self.w1, self.b1, self.d1, self.u1, self.scale, ids)), state, slots)
        return self.ops.linear_adapted(o.flatten(-2), self.w2, None, self.d2, self.u2, self.scale, ids)


def test_block_offline_then_live(ops):
    """The operators as a program uses them: a batch of recordings through the block, then the same people live, frame by frame on
    the states the recordings left -- equal to the recordings run on."""
    import torch
    block = Block(ops, 60, 2, 4, 32, 24, 3, 4, torch.float32)
    gen = torch.Generator().manual_seed(21)
    x = torch.randn(3, 60, 60, generator=gen).cuda()
    ids = torch.tensor([2, -1, 0], device="cuda", dtype=torch.int32)
    whole, end = block.sequence(x, ids, None, None)
    y, state = block.sequence(x[:, :50], ids, None, None)
    slots = torch.tensor([1, 2, 0], device="cuda", dtype=torch.int32)
    live = torch.empty_like(state)
    live[slots.long()] = state
    ys = [y] + [block.tick(x[:, t], ids, live, slots).unsqueeze(1) for t in range(50, 60)]
    # the same frames with other chunk borders: the state within 2 x the rule's own tolerance, outputs are sums of 96 of its
    # values with weights of magnitude 1/sqrt(96) and an adapter of at most twice that
    tol = 2 * delta_tol(60 + 10 * 32, 32, float(end.abs().max()) + 10.0) * 3 * math.sqrt(96)
    assert float((torch.cat(ys, 1) - whole).abs().max()) <= tol
    assert float((live[slots.long()] - end).abs().max()) <= tol


def test_operators_on_streams_and_in_captured_graphs(ops):
    """Two streams at once; a captured tick (adapters -> delta rule -> adapters) replayed several times with eager work between the
    replays; ids, slots and lengths are read on replay."""
    import torch
    block = Block(ops, 64, 2, 2, 64, 64, 4, 8, torch.bfloat16)
    gen = torch.Generator().manual_seed(22)
    xs = [torch.randn(6, 64, generator=gen).to(torch.bfloat16).cuda() for _ in range(5)]
    ids = torch.tensor([0, 1, 2, 3, -1, 0], device="cuda", dtype=torch.int32)
    slots = torch.arange(6, device="cuda", dtype=torch.int32)
    start = torch.randn(6, 2, 64, 64, generator=gen).cuda()
    eager_state, eager = start.clone(), []
    for i, x in enumerate(xs):
        if i == 3:
            ids = ids.flip(0)
        eager.append(block.tick(x, ids, eager_state, slots))
    ids = ids.flip(0)
    x, state = xs[0].clone(), start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.tick(x, ids, state, slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.tick(x, ids, state, slots)
        seq = ops.delta_rule(*block.split(ops.linear_adapted(x[None], block.w1, block.b1, block.d1, block.u1, block.scale, ids[:1])), ids[:1])[0]
    state.copy_(start)
    for i, step in enumerate(xs):
        if i == 3:
            ids.copy_(ids.flip(0))
        x.copy_(step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[i]), i
        n = max(0, int(ids[0]))
        assert not seq[:, n:].any() and (n == 0 or seq[:, :n].any())
        (eager_state @ eager_state).sum().item()
    assert torch.equal(state, eager_state)
    # two streams, one model: the operators share no workspace
    B, T = 3, 200
    args = [delta_inputs(30 + i, B, T, 2, 2, 64, 64, torch.float32) for i in range(2)]
    want = [ops.delta_rule(*a[:5], None, a[5]) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, a in zip(streams, args):
            with torch.cuda.stream(st):
                got.append(ops.delta_rule(*a[:5], None, a[5]))
        torch.cuda.synchronize()
        for (o, s), (wo, ws) in zip(got, want):
            assert torch.equal(o, wo) and torch.equal(s, ws)


def test_refusals(ops):
    import torch
    q, k, v, g, beta, s0 = delta_inputs(40, 2, 5, 2, 4, 16, 8, torch.float32)
    bad = [lambda: ops.delta_rule(q, k.bfloat16(), v, g, beta), lambda: ops.delta_rule(q.half(), k.half(), v.half(), g, beta),
           lambda: ops.delta_rule(q, k, v[:, :, :3], g[:, :, :3], beta[:, :, :3]), lambda: ops.delta_rule(q, k[:, :4], v, g, beta),
           lambda: ops.delta_rule(q, k, v, g[..., :2], beta), lambda: ops.delta_rule(q, k, v, g.double(), beta),
           lambda: ops.delta_rule(q, k, v, g, beta, [5, 6]), lambda: ops.delta_rule(q, k, v, g, beta, [5, -1]), lambda: ops.delta_rule(q, k, v, g, beta, [5]),
           lambda: ops.delta_rule(q, k, v, g, beta, None, s0[:, :2]), lambda: ops.delta_rule(q, k, v, g, beta, None, s0.double()),
           lambda: ops.delta_rule(q.cpu(), k, v, g, beta), lambda: ops.delta_rule(q.requires_grad_(), k, v, g, beta),
           lambda: ops.delta_rule(torch.zeros(1, 1, 1, 257, device="cuda"), torch.zeros(1, 1, 1, 257, device="cuda"), v[:1, :1, :1], g[:1, :1, :1], beta[:1, :1, :1])]
    q = q.detach()
    tick = [t[:, 0] for t in (q, k, v, g, beta)]
    bad += [lambda: ops.delta_rule_online(*tick, s0[:1]), lambda: ops.delta_rule_online(*tick, s0, [0, 2]), lambda: ops.delta_rule_online(*tick, s0, [0]),
            lambda: ops.delta_rule_online(*tick, s0.transpose(2, 3)), lambda: ops.delta_rule_online(*tick, s0.cpu()),
            lambda: ops.delta_rule_online(*tick, s0, torch.zeros(2, device="cuda"))]
    x, w, b, down, up, scale, ids = linear_inputs(41, 2, 3, 16, 24, 2, 4, torch.float32)
    bad += [lambda: ops.linear_adapted(x, w, b, down, up, scale, [0, 2]), lambda: ops.linear_adapted(x, w, b, down, up, scale, [0]),
            lambda: ops.linear_adapted(x, w, b, down, up[:, :23], scale, ids), lambda: ops.linear_adapted(x, w, b.bfloat16(), down, up, scale, ids),
            lambda: ops.linear_adapted(x[..., :15], w, b, down, up, scale, ids), lambda: ops.linear_adapted(x, w, b, down, up, scale.double(), ids),
            lambda: ops.linear_adapted(x, w, b, torch.zeros(2, 129, 16, device="cuda"), torch.zeros(2, 24, 129, device="cuda"), scale, ids),
            lambda: ops.linear_adapted(x, w, b[:3], down, up, scale, ids), lambda: ops.linear_adapted(x, w, b, down.cpu(), up, scale, ids)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError("call %d was not refused" % i)


BLOCKS = {"joints": (60, 256, 2, 72), "pose": (132, 256, 2, 96), "foot_contact": (132, 64, 2, 2), "velocity": (132, 256, 1, 72)}


def block_adapters(module, n, r1, r2, seed):
    """Adapters of magnitude 1/10 of the layers' own weights, on the host."""
    import torch
    n_in, H, dirs, n_out = BLOCKS[module]
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    layer = lambda K, M, r: (rn(n, r, K) / math.sqrt(K), 0.1 * rn(n, M, r) / math.sqrt(r), torch.rand(n, generator=gen) + 0.5)
    return {"linear1": layer(n_in, H, r1), "linear2": layer(dirs * H, n_out, r2)}


def merged(weights, prefix, adapters, a):
    """The block's weights with adapter `a` added to them (None: as they are)."""
    sd = dict(weights)
    if a is not None:
        for name, (down, up, scale) in adapters.items():
            key = prefix + name + ".weight"
            sd[key] = (sd[key].astype(np.float64) + float(scale[a]) * (up[a].double() @ down[a].double()).numpy()).astype(np.float32)
    return sd


@pytest.mark.parametrize("lstm_mode", [1, 0])
@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (2, 80), (40, 5)], ids=str)
@pytest.mark.parametrize("module", list(BLOCKS))
def test_block_of_the_model_with_adapters(ops, module, shape, lstm_mode):
    """rnn_forward with adapters equals, sequence by sequence, the block whose weights have the adapter added (rounding the sums of
    the weights is 2^-24 of them: nothing beside the 1e-4 that the network outputs are held to); ragged, on a carried state."""
    import torch
    from mobileposer_amd import synthetic
    from oracle import mp_oracle as O
    weights = synthetic.make_weights(0)
    n_in, H, dirs, n_out = BLOCKS[module]
    B, T = shape
    adapters = block_adapters(module, 3, 4, 8, 30)
    dev = {k: tuple(t.cuda() for t in v) for k, v in adapters.items()}
    gen = torch.Generator().manual_seed(31)
    x = torch.randn(B, T, n_in, generator=gen)
    state = [0.3 * torch.randn(2 * dirs, B, H, generator=gen) for _ in range(2)]
    lengths = [max(1, T - 3 * (b % 4)) for b in range(B)]
    lengths[0] = T
    ids = [2, -1, 0, 1][:B] if B <= 4 else [b % 4 - 1 for b in range(B)]
    ops.set_lstm_mode(lstm_mode)
    try:
        y, (h, c) = ops.rnn_forward(module, x.cuda(), lengths, [s.cuda() for s in state], dev, ids)
        one, _ = ops.rnn_forward(module, x.cuda(), lengths, None, {"linear2": dev["linear2"]}, torch.tensor(ids).cuda())
        plain, _ = ops.rnn_forward(module, x.cuda(), lengths, None)
        none, _ = ops.rnn_forward(module, x.cuda(), lengths, None, dev, [-1] * B)
    finally:
        ops.set_lstm_mode(1)
    assert float((none - plain).abs().max()) < 1e-4
    for b in {0, 1 % B, B // 2, B - 1}:
        a = None if ids[b] < 0 else ids[b]
        n = lengths[b]
        sd = merged(weights, O.PREFIX[module], adapters, a)
        wy, (wh, wc) = O.rnn_forward(sd, O.PREFIX[module], x[b:b + 1].numpy(), [n], tuple(s[:, b:b + 1].numpy() for s in state))
        assert np.abs(npy(y[b, :n]) - wy[0, :n]).max() < 1e-4
        assert np.abs(npy(h[:, b]) - wh[:, 0]).max() < 1e-4 and np.abs(npy(c[:, b]) - wc[:, 0]).max() < 1e-4
        sd = merged(weights, O.PREFIX[module], {"linear2": adapters["linear2"]}, a)
        wy, _ = O.rnn_forward(sd, O.PREFIX[module], x[b:b + 1].numpy(), [n])
        assert np.abs(npy(one[b, :n]) - wy[0, :n]).max() < 1e-4


def test_block_of_the_model_with_adapters_that_are_not_there(ops):
    """An id on the device that is no adapter's: that sequence's outputs are NaN, the others' are what they are without it; the call
    behind it is untouched."""
    import torch
    dev = {k: tuple(t.cuda() for t in v) for k, v in block_adapters("velocity", 2, 4, 8, 33).items()}
    x = torch.randn(3, 20, 132, generator=torch.Generator().manual_seed(34)).cuda()
    run = lambda ids: ops.rnn_forward("velocity", x, [20, 15, 20], None, dev, torch.tensor(ids, device="cuda", dtype=torch.int32))[0]
    want, got, after = run([1, 0, -1]), run([1, 2, -1]), run([1, 0, -1])
    assert torch.isnan(got[1, :15]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.equal(after, want)


def test_block_of_the_model_with_adapters_refusals(ops):
    import torch
    dev = {k: tuple(t.cuda() for t in v) for k, v in block_adapters("pose", 2, 4, 8, 32).items()}
    x = torch.zeros(2, 3, 132, device="cuda")
    down, up, scale = dev["linear1"]
    run = lambda adapters, ids: ops.rnn_forward("pose", x, [3, 3], None, adapters, ids)
    for adapters, ids in [({}, [0, 1]), ({"linear3": dev["linear1"]}, [0, 1]), (dev, None), (None, [0, 1]), (dev, [0, 2]), (dev, [0]),
                          ({"linear1": dev["linear2"]}, [0, 1]), ({"linear1": (down, up[:1], scale)}, [0, 1]), ({"linear1": (down, up, scale[:1])}, [0, 1]),
                          ({"linear1": (down.bfloat16(), up.bfloat16(), None)}, [0, 1]), ({"linear1": (down.cpu(), up, scale)}, [0, 1]),
                          ({"linear1": (down[:1], up[:1], None), "linear2": dev["linear2"]}, [0, 0])]:
        with pytest.raises(RuntimeError):
            run(adapters, ids)
    ops.set_lstm_mode(3)
    try:
        with pytest.raises(RuntimeError, match="mode 1 or 0"):
            run(dev, [0, 1])
    finally:
        ops.set_lstm_mode(1)


def test_foot_contact_block_with_adapters_in_the_split_mode(ops):
    """Mode 3 concerns the H = 256 blocks only: the H = 64 block takes adapters there and gives what it gives in mode 1."""
    import torch
    dev = {k: tuple(t.cuda() for t in v) for k, v in block_adapters("foot_contact", 2, 4, 8, 35).items()}
    x = torch.randn(3, 70, 132, generator=torch.Generator().manual_seed(36)).cuda()
    run = lambda: ops.rnn_forward("foot_contact", x, [70, 41, 70], None, dev, [0, -1, 1])[0]
    want = run()
    ops.set_lstm_mode(3)
    try:
        got = run()
    finally:
        ops.set_lstm_mode(1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(2, 3100, 128, 2050, 2, 20), (4, 300, 100, 70, 2, 5), (3, 1, 1024, 300, 3, 16)], ids=str)
def test_linear_adapted_captured(ops, shape):
    """Every kind of launch (large tiles straight to LDS, one launch, small tiles) in a graph: replays with other inputs and ids, the
    eager call between them."""
    import torch
    x, w, b, down, up, scale, ids = linear_inputs(14, *shape, torch.bfloat16)
    call = lambda: ops.linear_adapted(x, w, b, down, up, scale, ids, relu=True)
    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for i in range(4):
        x.copy_(x.roll(1, -1))
        ids.copy_((ids + 2) % (shape[4] + 1) - 1)
        graph.replay()
        got = y.clone()
        assert torch.equal(got, call())
        torch.cuda.synchronize()
