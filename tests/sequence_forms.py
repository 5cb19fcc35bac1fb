"""The sequence operators' formulas on the host: in 64 bits frame by frame, and in fp32 in the order in which the kernels sum (chunks of
32 frames, 32 products a step), with operands cut to a number of bf16 terms where a test wants to know what such a cut does.

Accuracy of the kernels is held to that of the fp32 form: the same products, each fp32 sum one rounding off, only in another order
within a step.  Two such sums' errors are alike in size, not equal: ALIKE = 3 in the root mean square over thousands of values; the
largest of them may differ by one more ratio of that kind (a maximum over 10^4 .. 10^5 values is 4 to 5 of their deviation, give or take a
tenth), LARGEST = 4.  An operand of two bf16 terms is off by up to 2^-18 of itself, 64 times an fp32 rounding."""
import math

import torch

ALIKE, LARGEST = 3.0, 4.0


def terms(x, n):
    """x as the sum of its first n bf16 terms, each the nearest to what the ones before leave (None: x itself)."""
    if n is None:
        return x
    left, out = x.clone(), torch.zeros_like(x)
    for _ in range(n):
        t = left.to(torch.bfloat16).to(x.dtype)
        out, left = out + t, left - t
    return out


def delta_inputs(seed, B, T, Hk, Hv, dk, dv, dtype):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    q, k, v = (t.to(dtype) for t in (unit(rn(B, T, Hk, dk)), unit(rn(B, T, Hk, dk)), rn(B, T, Hv, dv)))
    g = -torch.exp(torch.linspace(-4, 0, Hv)) * torch.rand(B, T, Hv, generator=gen)
    return q, k, v, g, torch.sigmoid(2 * rn(B, T, Hv)), 0.5 * rn(B, Hv, dk, dv)


def delta_exact(q, k, v, g, beta, state, scale):
    q, k, v, g, beta, S = (t.double() for t in (q, k, v, g, beta, state))
    rep = v.shape[2] // q.shape[2]
    o = torch.empty_like(v)
    for t in range(v.shape[1]):
        kt, qt = (x[:, t].repeat_interleave(rep, 1) for x in (k, q))
        S = S * g[:, t].exp()[..., None, None]
        u = beta[:, t][..., None] * (v[:, t] - (S * kt[..., None]).sum(2))
        S = S + kt[..., None] * u[..., None, :]
        o[:, t] = scale * (S * qt[..., None]).sum(2)
    return o, S


def delta_fp32(q, k, v, g, beta, state, scale, cut=None, out_cut=None):
    """The chunked form in fp32 (outputs not rounded further).  cut: terms of every operand; out_cut: of those that the outputs alone
    see (P, U beside it, S beside Q).  T has to be a multiple of 32."""
    q, k, v = q.float(), k.float(), v.float()
    C, rep, H = 32, v.shape[2] // q.shape[2], v.shape[2]
    out_cut = cut if out_cut is None else out_cut
    ct, co = (lambda x: terms(x, cut)), (lambda x: terms(x, out_cut))
    fold = lambda x: x.unflatten(1, (-1, C)).movedim(3, 1)                  # [B, H, n, C, ..]
    q, k, v = fold(q.repeat_interleave(rep, 2)), fold(k.repeat_interleave(rep, 2)), fold(v)
    beta, G = fold(beta[..., None])[..., 0], fold(g[..., None])[..., 0].double().cumsum(-1)
    low = torch.ones(C, C, dtype=torch.bool).tril()
    D = torch.where(low, (G[..., :, None] - G[..., None, :]).clamp_max(0).exp(), 0.0).float()
    A = (beta[..., None] * D * (ct(k) @ ct(k).transpose(-1, -2))).tril(-1)
    P = scale * D * (ct(q) @ ct(k).transpose(-1, -2))
    Ti = torch.linalg.solve_triangular(torch.eye(C) + A, torch.eye(C).expand_as(A), upper=False, unitriangular=True) * beta[..., None, :]
    eg, tail, whole = G.exp().float(), (G[..., -1:] - G).exp().float(), G[..., -1].exp().float()
    S, o = state, torch.empty(*v.shape)
    for n in range(v.shape[2]):
        R = v[:, :, n] - eg[:, :, n, :, None] * (ct(k[:, :, n]) @ ct(S))
        u = ct(Ti[:, :, n]) @ ct(R)
        o[:, :, n] = scale * eg[:, :, n, :, None] * (ct(q[:, :, n]) @ co(S)) + co(P[:, :, n]) @ co(u)
        S = whole[:, :, n, None, None] * S + ct(k[:, :, n]).transpose(-1, -2) @ ct(tail[:, :, n, :, None] * u)
    return o.movedim(1, 3).flatten(1, 2), S


def linear_inputs(seed, B, T, K, M, n, r, dtype, adapter=1.0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    x, w, b = rn(B, T, K), rn(M, K) / math.sqrt(K), rn(M)
    down, up = rn(n, r, K) / math.sqrt(K), adapter * rn(n, M, r) / math.sqrt(r)
    scale, ids = torch.rand(n, generator=gen) + 0.5, torch.randint(-1, n, (B,), generator=gen).to(torch.int32)
    return [t.to(dtype) for t in (x, w, b, down, up)] + [scale, ids]


def linear_exact(x, w, b, down, up, scale, ids):
    x, w, b, down, up = (t.double() for t in (x, w, b, down, up))
    y = x @ w.t() + b
    for i, a in enumerate(ids.tolist()):
        if a >= 0:
            y[i] += float(scale[a]) * ((x[i] @ down[a].t()) @ up[a].t())
    return y


def linear_fp32(x, w, b, down, up, scale, ids, cut=None, z_cut=None):
    """fp32, 32 products a step; cut: terms of every operand, z_cut: of scale Down x alone."""
    def product(a, m):
        a, m = terms(a, cut), terms(m, cut)
        acc = torch.zeros(*a.shape[:-1], m.shape[0])
        for k in range(0, a.shape[-1], 32):
            acc = acc + a[..., k:k + 32] @ m[:, k:k + 32].t()
        return acc
    x, w, b, down, up = (t.float() for t in (x, w, b, down, up))
    y = product(x, w)
    for i, a in enumerate(ids.tolist()):
        if a >= 0:
            z = terms(scale[a] * product(x[i], down[a]), z_cut)
            y[i] = y[i] + product(z, up[a])
    return y + b


def step_of(want):
    """The distance of bf16 numbers at `want`."""
    return torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -126))) - 7)


def held(got, want, plain):
    """The worst ratio of `got`'s error to its bound; `plain` is the fp32 form, both against the 64-bit `want`.  fp32: the root mean
    square and the largest error.  bf16: the sum of what is beyond half a step.  A value that was off by e before its rounding crosses
    the middle between two bf16 numbers with probability e / step and is then beyond half a step by e / 2 on average: e^2 / (2 step),
    at most e.  That grows with the square of the errors; a few crossings more than expected are a few of the largest e."""
    off, err = (plain.double() - want).abs(), (got.double() - want).abs()
    if got.dtype is torch.float32:
        return max(float(err.max() / (LARGEST * off.max())), float(err.pow(2).mean().sqrt() / (ALIKE * off.pow(2).mean().sqrt())))
    step = step_of(want)
    expected = torch.minimum(off, off * off / (2 * step)).sum()
    return float((err - step / 2).clamp_min(0).sum() / (ALIKE ** 2 * expected + LARGEST * off.max()))


DELTA = [(1, 96, 1, 2, 32, 32), (2, 160, 1, 1, 64, 64), (1, 320, 2, 4, 128, 128), (1, 96, 1, 1, 256, 40), (2, 128, 1, 2, 72, 41), (1, 1024, 1, 1, 64, 64), (1, 1024, 2, 2, 128, 96)]
LINEAR = [(2, 40, 64, 96, 2, 32), (7, 33, 132, 300, 3, 8), (130, 1, 600, 200, 5, 16), (1, 300, 512, 96, 1, 24)]
