"""Per-head edge attention in 64 bits (host), from its definition, and how far fp32 arithmetic may be from it."""
import math

import torch

from tests import mx8_oracle as Q8

U = 2.0 ** -24                     # fp32: half a step, relative


def forward(Q, K, V, E1, E2, nm, H, cap=0.0, groups=None):
    """Y, wV and (S', P) as (B,n,n,H), all float64; differentiable."""
    B, n, dx = Q.shape
    pm = (nm[:, :, None] & nm[:, None, :])[..., None]
    zero = torch.zeros((), dtype=torch.float64)
    e1, e2 = torch.where(pm, E1, zero), torch.where(pm, E2, zero)
    Y = Q[:, :, None] * K[:, None] / math.sqrt(dx // H) * (1 + e1) + e2
    S = Y.reshape(B, n, n, H, dx // H).sum(-1)
    if cap > 0:
        S = cap * torch.tanh(S / cap)
    if groups is not None:
        on = (groups[:, :, None] == groups[:, None, :]) & (groups >= 0)[:, :, None]
        S = torch.where(on[..., None], S, torch.full((), -math.inf, dtype=torch.float64))
    top = S.detach().amax(2, keepdim=True)
    top = torch.where(torch.isinf(top), zero, top)
    P = torch.exp(S - top)
    P = P / torch.where(P.sum(2, keepdim=True) > 0, P.sum(2, keepdim=True), torch.ones((), dtype=torch.float64))
    wV = torch.einsum('bijh,bjhc->bihc', P, V.reshape(B, n, H, dx // H)).reshape(B, n, dx)
    return Y, wV, S, P


def gradients(Q, K, V, E1, E2, nm, H, dY, dwV, cap=0.0, groups=None, e1_held=None):
    """dQ, dK, dV, dE1, dE2 by automatic differentiation of forward(); `e1_held`: the values of E1 that the backward pass has (8 bits): P, dE1 and
    dE2 are those of E1 itself, dQ and dK take the held values."""
    leaves = [t.detach().clone().requires_grad_(True) for t in (Q, K, V, E1, E2)]
    Y, wV, _, _ = forward(*leaves, nm, H, cap, groups)
    g = list(torch.autograd.grad((Y, wV), leaves, (dY, dwV)))
    if e1_held is not None:
        B, n, dx = Q.shape
        pm = (nm[:, :, None] & nm[:, None, :])[..., None]
        # the gradient of Y: dE2 without the mask
        Yl = Y.detach().requires_grad_(True)
        S = Yl.reshape(B, n, n, H, dx // H).sum(-1)
        if cap > 0:
            S = cap * torch.tanh(S / cap)
        if groups is not None:
            on = (groups[:, :, None] == groups[:, None, :]) & (groups >= 0)[:, :, None]
            S = torch.where(on[..., None], S, torch.full((), -math.inf, dtype=torch.float64))
        top = S.detach().amax(2, keepdim=True)
        P = torch.exp(S - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        P = P / P.sum(2, keepdim=True).clamp_min(1e-300)
        w = torch.einsum('bijh,bjhc->bihc', P, V.detach().reshape(B, n, H, dx // H)).reshape(B, n, dx)
        G = dY + torch.autograd.grad(w, Yl, dwV)[0]
        f = G * (1 + torch.where(pm, e1_held, torch.zeros((), dtype=torch.float64))) / math.sqrt(dx // H)
        g[0], g[1] = (f * K.detach()[:, None]).sum(2), (f * Q.detach()[:, :, None]).sum(1)
    return g


def held(E1):
    return Q8.quantize(E1.reshape(-1, E1.shape[-1]))[2].reshape(E1.shape)


def bounds(Q, K, V, E1, E2, nm, H, dY, dwV, out_eps, cap=0.0, groups=None, e1_held=None):
    """Elementwise bounds on |fp32 - 64 bits| of (Y, wV, dQ, dK, dV, dE1, dE2).  out_eps: half a step of the pair tensors' type, relative.

    Y: s Q, times K, 1 + E1, their product, the sum with E2: 5 roundings of A = |s Q K| (1 + |E1|) + |E2|.  S: those and the sum of df
    terms (8 in a lane, 4 exchanges): 17 U sum A; tanh and its two products: 6 U cap more.  P: the error of S (twice: its own and the
    sum's), S - max and the exponential's argument (4 U max |S - max|), the sum over n keys and the merges of slots and waves (n + 32) U:
    relative eps.  wV: eps sum P |V|.  dP: 13 U a, a = sum |dwV| |V|; D: (eps + 13 U) d, d = sum |dwV| sum P |V|; dS: P's eps on
    |dP - D| <= a + d, those two, and the tanh's factor (absolute error 2 dS' / cap + 3 U): P (3 eps + 40 U) (a + d) =: x.  G: x + 2 U |G|.
    dE2, dE1: that times 1 or |s Q K| (3 more roundings), then their type's.  dQ, dK, dV: sums of at most n + 64 terms in some order."""
    B, n, dx = Q.shape
    df = dx // H
    s = 1 / math.sqrt(df)
    heads = lambda t: t.reshape(t.shape[:-1] + (H, df))
    pm = (nm[:, :, None] & nm[:, None, :])[..., None]
    zero = torch.zeros((), dtype=torch.float64)
    e1, e2 = torch.where(pm, E1, zero).abs(), torch.where(pm, E2, zero).abs()
    qk = (Q[:, :, None] * K[:, None]).abs() * s
    A = qk * (1 + e1) + e2
    Y, wV, S, P = forward(Q, K, V, E1, E2, nm, H, cap, groups)
    fin = torch.where(torch.isinf(S), zero, S)
    dS = 17 * U * heads(A).sum(-1).max() + 6 * U * cap
    spread = float((fin.amax(2, keepdim=True) - fin).max())
    eps = 2 * dS + (4 * spread + n + 32) * U
    PV = torch.einsum('bijh,bjhc->bihc', P, heads(V).abs()).reshape(B, n, dx)
    out = [5 * U * A + out_eps * Y.abs(), eps * PV]
    a = torch.einsum('bihc,bjhc->bijh', heads(dwV).abs(), heads(V).abs())
    d = heads(dwV.abs() * PV).sum(-1)
    x = (P * (3 * eps + 40 * U) * (a + d[:, :, None])).repeat_interleave(df, -1)
    gr = gradients(Q, K, V, E1, E2, nm, H, dY, dwV, cap, groups)
    G = dY.abs() + (P * (a + d[:, :, None])).repeat_interleave(df, -1)        # at least |G|
    dG = x + 2 * U * G
    f = (1 + (e1 if e1_held is None else torch.where(pm, e1_held, zero).abs())) * s
    depth = (n + 64) * U
    out += [((dG + (5 * U + depth) * G) * f * K[:, None].abs()).sum(2), ((dG + (5 * U + depth) * G) * f * Q[:, :, None].abs()).sum(1)]
    out += [torch.einsum('bijh,bihc->bjhc', P * (eps + depth), heads(dwV).abs()).reshape(B, n, dx)]
    out += [(dG + 4 * U * G) * qk * (1 + out_eps) + out_eps * gr[3].abs(), dG * (1 + out_eps) + out_eps * gr[4].abs()]
    return out
