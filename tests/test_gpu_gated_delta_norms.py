"""The chunked gated delta rule's error in norm, chunk by chunk and head by head, for keys that lie in all directions and for keys that hardly differ.

Two bars.  For independent keys the roundings do not amplify one another: one to a type of half step h is h / sqrt(3) of its operand at most in the mean
square, the six operands and the result forward and the sixteen and the result backward are independent, so that sqrt(7 / 3) h and sqrt(17 / 3) h are
expected at most in a tensor; a chunk of one head has 64 rows of it and may be half as much above that again.  The gradient of a decay is the inner product of a state
with its adjoint, K V terms of either sign: its error goes by the root of the sum of their squares, whatever the sum itself has come to.

Correlated keys, and strengths beyond one, make the inverse of a chunk and the products with it large against their sum: r = X V - W S0 cancels, and so do the answers.  How
much is lost then is the roundings' doing, so they are carried out in 64 bits here, at the places that the kernels' heads name and nowhere else: a tensor's
error may be half as much again as theirs (sums in 32 bits, products of split factors).
"""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle
from tests.test_gpu_gated_delta import BF16, F16, HALF_STEP

pytestmark = pytest.mark.gpu

C = 64


def emulated(q, k, v, g, beta, s0, do, ds, dtype):
    """o, final state and the gradients of q, k, v, g, beta and s0, of one head (L, .), with the kernels' roundings."""
    rnd = lambda t: t.to(dtype).double()  # noqa: E731
    scale, state, chunks = q.shape[1] ** -0.5, s0, []
    for t0 in range(0, len(q), C):
        Q, K, V, B = (t[t0:t0 + C] for t in (q, k, v, beta))
        c = torch.cumsum(g[t0:t0 + C], 0)
        gam, suf = c.exp(), (c[-1] - c).exp()
        G = torch.exp((c[:, None] - c[None]).tril()).tril()
        X = torch.linalg.inv(torch.eye(len(Q), dtype=torch.float64) + (G * B * (K @ K.T)).tril(-1))
        P, X16 = rnd(scale * G * B * (Q @ K.T)), rnd(X)
        W, Wb, Y = rnd(rnd(X * gam) @ K), rnd(rnd(X.T * (B * suf)) @ K), rnd(P @ X16)
        Z, S = rnd(scale * gam[:, None] * Q - P @ W), rnd(state)
        r = X16 @ V - W @ S.T
        chunks.append((Q, K, B, G, gam, suf, Y, Wb, S, rnd(r), rnd(Y @ V + Z @ S.T)))
        state = gam[-1] * state + rnd(r * (B * suf)[:, None]).T @ K
    D, grads = ds, []
    for t0, (Q, K, B, G, gam, suf, Y, Wb, S, r, _) in zip(range((len(chunks) - 1) * C, -1, -C), reversed(chunks)):
        dO, D16 = do[t0:t0 + C], rnd(D)
        w = Y.T @ dO + Wb @ D16.T
        D = gam[-1] * D + dO.T @ rnd(scale * gam[:, None] * Q) - rnd(w * gam[:, None]).T @ K
        w = rnd(w)
        strict = torch.ones_like(G).tril(-1)
        y1, y2 = G * scale * (dO @ r.T), -strict * G * (w @ r.T)
        a1, a2 = y1 * B, y2 * B
        M = strict * (a1 * (Q @ K.T) + a2 * (K @ K.T))
        inq, ink, out = scale * gam[:, None] * (dO @ S), -gam[:, None] * (w @ S), suf[:, None] * (r @ D16)
        y1, y2, a1, a2 = (rnd(t) for t in (y1, y2, a1, a2))
        y = out + y1.T @ Q + y2.T @ K
        into, outof = (inq * Q + ink * K).sum(-1), B * (out * K).sum(-1)
        n = len(Q)
        dg = torch.stack([M[t:, :t].sum() + into[t:].sum() + outof[:t].sum() for t in range(n)]) + gam[-1] * (S * D16).sum()
        grads.append((inq + a1 @ K, B[:, None] * y + ink + a2 @ K, w, dg, (y * K).sum(-1)))
    grads = [torch.cat(t) for t in zip(*reversed(grads))]
    return [torch.cat([c[-1] for c in chunks]), state, *(rnd(t) for t in grads), D]


def inputs(kind, strength, nl, kd, vd, dtype, heads=2, state=0.2, final=0.1, back=1.0):
    gen = torch.Generator().manual_seed(nl + kd + vd)
    rn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    base, apart = rn(1, 1, heads, kd), {"independent": None, "correlated": 0.3, "equal": 0.0}[kind]
    k = rn(1, nl, heads, kd) if apart is None else base + apart * rn(1, nl, heads, kd)
    q = rn(1, nl, heads, kd) if apart is None else base + 0.5 * rn(1, nl, heads, kd)
    beta = torch.sigmoid(rn(1, nl, heads)) if strength is None else torch.full((1, nl, heads), strength, dtype=torch.float64)
    t = [unit(q), unit(k), rn(1, nl, heads, vd), -0.02 * rn(1, nl, heads).abs(), beta]
    init, do, ds = state * rn(1, heads, vd, kd), back * rn(1, nl, heads, vd), final * rn(1, heads, vd, kd)
    return [x.to(dtype).double() for x in t], init.float().double(), do.to(dtype).double(), ds.float().double()


NAMES = ("o", "state", "dq", "dk", "dv", "dg", "dbeta", "dinitial")


def call(ts, init, do, ds, dtype):
    from ssm_b200 import ops

    leaves = [t.to(dtype).cuda().requires_grad_(True) for t in ts] + [init.float().cuda().requires_grad_(True)]
    o, s = ops.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_final_state=True, keep_state_fp32=True)
    got = [o, s, *torch.autograd.grad([o, s], leaves, [do.to(dtype).cuda(), ds.float().cuda()])]
    return [t.detach().double().cpu() for t in got]


def exact(ts, init, do, ds):
    ref = [t.clone().requires_grad_(True) for t in (*ts, init)]
    o, s = lm_oracle.gated_delta(*ref[:5], None, ref[5])
    return [o.detach(), s.detach(), *torch.autograd.grad([o, s], ref, [do, ds])]


def decay_terms(ts, init, do, ds):
    """The root of the sum of squares of dg's terms <S'_t, dS'_t>: (1, L, H)."""
    q, k, v, g, beta = (t[0] for t in ts)
    scale, state, held = q.shape[-1] ** -0.5, init[0], []
    for t in range(len(q)):
        state = state * g[t].exp()[:, None, None]
        held.append(state)
        r = v[t] - torch.einsum("hvk,hk->hv", state, k[t])
        state = state + torch.einsum("hv,hk->hvk", beta[t][:, None] * r, k[t])
    d, size = ds[0], torch.empty_like(g)
    for t in range(len(q) - 1, -1, -1):
        d = d + scale * torch.einsum("hv,hk->hvk", do[0, t], q[t])
        w = beta[t][:, None] * torch.einsum("hvk,hk->hv", d, k[t])
        d = d - torch.einsum("hv,hk->hvk", w, k[t])
        size[t] = (held[t] * d).flatten(1).norm(dim=1)
        d = d * g[t].exp()[:, None, None]
    return size[None]


def by_chunk(t):
    """(1, L, H, ...) as rows of one chunk and head each."""
    t = t[0].transpose(0, 1).flatten(2) if t.dim() > 3 else t[0].transpose(0, 1)[..., None]
    return [t[h, i:i + C].flatten() for h in range(t.shape[0]) for i in range(0, t.shape[1], C)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kd,vd,nl", [(128, 128, 320), (64, 96, 200)])
@pytest.mark.parametrize("sizes", [dict(), dict(state=8.0), dict(final=8.0, back=0.01), dict(state=4.0, final=4.0, back=0.01)])
def test_independent_keys(dtype, kd, vd, nl, sizes):
    """Whatever dominates: the tokens, the initial state, the final state's gradient."""
    a = inputs("independent", None, nl, kd, vd, dtype, **sizes)
    got, want = call(*a, dtype), exact(*a)
    for name, x, y in zip(NAMES, got, want):
        bar = 1.5 * ((7 if name in ("o", "state") else 17) / 3) ** 0.5 * HALF_STEP[dtype]
        parts = zip([x.flatten()], [y.flatten()]) if name in ("state", "dinitial") else zip(by_chunk(x), by_chunk(y))
        size = by_chunk(decay_terms(*a)) if name == "dg" else None
        for i, (p, r) in enumerate(parts):
            off = float((p - r).norm() / (r.norm() if size is None else max(r.norm(), size[i].norm())))
            assert off <= bar, f"{name}, chunk and head {i}: {off:.2e} of its norm, {bar:.2e} allowed"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["independent", "correlated", "equal"])
@pytest.mark.parametrize("strength", [None, 1.0, 1.9])
def test_keys_that_hardly_differ_cost_what_the_roundings_cost(dtype, kind, strength):
    a = inputs(kind, strength, 512, 128, 128, dtype)
    got, want = call(*a, dtype), exact(*a)
    (q, k, v, g, beta), init, do, ds = a
    same = [emulated(q[0, :, h], k[0, :, h], v[0, :, h], g[0, :, h], beta[0, :, h], init[0, h], do[0, :, h], ds[0, h], dtype) for h in range(2)]
    for i, (name, x, y) in enumerate(zip(NAMES, got, want)):
        axis = 0 if name in ("state", "dinitial") else 1
        e = torch.stack([s[i] for s in same], axis)[None]
        off, theirs = float((x - y).norm() / y.norm()), float((e - y).norm() / y.norm())
        print(f"{dtype} {kind} {strength} {name}: {off:.2e}, by the roundings alone {theirs:.2e}")
        assert off <= 1.5 * theirs, f"{name}: {off:.2e} of its norm, {theirs:.2e} by the roundings alone"
