"""The gated delta rule on the GPU against its definition in 64 bits.

Tolerances, relative to the largest value of a tensor.  fp32: a token's update of the state rounds each element a handful of times (decay,
correction, and the K / 8 + 3 additions of the two products it needs); keys have norm one and strengths lie in (0, 1), so nothing
amplifies an earlier rounding, and after n tokens at most n (K / 8 + 8) half steps of 2^-24 of the largest value have come together
(the backward pass walks the same way again: twice that, and its sums over V or a chunk's pairs add V + 32 + 32).  16-bit
operands add half a step of the result's own rounding (2^-8 for bf16, 2^-11 for fp16), and where the tensor cores form the products,
half a step for each of the operands rounded on the way: the state, the rest, its weighted copies, the inverse and the pair matrix
forward (six), twice as many and their pair sums backward (sixteen).
"""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def tolerance(dtype, nl, kd, vd, back=False):
    t = max(nl, 1) * (kd / 8 + 8) * 2.0 ** -24
    if back:
        t = 2 * t + (vd + 64) * 2.0 ** -24
    return t if dtype == F32 else t + (17 if back else 7) * HALF_STEP[dtype]


def near(got, want, tol, what=""):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    if want.numel() == 0:
        return
    off, top = (got - want).abs().max().item(), want.abs().max().item()
    assert off <= tol * max(top, 1e-30) + 1e-30, f"{what}: off by {off:.3e} of {top:.3e}, {tol:.3e} allowed"


def inputs(nb, nl, nk, nh, kd, vd, dtype, seed=0, g_scale=0.3):
    """Rounded to `dtype`, as CPU doubles."""
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    unit = lambda t: t / t.norm(dim=-1, keepdim=True).clamp_min(1e-9)  # noqa: E731
    t = [unit(rn(nb, nl, nk, kd)), unit(rn(nb, nl, nk, kd)), rn(nb, nl, nh, vd), -g_scale * rn(nb, nl, nh).abs(), torch.sigmoid(rn(nb, nl, nh))]
    return [x.to(dtype).double() for x in t]


def on_gpu(ts, dtype, grad=False, g_dtype=None):
    got = [t.to(dtype).cuda() for t in ts]
    if g_dtype is not None:
        got[3] = ts[3].to(g_dtype).cuda()
    return [t.requires_grad_(grad) for t in got]


SHAPES = [  # batch, len, key heads, heads, K, V
    (1, 1, 1, 1, 128, 128), (2, 2, 1, 2, 64, 64), (1, 15, 2, 2, 128, 64), (1, 16, 1, 1, 64, 128), (3, 31, 1, 1, 32, 48), (1, 32, 2, 4, 128, 128),
    (2, 33, 1, 3, 80, 96), (1, 63, 1, 1, 128, 128), (1, 64, 1, 2, 128, 64), (2, 65, 2, 2, 64, 64), (1, 100, 1, 1, 1, 1), (1, 127, 3, 3, 128, 128),
    (2, 130, 1, 4, 128, 128), (1, 200, 2, 2, 7, 33), (1, 97, 1, 1, 200, 130), (1, 48, 1, 2, 256, 256), (1, 193, 2, 2, 64, 192),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nb,nl,nk,nh,kd,vd", SHAPES)
def test_forward_and_every_gradient(nb, nl, nk, nh, kd, vd, dtype):
    from ssm_b200 import ops

    ts = inputs(nb, nl, nk, nh, kd, vd, dtype, seed=nl + kd)
    gen = torch.Generator().manual_seed(5)
    init = torch.randn(nb, nh, vd, kd, generator=gen).double() * 0.2
    do = torch.randn(nb, nl, nh, vd, generator=gen).to(dtype).double()
    ds = torch.randn(nb, nh, vd, kd, generator=gen).double() * 0.1
    ref = [t.clone().requires_grad_(True) for t in (*ts, init)]
    o, s = lm_oracle.gated_delta(*ref[:5], None, ref[5])
    want = torch.autograd.grad([o, s], ref, [do, ds])
    leaves = on_gpu(ts, dtype, True) + [init.float().cuda().requires_grad_(True)]
    got_o, got_s = ops.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_final_state=True, keep_state_fp32=True)
    assert got_o.dtype == dtype and got_s.dtype == F32
    near(got_o, o, tolerance(dtype, nl, kd, vd), "o")
    near(got_s, s, tolerance(dtype, nl, kd, vd), "state")
    with torch.no_grad():  # nothing is kept for a backward pass
        again = ops.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_final_state=True, keep_state_fp32=True)
    near(again[0], o, tolerance(dtype, nl, kd, vd), "o without gradients")
    near(again[1], s, tolerance(dtype, nl, kd, vd), "state without gradients")
    got = torch.autograd.grad([got_o, got_s], leaves, [do.to(dtype).cuda(), ds.float().cuda()])
    for name, x, y, leaf in zip(("q", "k", "v", "g", "beta", "initial"), got, want, leaves):
        assert x.dtype == leaf.dtype
        near(x, y, tolerance(dtype, nl, kd, vd, True), "gradient of " + name)


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 48, 40), (BF16, 128, 128), (F16, 128, 64), (BF16, 64, 64)])
@pytest.mark.parametrize("cuts,where", [([0, 70, 70, 71, 200], "cuda64"), ([0, 0, 33], "cuda32"), ([0, 64, 128, 150], "host"), ([0, 1, 2, 3, 4], "cuda64"), ([0, 0], "cuda64")])
def test_packed_sequences(dtype, kd, vd, cuts, where):
    """Sequences of any length, none among them, and rows behind the last."""
    from ssm_b200 import ops

    nl, nh, nk, seqs = 200, 2, 1, len(cuts) - 1
    ts = inputs(1, nl, nk, nh, kd, vd, dtype, seed=len(cuts))
    gen = torch.Generator().manual_seed(6)
    init = torch.randn(seqs, nh, vd, kd, generator=gen).double() * 0.2
    do = torch.randn(1, nl, nh, vd, generator=gen).to(dtype).double()
    ds = torch.randn(seqs, nh, vd, kd, generator=gen).double() * 0.1
    ref = [t.clone().requires_grad_(True) for t in (*ts, init)]
    o, s = lm_oracle.gated_delta(*ref[:5], None, ref[5], cuts)
    want = torch.autograd.grad([o + 0 * sum(t.sum() for t in ref), s], ref, [do, ds])  # a gradient of zero where there is no token at all
    leaves = on_gpu(ts, dtype, True) + [init.float().cuda().requires_grad_(True)]
    cu = torch.tensor(cuts, dtype=torch.int32 if where == "cuda32" else torch.int64)
    cu = cu if where == "host" else cu.cuda()
    got_o, got_s = ops.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_final_state=True, keep_state_fp32=True, cu_seqlens=cu)
    longest = max(b - a for a, b in zip(cuts, cuts[1:]))
    near(got_o, o, tolerance(dtype, longest, kd, vd), "o")
    near(got_s, s, tolerance(dtype, longest, kd, vd), "state")
    assert not got_o[:, cuts[-1]:].any()
    with torch.no_grad():
        again = ops.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_final_state=True, keep_state_fp32=True, cu_seqlens=cu)
    near(again[0], o, tolerance(dtype, longest, kd, vd), "o without gradients")
    near(again[1], s, tolerance(dtype, longest, kd, vd), "state without gradients")
    assert not again[0][:, cuts[-1]:].any()
    got = torch.autograd.grad([got_o, got_s], leaves, [do.to(dtype).cuda(), ds.float().cuda()])
    for name, x, y in zip(("q", "k", "v", "g", "beta", "initial"), got, want):
        near(x, y, tolerance(dtype, longest, kd, vd, True), "gradient of " + name)
        if name != "initial":
            assert not x[:, cuts[-1]:].any(), name


@pytest.mark.parametrize("nb,nl,nk,nh,kd,vd,cuts", [
    (3, 500, 4, 8, 128, 64, None), (4, 330, 4, 8, 64, 128, None), (5, 260, 4, 8, 128, 192, None), (2, 410, 16, 16, 72, 88, None),
    (1, 1500, 6, 12, 128, 72, [0, 3, 70, 71, 200, 200, 520, 1111, 1400]), (1, 1500, 12, 12, 64, 128, [0, 640, 641, 1300]),
])
def test_more_chunks_than_blocks_side_by_side(nb, nl, nk, nh, kd, vd, cuts):
    """The gradients' blocks take several chunks each: slices of 64 columns, one to three of them, whole and ragged, and chunks of no sequence."""
    from ssm_b200 import ops

    ts = inputs(nb, nl, nk, nh, kd, vd, BF16, seed=nl)
    gen = torch.Generator().manual_seed(11)
    do = torch.randn(nb, nl, nh, vd, generator=gen).to(BF16).double()
    ref = [t.clone().requires_grad_(True) for t in ts]
    o, _ = lm_oracle.gated_delta(*ref, cu_seqlens=cuts)
    want = torch.autograd.grad(o, ref, do)
    leaves = on_gpu(ts, BF16, True)
    got_o = ops.gated_delta_scan(*leaves, cu_seqlens=None if cuts is None else torch.tensor(cuts).cuda())
    longest = nl if cuts is None else max(b - a for a, b in zip(cuts, cuts[1:]))
    near(got_o, o, tolerance(BF16, longest, kd, vd), "o")
    got = torch.autograd.grad(got_o, leaves, do.to(BF16).cuda())
    for name, x, y in zip(("q", "k", "v", "g", "beta"), got, want):
        near(x, y, tolerance(BF16, longest, kd, vd, True), "gradient of " + name)
        if cuts is not None:
            assert not x[:, cuts[-1]:].any(), name


@pytest.mark.parametrize("nb,nl,nk,nh", [(1, 8, 8, 16), (1, 9, 8, 16), (40, 4, 2, 4), (40, 5, 4, 4), (2, 1, 1, 1)])
def test_a_few_tokens_without_gradients(nb, nl, nk, nh):
    """On both sides of the choice between chunks and single tokens, a state carried on in place of a longer call."""
    from ssm_b200 import ops

    kd = vd = 128
    ts = inputs(nb, 2 * nl, nk, nh, kd, vd, BF16, seed=nb + nl)
    o, s = lm_oracle.gated_delta(*ts)
    x = on_gpu(ts, BF16)
    first = ops.gated_delta_scan(*[t[:, :nl] for t in x], return_final_state=True, keep_state_fp32=True)
    second = ops.gated_delta_scan(*[t[:, nl:] for t in x], initial_state=first[1], return_final_state=True, keep_state_fp32=True)
    near(torch.cat([first[0], second[0]], 1), o, tolerance(BF16, 2 * nl, kd, vd), "o")
    near(second[1], s, tolerance(BF16, 2 * nl, kd, vd), "state")


@pytest.mark.parametrize("cuts", [[0, 90, 40, 120], [5, -3, 500, 60], [0, 1 << 40, 0, 0], [100, 100, 100, 100]])
def test_boundaries_on_the_device_that_break_the_rule_stay_inside(cuts):
    """Entries are clamped to rise from 0 to at most L: the call answers as for the clamped ones."""
    from ssm_b200 import ops

    nl = 120
    fixed, at = [0], 0
    for c in cuts[1:]:
        at = max(at, min(nl, max(0, c)))
        fixed.append(at)
    for dtype in (F32, BF16):
        x = on_gpu(inputs(1, nl, 2, 2, 128, 64, dtype), dtype)
        a = ops.gated_delta_scan(*x, return_final_state=True, cu_seqlens=torch.tensor(cuts).cuda())
        b = ops.gated_delta_scan(*x, return_final_state=True, cu_seqlens=torch.tensor(fixed).cuda())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(ValueError, match="cu_seqlens"):
        ops.gated_delta_scan(*x, cu_seqlens=torch.tensor([0, 90, 40, 120]))


def test_many_sequences_and_boundaries():
    from ssm_b200 import ops

    gen = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 4, (2600,), generator=gen)  # more than one round of the table's threads, a third of them nearly empty
    cu = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(lens, 0)])
    nl = int(cu[-1]) + 40
    for dtype, kd, vd in ((F32, 8, 8), (BF16, 128, 64)):
        ts = inputs(1, nl, 1, 1, kd, vd, dtype)
        o, s = lm_oracle.gated_delta(*ts, cu_seqlens=cu)
        got = ops.gated_delta_scan(*on_gpu(ts, dtype), return_final_state=True, keep_state_fp32=True, cu_seqlens=cu.cuda())
        near(got[0], o, tolerance(dtype, 4, kd, vd))
        near(got[1], s, tolerance(dtype, 4, kd, vd))


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 64, 64), (BF16, 128, 128), (F16, 64, 64)])
def test_resets_strong_decays_and_idle_tokens(dtype, kd, vd):
    """g of -inf and of -200 start anew, beta of zero writes nothing, keys of zero: all finite, the gradients too."""
    from ssm_b200 import ops

    nl = 150
    ts = inputs(1, nl, 1, 2, kd, vd, dtype)
    q, k, v, g, beta = ts
    g[0, 20, 0] = g[0, 64, 1] = g[0, 100, 0] = -float("inf")
    g[0, 70:90, 1] = -200.0
    beta[0, 30:40] = 0.0
    k[0, 50:55] = 0.0
    do = torch.randn(1, nl, 2, vd, generator=torch.Generator().manual_seed(1)).to(dtype).double()
    ref = [t.clone().requires_grad_(True) for t in ts]
    o, s = lm_oracle.gated_delta(*ref)
    want = torch.autograd.grad(o, ref, do)
    leaves = on_gpu(ts, dtype, True)
    got_o, got_s = ops.gated_delta_scan(*leaves, return_final_state=True)
    near(got_o, o, tolerance(dtype, nl, kd, vd), "o")
    near(got_s, s, tolerance(dtype, nl, kd, vd), "state")
    for name, x, y in zip(("q", "k", "v", "g", "beta"), torch.autograd.grad(got_o, leaves, do.to(dtype).cuda()), want):
        near(x, y, tolerance(dtype, nl, kd, vd, True), "gradient of " + name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_decay_with_a_scale_and_mixed_types(dtype):
    from ssm_b200 import ops

    kd, vd, nl = 128, 128, 80
    q, k, v, _, beta = inputs(2, nl, 2, 2, kd, vd, dtype)
    ref = [t.clone().requires_grad_(True) for t in (q, k, v, beta)]
    o, _ = lm_oracle.gated_delta(*ref[:3], None, ref[3], 0.7)
    want = torch.autograd.grad(o.square().sum(), ref)
    leaves = [q.float().cuda(), k.to(dtype).cuda(), v.to(dtype).cuda(), beta.float().cuda()]  # q in another type than v: read in v's
    leaves = [t.requires_grad_(True) for t in leaves]
    got = ops.gated_delta_scan(*leaves[:3], None, leaves[3], scale=0.7)
    near(got, o, tolerance(dtype, nl, kd, vd))
    grads = torch.autograd.grad(got, leaves, (2 * o).to(dtype).cuda())
    for x, y, leaf in zip(grads, want, leaves):
        assert x.dtype == leaf.dtype
        near(x, y, tolerance(dtype, nl, kd, vd, True) + HALF_STEP[dtype])  # the incoming gradient is rounded too


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_operands_of_any_layout_are_read_where_they_lie_or_copied(dtype):
    """Slices of one projection, heads before tokens, an odd offset, a broadcast head: the same answers as dense operands."""
    from ssm_b200 import ops

    nb, nl, nh, d = 2, 75, 4, 64
    ts = inputs(nb, nl, nh, nh, d, d, dtype)
    dense = on_gpu(ts, dtype)
    want = ops.gated_delta_scan(*dense)
    fused = torch.cat([t.reshape(nb, nl, -1) for t in dense[:3]], -1)
    q, k, v = (t.view(nb, nl, nh, d) for t in fused.split(nh * d, -1))
    assert torch.equal(ops.gated_delta_scan(q, k, v, dense[3], dense[4]), want)
    by_head = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense]
    assert torch.equal(ops.gated_delta_scan(*by_head), want)
    odd = [torch.empty(t.numel() + 3, dtype=dtype, device="cuda")[3:].view(t.shape).copy_(t) for t in dense]
    assert torch.equal(ops.gated_delta_scan(*odd), want)
    inner = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in dense[:3]]
    assert torch.equal(ops.gated_delta_scan(*inner, dense[3], dense[4]), want)
    one = dense[1][:, :, :1]
    a = ops.gated_delta_scan(one.expand(-1, -1, nh, -1), one.expand(-1, -1, nh, -1), *dense[2:])
    b = ops.gated_delta_scan(one, one, *dense[2:])
    assert torch.equal(a, b)


def test_gradients_against_differences():
    """A step along a direction changes the loss by the gradient's product with it.  fp32, central differences with h = 2^-6: the loss sums
    3000 terms of size one with errors of 1e-6 each and of either sign, so its difference is off by 1e-4 / 2h = 3e-3, plus h^2 of the third derivative."""
    from ssm_b200 import ops

    ts = inputs(1, 96, 1, 2, 32, 16, F32)
    gen = torch.Generator().manual_seed(3)
    do = torch.randn(1, 96, 2, 16, generator=gen).cuda()
    leaves = on_gpu(ts, F32, True)
    grads = torch.autograd.grad(ops.gated_delta_scan(*leaves), leaves, do)
    h = 2.0 ** -6
    for i, x in enumerate(leaves):
        d = torch.randn(x.shape, generator=gen).cuda()
        d /= d.norm()
        f = lambda s: float((ops.gated_delta_scan(*[t.detach() + (s * d if j == i else 0) for j, t in enumerate(leaves)]).double() * do).sum())  # noqa: E731
        diff, want = (f(h) - f(-h)) / (2 * h), float((grads[i] * d).sum())
        assert abs(diff - want) <= 5e-3 + 1e-2 * float(grads[i].norm()) * h, (i, diff, want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nb,nk,nh,kd,vd", [(1, 1, 1, 128, 128), (3, 2, 4, 64, 96), (2, 1, 3, 7, 5), (5, 2, 2, 256, 33), (2, 1, 1, 1, 1), (4, 1, 2, 36, 64)])
def test_step(nb, nk, nh, kd, vd, dtype):
    from ssm_b200 import ops

    q, k, v, g, beta = (t[:, 0] for t in inputs(nb, 1, nk, nh, kd, vd, dtype, seed=kd))
    state = torch.randn(nb, nh, vd, kd, generator=torch.Generator().manual_seed(2)).double()
    o, s = lm_oracle.gated_delta(q[:, None], k[:, None], v[:, None], g[:, None], beta[:, None], None, state)
    st = state.float().cuda()
    x = on_gpu((q, k, v, g, beta), dtype, g_dtype=F32)
    got = ops.gated_delta_step(st, *x)
    one = (kd / 8 + 8) * 2.0 ** -24
    near(st, s, 4 * one, "state")
    near(got, o[:, 0], 4 * one + HALF_STEP[dtype], "o")
    # slices of a wider projection, a state in another order
    wide = torch.cat([t.reshape(nb, -1) for t in x[:3]], 1)
    parts = [t.view(nb, -1, n) for t, n in zip(wide.split([nk * kd, nk * kd, nh * vd], 1), (kd, kd, vd))]
    st2 = state.float().cuda().transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(ops.gated_delta_step(st2, *parts, *x[3:]), got) and torch.equal(st2, st)


def test_step_with_gradients_and_refusals():
    from ssm_b200 import ops

    ts = inputs(2, 1, 1, 2, 16, 8, F32)
    ref = [t.clone().requires_grad_(True) for t in ts]
    s0 = torch.randn(2, 2, 8, 16, generator=torch.Generator().manual_seed(2)).double()
    o, s = lm_oracle.gated_delta(*ref, None, s0)
    want = torch.autograd.grad(o.sum(), ref)
    state = s0.float().cuda()
    leaves = [t[:, 0].detach().requires_grad_(True) for t in on_gpu(ts, F32)]
    got = ops.gated_delta_step(state, *leaves)
    near(state, s, 1e-5)
    for x, y in zip(torch.autograd.grad(got.sum(), leaves), want):
        near(x, y[:, 0], tolerance(F32, 1, 16, 8, True))
    x = [t.detach() for t in leaves]
    with pytest.raises(ValueError, match="float32"):
        ops.gated_delta_step(state.half(), *x)
    with pytest.raises(ValueError):
        ops.gated_delta_step(state[:1], *x)
    with pytest.raises(ValueError, match="not built"):
        ops.gated_delta_scan(*[t.double().cuda() for t in ts])
    with pytest.raises(ValueError, match="256"):
        ops.gated_delta_scan(*on_gpu(inputs(1, 2, 1, 1, 257, 4, F32), F32))
    with pytest.raises(ValueError, match="batch of one"):
        ops.gated_delta_scan(*on_gpu(ts, F32), cu_seqlens=torch.tensor([0, 1]))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_delta_scan(*on_gpu(ts, F32)[:4], ts[4].float())


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 32, 32), (BF16, 128, 128)])
def test_prefill_then_steps_continue_one_another(dtype, kd, vd):
    """Prefill of a prompt, then token by token, as a program decodes: the answers of the whole sequence at once."""
    from ssm_b200 import ops

    nb, nl, cut = 2, 90, 77
    ts = inputs(nb, nl, 1, 2, kd, vd, dtype)
    want, s = lm_oracle.gated_delta(*ts)
    x = on_gpu(ts, dtype, g_dtype=F32)
    o, state = ops.gated_delta_scan(*[t[:, :cut] for t in x], return_final_state=True, keep_state_fp32=True)
    outs = [o] + [ops.gated_delta_step(state, *[t[:, i] for t in x])[:, None] for i in range(cut, nl)]
    near(torch.cat(outs, 1), want, tolerance(dtype, nl, kd, vd))
    near(state, s, tolerance(dtype, nl, kd, vd))


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 32, 32), (BF16, 128, 128), (BF16, 64, 64)])
def test_nothing_to_do(dtype, kd, vd):
    from ssm_b200 import ops

    for nb, nl in ((0, 5), (2, 0)):
        leaves = on_gpu(inputs(nb, nl, 1, 1, kd, vd, dtype), dtype, True)
        init = torch.randn(nb, 1, vd, kd, device="cuda").requires_grad_(True)
        o, s = ops.gated_delta_scan(*leaves, initial_state=init, return_final_state=True, keep_state_fp32=True)
        assert o.shape == (nb, nl, 1, vd) and torch.equal(s, init)
        got = torch.autograd.grad([o.float().sum() + s.sum()], [*leaves, init])
        assert torch.equal(got[5], torch.ones_like(init))
    x = on_gpu(inputs(1, 4, 1, 1, kd, vd, dtype), dtype)
    o, s = ops.gated_delta_scan(*x, return_final_state=True, cu_seqlens=torch.tensor([0, 0, 0]).cuda())
    assert not o.any() and not s.any()


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 32, 48), (BF16, 128, 128), (F16, 64, 64)])
def test_repeats_other_streams_and_graphs_give_the_same_bits(dtype, kd, vd):
    from ssm_b200 import ops

    ts = inputs(2, 150, 1, 2, kd, vd, dtype)
    do = torch.randn(2, 150, 2, vd, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    leaves = on_gpu(ts, dtype, True)

    def go(ls):
        o, s = ops.gated_delta_scan(*ls, return_final_state=True)
        return [o, s, *torch.autograd.grad(o, ls, do)]

    want = [t.detach().clone() for t in go(leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [t.detach().clone() for t in go(leaves)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    # two calls under way at once, on two streams
    streams = [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(go(leaves))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    # captured on the capture stream, with leaves of its own; replayed on changed inputs
    fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
    with torch.cuda.stream(side):
        go(fresh)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept = go(fresh)
    with torch.no_grad():
        for t in fresh:
            t.zero_()
    graph.replay()
    with torch.no_grad():
        for t, x in zip(fresh, leaves):
            t.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_edits_and_second_derivatives_raise():
    from ssm_b200 import ops

    leaves = on_gpu(inputs(1, 20, 1, 1, 16, 16, F32), F32, True)
    k = leaves[1] * 1.0
    o = ops.gated_delta_scan(leaves[0], k, *leaves[2:])
    k.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified in place"):
        o.sum().backward()
    o = ops.gated_delta_scan(*leaves)
    (dv,) = torch.autograd.grad(o.sum(), leaves[2], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(dv.sum(), leaves[0])


def test_a_long_chain_in_16_bits():
    """4000 tokens of one head: what was rounded early does not grow."""
    from ssm_b200 import ops

    ts = inputs(1, 4000, 1, 1, 128, 128, BF16, g_scale=0.02)
    o, s = lm_oracle.gated_delta(*ts)
    got = ops.gated_delta_scan(*on_gpu(ts, BF16, g_dtype=F32), return_final_state=True, keep_state_fp32=True)
    near(got[0], o, tolerance(BF16, 1, 128, 128))
    near(got[1], s, tolerance(BF16, 1, 128, 128))


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 24, 40), (BF16, 128, 128), (F16, 64, 72)])
def test_nan_and_inf_stay_in_their_sequence(dtype, kd, vd):
    """A sequence of NaN and infinities between others, in the same chunks of rows, and rows of NaN behind the last one."""
    from ssm_b200 import ops

    cuts, nl, nh = [0, 40, 75, 170, 171], 200, 2
    ts = inputs(1, nl, 1, nh, kd, vd, dtype)
    do = torch.randn(1, nl, nh, vd, generator=torch.Generator().manual_seed(3)).to(dtype).double()
    cu = torch.tensor(cuts).cuda()

    def call(spoil):
        leaves = on_gpu(ts, dtype)
        go = do.to(dtype).cuda()
        if spoil:
            for t in (*leaves, go):
                t[:, 40:75] = float("nan")
                t[:, 60] = float("inf")
                t[:, 171:] = float("nan")
        leaves = [t.requires_grad_(True) for t in leaves]
        o, s = ops.gated_delta_scan(*leaves, return_final_state=True, keep_state_fp32=True, cu_seqlens=cu)
        with torch.no_grad():
            again = ops.gated_delta_scan(*leaves, return_final_state=True, keep_state_fp32=True, cu_seqlens=cu)
        return [o, s, *again, *torch.autograd.grad(o, leaves, go)]

    clean, spoilt = call(False), call(True)
    keep = torch.tensor([i for i in range(nl) if not 40 <= i < 75], device="cuda")
    for i, (x, y) in enumerate(zip(clean, spoilt)):
        if i in (1, 3):  # states
            assert torch.equal(x[[0, 2, 3]], y[[0, 2, 3]]) and not torch.isfinite(y[1]).all()
        else:
            assert torch.equal(x[:, keep], y[:, keep]), i


def test_a_step_on_a_state_that_a_graph_keeps_is_noticed():
    from ssm_b200 import ops

    x = on_gpu(inputs(1, 70, 1, 2, 64, 64, BF16), BF16, True)
    state = torch.randn(1, 2, 64, 64, device="cuda")
    o = ops.gated_delta_scan(*x, initial_state=state)
    with torch.no_grad():
        ops.gated_delta_step(state, *[t[:, 0] for t in x])
    with pytest.raises(RuntimeError, match="modified in place"):
        o.sum().backward()
    with torch.inference_mode():  # no version counter there
        held = torch.zeros(1, 2, 64, 64, device="cuda")
        ops.gated_delta_step(held, *[t[:, 0] for t in x])
        assert held.any()
