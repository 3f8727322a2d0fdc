"""``ops.fused_block_norm`` against its definition in 64 bits.

Tolerances.  All sums and products are held in 32 bits: a result of at most a few dozen roundings of 2^-24, of terms whose sizes add up to at most twenty times
the result's rms for these inputs, is off by 2^-24 * 1000 = 6e-5 of the rms at the worst element; sums over a thousand rows keep that relative to the sum
of the terms' sizes, some thirty times the rms of a sum of random terms: 2e-3.  To that comes half a step of the type that the result is rounded to.
A row of one column is an exception for the gradient of x: RMSNorm's x / sqrt(x^2 + eps) hardly depends on x there, and g - h (g h) = g (1 - h^2) is eps / x^2, 1e-4, of the terms it is
the difference of.  Its error is one of 2^-24 of those terms, so they stand in the place of the result."""

from __future__ import annotations

import pytest
import torch

from oracle import training_oracle as oracle
from ssm_b200 import ops

pytestmark = pytest.mark.gpu

NAMES = ("x", "residual", "post_weight", "weight", "post_bias", "bias", "gate")


def make(nb, nl, d, dtype, gate="none", biases=False, residual=torch.float32, params=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    params = dtype if params is None else params
    t = {"x": (0.3 * rn(nb, nl, d)).to(dtype), "residual": None if residual is None else (2 * rn(nb, nl, d)).to(residual),
         "post_weight": (1 + 0.1 * rn(d)).to(params), "weight": (1 + 0.1 * rn(d)).to(params),
         "post_bias": (0.1 * rn(d)).to(params) if biases else None, "bias": (0.1 * rn(d)).to(params) if biases else None}
    shape = {"none": None, "channel": (d,), "sequence": (nb, d), "sequence3": (nb, 1, d), "token": (nb, nl, d)}[gate]
    t["gate"] = None if shape is None else (0.5 + 0.3 * rn(*shape)).to(dtype)
    t["dy"], t["dr"] = rn(nb, nl, d).to(dtype), rn(nb, nl, d)
    return t


def call(space, t, **kw):
    return space.fused_block_norm(t["x"], t["residual"], t["post_weight"], t["weight"], t["post_bias"], t["bias"], t["gate"], residual_scale=0.7, **kw)


def near(got, want, what, sums=False, terms=None):
    want = want.double()
    if want.numel() == 0:
        assert got.shape == want.shape
        return
    eps = torch.finfo(got.dtype).eps / 2
    rms = (want if terms is None else terms).pow(2).mean().sqrt()
    err = (got.double() - want).abs()
    assert (err <= eps * want.abs() + (2e-3 if sums else 6e-5) * rms).all(), f"{what}: {float((err / (rms + 1e-30)).max())}"


def check(t, **kw):
    leaves = {n: t[n].detach().requires_grad_(True) for n in NAMES if t[n] is not None}
    y, r = call(ops, {**t, **leaves}, **kw)
    got = torch.autograd.grad([y, r], list(leaves.values()), [t["dy"].to(y.dtype), t["dr"].to(r.dtype)])
    wide = {n: v.detach().double().requires_grad_(True) for n, v in leaves.items()}
    wy, wr = call(oracle, {**t, **wide}, **kw)
    want = torch.autograd.grad([wy, wr], list(wide.values()), [t["dy"].to(y.dtype).double(), t["dr"].to(r.dtype).double()])
    assert y.dtype == t["x"].dtype and r.dtype == (torch.float32 if kw.get("residual_in_fp32", True) else t["x"].dtype)
    near(y.detach(), wy.detach(), "y")
    near(r.detach(), wr.detach(), "r")
    for n, g, w in zip(leaves, got, want):
        assert g.dtype == leaves[n].dtype and g.shape == leaves[n].shape
        terms = None
        if n == "x" and t["x"].shape[-1] == 1:
            x = t["x"].double()
            terms = want[list(leaves).index("residual")] * 0.7 * t["gate"].double() * t["post_weight"].double() * (x * x + 1e-5).rsqrt()
        near(g, w, "d" + n, sums=g.numel() < t["x"].numel(), terms=terms)
    with torch.no_grad():
        y2, r2 = call(ops, t, **kw)
    assert torch.equal(y2, y) and torch.equal(r2, r)


@pytest.mark.parametrize("d", [1, 7, 64, 100, 257, 768, 1001, 2560, 4100, 8192])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_widths(d, dtype):
    check(make(2, 5, d, dtype, "channel", d % 2 == 0), is_rms=d == 1)


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "sequence3", "token"])
@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("biases", [True, False])
def test_gates(gate, rms, biases):
    check(make(3, 67, 320, torch.bfloat16, gate, biases), is_rms=rms, eps=1e-3, post_eps=1e-6)


@pytest.mark.parametrize("nb,nl", [(1, 1), (1, 3000), (7, 1), (2500, 1), (5, 421), (700, 3), (1, 0), (0, 4)])
@pytest.mark.parametrize("gate", ["channel", "sequence"])
def test_rows_and_sequences(nb, nl, gate):
    check(make(nb, nl, 96, torch.float32, gate))


@pytest.mark.parametrize("residual", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp32", [True, False])
@pytest.mark.parametrize("d", [128, 130])
def test_types_of_the_stream(residual, fp32, d):
    check(make(2, 9, d, torch.bfloat16, "token", True, residual, torch.float32), residual_in_fp32=fp32)


def test_only_one_output_is_used():
    t = make(2, 33, 256, torch.bfloat16, "sequence")
    for which in (0, 1):
        x = t["x"].clone().requires_grad_(True)
        w = t["weight"].clone().requires_grad_(True)
        out = call(ops, {**t, "x": x, "weight": w})[which]
        grads = torch.autograd.grad(out, [x, w], t["dy" if which == 0 else "dr"])
        xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
        want = torch.autograd.grad(call(oracle, {**t, "x": xd, "weight": wd})[which], [xd, wd], t["dy" if which == 0 else "dr"].double(), allow_unused=True)
        near(grads[0], want[0], "dx")
        if which == 0:
            near(grads[1], want[1], "dw", sums=True)
        else:
            assert not grads[1].any()


def test_strides_offsets_and_odd_places():
    t = make(3, 10, 64, torch.bfloat16, "token")
    want = call(ops, t)
    odd = torch.empty(3 * 10 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(3, 10, 64).copy_(t["x"])
    moved = {**t, "x": odd, "residual": t["residual"].transpose(0, 1).contiguous().transpose(0, 1), "gate": torch.cat([t["gate"], t["gate"]], -1)[..., :64]}
    for a, b in zip(call(ops, moved), want):
        near(a, b, "moved")
    broad = {**t, "gate": t["gate"][:1, :1].expand(3, 10, 64)}
    for a, b in zip(call(ops, broad), call(ops, {**t, "gate": t["gate"][0, 0]})):
        assert torch.equal(a, b)


def test_gradients_against_differences():
    """Central differences of the 32-bit forward pass: a step of 1e-2 on values of size one leaves (1e-2)^2 of curvature and 2^-24 * |sum| / 1e-2 of rounding, the sum of
    some 400 terms of size one: 1e-2 in all."""
    t = make(2, 3, 64, torch.float32, "sequence", True)
    leaves = [t[n].requires_grad_(True) for n in NAMES]
    f = lambda: sum((o * g).double().sum() for o, g in zip(call(ops, t, is_rms=False), (t["dy"], t["dr"])))  # noqa: E731
    grads = torch.autograd.grad(f(), leaves)
    gen = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        for leaf, g in zip(leaves, grads):
            dir = torch.randn(leaf.shape, device="cuda", generator=gen)
            dir /= dir.norm()
            leaf += 1e-2 * dir
            up = f()
            leaf -= 2e-2 * dir
            down = f()
            leaf += 1e-2 * dir
            assert abs(float((up - down) / 2e-2 - (g.double() * dir.double()).sum())) < 1e-2


def test_a_row_that_is_not_finite_stays_alone():
    t = make(2, 8, 128, torch.bfloat16, "token")
    want = call(ops, t)
    bad = {**t, "x": t["x"].clone(), "residual": t["residual"].clone()}
    bad["x"][0, 3, 5] = float("nan")
    bad["residual"][1, 2] = float("inf")
    x = bad["x"].requires_grad_(True)
    y, r = call(ops, bad)
    keep = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[1, 2] = False
    assert torch.equal(y[keep], want[0][keep]) and torch.equal(r[keep], want[1][keep])
    assert y[0, 3].isnan().all() and y[1, 2].isnan().all()
    dx = torch.autograd.grad(y, x, t["dy"])[0]
    assert dx[keep].isfinite().all()


def test_repeats_streams_and_graphs_give_the_same_bits():
    t = make(4, 50, 640, torch.bfloat16, "sequence")
    leaves = [t[n].requires_grad_(True) for n in ("x", "residual", "post_weight", "weight", "gate")]

    def once():
        y, r = call(ops, t)
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], leaves, [t["dy"], t["dr"]])]

    want = once()
    for a, b in zip(once(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
        once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for _ in range(2):
        for o in out:
            o.zero_()
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_an_edit_between_forward_and_backward_is_an_error():
    t = make(1, 4, 64, torch.float32)
    x = t["x"].clone().requires_grad_(True)
    y, _ = call(ops, {**t, "x": x})
    t["residual"].add_(1)
    with pytest.raises(RuntimeError, match="modified in place"):
        y.sum().backward()


def test_second_derivatives_are_refused():
    t = make(1, 2, 64, torch.float32)
    x = t["x"].clone().requires_grad_(True)
    g = torch.autograd.grad(call(ops, {**t, "x": x})[0].sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


@pytest.mark.parametrize("d", [97, 1001, 4101])
@pytest.mark.parametrize("nb,nl", [(5, 421), (700, 3), (1, 1500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_widths_with_a_gate_per_sequence_whose_rows_several_blocks_share(dtype, nb, nl, d):
    check(make(nb, nl, d, dtype, "sequence", True), is_rms=False)
