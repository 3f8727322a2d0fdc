"""The gated delta rule and the token losses inside ``torch.jit.trace`` and under forward mode, like the operators beside them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cases():
    from ssm_b200 import ops

    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    half = lambda *s: r(*s).bfloat16()  # noqa: E731
    targets, ids = torch.arange(6, device="cuda"), torch.arange(18, device="cuda").view(6, 3)
    teacher = r(6, 3)

    def step(state, q, k, v, b):  # the state an argument: the copy of a constant is a constant to the traced graph, which does not see it written
        held = state.clone()
        return ops.gated_delta_step(held, q, k, v, None, torch.sigmoid(b)) + held.sum(-1).to(v.dtype)

    return {
        "scan": (lambda q, k, v, b: ops.gated_delta_scan(q, k, v, None, torch.sigmoid(b), scale=0.1), lambda: (0.1 * half(1, 90, 1, 64), 0.1 * half(1, 90, 1, 64), half(1, 90, 2, 64), half(1, 90, 2))),
        "scan_state": (lambda q, k, v, b: sum(t.sum() for t in ops.gated_delta_scan(q, k, v, -torch.sigmoid(b), torch.sigmoid(b), return_final_state=True)),
                       lambda: (0.1 * r(1, 20, 1, 24), 0.1 * r(1, 20, 1, 24), r(1, 20, 2, 8), r(1, 20, 2))),
        "step": (step, lambda: (r(2, 2, 64, 64), 0.1 * r(2, 1, 64), 0.1 * r(2, 1, 64), r(2, 2, 64), r(2, 2))),
        "logp": (lambda x: sum(t.float().sum(-1) if t.dim() > 1 else t for t in ops.token_log_probs(x, targets, 0.7, 3, True)[:3]), lambda: (r(6, 900),)),
        "distill": (lambda x: ops.topk_distill_loss(x, teacher, ids, 2.0), lambda: (r(6, 900),)),
    }


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("op", ["scan", "scan_state", "step", "logp", "distill"])
def test_traced_operators_run_on_their_arguments(op, grad):
    fn, make = _cases()[op]
    torch.manual_seed(1)
    traced = torch.jit.trace(fn, make(), check_trace=False)
    ins = [t.requires_grad_(grad) for t in make()]
    want = fn(*ins)
    junk = [torch.full_like(want, 7.0) for _ in range(4)]  # memory that an output left unwritten would show
    del junk
    got = traced(*ins)
    if not grad:
        assert torch.equal(got, want)
    else:  # the step's gradients come by way of the scan, whose sums run in another order than the step's
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
        weight = torch.randn_like(want)
        for a, b in zip(torch.autograd.grad((got * weight).sum(), ins), torch.autograd.grad((want * weight).sum(), ins)):
            torch.testing.assert_close(a, b, rtol=2e-2 if op == "scan" else 1e-4, atol=1e-2 if op == "scan" else 1e-4)


def test_a_traced_step_moves_its_state():
    """The state of the traced call, not a copy of it."""
    from ssm_b200 import ops

    def fn(state, q, k, v, b):
        return ops.gated_delta_step(state, q, k, v, None, b)

    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    make = lambda: (r(2, 2, 32, 16), 0.2 * r(2, 1, 16), 0.2 * r(2, 1, 16), r(2, 2, 32), torch.rand(2, 2, device="cuda"))  # noqa: E731
    traced = torch.jit.trace(fn, make(), check_trace=False)
    ins = make()
    mine, theirs = ins[0].clone(), ins[0].clone()
    want, got = fn(mine, *ins[1:]), traced(theirs, *ins[1:])
    assert torch.equal(got, want) and torch.equal(theirs, mine) and not torch.equal(mine, ins[0])


@pytest.mark.parametrize("which", range(5))
def test_a_step_s_tangents_are_refused(which):
    import torch.autograd.forward_ad as fwad

    from ssm_b200 import ops

    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    ins = [r(1, 2, 8, 16), r(1, 1, 16), r(1, 1, 16), r(1, 2, 8), r(1, 2), torch.rand(1, 2, device="cuda")]
    for grad in (torch.enable_grad(), torch.no_grad()):
        with fwad.dual_level(), grad:
            args = list(ins)
            args[which + 1] = fwad.make_dual(ins[which + 1], torch.ones_like(ins[which + 1]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.gated_delta_step(*args)
