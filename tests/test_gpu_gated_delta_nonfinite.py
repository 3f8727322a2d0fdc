"""Values that are not finite in the gated delta rule: they reach what depends on them, in every kernel that a call can take, and nothing before."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_gated_delta import BF16, F16, F32, inputs, on_gpu

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 64, 48), (BF16, 128, 128), (F16, 64, 64)])
@pytest.mark.parametrize("at", [0, 70, 149])
def test_a_decay_that_is_not_a_number_shows(dtype, kd, vd, at):
    """In one head, at one token: that head's answers from there on and its state, the gradients; the other head and tokens as before."""
    from ssm_b200 import ops

    ts = inputs(1, 150, 1, 2, kd, vd, dtype)

    def call(spoil):
        leaves = on_gpu(ts, dtype)
        if spoil:
            leaves[3][0, at, 1] = NAN
        with torch.no_grad():
            first = ops.gated_delta_scan(*leaves, return_final_state=True, keep_state_fp32=True)
        leaves = [t.requires_grad_(True) for t in leaves]
        again = ops.gated_delta_scan(*leaves, return_final_state=True, keep_state_fp32=True)
        return [*first, *again], torch.autograd.grad(again[0].float().sum(), leaves)

    (clean, grads), (spoilt, bad) = call(False), call(True)
    for i in (0, 2):
        assert torch.equal(clean[i][:, :, 0], spoilt[i][:, :, 0])
        assert torch.isnan(spoilt[i][:, at:, 1]).all()
        whole = at // 64 * 64
        assert torch.equal(clean[i][:, :whole, 1], spoilt[i][:, :whole, 1])
    for i in (1, 3):
        assert torch.equal(clean[i][:, 0], spoilt[i][:, 0]) and torch.isnan(spoilt[i][:, 1]).all()
    assert torch.isnan(bad[3][:, at, 1]).all() and torch.equal(bad[3][:, :, 0], grads[3][:, :, 0])


def _spoil(leaves, name, value, at, head=1):
    q, k, v, g, beta = leaves
    if name == "v":
        v[0, at, head, 3] = value
    elif name in "qk":
        (q if name == "q" else k)[0, at, head, 5] = value
    else:
        (g if name == "g" else beta)[0, at, head] = value


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype,kd,vd", [(F32, 64, 48), (BF16, 128, 128), (BF16, 64, 192), (F16, 128, 64), (F16, 72, 40)])
@pytest.mark.parametrize("name,value", [("q", NAN), ("k", NAN), ("k", -INF), ("v", NAN), ("v", INF), ("g", NAN), ("beta", NAN), ("beta", INF)])
def test_nothing_before_a_value_that_is_not_finite_changes(name, value, dtype, kd, vd, train):
    """Tokens before it give the same bits, its own column of v (or its head) gives nothing finite from it on."""
    from ssm_b200 import ops

    nl = 200
    ts = inputs(1, nl, 2, 2, kd, vd, dtype, seed=3)

    def call(at):
        leaves = on_gpu(ts, dtype)
        if at is not None:
            _spoil(leaves, name, value, at)
        leaves = [t.requires_grad_(train) for t in leaves]
        return [t.detach() for t in ops.gated_delta_scan(*leaves, return_final_state=True, keep_state_fp32=True)]

    o, s = call(None)
    for at in (0, 15, 17, 63, 64, 100, 199):
        bo, bs = call(at)
        assert torch.equal(o[:, :, 0], bo[:, :, 0]) and torch.equal(s[:, 0], bs[:, 0]), at
        assert torch.equal(o[:, :at, 1], bo[:, :at, 1]), at
        if name == "q":  # its own answer alone
            assert not torch.isfinite(bo[:, at, 1]).any() and torch.equal(o[:, at + 1:], bo[:, at + 1:]) and torch.equal(s, bs), at
        elif name == "v":
            others = torch.arange(vd, device="cuda") != 3
            assert torch.equal(o[:, :, 1, others], bo[:, :, 1, others]) and torch.equal(s[:, 1, others], bs[:, 1, others]), at
            assert not torch.isfinite(bo[:, at:, 1, 3]).any() and not torch.isfinite(bs[:, 1, 3]).any(), at
        else:
            assert not torch.isfinite(bo[:, at + 1:, 1]).any() and not torch.isfinite(bs[:, 1]).any(), at


@pytest.mark.parametrize("dtype,kd,vd", [(F32, 32, 32), (BF16, 128, 128), (F16, 64, 64)])
def test_a_padded_batch_with_garbage_behind_its_sequences(dtype, kd, vd):
    """Prompts of several lengths in one dense batch, what lies behind each of them never written: each answers as without it."""
    from ssm_b200 import ops

    lens = [150, 97, 1, 128, 40]
    leaves = on_gpu(inputs(len(lens), 150, 1, 2, kd, vd, dtype), dtype)
    want = ops.gated_delta_scan(*leaves)
    for t in leaves:
        for b, n in enumerate(lens):
            t[b, n:] = NAN
    got = ops.gated_delta_scan(*leaves)
    for b, n in enumerate(lens):
        assert torch.equal(got[b, :n], want[b, :n]), n


@pytest.mark.parametrize("dtype,kd,vd", [(BF16, 128, 128), (F16, 64, 64)])
def test_several_columns_and_chunks_of_values_that_are_not_finite(dtype, kd, vd):
    """Each column of v from its first such value on, in chunks one behind the other, packed sequences among them."""
    from ssm_b200 import ops

    nl, cuts = 330, [0, 100, 101, 330]
    ts = inputs(1, nl, 1, 1, kd, vd, dtype)
    clean = ops.gated_delta_scan(*on_gpu(ts, dtype), cu_seqlens=torch.tensor(cuts).cuda(), return_final_state=True, keep_state_fp32=True)
    leaves = on_gpu(ts, dtype)
    gen = torch.Generator().manual_seed(7)
    first = torch.full((3, vd), nl)
    for _ in range(40):
        t, c = int(torch.randint(0, nl, (1,), generator=gen)), int(torch.randint(0, vd, (1,), generator=gen))
        leaves[2][0, t, 0, c] = [NAN, INF, -INF][t % 3]
        seq = sum(t >= e for e in cuts[1:])
        first[seq, c] = min(int(first[seq, c]), t)
    got = ops.gated_delta_scan(*leaves, cu_seqlens=torch.tensor(cuts).cuda(), return_final_state=True, keep_state_fp32=True)
    at = torch.arange(nl)
    seq = sum((at >= e).long() for e in cuts[1:-1])
    lost = (at[:, None] >= first[seq]).cuda()
    assert torch.equal(got[0][0, :, 0][~lost], clean[0][0, :, 0][~lost]) and not torch.isfinite(got[0][0, :, 0][lost]).any()
    gone = (first < nl).cuda()
    assert torch.equal(got[1][:, 0][~gone], clean[1][:, 0][~gone]) and not torch.isfinite(got[1][:, 0][gone]).any()
