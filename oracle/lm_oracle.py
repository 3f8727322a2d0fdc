"""The operators beside the state-space ones, from their definitions, on CPU tensors in whatever type they come in (double in the tests);
differentiable through autograd.  Test infrastructure only."""

from __future__ import annotations

import torch


def gated_delta(q, k, v, g, beta, scale=None, initial_state=None, cu_seqlens=None):
    """``(o, final states)`` of the gated delta rule, token by token; shapes as in ``ssm_b200.ops.gated_delta_scan``."""
    if cu_seqlens is not None:
        cu = [int(c) for c in cu_seqlens]
        outs, states = [], []
        for i, (a, b) in enumerate(zip(cu, cu[1:])):
            cut = lambda t: None if t is None else t[:, a:b]  # noqa: E731
            o, s = gated_delta(cut(q), cut(k), cut(v), cut(g), cut(beta), scale, None if initial_state is None else initial_state[i:i + 1])
            outs.append(o)
            states.append(s)
        outs.append(torch.zeros_like(v[:, cu[-1]:]))
        return torch.cat(outs, 1), torch.cat(states)
    nb, nl, nh, vd = v.shape
    kd, rep = k.shape[3], nh // k.shape[2]
    scale = kd ** -0.5 if scale is None else scale
    state = v.new_zeros(nb, nh, vd, kd) if initial_state is None else initial_state
    o = []
    for t in range(nl):
        kt, qt = k[:, t].repeat_interleave(rep, 1), q[:, t].repeat_interleave(rep, 1)
        if g is not None:
            state = state * torch.exp(g[:, t])[..., None, None]
        r = v[:, t] - torch.einsum("bhvk,bhk->bhv", state, kt)
        state = state + torch.einsum("bhv,bhk->bhvk", beta[:, t, :, None] * r, kt)
        o.append(scale * torch.einsum("bhvk,bhk->bhv", state, qt))
    return (torch.stack(o, 1) if o else torch.zeros_like(v)), state


def token_log_probs(logits, targets, temperature=1.0, top_k=0, ignore_index=-100):
    """``(log p[target], entropy, top log probabilities, their ids)``."""
    logp = torch.log_softmax(logits / temperature, -1)
    kept = targets != ignore_index
    at = torch.where(kept, targets, torch.zeros_like(targets))
    got = torch.where(kept, torch.gather(logp, -1, at[..., None])[..., 0], torch.zeros((), dtype=logits.dtype))
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp.clamp_min(torch.finfo(logp.dtype).min), torch.zeros((), dtype=logits.dtype)).sum(-1)
    _, ids = torch.sort(logits.detach(), dim=-1, descending=True, stable=True)
    ids = ids[..., :top_k]
    return got, entropy, torch.gather(logp, -1, ids), ids


def topk_distill_loss(logits, teacher_logits, teacher_ids, temperature=1.0):
    """Divergence of the student from the teacher's renormalised top tokens."""
    logq = torch.log_softmax(logits / temperature, -1)
    kept = teacher_ids >= 0
    t = torch.where(kept, teacher_logits, torch.full((), -float("inf"), dtype=teacher_logits.dtype)) / temperature
    empty = (t == -float("inf")).all(-1, keepdim=True)
    logt = torch.log_softmax(torch.where(empty, torch.zeros_like(t), t), -1)
    pt = torch.where(empty, torch.zeros_like(t), torch.exp(logt))
    term = pt * (logt.clamp_min(torch.finfo(logt.dtype).min) - torch.gather(logq, -1, teacher_ids.clamp_min(0)))
    return torch.where(pt > 0, term, torch.zeros_like(term)).sum(-1)


def namespace():
    """The state-space oracle's operators with these beside them, under the names and signatures of ``ssm_b200.ops``."""
    from types import SimpleNamespace

    from . import ssm_oracle

    def gated_delta_scan(q, k, v, g, beta, scale=None, initial_state=None, return_final_state=False, keep_state_fp32=False, cu_seqlens=None):
        o, s = gated_delta(q, k, v, g, beta, scale, initial_state, cu_seqlens)
        return (o, s) if return_final_state else o

    def gated_delta_step(state, q, k, v, g, beta, scale=None):
        o, s = gated_delta(q[:, None], k[:, None], v[:, None], None if g is None else g[:, None], beta[:, None], scale, state.clone())
        with torch.no_grad():
            state.copy_(s)
        return o[:, 0]

    def log_probs(logits, targets, temperature=1.0, top_k=0, return_entropy=False, ignore_index=-100):
        got = token_log_probs(logits, targets, temperature, top_k, ignore_index)
        out = got[:1] + (got[1:2] if return_entropy else ()) + (got[2:] if top_k else ())
        return out if len(out) > 1 else out[0]

    return SimpleNamespace(**{n: f for n, f in vars(ssm_oracle).items() if not n.startswith("_")}, gated_delta_scan=gated_delta_scan,
                           gated_delta_step=gated_delta_step, token_log_probs=log_probs, topk_distill_loss=topk_distill_loss)
