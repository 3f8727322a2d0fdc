"""What a training step runs around the mixers, from the definitions, on CPU tensors (in 64 bits where the tests want them): the norms around a
block, cross entropy from hidden states, the norm over many tensors with clipping.  The functions have the arguments of ``ssm_b200.ops``."""

from __future__ import annotations

import math

import torch


def _norm(x, weight, bias, is_rms, eps):
    if not is_rms:
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return x if bias is None else x + bias


def fused_block_norm(x, residual, post_weight, weight, post_bias=None, bias=None, gate=None, residual_scale=1.0, is_rms=True, eps=1e-5, post_eps=None,
                     residual_in_fp32=True):
    wide = lambda t: t if t is None or t.dtype == torch.float64 else t.float()  # noqa: E731
    n = _norm(wide(x), wide(post_weight), wide(post_bias), is_rms, eps if post_eps is None else post_eps)
    if gate is not None:
        gate = wide(gate)
        n = n * (gate[:, None] if gate.dim() == 2 else gate)
    r = residual_scale * n
    if residual is not None:
        r = wide(residual) + r
    y = _norm(r, wide(weight), wide(bias), is_rms, eps)
    return y.to(x.dtype), r if x.dtype == torch.float64 else r.to(torch.float32 if residual_in_fp32 else x.dtype)


def linear_cross_entropy(hidden, weight, targets, ignore_index=-100, reduction="none", return_log_z=False):
    kept = targets != ignore_index
    z = (hidden if hidden.dtype == torch.float64 else hidden.float()) @ (weight if weight.dtype == torch.float64 else weight.float()).t()
    z = torch.where(kept[..., None], z, torch.zeros((), dtype=z.dtype, device=z.device))  # what lies in rows left out does no harm
    log_z = torch.logsumexp(z, -1)
    at = torch.where(kept, targets, torch.zeros_like(targets)).long()
    bad = (at < 0) | (at >= weight.shape[0])
    loss = log_z - torch.gather(z, -1, at.clamp(0, weight.shape[0] - 1)[..., None])[..., 0]
    none = torch.zeros((), dtype=z.dtype, device=z.device)
    loss = loss + torch.where(bad, none + math.nan, none)
    loss, log_z = torch.where(kept, loss, none), torch.where(kept, log_z, none)
    if reduction != "none":
        loss = loss.sum()
    if reduction == "mean":
        loss = loss / kept.sum().clamp(min=1)
    return (loss, log_z) if return_log_z else loss


def global_norm(tensors, norm_type=2.0):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    flat = [t.detach().double().reshape(-1) for t in tensors if t.numel()]
    if not flat:
        return torch.zeros(())
    flat = torch.cat(flat)
    return (flat.abs().max() if norm_type == math.inf else flat.pow(2).sum().sqrt()).float()


def clip_global_norm_(tensors, max_norm, norm_type=2.0):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    norm = global_norm(tensors, norm_type)
    c = max_norm / (norm.double() + 1e-6)
    if not c >= 1 and max_norm != math.inf:
        for t in tensors:
            t.detach().copy_(t.detach().double() * c)
    return norm


def namespace():
    """The oracle's operators under one roof, as ``ssm_b200.ops`` has them."""
    from . import lm_oracle

    ns = lm_oracle.namespace()
    for fn in (fused_block_norm, linear_cross_entropy, global_norm, clip_global_norm_):
        setattr(ns, fn.__name__, fn)
    return ns
