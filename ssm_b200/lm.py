"""Language-model wrapper on the B200 operators: ``MixerModel`` / ``MambaLMHeadModel`` with the constructor and
call signatures of the upstream classes (src/ssm/models/lm.py:175-392, 395-520; configuration
src/ssm/models/config.py), built from this package's mixer blocks.

Every layer is upstream's fused-add-norm block (src/ssm/modules/block.py:109-131): ``residual = hidden + residual``
and ``hidden = norm(residual)`` are ONE call of ``fused_layer_norm(..., return_residual=True)`` (upstream routes that
to an external Triton kernel), followed by the mixer; the final norm folds the last residual add the same way
(lm.py:378-387).  The residual stream is kept in fp32 when ``residual_in_fp32``.  Mixers: ``ssm_cfg["layer"]`` selects
``"Mamba1"`` (selective scan) or ``"Mamba2"`` (state-space-dual scan with a d_state axis, upstream Mamba-2 layout); beyond upstream ``"GatedDelta"``
(the gated delta rule).
Attention layers and the gated MLP of upstream's hybrid configurations are outside the operator hot path and are
rejected.  Beyond upstream: ``forward(..., sharded=True, group=pg)`` runs a Mamba-2 stack on one contiguous shard of a
sequence split over ranks (`ssm_b200.seqpar`), and ``step`` decodes one token against caches allocated by
``allocate_inference_cache``; ``MambaLMHeadModel.score`` gives the log probabilities of given tokens and ``distill_loss`` the divergence from a
teacher's top logits, both differentiable; ``loss`` is the cross entropy of the next token without the logits, ``clip_grad_norm_`` clips all gradients by their
norm; ``ssm_cfg["post_norm"]`` puts a norm after every mixer, with a learned gate (``"post_gate"``) and a factor (``"residual_scale"``), one call with the
residual add and the next layer's norm.
"""

from __future__ import annotations

from collections import namedtuple
from dataclasses import dataclass, field
from typing import Any, Optional

import torch
from torch import Tensor, nn

from .mixer import GatedDeltaBlock, Mamba1Block, Mamba2Block

CausalLMOutput = namedtuple("CausalLMOutput", ["logits"])


def _default_ssm_cfg() -> dict:
    return {"layer": "Mamba1", "dt_rank": "auto", "dt_min": 1e-3, "dt_max": 1e-1, "dt_init_floor": 1e-4}


@dataclass
class MambaConfig:
    """Same fields and defaults as upstream's ``MambaConfig`` (src/ssm/models/config.py)."""

    d_model: int = 2560
    d_intermediate: int = 0
    n_layer: int = 64
    vocab_size: int = 50277
    ssm_cfg: dict = field(default_factory=_default_ssm_cfg)
    attn_layer_idx: list = field(default_factory=list)
    attn_cfg: dict = field(default_factory=dict)
    rms_norm: bool = True
    residual_in_fp32: bool = True
    fused_add_norm: bool = True
    pad_vocab_size_multiple: int = 8
    tie_embeddings: bool = True


@dataclass
class InferenceCache:
    """Per-layer decode state (what upstream keeps in ``InferenceParams.layer_states``)."""

    layer_states: dict
    seqlen_offset: int = 0


class MixerModel(nn.Module):
    """Embedding, ``n_layer`` fused-add-norm mixer blocks, final norm (upstream ``MixerModel``, lm.py:175-392)."""

    def __init__(self, *, d_model: int, n_layer: int, d_intermediate: int, vocab_size: int, ssm_cfg: Optional[dict] = None,
                 attn_layer_idx: Optional[list] = None, attn_cfg: Optional[dict] = None, norm_epsilon: float = 1e-5, rms_norm: bool = False,
                 initializer_cfg: Optional[dict] = None, fused_add_norm: bool = False, residual_in_fp32: bool = False, device=None, dtype=None,
                 ops: Any = None) -> None:
        super().__init__()
        if attn_layer_idx or d_intermediate:
            raise ValueError("attention layers and the gated MLP are not part of the state-space operator path")
        del attn_cfg, fused_add_norm  # the add + norm of every layer always runs as one fused operator call
        cfg = dict(ssm_cfg or {})
        kind = cfg.pop("layer", "Mamba1")
        cfg.pop("dt_init", None)
        self.post_norm, post_gate = bool(cfg.pop("post_norm", False)), bool(cfg.pop("post_gate", False))
        self.residual_scale = float(cfg.pop("residual_scale", 1.0))
        if not self.post_norm and (post_gate or self.residual_scale != 1.0):
            raise ValueError("ssm_cfg['post_gate'] and ['residual_scale'] belong to ['post_norm']")
        if kind in ("Mamba2", "GatedDelta"):
            cfg.pop("dt_rank", None)  # one step size per head, projected straight from the input
        if kind not in ("Mamba1", "Mamba2", "GatedDelta"):
            raise ValueError("ssm_cfg['layer'] must be 'Mamba1', 'Mamba2' or 'GatedDelta'")
        self.kind, self.rms_norm, self.eps, self.residual_in_fp32 = kind, bool(rms_norm), norm_epsilon, bool(residual_in_fp32)
        self.d_model = d_model
        self._ops = ops
        kw = dict(device=device, dtype=dtype)
        self.embedding = nn.Embedding(vocab_size, d_model, **kw)
        std = (initializer_cfg or {}).get("initializer_range", 0.02)
        nn.init.normal_(self.embedding.weight, std=std)
        block = {"Mamba1": Mamba1Block, "Mamba2": Mamba2Block, "GatedDelta": GatedDeltaBlock}[kind]
        # a block's own norm weight (`norm_w` / `pre_norm_w`) serves as the pre-norm of its layer
        self.layers = nn.ModuleList([block(d_model, eps=norm_epsilon, ops=ops, **cfg, **kw) for _ in range(n_layer)])
        self.norm_f_weight = nn.Parameter(torch.ones(d_model, **kw))
        self.norm_f_bias = None if rms_norm else nn.Parameter(torch.zeros(d_model, **kw))
        if not rms_norm:
            for layer in self.layers:
                layer.norm_b = nn.Parameter(torch.zeros(d_model, **kw))
        if self.post_norm:
            for layer in self.layers:
                layer.post_norm_w = nn.Parameter(torch.ones(d_model, **kw))
                if not rms_norm:
                    layer.post_norm_b = nn.Parameter(torch.zeros(d_model, **kw))
                if post_gate:
                    layer.post_gate = nn.Parameter(torch.ones(d_model, **kw))
        rescale = (initializer_cfg or {}).get("rescale_prenorm_residual", True)
        if rescale:  # upstream divides the output projections by sqrt(n_layer) (lm.py:80-98)
            with torch.no_grad():
                for layer in self.layers:
                    layer.out_proj /= n_layer ** 0.5

    def _namespace(self):
        if self._ops is not None:
            return self._ops
        from . import ops

        return ops

    def _pre_norm(self, layer):
        return (layer.norm_w if self.kind == "Mamba1" else layer.pre_norm_w), getattr(layer, "norm_b", None)

    def _norm(self, ops, before, hidden: Tensor, residual: Optional[Tensor], w: Tensor, b: Optional[Tensor]):
        """The stream behind layer ``before`` (``None``: behind the embedding), and its norm for what comes next."""
        if before is not None and self.post_norm:
            return ops.fused_block_norm(hidden, residual, before.post_norm_w, w, post_bias=getattr(before, "post_norm_b", None), bias=b, gate=getattr(before, "post_gate", None),
                                        residual_scale=self.residual_scale, is_rms=self.rms_norm, eps=self.eps, residual_in_fp32=self.residual_in_fp32)
        return ops.fused_layer_norm(hidden, w, b, residual=residual, is_rms=self.rms_norm, eps=self.eps, prenorm=True, residual_in_fp32=self.residual_in_fp32, return_residual=True)

    def allocate_inference_cache(self, batch_size: int, max_seqlen: int = 0, dtype: Optional[torch.dtype] = None, **kwargs) -> InferenceCache:
        del max_seqlen, kwargs  # state-space layers keep a fixed-size state
        return InferenceCache({i: layer.allocate_inference_cache(batch_size, dtype) for i, layer in enumerate(self.layers)})

    def forward(self, input_ids: Tensor, *, inference_params: Optional[InferenceCache] = None, sharded: bool = False, group=None) -> Tensor:
        """``input_ids (B, L)`` -> hidden states ``(B, L, d_model)`` after the final norm.  With ``inference_params`` and
        ``L == 1`` the call advances the caches by one token (decode)."""
        ops = self._namespace()
        hidden = self.embedding(input_ids)
        residual = before = None
        decode = inference_params is not None and input_ids.shape[1] == 1
        if inference_params is not None and not decode:
            raise ValueError("prefill into a cache is not built: feed the prompt token by token, or run forward() without a cache")
        for i, layer in enumerate(self.layers):
            w, b = self._pre_norm(layer)
            hidden, residual = self._norm(ops, before, hidden, residual, w, b)
            before = layer
            if decode:
                hidden = layer.mixer_step(hidden[:, 0], inference_params.layer_states[i]).unsqueeze(1)
            elif self.kind == "Mamba2":
                hidden = layer.mixer_forward(hidden, sharded=sharded, group=group)
            else:
                if sharded:
                    raise ValueError("sequence-sharded prefill is built for Mamba2 layers")
                hidden = layer.mixer_forward(hidden)
        if inference_params is not None:
            inference_params.seqlen_offset += input_ids.shape[1]
        if self.post_norm and before is not None:
            return self._norm(ops, before, hidden, residual, self.norm_f_weight, self.norm_f_bias)[0]
        return ops.fused_layer_norm(hidden, self.norm_f_weight, self.norm_f_bias, residual=residual, is_rms=self.rms_norm, eps=self.eps,
                                    prenorm=True, residual_in_fp32=self.residual_in_fp32)


class MambaLMHeadModel(nn.Module):
    """Backbone plus (tied) output head; ``forward`` returns ``CausalLMOutput(logits)`` (upstream lm.py:395-520)."""

    def __init__(self, config: MambaConfig, initializer_cfg: Optional[dict] = None, device=None, dtype=None, ops: Any = None) -> None:
        super().__init__()
        self.config = config
        vocab = config.vocab_size
        if vocab % config.pad_vocab_size_multiple:
            vocab += config.pad_vocab_size_multiple - vocab % config.pad_vocab_size_multiple
        self.backbone = MixerModel(d_model=config.d_model, n_layer=config.n_layer, d_intermediate=config.d_intermediate, vocab_size=vocab,
                                   ssm_cfg=config.ssm_cfg, attn_layer_idx=config.attn_layer_idx, attn_cfg=config.attn_cfg, rms_norm=config.rms_norm,
                                   fused_add_norm=config.fused_add_norm, residual_in_fp32=config.residual_in_fp32, initializer_cfg=initializer_cfg,
                                   device=device, dtype=dtype, ops=ops)
        self.lm_head = nn.Linear(config.d_model, vocab, bias=False, device=device, dtype=dtype)
        self.tie_weights()

    def tie_weights(self) -> None:
        if self.config.tie_embeddings:
            self.lm_head.weight = self.backbone.embedding.weight

    def allocate_inference_cache(self, batch_size: int, max_seqlen: int = 0, dtype: Optional[torch.dtype] = None, **kwargs) -> InferenceCache:
        return self.backbone.allocate_inference_cache(batch_size, max_seqlen, dtype=dtype, **kwargs)

    def forward(self, input_ids: Tensor, position_ids: Optional[Tensor] = None, inference_params: Optional[InferenceCache] = None,
                num_last_tokens: int = 0, **mixer_kwargs) -> CausalLMOutput:
        del position_ids
        if input_ids.dim() != 2:
            raise ValueError("input_ids must be a 2D tensor of shape (batch, seqlen)")
        hidden = self.backbone(input_ids, inference_params=inference_params, **mixer_kwargs)
        if num_last_tokens > 0:
            hidden = hidden[:, -num_last_tokens:, :]
        return CausalLMOutput(logits=self.lm_head(hidden))

    @staticmethod
    def _whole(what: str, mixer_kwargs: dict) -> None:
        if mixer_kwargs.get("sharded"):
            raise ValueError(f"{what}: a shard of a sequence has neither the distribution before its first token nor the token behind its last one")
        if mixer_kwargs.get("inference_params") is not None or mixer_kwargs.get("num_last_tokens"):
            raise ValueError(f"{what} runs over the whole sequence: inference_params and num_last_tokens are not taken")

    @staticmethod
    def _next(tokens: Tensor, ignore_index: int) -> Tensor:
        """What each position predicts; the last one nothing."""
        return torch.cat([tokens[:, 1:], torch.full_like(tokens[:, :1], ignore_index)], 1)

    def loss(self, input_ids: Tensor, labels: Optional[Tensor] = None, ignore_index: int = -100, reduction: str = "mean", return_log_z: bool = False, **mixer_kwargs):
        """Cross entropy of a sequence's own next tokens, without the logits (``ops.linear_cross_entropy`` of the hidden states and the head): the mean over the
        positions that count, their sum, or with ``reduction="none"`` one per position ``(B, L - 1)``; ``labels (B, L)`` in the place of the tokens, those equal to ``ignore_index``
        left out; with ``return_log_z`` the log of the partition sums ``(B, L - 1)`` behind it.  A whole sequence at once; over all of the head's columns, padded ones too."""
        self._whole("loss", mixer_kwargs)
        if input_ids.dim() != 2:
            raise ValueError("input_ids must be a 2D tensor of shape (batch, seqlen)")
        hidden = self.backbone(input_ids, **mixer_kwargs)
        targets = self._next(input_ids if labels is None else labels, ignore_index)
        got = self.backbone._namespace().linear_cross_entropy(hidden, self.lm_head.weight, targets, ignore_index, reduction, return_log_z)
        loss, *log_z = got if return_log_z else (got,)
        loss = loss[:, :-1] if reduction == "none" else loss
        return (loss, log_z[0][:, :-1]) if return_log_z else loss

    def clip_grad_norm_(self, max_norm: float, norm_type: float = 2.0) -> Tensor:
        """Clips the gradients of all parameters by their common norm, which is returned (``ops.clip_global_norm_``); parameters without one are left out."""
        return self.backbone._namespace().clip_global_norm_([p.grad for p in self.parameters() if p.grad is not None], max_norm, norm_type)

    def score(self, input_ids: Tensor, labels: Optional[Tensor] = None, temperature: float = 1.0, top_k: int = 0, return_entropy: bool = False,
              ignore_index: int = -100, **mixer_kwargs):
        """Log probabilities of a sequence's own tokens, each given those before it: ``input_ids (B, L)`` -> ``(B, L - 1)`` fp32, with the entropies and
        the ``top_k`` alternatives behind them as in ``ops.token_log_probs``.  ``labels (B, L)`` in the place of the tokens; those equal to
        ``ignore_index`` give 0.  A whole sequence at once: no shard of one, no cache; over all of the head's columns, padded ones too."""
        self._whole("score", mixer_kwargs)
        logits = self.forward(input_ids, **mixer_kwargs).logits
        targets = self._next(input_ids if labels is None else labels, ignore_index)
        got = self.backbone._namespace().token_log_probs(logits, targets, temperature, top_k, return_entropy, ignore_index)
        return tuple(t[:, :-1] for t in got) if isinstance(got, tuple) else got[:, :-1]

    def distill_loss(self, input_ids: Tensor, teacher_logits: Tensor, teacher_ids: Tensor, temperature: float = 1.0, **mixer_kwargs) -> Tensor:
        """Divergence of this model's distributions from a teacher's top logits ``(B, L, k)`` with their ids, per position: ``(B, L)`` fp32
        (``ops.topk_distill_loss``)."""
        logits = self.forward(input_ids, **mixer_kwargs).logits
        return self.backbone._namespace().topk_distill_loss(logits, teacher_logits, teacher_ids, temperature)

    @torch.no_grad()
    def generate(self, input_ids: Tensor, max_length: int, cuda_graph: bool = False) -> Tensor:
        """Greedy decoding: the prompt is fed token by token into fresh caches, then ``max_length - prompt`` tokens are
        produced.  ``cuda_graph=True`` captures one decode step and replays it (what upstream's generation driver does,
        src/ssm/utils/generation.py:187-315)."""
        nb, plen = input_ids.shape
        cache = self.allocate_inference_cache(nb)
        tok = input_ids[:, :1].clone()
        logits = None
        step = lambda: self.forward(tok, inference_params=cache).logits[:, -1]  # noqa: E731
        graph = None
        if cuda_graph:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            snapshot = [[t.clone() for t in _flat(cache.layer_states[i])] for i in cache.layer_states]
            with torch.cuda.stream(side):
                for _ in range(2):
                    step()
            torch.cuda.current_stream().wait_stream(side)
            for saved, i in zip(snapshot, cache.layer_states):  # the warm-up steps advanced the caches: restore them
                for dst, src in zip(_flat(cache.layer_states[i]), saved):
                    dst.copy_(src)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                logits = step()
            for saved, i in zip(snapshot, cache.layer_states):
                for dst, src in zip(_flat(cache.layer_states[i]), saved):
                    dst.copy_(src)
        out = [input_ids]
        for t in range(max_length - 1):
            tok.copy_(input_ids[:, t:t + 1] if t < plen else nxt)
            if graph is not None:
                graph.replay()
            else:
                logits = step()
            nxt = logits.argmax(-1, keepdim=True)
            if t + 1 >= plen:
                out.append(nxt.clone())
        return torch.cat(out, dim=1)


def _flat(state):
    if isinstance(state, Tensor):
        return [state]
    return [t for s in state for t in _flat(s)]
