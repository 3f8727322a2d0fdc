"""The gated delta block and the head's losses where their surroundings are unusual, on the CPU oracle's operators."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle
from ssm_b200.mixer import GatedDeltaBlock


@pytest.mark.parametrize("cast,kept", [(lambda m: m.to(torch.bfloat16), torch.float32), (lambda m: m.half(), torch.float32), (lambda m: m.double(), torch.float64),
                                       (lambda m: m.to(torch.bfloat16).float(), torch.float32)])
def test_a_cast_block_scales_its_keys_to_norm_one(cast, kept):
    """``K ** -0.5`` has no 16-bit form for most K: the factor stays in 32 bits or more, and out of the state dict."""
    m = cast(GatedDeltaBlock(16, d_state=24, headdim=8, ops=lm_oracle.namespace()))
    want = torch.full((24,), 24 ** -0.5, dtype=kept)
    assert m.unit.dtype == kept and torch.equal(m.unit, want) and "unit" not in m.state_dict()


def test_a_block_made_without_memory_has_its_factor_once_it_gets_some():
    m = GatedDeltaBlock(16, d_state=24, headdim=8, device="meta", ops=lm_oracle.namespace()).to_empty(device="cpu")
    assert torch.equal(m.unit, torch.full((24,), 24 ** -0.5))


@pytest.mark.parametrize("layer", ["Mamba2", "GatedDelta"])
def test_a_shard_of_a_sequence_cannot_be_scored(layer):
    """The token behind a shard's last one, and the distribution before its first, are another rank's."""
    from ssm_b200.lm import MambaConfig, MambaLMHeadModel

    cfg = MambaConfig(d_model=32, n_layer=1, vocab_size=50, ssm_cfg=dict(layer=layer, d_state=16, headdim=16))
    model = MambaLMHeadModel(cfg, ops=lm_oracle.namespace())
    with pytest.raises(ValueError, match="shard"):
        model.score(torch.zeros(1, 8, dtype=torch.long), sharded=True)
    for kw in (dict(num_last_tokens=3), dict(inference_params=model.allocate_inference_cache(1))):
        with pytest.raises(ValueError, match="whole sequence"):
            model.score(torch.zeros(1, 8, dtype=torch.long), **kw)
