"""A refused ``HybridBlock.weight_loader`` leaves the block as it was."""

import pytest
import torch

from moe_inference_verify_microbench_b200.hybrid import HybridBlock


@pytest.mark.parametrize("options,extra", [
    ({}, "attn_post_norm_weight"), ({}, "moe_gate"), ({"post_norm": True}, "attn_gate")])
def test_refused_load_changes_nothing(options, extra):
    block = HybridBlock(64, 64, 2, 2, 32, 4, 2, 1, 0, None, 1, 0, None, **options)
    for p in block.parameters():
        p.data.fill_(3.0)
    z = lambda *s: torch.zeros(*s)
    w = [z(64, 64)] * 4
    args = (z(64), z(64, 64), z(64, 64), z(64, 64), z(64, 64), z(64), z(4, 64), w, w, w)
    with pytest.raises(ValueError, match="no " + extra.replace("_weight", "")):
        block.weight_loader(*args, **{extra: z(64)})
    assert all(bool((p == 3.0).all()) for p in block.parameters())
