"""Sizes that the 4-bit layout does not have are refused when a module is made, not in its
first forward."""

import pytest

from moe_inference_verify_microbench_b200 import PermutedSparseMoE


@pytest.mark.parametrize("hidden,intermediate,group", [(96, 64, 32), (64, 96, 32), (160, 64, 32),
                                                       (8256, 64, 64), (64, 8256, 64)])
def test_sizes_without_a_layout(hidden, intermediate, group):
    with pytest.raises(ValueError, match="64"):
        PermutedSparseMoE(hidden, intermediate, 16, 2, expert_weights="w4", group_size=group)
    PermutedSparseMoE(hidden, intermediate, 2, 2)  # bf16: no such layout


@pytest.mark.parametrize("hidden,intermediate,group", [(64, 192, 32), (8192, 64, 64)])
def test_sizes_with_one(hidden, intermediate, group):
    PermutedSparseMoE(hidden, intermediate, 1, 1, expert_weights="w4", group_size=group)
