"""Sizes that do not fit the C types of llmrs_cuda_rope_frequencies are refused, not cut to 32 bits; host only."""
import pytest

from llm_rs_b200 import RopeScaling, rope_frequencies


@pytest.mark.parametrize("kw", [dict(rotary_dim=(1 << 32) + 64), dict(rotary_dim=-64), dict(original_context=(1 << 32) + 8192),
                                dict(original_context=-1)])
def test_sizes_beyond_32_bits(cuda_lib, kw):
    args = dict(rotary_dim=64, rope_theta=10000.0, kind=RopeScaling.YARN, factor=2.0, original_context=4096, low=1.0, high=32.0) | kw
    with pytest.raises(ValueError):
        rope_frequencies(**args)
