"""What the fused blocks are as torch modules (CPU)."""

from __future__ import annotations

import io

import pytest
import torch

from opake_amd.exceptions import ConfigurationError
from opake_amd.lora import LoRABlock
from opake_amd.moe import RoutedLM, TopKMoE
from opake_amd.transformer import BlockLM, LlamaBlock, RotaryFrequencies


@pytest.mark.parametrize("make", [
    lambda d, **kw: LlamaBlock(d, 2, 8, device="meta", **kw),
    lambda d, **kw: BlockLM(7, d, 2, 8, device="meta", **kw),
    lambda d, **kw: LoRABlock(d, 2, 1, 8, 2, device="meta", **kw),
    lambda d, **kw: RoutedLM(7, d, 2, 8, 4, 3, device="meta", **kw)])
def test_heads_that_attention_does_not_take_are_refused_when_the_block_is_made(make):
    make(512, fused=True)
    make(528), make(6)
    for d in (528, 6):  # 264 wide, and three
        with pytest.raises(ConfigurationError):
            make(d, fused=True)
    assert RotaryFrequencies(512).freqs.shape == (256,)  # (rotary takes them)


@pytest.mark.parametrize("make,x", [
    (lambda: LlamaBlock(8, 2, 6), (2, 3, 8)), (lambda: LoRABlock(8, 2, 1, 6, 2), (2, 3, 8)),
    (lambda: TopKMoE(8, 6, 3), (2, 3, 8))])
def test_blocks_pickled_before_there_were_fused_ones(make, x):
    """Their dictionaries lack ``fused``: they run as they did."""
    block, x = make(), torch.randn(*x)
    with torch.no_grad():
        want = block(x)
        for m in block.modules():
            m.__dict__.pop("fused", None)
        buffer = io.BytesIO()
        torch.save(block, buffer)
        buffer.seek(0)
        assert torch.equal(torch.load(buffer, weights_only=False)(x), want)
