"""What a ``TopKMoE`` is as a torch module (CPU)."""

from __future__ import annotations

import pytest
import torch

from opake_amd.moe import TopKMoE


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(),
                                  lambda m: m.double(), lambda m: m.to("meta").bfloat16()],
                         ids=["to", "half", "double", "meta"])
def test_casts_leave_the_route_bias_float32(cast):
    """A balancing rule's steps are far below bfloat16's, and the choice takes float32."""
    moe = TopKMoE(8, 4, 4, 2, routing={})
    moe.route_bias.copy_(torch.tensor([1.001, -0.003, 0.0, 2.0**-20]))
    want = moe.route_bias.clone()
    cast(moe)
    assert moe.route_bias.dtype == torch.float32 and moe.router.weight.dtype != torch.float32
    assert moe.route_bias.device == moe.router.weight.device
    assert moe.route_bias.is_meta or torch.equal(moe.route_bias, want)
    assert "route_bias" in moe.state_dict()
    plain = TopKMoE(8, 4, 4, 2).to(torch.bfloat16)
    assert not hasattr(plain, "route_bias") and plain.router.weight.dtype == torch.bfloat16
