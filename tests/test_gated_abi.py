"""What the gated projections' entry points answer before anything is launched (CPU)."""

from __future__ import annotations

import pytest

from opake_amd import _native as nat


@pytest.fixture()
def lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("native library not built")
    return nat.load()


@pytest.mark.parametrize("code", [nat.DPC_BF16, nat.DPC_F32])
@pytest.mark.parametrize("D,F", [(2048, 8192), (1024, 1408), (1001, 512), (64, 512), (16, 8),
                                 (1, 1), (1 << 20, 1 << 19)])
def test_no_token(lib, code, D, F):
    """No workspace and nothing to do, whatever the widths."""
    assert lib.dpc_gated_linear_workspace_bytes(0, D, F, code) == 0
    assert lib.dpc_gated_linear(0, 0, 0, D, F, code, nat.ACT_SILU, 0, 0, 0, 0, 0, 0) == nat.DPC_OK
    assert lib.dpc_gated_linear_act_grad(0, 0, 0, 0, F, code, nat.ACT_SILU, 0, 0) == nat.DPC_OK
    for want in ((1, 0), (0, 1), (1, 1), (0, 0)):
        assert lib.dpc_gated_linear_grad_workspace_bytes(0, D, F, code, *want) == 0
    assert lib.dpc_gated_linear_grad(0, 0, 0, 0, D, F, code, 256, 256, 0, 0, 0) == nat.DPC_OK


def test_workspaces_of_few_tokens(lib):
    for code, N in ((nat.DPC_BF16, 1), (nat.DPC_BF16, 33), (nat.DPC_F32, 1), (nat.DPC_F32, 65)):
        for D, F in ((2048, 8192), (1001, 512), (64, 512)):
            assert lib.dpc_gated_linear_workspace_bytes(N, D, F, code) > 0
            assert lib.dpc_gated_linear_grad_workspace_bytes(N, D, F, code, 1, 1) > 0
