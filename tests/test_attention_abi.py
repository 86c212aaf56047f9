"""What the attention entry points refuse before anything is launched (CPU)."""

from __future__ import annotations

import pytest

from opake_amd import _native as nat


@pytest.fixture()
def lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("native library not built")
    return nat.load()


def _strides(*s):
    return (nat._c_i64 * len(s))(*s)


def test_forward(lib):
    ok = _strides(*([1 << 12, 64, 16] * 3))

    def call(B=1, T=4, S=4, H=4, KV=2, h=16, code=nat.DPC_BF16, causal=1, window=0, scale=1.0,
             q=256, k=256, v=256, out=256, strides=ok, size=0):
        return lib.dpc_attention(q, k, v, strides, B, T, S, H, KV, h, code, 0, 0, causal, window,
                                 scale, out, 0, 0, 0, size, 0)

    assert call(B=0) == call(T=0) == nat.DPC_OK  # nothing to do
    for bad in (dict(H=3), dict(KV=0), dict(h=0), dict(h=12), dict(h=264), dict(B=-1), dict(T=-1),
                dict(T=1 << 25), dict(code=nat.DPC_F16), dict(window=-1),
                dict(window=3, causal=0), dict(scale=0.0), dict(scale=float("nan")),
                dict(scale=1e300), dict(q=0), dict(k=0), dict(v=264), dict(out=0),
                dict(B=1 << 29, T=1 << 20),
                dict(strides=_strides(1 << 12, 64, 17, *([1 << 12, 64, 16] * 2)))):
        assert call(**bad) == nat.DPC_EINVAL, bad
    assert call(T=1, S=1 << 14) == nat.DPC_ENOSPC  # keys in splits
    for far in (_strides(1 << 12, 1 << 30, 16, *([1 << 12, 64, 16] * 2)),
                _strides(*([1 << 12, 64, 16] * 2), 1 << 12, 8, 16)):  # values overlap
        assert call(strides=far) == nat.DPC_ENOTSUP


def test_gradient(lib):
    ok = _strides(*([1 << 12, 64, 16] * 4))

    def call(T=4, dk=256, dv=256, state=256, size=0, ws=0, kept=1 << 20):
        return lib.dpc_attention_grad(256, 256, 256, 256, 256, ok, 1, T, 4, 4, 2, 16, nat.DPC_BF16,
                                      0, 0, 1, 0, 1.0, state, kept, 256, dk, dv, ws, size, 0)

    for bad in (dict(state=0), dict(dk=0), dict(dv=0), dict(dk=8), dict(ws=8, size=1 << 20)):
        assert call(**bad) == nat.DPC_EINVAL, bad
    assert call() == call(size=1 << 20, ws=256, kept=8) == nat.DPC_ENOSPC


def test_workspaces(lib):
    def size(B, T, S, H, KV, h, code=nat.DPC_BF16):
        return lib.dpc_attention_workspace_bytes(B, T, S, H, KV, h, code)

    assert size(16, 1024, 1024, 16, 16, 128) == 0  # whole row tiles
    assert size(0, 1, 1, 1, 1, 8) == size(1, 0, 1, 1, 1, 8) == 0
    assert size(1, 1, 64, 1, 1, 64) == 0
    assert size(1, 1, 512, 1, 1, 64) == 4 * (64 * 4 + 8)  # one split of four waves
    assert lib.dpc_attention_grad_workspace_bytes(2, 3, 4) == 96
    assert lib.dpc_attention_state_bytes(2, 3, 4, 16, nat.DPC_BF16) == 256 + 24 * 16
    assert lib.dpc_attention_state_bytes(2, 3, 4, 16, nat.DPC_F32) == 256 + 96
