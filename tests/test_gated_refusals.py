"""Derivatives that ``gated_linear`` does not have are refused before any launch (CPU: the
launch is replaced)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from opake_amd import _native as nat
from opake_amd import gated


@pytest.fixture()
def launches(monkeypatch):
    if not nat.LIB_PATH.exists():
        pytest.skip("native library not built")
    made = []
    monkeypatch.setattr(nat, "require_device", lambda *tensors: None)
    monkeypatch.setattr(nat, "call_on", lambda dev, name, *args: made.append(name))
    return made


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("leaf", [True, False])
def test_tangents(launches, grad, leaf):
    x, w = torch.ones(3, 16), torch.ones(8, 16, requires_grad=leaf)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        for a, b in ((fwd.make_dual(x, x), w), (x, fwd.make_dual(w, w.detach()))):
            with pytest.raises(NotImplementedError):
                gated.gated_linear(a, b)
        del launches[:]
        gated.gated_linear(x, w)  # none here: as outside
    assert launches == ["dpc_gated_linear"]


def test_function_transforms(launches):
    x, w = torch.ones(2, 3, 16), torch.ones(8, 16)
    for f in (torch.func.vmap(lambda t: gated.gated_linear(t, w)),
              torch.func.grad(lambda t: gated.gated_linear(t, w).sum()),
              lambda t: torch.func.jvp(lambda u: gated.gated_linear(u, w), (t,), (t,))):
        with pytest.raises(RuntimeError):  # (NotImplementedError is one)
            f(x)
    assert not launches
