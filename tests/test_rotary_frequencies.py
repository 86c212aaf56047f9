"""Rotary frequencies and their scalings (CPU), and the entry points' own refusals."""

from __future__ import annotations

import math

import pytest
import torch

from opake_amd import _native as nat
from opake_amd.exceptions import ConfigurationError, InputTypeError
from opake_amd.rotary import rotary_frequencies


def _plain(dims, base):
    return [base ** (-2.0 * i / dims) for i in range(dims // 2)]


def test_plain_and_linear():
    f, a = rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and a == 1.0
    torch.testing.assert_close(f, torch.tensor(_plain(64, 10000.0), dtype=torch.float64))
    g, a = rotary_frequencies(64, 10000.0, scaling=dict(kind="linear", factor=4))
    torch.testing.assert_close(g, f / 4)
    assert a == 1.0


def test_ntk_keeps_the_highest_and_divides_the_lowest():
    f, _ = rotary_frequencies(128, 500000.0)
    g, _ = rotary_frequencies(128, 500000.0, scaling=dict(kind="ntk", factor=8.0))
    assert g[0] == f[0] == 1.0
    assert math.isclose(g[-1].item() * 8.0, f[-1].item(), rel_tol=1e-12)
    assert bool((g <= f).all())


@pytest.mark.parametrize("kind", ["bands", "ramp"])
def test_bands(kind):
    opts = dict(kind=kind, factor=8.0, low=1.0, high=4.0, original=8192)
    f, _ = rotary_frequencies(128, 500000.0)
    g, a = rotary_frequencies(128, 500000.0, scaling=opts)
    turns = 8192 * f / (2 * math.pi)
    torch.testing.assert_close(g[turns > 8.0], f[turns > 8.0])
    torch.testing.assert_close(g[turns < 0.5], f[turns < 0.5] / 8.0)
    between = (turns < 3.9) & (turns > 1.1)
    assert between.any() and bool((g[between] < f[between]).all())
    assert bool((g[between] > f[between] / 8.0).all())
    assert math.isclose(a, 1.0 if kind == "bands" else 0.1 * math.log(8.0) + 1.0)
    if kind == "bands":
        mix = (turns[between] - 1.0) / 3.0
        torch.testing.assert_close(g[between], f[between] * (mix + (1 - mix) / 8.0))
    same, _ = rotary_frequencies(128, 500000.0, scaling=dict(opts, factor=1.0))
    torch.testing.assert_close(same, f)


def test_refusals():
    for kw in (dict(dims=0), dict(dims=3), dict(dims=4096), dict(dims=4, base=1.0),
               dict(dims=4, base=math.inf), dict(dims=4, scaling={}),
               dict(dims=4, scaling=dict(kind="cubic", factor=2.0)),
               dict(dims=4, scaling=dict(kind="linear")),
               dict(dims=4, scaling=dict(kind="linear", factor=0.5)),
               dict(dims=4, scaling=dict(kind="linear", factor=2.0, low=1.0)),
               dict(dims=2, scaling=dict(kind="ntk", factor=2.0)),
               dict(dims=4, scaling=dict(kind="bands", factor=2.0, low=4.0, high=1.0,
                                         original=10))):
        with pytest.raises(ConfigurationError):
            rotary_frequencies(**kw)
    for kw in (dict(dims=4.0), dict(dims=True), dict(dims=4, base="a"),
               dict(dims=4, scaling=dict(kind="linear", factor="2"))):
        with pytest.raises(InputTypeError):
            rotary_frequencies(**kw)


def test_entry_points_refuse_without_a_device():
    if not nat.LIB_PATH.exists():
        pytest.skip("native library not built")
    lib = nat.load()
    st = (nat._c_i64 * 6)(64, 16, 4, 0, 0, 0)

    def rotary(B=1, T=1, H=4, KV=0, h=4, code=nat.DPC_F32, pairs=2, q=16, out=32, k=0):
        return lib.dpc_rotary(q, k, B, T, H, KV, h, code, st, 0, 0, 0, 64, pairs, 0, 1.0, 0, out,
                              0, 0)

    assert rotary(B=0) == rotary(T=0) == nat.DPC_OK  # nothing to do
    for bad in (dict(h=0), dict(h=4096), dict(pairs=3), dict(pairs=-1), dict(H=0), dict(B=-1),
                dict(code=nat.DPC_F16), dict(q=0), dict(out=0), dict(KV=1), dict(H=1 << 22)):
        assert rotary(**bad) == nat.DPC_EINVAL, bad
