"""Frequencies of the position rotation (host code, no GPU)."""
from __future__ import annotations

import math

import pytest

from turbocider_b200 import cuda as tcc


def plain(d, theta):
    return [theta ** (-2 * i / d) for i in range(d // 2)]


@pytest.mark.parametrize("d", [2, 8, 64, 128])
def test_plain_and_linear(d):
    f, a = tcc.rope_freqs(d, 1e4)
    assert a == 1.0 and f.tolist() == pytest.approx(plain(d, 1e4), rel=1e-14)
    f, a = tcc.rope_freqs(d, 1e4, "linear", factor=4.0)
    assert a == 1.0 and f.tolist() == pytest.approx([x / 4 for x in plain(d, 1e4)], rel=1e-14)


def test_ntk_stretches_the_slowest_pair_by_the_factor():
    f, a = tcc.rope_freqs(128, 1e4, "ntk", factor=8.0)
    p = plain(128, 1e4)
    assert a == 1.0 and f[0] == 1.0 and float(f[-1]) == pytest.approx(p[-1] / 8, rel=1e-12)


@pytest.mark.parametrize("scaling", ["yarn", "bands"])
def test_ramps(scaling):
    d, theta, factor, length = 128, 1e6, 16.0, 32768.0
    f, a = tcc.rope_freqs(d, theta, scaling, factor=factor, trained_length=length, beta_fast=32.0, beta_slow=1.0)
    assert a == pytest.approx(0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0, rel=1e-6)
    low = max(math.floor(d * math.log(length / (32 * 2 * math.pi)) / (2 * math.log(theta))), 0)
    high = min(math.ceil(d * math.log(length / (2 * math.pi)) / (2 * math.log(theta))), d - 1)
    for i, (got, p) in enumerate(zip(f.tolist(), plain(d, theta))):
        if scaling == "yarn":
            keep = 1 - min(max((i - low) / (high - low), 0), 1)
        else:
            keep = min(max((length * p / (2 * math.pi) - 1) / 31, 0), 1)
        assert got == pytest.approx(p * keep + p / factor * (1 - keep), rel=1e-12)
    assert float(f[0]) == 1.0 and float(f[-1]) == pytest.approx(plain(d, theta)[-1] / factor, rel=1e-12)


@pytest.mark.parametrize("kw,match", [
    (dict(rotary_dim=0), "even"), (dict(rotary_dim=7), "even"), (dict(rotary_dim=8, theta=0.0), "theta"),
    (dict(rotary_dim=8, theta=math.inf), "theta"), (dict(rotary_dim=8, scaling="linear", factor=0.5), "factor"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0), "trained_length"), (dict(rotary_dim=8, scaling="x"), "unknown"),
    (dict(rotary_dim=2, scaling="ntk", factor=2.0), "above 2"),
    (dict(rotary_dim=8, scaling="bands", factor=2.0, trained_length=1.0, beta_fast=1.0, beta_slow=2.0), "beta")])
def test_refusals(kw, match):
    with pytest.raises(tcc.BackendError, match=match):
        tcc.rope_freqs(**kw)


def test_entry_points_refuse_null_arguments():
    lib = tcc.lib()
    assert lib.tc_cuda_qk_norm_rope(None, None, None, 0, 0, 0, 0, 0.0, None, None) == 1
    assert lib.tc_cuda_kv_append(None, None, None, None, None, None, 0, 0.0, None, None) == 1
    assert lib.tc_cuda_paged_attention(None, None, None, None, None) == 1
    assert lib.tc_cuda_last_error().decode() == "null argument"
