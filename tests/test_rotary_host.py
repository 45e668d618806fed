"""What a Rotary holds and which scalings it takes (no GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from tritonkv_amd import rotary as ro


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_rotary_keeps_frequencies_of_its_own(dtype):
    """Those of a tensor that is changed later stay what its turns say."""
    w = torch.tensor([1.0, 0.25, 0.01], dtype=dtype)
    rot = ro.Rotary(inv_freq=w)
    before = rot.inv_freq.clone()
    w.mul_(2)
    assert torch.equal(rot.inv_freq, before) and torch.equal(rot.turns, ro._turns(before))


LLAMA3 = dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
YARN = dict(factor=16.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("kind,rest", [("linear", dict(factor=4.0)), ("ntk", dict(factor=4.0)), ("llama3", LLAMA3),
                                       ("yarn", YARN)])
def test_a_scaling_may_name_its_type_as_models_do(kind, rest):
    want = ro.rotary_frequencies(64, 1e4, dict(type=kind, **rest))
    assert ro.rotary_frequencies(64, 1e4, dict(rope_type=kind, **rest)) == want
    assert ro.rotary_frequencies(64, 1e4, dict(rope_type=kind, type=kind, **rest)) == want
    with pytest.raises(ValueError, match="type"):
        ro.rotary_frequencies(64, 1e4, dict(rope_type=kind, type="other", **rest))
    for missing in ({}, dict(type=None), dict(rope_type="other")):
        with pytest.raises(ValueError, match="type"):
            ro.rotary_frequencies(64, 1e4, dict(**missing, **rest))
    with pytest.raises(ValueError, match=f"'{kind}'.*'factor'"):
        ro.rotary_frequencies(64, 1e4, dict(rope_type=kind))


@pytest.mark.parametrize("scaling,name", [
    (dict(type="yarn", mscale=0.707, **YARN), "mscale"), (dict(type="yarn", truncate=False, **YARN), "truncate"),
    (dict(type="linear", factor=4.0, attention_factor=1.2), "attention_factor"),
    (dict(type="ntk", factor=4.0, beta_fast=32), "beta_fast"), (dict(type="llama3", mscale=1.0, **LLAMA3), "mscale"),
    (dict(type="yarn", long_factor=[1.0], **YARN), "long_factor")])
def test_entries_that_a_scaling_does_not_know_are_refused(scaling, name):
    """They would change the angles, and were passed over."""
    with pytest.raises(ValueError, match=name):
        ro.rotary_frequencies(64, 1e4, scaling)
    del scaling[name]
    ro.rotary_frequencies(64, 1e4, scaling)


def test_entries_that_a_scaling_knows_are_taken():
    ro.rotary_frequencies(64, 1e4, dict(type="linear", factor=4.0, original_max_position_embeddings=4096))
    f, a = ro.rotary_frequencies(64, 1e4, dict(type="yarn", beta_fast=16, beta_slow=2, attention_factor=1.0, **YARN))
    assert a == 1.0 and not any(math.isnan(w) for w in f)
