"""The rotary table's scalings with all the keys that model configurations
give them, against their definitions in plain Python."""

import math

import pytest
import torch

from torch_mcpu_b200 import ops


def turn(reach, part, base, frequencies, amplitude=1.0):
    angle = [[p * f for f in frequencies] for p in range(reach)]
    a = torch.tensor(angle, dtype=torch.float64)
    return torch.cat([a.cos() * amplitude, a.sin() * amplitude], 1)


def inverse(part, base):
    return [base ** (-2 * i / part) for i in range(part // 2)]


def yarn(part, base, factor, original, fast=32.0, slow=1.0, whole=True):
    """Dimensions that turn more than `fast` times over the original length keep their frequency, those below `slow` times are
    stretched by the factor, blended linearly between; the ends are whole dimensions unless `whole` is false."""
    def dimension(turns):
        return part * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = dimension(fast), dimension(slow)
    if whole:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, part - 1)
    out = []
    for i, f in enumerate(inverse(part, base)):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(f / factor * ramp + f * (1 - ramp))
    return out


def m(factor, mscale):
    return 0.1 * mscale * math.log(factor) + 1.0


YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
FORMS = [  # extra keys, amplitude, ends of the ramp
    ({}, m(40, 1), {}),
    ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0, {}),  # DeepSeek-V3
    ({"mscale": 0.707, "mscale_all_dim": 0.707, "beta_fast": 32, "beta_slow": 1}, 1.0, {}),  # DeepSeek-V2
    ({"mscale": 1.0, "mscale_all_dim": 0.5}, m(40, 1) / m(40, 0.5), {}),
    ({"mscale": 1.3, "mscale_all_dim": 0.0}, m(40, 1.3), {}),
    ({"attention_factor": 0.9}, 0.9, {}),
    ({"attention_factor": 0.9, "mscale": 1.0, "mscale_all_dim": 1.0}, 0.9, {}),
    ({"attention_factor": None, "mscale": None, "mscale_all_dim": None}, m(40, 1), {}),
    ({"truncate": False}, m(40, 1), {"whole": False}),
    ({"truncate": True}, m(40, 1), {}),
    ({"beta_fast": 20, "beta_slow": 2, "truncate": False, "mscale": 1.0, "mscale_all_dim": 1.0}, 1.0, {"fast": 20, "slow": 2, "whole": False}),
]


@pytest.mark.parametrize("more,amplitude,ends", FORMS)
@pytest.mark.parametrize("named", ["rope_type", "type"])
def test_yarn(more, amplitude, ends, named):
    part, base, reach = 64, 10000.0, 300
    scaling = {**YARN, **more}
    scaling[named] = scaling.pop("rope_type")
    got = ops.rotary_cos_sin_cache(reach, part, base, scaling).double()
    want = turn(reach, part, base, yarn(part, base, 40.0, 4096.0, **ends), amplitude)
    assert ((got - want).abs() <= 2.0 ** -24 * 1.5 + 1e-11).all()  # one rounding to fp32, of values up to 1.5


def test_yarn_that_does_not_stretch():
    scaling = {"type": "yarn", "factor": 1.0, "original_max_position_embeddings": 4096, "mscale": 0.7, "mscale_all_dim": 0.2}
    got = ops.rotary_cos_sin_cache(64, 64, 10000.0, scaling).double()
    assert ((got - turn(64, 64, 10000.0, inverse(64, 10000.0))).abs() <= 2.0 ** -24 + 1e-11).all()


def test_keys_that_say_what_the_call_says():
    part, base = 64, 10000.0
    plain = ops.rotary_cos_sin_cache(64, part, base)
    assert torch.equal(plain, ops.rotary_cos_sin_cache(64, part, base, {"rope_type": "default", "rope_theta": 10000.0}))
    assert torch.equal(plain, ops.rotary_cos_sin_cache(64, part, base, {"rope_type": "default", "rope_theta": 10000, "partial_rotary_factor": 0.5}))
    linear = {"type": "linear", "factor": 2.0}
    more = {**linear, "original_max_position_embeddings": 2048, "rope_theta": 10000.0, "attention_factor": None}
    assert torch.equal(ops.rotary_cos_sin_cache(64, part, base, linear), ops.rotary_cos_sin_cache(64, part, base, more))


@pytest.mark.parametrize("scaling,why", [
    ({**YARN, "attn_factor": 1.2}, "attn_factor"), ({**YARN, "extrapolation_factor": 0.5}, "extrapolation_factor"),
    ({**YARN, "mscale": 1.0}, "mscale_all_dim"), ({**YARN, "mscale_all_dim": 1.0}, "mscale"),
    ({**YARN, "low_freq_factor": 1.0}, "low_freq_factor"), ({"rope_type": "linear", "factor": 2.0, "beta_fast": 3}, "beta_fast"),
    ({"rope_type": "linear", "factor": 2.0, "rope_theta": 500000.0}, "rope_theta"),
    ({"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 32, "alpha": 3.0}, "alpha"),
    ({"rope_type": "linear", "type": "yarn", "factor": 2.0}, "type"), ({"rope_type": "default", "mrope_section": [16, 24, 24]}, "mrope_section")])
def test_keys_that_are_not_understood_are_refused(scaling, why):
    with pytest.raises(RuntimeError, match=why):
        ops.rotary_cos_sin_cache(64, 64, 10000.0, scaling)
