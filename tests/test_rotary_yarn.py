"""The factor that yarn scaling puts on cos and sin (no GPU needed)."""
import math

import pytest

from amass_kv_b200.rotary import Rotary

YARN = dict(type="yarn", factor=16.0, original_max_position=4096)


def test_factor():
    assert math.isclose(Rotary("cpu", rotary_dim=64, scaling=YARN).mscale,
                        0.1 * math.log(16) + 1)
    rot = Rotary("cpu", rotary_dim=64,
                 scaling=dict(YARN, attention_factor=None))
    assert math.isclose(rot.mscale, 0.1 * math.log(16) + 1)
    rot = Rotary("cpu", rotary_dim=64,
                 scaling=dict(YARN, attention_factor=0.75))
    assert rot.mscale == 0.75


@pytest.mark.parametrize("kw", [dict(mscale=0.707), dict(mscale=1.0),
                                dict(mscale=1.0, mscale_all_dim=1.0),
                                dict(mscale_all_dim=1.0)])
def test_arguments_of_the_factor_are_refused(kw):
    """Model configurations give these to a formula for the factor; taken for
    the factor itself they would turn out another embedding."""
    with pytest.raises(ValueError, match="attention_factor"):
        Rotary("cpu", rotary_dim=64, scaling=dict(YARN, **kw))


@pytest.mark.parametrize("m", [0.0, -1.0, float("nan"), float("inf")])
def test_factors_that_are_none(m):
    with pytest.raises(ValueError, match="attention_factor"):
        Rotary("cpu", rotary_dim=64, scaling=dict(YARN, attention_factor=m))
