"""A head's configuration is checked where its plan is made."""
import pytest

from plow_amd import layer


@pytest.mark.parametrize("bad", [{"enc": "int4"}, {"enc": "fp8blk"}, {"scale": 0.0}, {"scale": -1.0}, {"n_alt": 65}])
def test_heads_that_cannot_be_served(bad):
    """An encoding that the head has no product for must not run as bf16, a factor of 0 not as 1."""
    with pytest.raises(ValueError):
        layer.plan_head(layer.HeadConfig("h", T=2, H=256, V=100, **bad))


def test_heads_that_can():
    for good in ({}, {"enc": "int4g"}, {"scale": 0.5}, {"n_alt": 64}):
        assert len(layer.plan_head(layer.HeadConfig("h", T=2, H=256, V=100, **good)).insts) == 3
