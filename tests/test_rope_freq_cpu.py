"""Rotary frequencies: what has no ramp is refused."""
import pytest

from halftone_quantizedkvcache_b200 import kernels


@pytest.mark.parametrize("bad", [dict(theta=1.0), dict(theta=0.5), dict(beta_fast=0.0), dict(beta_slow=-1.0),
                                 dict(beta_slow=0.0)])
def test_yarn_without_a_ramp(bad):
    """The ramp's ends are logarithms to the base theta of lengths over beta."""
    with pytest.raises(ValueError):
        kernels.rope_inv_freq(64, scaling="yarn", factor=2.0, original_len=4096, device="cpu", **bad)


def test_other_scalings_do_not_need_one():
    for scaling in (None, "linear"):
        f, m = kernels.rope_inv_freq(64, 1.0, scaling=scaling, device="cpu")
        assert m == 1.0 and (f == 1.0).all()
