"""Frequency factors at the ends of their arguments."""
import math

import numpy as np
import pytest

from webgpu_amd.rope import llama3_factors, yarn_factors


@pytest.mark.parametrize("theta", [1.0, 0.5, 0.0, -1e4, math.inf, math.nan])
def test_yarn_factors_refuse_a_base_without_a_ramp(theta):
    """With a base of 1 all pairs turn alike, and below it later ones turn faster: the pair that turns a given number of
    times, dim ln(original / (2 pi turns)) / (2 ln theta), is none or lies on the wrong side."""
    with pytest.raises(ValueError):
        yarn_factors(64, theta, 2.0, 4096)


@pytest.mark.parametrize("theta", [0.0, -1e4, math.inf, math.nan])
def test_llama3_factors_refuse_a_base_that_is_no_positive_number(theta):
    with pytest.raises(ValueError):
        llama3_factors(64, theta, 8.0, 1.0, 4.0, 8192)


def test_factors_of_bases_near_one():
    f, m = yarn_factors(64, 1.001, 2.0, 4096)  # every pair turns hundreds of times
    assert np.all(f == 1) and m == 0.1 * math.log(2) + 1
    assert np.all(llama3_factors(64, 1.0, 8.0, 1.0, 4.0, 8192) == 1)
