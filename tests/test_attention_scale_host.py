"""Scales whose product with log2(e), the kernels' multiplier of a score, passes fp32's range are
refused (nothing is launched): it would be infinite, and 0 * infinity makes NaN of finite scores."""
import ctypes

import numpy as np
import pytest

from test_attention_host import ATTENTION, dll, error  # noqa: F401  (dll is a fixture)


@pytest.mark.parametrize("scale", [2.4e38, 2.9e38, 3e38, 3.4e38])
def test_scales_beyond_the_multiplier_are_refused(pkg, dll, scale):  # noqa: F811
    change = {"scale": ctypes.c_float(scale)}
    assert dll.w4a16_kv_attention(*{**ATTENTION, **change}.values()) == 1 and "scale" in error(pkg)


def test_the_layers_limit_is_below_the_librarys():
    from test_attention_host import attn
    assert np.isfinite(np.float32(attn.MAX_SCALE) * np.float32(1.44269504))
