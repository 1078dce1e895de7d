"""Block tables that reach 2^31 tokens: the kernels count keys in 32 bits and round them up to tiles,
so the C ABI refuses tables whose last tokens those sums could pass (nothing is launched)."""
import pytest

from test_attention_host import ATTENTION, STEP, dll, error  # noqa: F401  (dll is a fixture)

REACH = 2 ** 31 - 1 - 2 ** 19


@pytest.mark.parametrize("block", [16, 64, 256])
def test_reach_is_bounded(pkg, dll, block):  # noqa: F811
    """The largest table below the limit is taken, the next one refused by every call that reads it."""
    width = REACH // block
    assert dll.w4a16_kv_attention_workspace(1, 1, 1, 1, 64, block, width, 1) > 0
    assert dll.w4a16_kv_attention_workspace(1, 1, 1, 1, 64, block, width + 1, 1) == 0
    for over in (width + 1, 2 ** 31 // block, 2 ** 31 - 1):
        change = dict(width=over, stride=over, block=block)
        assert dll.w4a16_kv_step(*{**STEP, **change}.values()) == 2 and "reach" in error(pkg)
        assert dll.w4a16_kv_attention(*{**ATTENTION, **change}.values()) == 2 and "reach" in error(pkg)


def test_sums_behind_the_reach_stay_below_2_31():
    """What the kernels add to a key count or position: a unit of 128 keys with two more in flight, a
    tile of 64 keys with three more, and a step's 2^18 rows rounded up to a block of 256."""
    for more in (128 - 1 + 2 * 128, 64 + 3 * 64 + 12, 2 ** 18 + 255):
        assert REACH + more < 2 ** 31
