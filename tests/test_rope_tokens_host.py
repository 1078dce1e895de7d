"""The most tokens that a norm-and-rotation call takes, on the CPU (nothing is launched)."""
import ctypes

import pytest

P = 1 << 20  # a pointer that no refused call follows
ROPE = dict(q=P, qt=4096, qh=128, k=P, kt=4096, kh=128, positions=P, table=P, table_rows=64, rotary=128, qw=P, kw=P,
            eps=ctypes.c_float(1e-6), q_out=P, k_out=P, T=3, H=32, KV=8, D=128, stream=None)
APPEND = dict(q=P, qt=4096, qh=128, k=P, kt=4096, kh=128, v=P, vt=4096, vh=128, cache=P, slots=P, positions=P, table=P,
              table_rows=64, rotary=128, qw=None, kw=None, eps=ctypes.c_float(1e-6), q_out=P, k_out=None, T=3, H=32, KV=8, D=128,
              blocks=4, block=16, stream=None)


@pytest.mark.parametrize("tokens", [(1 << 26) - 31, 1 << 26, 1 << 28, 1 << 30])
def test_more_tokens_than_a_launch_has_threads_for(pkg, tokens):
    """64 threads a token in workgroups of 256, 8 of them at a time, and a launch has fewer than 2^32: more tokens are
    refused by name, not by the launch."""
    assert 256 * ((-(-tokens // 4) + 7) // 8 * 8) >= 2 ** 32
    dll = pkg.lib().dll
    assert dll.w4a16_qk_norm_rope(*{**ROPE, "T": tokens}.values()) == 2 and "too many" in pkg.lib().last_error()
    assert dll.w4a16_kv_append(*{**APPEND, "T": tokens}.values()) == 2 and "too many" in pkg.lib().last_error()


def test_the_most_tokens(pkg):
    tokens = (1 << 26) - 32
    assert 256 * ((-(-tokens // 4) + 7) // 8 * 8) < 2 ** 32
    assert pkg.lib().dll.w4a16_qk_norm_rope(*{**ROPE, "T": tokens, "q": None}.values()) == 1 and "null" in pkg.lib().last_error()
