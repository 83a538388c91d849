"""Sizes and addresses that the hybrid layers' entry points have to refuse or answer without any device work."""
import pytest

from genllm_amd import _lib

INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("shape", [
    (1, 100, 1, 1, 64, 8), (1, 100, 1, 1, 64, 15), (1, 100, 1, 1, 8, 64), (1, 100, 1, 1, 96, 128), (1, 100, 1, 1, 128, 256),
    (INT_MAX, INT_MAX, 1, INT_MAX, INT_MAX, INT_MAX), (INT_MAX, 100, 1, INT_MAX, 128, 128), (1 << 16, 100, 8, 16, 64, 64),
    (1, (1 << 30) + 1, 1, 1, 64, 64), (0, 100, 1, 1, 64, 64), (1, 0, 1, 1, 64, 64), (1, 100, 0, 1, 64, 64), (1, 100, 1, -1, 64, 64)])
def test_workspace_of_sizes_that_are_not_served(shape):
    """None, for any sizes at all: a caller asks before the call itself refuses them."""
    assert _lib.lib().genllm_gated_delta_workspace_bytes(*shape) == 0


def test_workspace_at_the_limits():
    f = _lib.lib().genllm_gated_delta_workspace_bytes
    assert f(1, 12, 16, 32, 128, 128) == 0 and f(1, 1 << 30, 16, 32, 128, 128) > 0
    assert 0 < f(1 << 15, 64, 16, 16, 64, 64) < 1 << 30 and f(1, 64, 1, 1 << 19, 64, 64) > 0
