"""What spanqr_linear_cross_entropy_workspace takes, seen from outside, without a GPU."""
import pytest

from spanqr_amd import _lib

BF16 = 1


def need(N, H, V, grads, most=4 << 30):
    return _lib.lib().spanqr_linear_cross_entropy_workspace(BF16, N, H, V, grads, most)


@pytest.mark.parametrize("H,V", [(64, 1000), (8, 512), (8, 16)])
def test_tokens_of_one_launch(H, V):
    """A piece of the tokens is one launch with a workgroup a token, and a launch has fewer than 2^32 threads: whatever the
    workspace holds, 2^23 tokens are taken at a time. Behind those only the tokens' losses grow."""
    most = 1 << 23
    one = need(most, H, V, 0)
    for N in (1 << 24, 1 << 25, (1 << 24) + 77):
        assert 0 < need(N, H, V, 0) <= one + 4 * (N - most) + 256, N


def test_tiles_of_one_launch():
    """the same for the products' tiles, of 2^16 logits at most"""
    huge = 1 << 45
    V = 1 << 22
    one = need((1 << 18) - 256, 8, V, 0, huge)      # 2^24 tiles but 2^14
    N = 1 << 21
    assert 0 < need(N, 8, V, 0, huge) <= one + 4 * N


def test_tokens_are_counted_in_int():
    assert need((1 << 31) - 1, 8, 16, 0) > 0
    assert need(1 << 31, 8, 16, 0) == -1   # SPANQR_EINVAL
