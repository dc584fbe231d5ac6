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


def p_bytes(N, V):
    return 2 * N * ((V + 63) // 64 * 64)


@pytest.mark.parametrize("N,H,V", [(65536, 5120, 32000), (8192, 5120, 1000), (16384, 5120, 128000), (300, 4096, 1000)])
def test_only_what_is_used(N, H, V):
    """beside the exponentials and their statistics (16 bytes for 64 columns at most) nothing of their size that no launch touches"""
    rest = N * (16 * (V // 64 + 1) + 16) + 4 * 128 * H + 4096
    whole = need(N, H, V, 3, 1 << 45)
    assert p_bytes(N, V) <= whole <= p_bytes(N, V) + rest + (4 * 16384 * H if N == 300 else 0)


def test_pieces_take_no_more_than_the_whole():
    """dW over pieces has sums in fp32 that all tokens at once do without"""
    for N in (257, 300, 500, 900, 4000):
        for H, V in ((4096, 1000), (1024, 50257), (5120, 512)):
            for most in (0, 10 << 20, 100 << 20):
                assert need(N, H, V, 3, most) <= max(most, need(N, H, V, 3, 1 << 45)), (N, H, V, most)


@pytest.mark.parametrize("grads", [0, 1, 2, 3])
def test_what_fits_for_some_fits_for_fewer(grads):
    """a workspace for N tokens, whole or in pieces, is enough for fewer (all of the workspace but the sums of dx's parts,
    which adapt to it, is what the least query gives)"""
    for H, V in ((768, 32000), (64, 100), (5120, 1000), (1000, 50257)):
        last = 0
        for N in (1, 2, 16, 17, 31, 32, 33, 63, 64, 65, 100, 256, 257, 512, 1000, 4096, 10000, 40000):
            least = need(N, H, V, grads, 1 << 45)
            if not grads & 1:
                assert least >= last, (H, V, N)
            last = least
            for most in (64 << 20, 1 << 30):
                got = need(N, H, V, grads, most)
                # the same call again, with what the query gave as its bound, needs no more
                assert need(N, H, V, grads, got) <= got, (H, V, N, most)
