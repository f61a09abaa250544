"""CPU checks of what the head's backward asks for over long batches, where a piece of the vocabulary shrinks no
further."""
import pytest

from pragnosia_amd._lib import lm_lib

LIMIT, WORDS = 144 << 20, 1024  # bytes of a piece's dl, and the least words of one


@pytest.mark.parametrize("n,V,d", [(16384, 32768, 768), (73728, 32768, 768), (131072, 32768, 768), (131073, 1003, 128),
                                   (1 << 20, 8192, 768), (1 << 22, 512, 64), (1 << 24, 24, 8)])
def test_workspace_of_long_batches(n, V, d):
    """dl: 144 MB, or 2 KB a token, and a tile more (a quarter); dh's fp32 sums where there are several pieces; dW's by
    ranges of tokens, 64 at most; 32 bytes a token of row data."""
    dl = 1.25 * max(LIMIT, 2 * WORDS * (n + 255))
    words = max(WORDS, LIMIT // (2 * n)) + 256
    most = dl + 4 * n * d + 64 * 4 * min(words, V) * d + 32 * n + 4096
    got = lm_lib().pragnosia_head_bwd_workspace_bytes(n, V, d)
    assert 0 < got <= most
    assert got >= 32 * n
