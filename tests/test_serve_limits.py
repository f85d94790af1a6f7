"""CPU: sizes at the ends of the serving operators' 32- and 64-bit arithmetic (include/popcorn_serve.h)."""
import ctypes

import pytest

import popcorn_b200 as pc

FAKE = 0x1000  # never dereferenced


def _cache(page_size=16, dim=64):
    return pc.KvCacheStruct(FAKE, FAKE, FAKE, FAKE, 4, 2, page_size, dim)


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
def test_tables_of_nearly_2_to_31_tokens_are_refused(lib, page_size):
    """A step of the kernel for prompts ends up to 127 tokens behind the last one, and the next one 128 further: tables
    whose tokens leave no room for that below 2^31 are refused."""
    c = _cache(page_size)
    for spare in (0, 64, 65, 128, 192, 255):
        width = ((1 << 31) - 1 - spare) // page_size
        if width * page_size <= (1 << 31) - 1 - 256:
            continue
        assert lib.popcornKvAttention(FAKE, None, FAKE, 256, 64, pc.TYPE_F16, ctypes.byref(c), FAKE, width, FAKE, FAKE, 1, 100,
                                      100, 4, 1, 0, 0.1, None, 0, None) == pc.POPCORN_ERROR_INVALID_VALUE, width


@pytest.mark.parametrize("kind", [pc.TYPE_F32, pc.TYPE_F16, pc.TYPE_BF16])
@pytest.mark.parametrize("group", [1, 2, 4, 16])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_max_tokens_past_all_tokens_is_all_tokens(lib, kind, group, dim):
    """One sequence cannot have more queries than there are: larger bounds, up to the largest int64, take the same
    kernels, and so the same workspace."""
    c = _cache(dim=dim)
    size = lambda seqs, tokens, most: lib.popcornKvAttentionWorkspace(ctypes.byref(c), kind, seqs, tokens, most, 2 * group)  # noqa: E731
    for seqs, tokens in ((1, 1), (1, 300), (3, 40), (7, 5000)):
        want = size(seqs, tokens, tokens)
        assert want > 0
        for most in (tokens + 1, 1 << 31, 1 << 60, 1 << 62, (1 << 63) - 1):
            assert size(seqs, tokens, most) == want, (seqs, tokens, most)
