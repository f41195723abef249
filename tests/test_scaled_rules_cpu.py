"""Into how many shares the attention over 8-bit rows cuts its walks, at the sizes that the rules' own notes speak of."""

import pytest

from llmoxide_b200 import kernels


@pytest.mark.parametrize("n_seqs, past, head_dim, want", [
    (64, 2048, 128, 1), (8, 2048, 128, 6), (64, 16001, 128, 4), (1, 32768, 128, 48), (1, 32768, 64, 48), (2, 32768, 128, 8),
    (4, 32768, 128, 8), (8, 32768, 128, 6), (2, 8192, 128, 8), (1, 200, 64, 1)])
def test_single_tokens(n_seqs, past, head_dim, want):
    assert kernels.scaled_decode_shares(n_seqs, 8, 4, past // 64 + 1, head_dim, 0) == want


def test_single_tokens_always_have_a_share_of_some_pages():
    for n_seqs in (1, 2, 3, 5, 8, 17, 64, 500):
        for heads, group in ((1, 1), (8, 4), (2, 16), (4, 9)):
            for pages in (1, 2, 5, 33, 192, 600):
                for head_dim in (64, 128, 256):
                    n = kernels.scaled_decode_shares(n_seqs, heads, group, pages, head_dim, 0)
                    assert 1 <= n <= 48 and (n == 1 or pages >= 4 * n)


@pytest.mark.parametrize("n_seqs, new, past, want", [(1, 33, 32735, 18), (1, 2048, 6144, 1), (1, 512, 8000, 2)])
def test_several_tokens(n_seqs, new, past, want):
    pages = (new + past + 63) // 64
    assert kernels.scaled_chunk_shares(n_seqs, 8, 4 * new, pages, True, n_seqs * new * 4096) == want


def test_only_those_that_ask_get_scales():
    """An entry whose own numbers are of 8 bits, as another kind of layer may keep them, is stored as it is."""
    import torch

    from llmoxide_b200.cache import Cache, PAGE
    from llmoxide_b200.cache.storage import KVNeed
    for dtype in (torch.int8, torch.float8_e4m3fn):
        plain = Cache([(KVNeed(2, 32, dtype=dtype), None)], 1, 2 * PAGE, torch.float32, torch.device("cpu"))
        assert plain.bytes() == 2 * 2 * PAGE * 2 * 32 and plain.view(0).k_scale is None and plain.view(0).v_scale is None
        rows = Cache([(KVNeed(2, 32, dtype=dtype, scaled=True), None)], 1, 2 * PAGE, torch.float32, torch.device("cpu"))
        assert rows.bytes() == 2 * 2 * PAGE * 2 * (32 + 4) and rows.view(0).k_scale.shape == rows.view(0).k.shape[:3]
        rows.wipe(), plain.wipe()
