"""Arguments of the paged front end that have no meaning: numbers beyond their fields, calls of a closed cache."""
import numpy as np
import pytest
import torch

from helpers import pkg


def test_numbers_beyond_their_fields_are_refused():
    P = pkg()
    for kw in (dict(layers=(1 << 32) + 1), dict(layers=-1), dict(page_rows=(1 << 32) + 16), dict(max_sequences=(1 << 32) + 1),
               dict(num_kv_heads=(1 << 64) + 2), dict(head_dim=-64), dict(page_count=-1), dict(max_table_pages=-1), dict(device=1 << 32),
               dict(storage_bytes=-1, storage_ptr=1 << 20)):
        with pytest.raises(ValueError, match="out of range"):
            P.PagedKv(**{**dict(layers=1, num_kv_heads=2, head_dim=64, page_count=4), **kw})
    with pytest.raises(ValueError, match="out of range"):
        P.PagedKv.bytes_for((1 << 32) + 1, 2, 64, page_count=4)
    for rotary_dim, device in (((1 << 32) + 64, 0), (-64, 0), (64, 1 << 32)):
        with pytest.raises(ValueError, match="out of range"):
            P.Rotation(rotary_dim, device=device)
    for heads in (-1, (1 << 32) + 2):
        with pytest.raises(ValueError, match="out of range"):
            P.Rows(1 << 20, "f16", heads)
    assert P.Rows(0, "f16", 0).raw.heads == 0  # (the library's to refuse)
    assert P.PagedKv.bytes_for(3, 2, 64, page_count=4, page_rows=32) == 3 * 4 * 2 * 2 * 32 * 64 * 2


@pytest.mark.gpu
def test_a_closed_cache_says_so():
    P = pkg()
    cache = P.PagedKv(1, 1, 64, page_count=4, page_rows=16)
    x = P.Rows.of(torch.ones(1, 1, 64, dtype=torch.float16, device="cuda"))
    cache.set_batch([(5, 1)], [np.array([1], np.uint32)])
    cache.close()
    for call in (lambda: cache.set_batch([(5, 1)], [[1]]), lambda: cache.set_batch([(5, 1)], [np.array([1], np.uint32)]),
                 lambda: cache.append_device(0, x, x), lambda: cache.attention_device(0, x, x),
                 lambda: cache.attention_step_device(0, x, x, x, x), lambda: cache.set_stream(0), cache.synchronize):
        with pytest.raises(ValueError, match="closed"):
            call()
    assert cache.storage_ptr() == 0
    cache.close()
