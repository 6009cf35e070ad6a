"""Tree speculation without a GPU: refusals, rules and failures at the edges of the operators' arguments."""
import pytest
import torch

from carbon_b200.ops import spec


def test_cache_rows_refuse_an_address_between_words():
    """The kernel moves rows in words of 4 bytes at least: a contiguous view that starts inside one is refused."""
    flat = torch.zeros(16 * 8 + 4, dtype=torch.uint8)
    base = flat.data_ptr()
    for off in range(4):
        view = flat[off:off + 128].view(16, 8)
        assert view.is_contiguous()
        if (base + off) % 4:
            with pytest.raises(ValueError, match="4-byte boundary"):
                spec.CacheRows([view])
            with pytest.raises(ValueError, match="4-byte boundary"):
                spec.CacheRows([torch.zeros(16, 4), view])
        else:
            spec.CacheRows([view])
