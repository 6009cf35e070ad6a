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


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16])
def test_rows_off_a_16_byte_boundary_are_refused(dtype):
    """What tree_mla asks of its cache before a launch (the row kernels read 16 bytes at a time)."""
    flat = torch.zeros(656 * 4 + 16, dtype=dtype)
    for off in range(0, 17):
        rows = flat[off:off + 656 * 4].view(4, 656)
        if rows.data_ptr() % 16:
            with pytest.raises(ValueError, match="16-byte boundary"):
                spec._aligned("tree_mla: kv", rows)
        else:
            spec._aligned("tree_mla: kv", rows)
