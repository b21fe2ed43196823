"""What the operators of drafted tokens refuse beside shapes and pointers (no GPU needed)."""
import pytest
import torch

import oasr_b200 as ob


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.bool, torch.uint32])
@pytest.mark.parametrize("name", ["path", "counts", "offset", "block_table"])
def test_commit_drafts_takes_whole_numbers_only(dtype, name):
    """Rows are moved in place: what is not a whole number is refused, and not rounded to one."""
    index = dict(path=torch.zeros(2, 3, dtype=torch.int32), counts=torch.zeros(2, dtype=torch.int64), offset=torch.zeros(2, dtype=torch.int32), block_table=torch.zeros(2, 1, dtype=torch.int32))
    bad = index | {name: index[name].to(dtype)}
    with pytest.raises(ValueError, match=f"{name} must be whole numbers"):
        ob.commit_drafts((torch.zeros(4, 16, 2, 8),), **bad)
    with pytest.raises(ValueError, match=f"{name} must be whole numbers"):
        ob.commit_drafts_q4(ob.PagedKVCacheQ4.empty_pools(4, 1, 16, 64, device="cpu"), **bad)


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_commit_drafts_takes_all_of_them(dtype):
    """(up to the check that everything is on a GPU)"""
    i = torch.zeros(2, 3, dtype=dtype)
    with pytest.raises(RuntimeError, match="CUDA"):
        ob.commit_drafts((torch.zeros(4, 16, 2, 8),), i, i[:, 0], i, i[:, 0])
