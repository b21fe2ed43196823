"""What the operators of drafted tokens refuse beside shapes and pointers (no GPU needed)."""
import pytest
import torch

import oasr_b200 as ob
from oasr_b200 import _lib
from tests.test_drafts_args import commit, refused


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


@pytest.mark.parametrize("second,first", [((1 << 20, 2, 1, 256), (1 << 20, 2, 1, 256)), ((1 << 20, 1, 2, 64), ((1 << 20) + 16384 - 64, 1, 1, 64)), (((1 << 20) + 32768, 1, 1, 256), (1 << 20, 2, 1, 256)),
                                          ((1 << 20, 1, 1, 256), ((1 << 20) + 32752, 1, 1, 16))])
def test_commit_drafts_refuses_pools_that_share_memory(first, second):
    """8 pages of 16 rows: a pool twice, a layer of another, and one row of overlap."""
    for pools in ((first, second), (second, first), (second, (1 << 30, 3, 1, 16), first)):
        refused("commit_drafts", commit(n=len(pools), pools=(_lib.DraftPool * len(pools))(*[_lib.DraftPool(*p) for p in pools])), _lib.ERR_INVALID)


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (2, 0, 1), (0, 2, 1)])
def test_commit_drafts_takes_layers_of_one_allocation(order):
    """Side by side is not shared: the pools are not what this call is refused for."""
    pools = (_lib.DraftPool * 4)(*[_lib.DraftPool((1 << 20) + i * 8 * 16 * 256, 1, 1, 256) for i in order], _lib.DraftPool(1 << 30, 0, 1, 16))
    refused("commit_drafts", commit(n=4, pools=pools), _lib.ERR_INVALID)
    assert "bad pool" in _lib.last_error()
    pools[3] = _lib.DraftPool((1 << 20) + 8 * 16 * 256 * 3 - 1, 1, 1, 1)
    refused("commit_drafts", commit(n=4, pools=pools), _lib.ERR_INVALID)
    assert f"pools {order.index(2)} and 3 share memory" in _lib.last_error()


def test_a_refused_device_leaves_no_workspace_size_behind(monkeypatch):
    """The size is asked for on the current device: a call that is refused for another one must not keep an answer under that one's name."""
    from oasr_b200 import attention

    def refuse(t):
        raise RuntimeError("not the current device")
    monkeypatch.setattr(attention, "_one_device", lambda *t: None)
    monkeypatch.setattr(attention, "_stream", refuse)
    before = attention._tree_workspace.cache_info().currsize
    pool, i32 = torch.zeros(4, 16, 3, 64).bfloat16(), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="not the current device"):
        ob.fmha_tree(torch.zeros(1, 21, 11, 64).bfloat16(), pool, pool, softmax_scale=1.0, block_table=i32, cache_seqlens=i32[0, :1])
    assert attention._tree_workspace.cache_info().currsize == before
