"""Accepted rows moved where pools are one, or lie together."""
import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import pages
from tests.test_gpu_drafts import i32, moved

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["function", "cache", "layers"])
def test_keys_that_are_the_values_move_once(how):
    """Paths of hundreds of rows, so that a second move would meet rows that the first has moved; the layers of one tensor one by one."""
    block, T = 16, 400
    bt, n = pages(7, 2, 32)
    path = [list(range(0, T, 2)) + [-1] * (T // 2), [0] + list(range(100, T)) + [-1] * 99]
    counts, offset = [200, 301], [100, 3]
    pool = torch.randint(0, 255, (3, n, block, 2, 64), generator=torch.Generator().manual_seed(1)).to(torch.float16)
    want = moved(pool, bt, offset, path, counts, block, False)
    dev = pool.cuda()
    for _ in range(5):
        dev.copy_(pool)
        if how == "function":
            ob.commit_drafts((dev, dev), bt.cuda(), i32(offset), i32(path), i32(counts))
        elif how == "cache":
            for layer in dev:
                ob.PagedKVCache(layer, layer, bt.cuda(), i32([500, 500]), block).commit_drafts(i32(offset), i32(path), i32(counts))
        else:
            ob.commit_drafts([dev[i] for i in (1, 0, 2)], bt.cuda(), i32(offset), i32(path), i32(counts))
        assert torch.equal(dev.cpu(), want)


def test_pools_that_share_memory_are_refused():
    pool = torch.zeros(3, 8, 16, 2, 64, dtype=torch.float16, device="cuda")
    rest = dict(block_table=i32([[0, 1]]), offset=0, path=i32([[0, 2]]), counts=i32([2]))
    for pools in ((pool, pool.view_as(pool)), (pool, pool[1]), (pool[1], pool), (pool[0], pool[1], pool[0])):
        with pytest.raises(RuntimeError, match="share memory"):
            ob.commit_drafts(pools, **rest)
