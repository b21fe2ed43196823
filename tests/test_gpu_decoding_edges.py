"""The decoding operators where they can go wrong."""
import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import EPS, chunk, rand

pytestmark = pytest.mark.gpu


# ---- 4-bit codes --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("frames", [1, 3, 5, 7, 31])
@pytest.mark.parametrize("H,Hkv,D,R,inter", [(4, 1, 128, 128, False), (3, 3, 64, 64, False), (2, 1, 64, 32, False), (5, 2, 96, 32, False), (1, 1, 128, 96, False), (2, 3, 32, 16, False),
                                             (1, 2, 256, 192, False), (3, 1, 512, 512, False), (4, 2, 128, 64, True), (0, 1, 64, 64, False)])
def test_codes_do_not_depend_on_the_rows_beside_them(frames, H, Hkv, D, R, inter):
    """A frame gets the same codes, scales and query alone (a warp then holds queries, keys and values) and among 32 (one kind a warp)."""
    dt = torch.bfloat16
    q, k, v = chunk(11, 32, max(H, 1), Hkv, 1, D, dt, False)
    v = v * 3                                             # its scales are not the keys'
    table = ob.rope_table(64, R)
    off = (torch.arange(32, dtype=torch.int32) % 16).cuda()
    bt = torch.arange(32, dtype=torch.int32, device="cuda")[:, None]
    kw = (1 + 0.2 * rand(3, D)).to(dt).cuda()
    got = []
    for n in (frames, 32):
        pools = ob.PagedKVCacheQ4.empty_pools(32, Hkv, 16, D, dt)
        out = ob.write_kv_rope_q4(*pools, bt[:n], k[:n], v[:n], off[:n], table, q=q[:n] if H else None, k_weight=kw, eps=EPS, interleaved=inter)
        got.append([p[:frames] for p in pools] + ([out[:frames]] if H else []))
    assert all(torch.equal(a, b) for a, b in zip(*got))
