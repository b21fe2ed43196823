"""The entry points of drafted tokens refuse bad shapes, sizes and pointers before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

import oasr_b200 as ob
from oasr_b200 import _lib

P16 = ctypes.c_void_p(4096)     # never followed: every call here is refused
ODD = ctypes.c_void_p(4097)
EIGHT = ctypes.c_void_p(4104)
S = (ctypes.c_int64 * 3)(4096, 64, 512)
S_ODD = (ctypes.c_int64 * 3)(4096, 63, 512)


def refused(name, args, code):
    assert getattr(_lib.load(), "oasr_b200_" + name)(*args) == code, (name, _lib.last_error())


@pytest.mark.parametrize("how,code", [(dict(B=-1), -1), (dict(T=-1), -1), (dict(T=1025, words=33), -5), (dict(words=2), -1), (dict(mask=None), -1), (dict(depth=None), -1),
                                      (dict(parents=None), -1), (dict(parents=ODD), -3), (dict(B=1 << 31), -1)])
def test_draft_tree(how, code):
    refused("draft_tree", (dict(mask=P16, depth=P16, parents=P16, B=2, T=32, words=1, stream=None) | how).values(), code)


def tree(**how):
    a = dict(out=P16, os=S, q=P16, qs=S, k=P16, v=P16, bt=P16, lens=P16, starts=None, q_lens=None, mask=P16, ms=1, words=1, work=P16, size=1 << 40, per=4, block=16, blocks=8,
             B=2, H=4, Hkv=2, T=5, D=64, scale=0.1, dtype=_lib.DT_BF16, stream=None) | how
    return list(a.values())


@pytest.mark.parametrize("how,code", [
    (dict(B=-1), -1), (dict(H=3), -1), (dict(Hkv=0), -1), (dict(D=96), -5), (dict(block=8), -5), (dict(block=24), -5), (dict(block=0), -5), (dict(blocks=0), -1), (dict(lens=None), -1),
    (dict(bt=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(qs=S_ODD), -3), (dict(os=S_ODD), -3), (dict(out=EIGHT), -3), (dict(k=EIGHT), -3), (dict(mask=ODD), -3), (dict(B=70000), -1),
    (dict(per=1 << 30), -1), (dict(T=1 << 15, words=1 << 10), -1), (dict(words=0), -1), (dict(T=33), -1), (dict(ms=-1), -1), (dict(dtype=_lib.DT_F32), -2), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(per=1 << 12, size=16), -1), (dict(per=1 << 12, work=None), -1), (dict(per=1 << 12, work=EIGHT), -3)])
def test_fmha_tree(how, code):
    refused("fmha_tree", tree(**how), code)


def test_fmha_tree_workspace():
    need = _lib.load().oasr_b200_fmha_tree_workspace_bytes
    assert need(1, 8, 8, 1, 64, 4, 16, 4) == 0                       # a short cache is not split
    assert need(1, 8, 2, 5, 128, 4096, 16, 4096) > 0
    for bad in [(0, 8, 8, 1, 64, 4096, 16), (1, 8, 3, 1, 64, 4096, 16), (1, 8, 8, 1, 96, 4096, 16), (1, 8, 8, 0, 64, 4096, 16), (1, 8, 0, 1, 64, 4096, 16), (1, 8, 8, 1, 64, 4096, 0)]:
        assert need(*bad, 4096) == 0
    refused("set_tunable", (b"fmha_tree_path", 3), -1)


def verify(**how):
    a = dict(tokens=P16, path=P16, counts=P16, logits=P16, lb=1000, ln=100, drafts=P16, parents=P16, ps=5, u=P16, probs=None, pb=0, pn=0, temps=None, temp=1.0, B=2, T=5, V=100,
             dtype=_lib.DT_BF16, stream=None) | how
    return list(a.values())


@pytest.mark.parametrize("how,code", [(dict(B=-1), -1), (dict(T=-1), -1), (dict(V=0), -1), (dict(T=1025), -5), (dict(V=1 << 27), -1), (dict(B=1 << 24), -1), (dict(logits=None), -1),
                                      (dict(tokens=None), -1), (dict(u=None), -1), (dict(parents=None), -1), (dict(temp=float("nan")), -1), (dict(temp=float("inf")), -1),
                                      (dict(dtype=_lib.DT_INT8), -2), (dict(logits=ODD), -3), (dict(u=ODD), -3), (dict(probs=ODD), -3), (dict(temps=ODD), -3)])
def test_verify_drafts(how, code):
    refused("verify_drafts", verify(**how), code)


def commit(pool=(4096, 2, 1, 256), **how):
    pools = (_lib.DraftPool * 1)(_lib.DraftPool(*pool))
    a = dict(pools=pools, n=1, bt=P16, offset=P16, path=P16, counts=P16, B=2, T=5, per=4, block=16, blocks=8, stream=None) | how
    return list(a.values())


@pytest.mark.parametrize("how,code", [
    (dict(B=-1), -1), (dict(n=-1), -1), (dict(block=0), -1), (dict(blocks=0), -1), (dict(per=-1), -1), (dict(B=70000), -1), (dict(T=1 << 23), -1), (dict(pools=None), -1), (dict(bt=None), -1),
    (dict(path=None), -1), (dict(counts=None), -1), (dict(offset=ODD), -3), (dict(pool=(None, 1, 1, 16)), -1), (dict(pool=(4096, 0, 1, 16)), -1), (dict(pool=(4096, 1, 0, 16)), -1),
    (dict(pool=(4096, 1, 1, 0)), -1), (dict(pool=(4096, 1, 1, 1 << 31)), -1)])
def test_commit_drafts(how, code):
    refused("commit_drafts", commit(**how), code)


def test_empty_calls_need_no_gpu():
    lib = _lib.load()
    assert lib.oasr_b200_draft_tree(None, None, None, 0, 5, 1, None) == 0 and lib.oasr_b200_draft_tree(None, None, None, 5, 0, 0, None) == 0
    assert lib.oasr_b200_fmha_tree(*tree(B=0, q=None)) == 0 and lib.oasr_b200_fmha_tree(*tree(T=0)) == 0
    assert lib.oasr_b200_verify_drafts(*verify(B=0, logits=None)) == 0 and lib.oasr_b200_verify_drafts(*verify(T=0)) == 0
    assert lib.oasr_b200_commit_drafts(*commit(n=0, pools=None)) == 0 and lib.oasr_b200_commit_drafts(*commit(T=0)) == 0 and lib.oasr_b200_commit_drafts(*commit(per=0)) == 0


def test_cpu_tensors_are_refused():
    i32 = torch.zeros(1, 2, dtype=torch.int32)
    pool, x, lens = torch.zeros(2, 16, 1, 64).bfloat16(), torch.zeros(1, 1, 2, 64).bfloat16(), torch.ones(1, dtype=torch.int32)
    for call in (lambda: ob.draft_tree(i32), lambda: ob.fmha_tree(x, pool, pool, softmax_scale=1.0, block_table=i32, cache_seqlens=lens),
                 lambda: ob.verify_drafts(torch.zeros(1, 2, 8), i32, i32, torch.zeros(1, 2)), lambda: ob.commit_drafts((pool, pool), i32, lens, i32, lens),
                 lambda: ob.commit_drafts_q4(ob.PagedKVCacheQ4.empty_pools(2, 1, 16, 64, device="cpu"), i32, lens, i32, lens)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_bad_shapes_are_refused():
    i32, u = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    x = torch.zeros(2, 3, 8)
    for bad in (lambda: ob.draft_tree(i32[None]), lambda: ob.draft_tree(u), lambda: ob.verify_drafts(x[0], i32, i32, u), lambda: ob.verify_drafts(x, i32[:1], i32, u),
                lambda: ob.verify_drafts(x, i32, i32[:, :2], u), lambda: ob.verify_drafts(x, i32, i32, u.double()), lambda: ob.verify_drafts(x, i32, i32, u[:1]),
                lambda: ob.verify_drafts(x, i32, i32, u, temperature=u[0, :2].double()), lambda: ob.verify_drafts(x, i32, i32, u, temperature=u[0]),
                lambda: ob.verify_drafts(x, i32, i32, u, draft_probs=x[:, :2]), lambda: ob.verify_drafts(x, i32, i32, u, draft_probs=x.double()),
                lambda: ob.verify_drafts(x, i32.float(), i32, u), lambda: ob.verify_drafts(x[:, :, :0], i32, i32, u)):
        with pytest.raises(RuntimeError):
            bad()
    pool, path, counts = torch.zeros(4, 16, 2, 8), i32, torch.zeros(2, dtype=torch.int32)
    for bad in (dict(pools=()), dict(pools=(pool[:, :, :, ::2],)), dict(pools=(pool[0],)), dict(pools=(pool, pool[:, :8].contiguous())), dict(path=path[0]), dict(counts=counts[:1]),
                dict(offset=counts[:1]), dict(block_table=i32[:1])):
        with pytest.raises(ValueError):
            ob.commit_drafts(**(dict(pools=(pool,), block_table=i32, offset=counts, path=path, counts=counts) | bad))
