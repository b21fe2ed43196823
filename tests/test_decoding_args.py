"""The decoding operators' entry points refuse bad shapes, sizes and pointers before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

import oasr_b200 as ob
from oasr_b200 import _lib

P16 = ctypes.c_void_p(4096)     # never followed: every call here is refused
ODD = ctypes.c_void_p(4098)
S = (ctypes.c_int64 * 3)(4096, 64, 512)
S_ODD = (ctypes.c_int64 * 3)(4096, 63, 512)


def refused(name, args, code):
    assert getattr(_lib.load(), "oasr_b200_" + name)(*args) == code, (name, _lib.last_error())


def qk(**how):
    a = dict(q_out=P16, k_out=P16, q=P16, k=P16, qw=P16, kw=P16, table=P16, rows=8, rotary=64, pos=P16, i64=1, N=4, H=2, Hkv=1, D=64, s1=128, s2=64, s3=128, s4=64,
             s5=128, s6=64, s7=128, s8=64, eps=1e-6, inter=0, dtype=_lib.DT_BF16, stream=None) | how
    return list(a.values())


@pytest.mark.parametrize("how,code", [
    (dict(N=-1), -1), (dict(H=0), -1), (dict(Hkv=-1), -1), (dict(rows=0), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(table=None), -1), (dict(pos=None), -1),
    (dict(H=65535), -1), (dict(N=1 << 31), -1), (dict(D=72), -5), (dict(D=528), -5), (dict(rotary=24), -5), (dict(rotary=128), -5), (dict(rotary=0), -5), (dict(s2=60), -3),
    (dict(s8=4), -3), (dict(q=ODD), -3), (dict(kw=ODD), -3), (dict(pos=ODD), -3), (dict(dtype=_lib.DT_INT8), -2)])
def test_qk_norm_rope(how, code):
    refused("qk_norm_rope", qk(**how), code)


def write(q4, **how):
    a = dict(q_out=P16, qo=S, kc=P16) | (dict(ks=P16) if q4 else {}) | dict(vc=P16) | (dict(vs=P16) if q4 else {})
    a |= dict(q=P16, qs=S, k=P16, kst=S, v=P16, vst=S, qw=None, kw=None, table=P16, rows=8, rotary=64, bt=P16, off=P16, rope=None, lens=None, B=2, H=2, Hkv=1, T=3, D=64,
              per=4, block=16, blocks=8, eps=1e-6, inter=0, dtype=_lib.DT_BF16, stream=None)
    return list((a | how).values())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("how,code", [
    (dict(B=-1), -1), (dict(Hkv=0), -1), (dict(block=0), -1), (dict(blocks=0), -1), (dict(rows=0), -1), (dict(kc=None), -1), (dict(v=None), -1), (dict(bt=None), -1),
    (dict(off=None), -1), (dict(q=None), -1), (dict(q_out=None), -1), (dict(qs=None), -1), (dict(B=1 << 20, T=1 << 20), -1), (dict(D=40), -5), (dict(rotary=40), -5),
    (dict(kst=S_ODD), -3), (dict(qo=S_ODD), -3), (dict(v=ODD), -3), (dict(kc=ODD), -3), (dict(dtype=_lib.DT_F32), -2)])
def test_write_kv_rope(q4, how, code):
    refused("write_kv_rope_q4" if q4 else "write_kv_rope", write(q4, **how), code)


def test_write_kv_rope_q4_needs_whole_groups_and_scales():
    refused("write_kv_rope_q4", write(True, D=80, rotary=16), -5)
    refused("write_kv_rope_q4", write(True, ks=None), -1)


def test_gather():
    def args(**how):
        return list((dict(k=P16, v=P16, kc=P16, ks=P16, vc=P16, vs=P16, bt=P16, start=None, B=1, Hkv=1, T=4, D=64, per=2, block=16, blocks=4, dtype=_lib.DT_F16, stream=None) | how).values())
    for how, code in [(dict(T=-1), -1), (dict(D=48), -5), (dict(D=1024), -5), (dict(bt=None), -1), (dict(k=ODD), -3), (dict(dtype=_lib.DT_F32), -2), (dict(T=1 << 32), -1)]:
        refused("paged_kv_gather_q4", args(**how), code)


def test_fmha_q4():
    def args(**how):
        return list((dict(out=P16, os=S, q=P16, qs=S, kc=P16, ks=P16, vc=P16, vs=P16, bt=P16, lens=P16, starts=None, q_lens=None, per=4, block=16, blocks=8, B=2, H=4, Hkv=2, T=1,
                          D=64, scale=0.1, causal=0, dtype=_lib.DT_BF16, stream=None) | how).values())
    for how, code in [(dict(B=-1), -1), (dict(H=3), -1), (dict(D=96), -5), (dict(block=8), -5), (dict(block=24), -5), (dict(lens=None), -1), (dict(bt=None), -1), (dict(vs=None), -1),
                      (dict(qs=S_ODD), -3), (dict(os=S_ODD), -3), (dict(out=ODD), -3), (dict(ks=ODD), -3), (dict(B=70000), -1), (dict(per=1 << 30), -1), (dict(block=1 << 26), -1),
                      (dict(dtype=_lib.DT_F32), -2)]:
        refused("fmha_q4", args(**how), code)
    refused("set_tunable", (b"fmha_q4_path", 3), -1)


def test_token_log_probs():
    def args(**how):
        return list((dict(lp=P16, ent=P16, top=P16, ids=P16, x=P16, tok=P16, i64=1, rows=4, V=100, stride=104, n=1, k=2, dtype=_lib.DT_F32, stream=None) | how).values())
    for how, code in [(dict(V=0), -1), (dict(V=262145, stride=262145), -5), (dict(stride=99), -1), (dict(k=33), -1), (dict(V=2, k=3), -1), (dict(k=-1), -1), (dict(x=None), -1),
                      (dict(tok=None), -1), (dict(lp=None), -1), (dict(ids=None), -1), (dict(dtype=_lib.DT_INT8), -2), (dict(x=ODD), -3)]:
        refused("token_log_probs", args(**how), code)


def test_empty_calls_need_no_gpu():
    lib = _lib.load()
    assert lib.oasr_b200_qk_norm_rope(*qk(N=0, q=None)) == 0
    assert lib.oasr_b200_write_kv_rope(*write(False, T=0)) == 0 and lib.oasr_b200_write_kv_rope_q4(*write(True, B=0)) == 0


def test_cpu_tensors_are_refused():
    q, table, pos = torch.zeros(2, 1, 64).bfloat16(), ob.rope_table(4, 64, device="cpu"), torch.zeros(2, dtype=torch.int64)
    pools = ob.PagedKVCacheQ4.empty_pools(2, 1, 16, 64, device="cpu")
    bt, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 1, 64).bfloat16()
    for call in (lambda: ob.qk_norm_rope(q, None, table, pos), lambda: ob.write_kv_rope_q4(*pools, bt, x, x, lens, table),
                 lambda: ob.write_kv_rope(*[torch.zeros(2, 16, 1, 64).bfloat16()] * 2, bt, x, x, lens, table), lambda: ob.gather_paged_kv_q4(*pools, bt, None, 4),
                 lambda: ob.fmha_q4(x, *pools, softmax_scale=1.0, block_table=bt, cache_seqlens=lens), lambda: ob.token_log_probs(torch.zeros(2, 8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_rope_table():
    t = ob.rope_table(5, 32, base=100.0, device="cpu")
    want = torch.arange(5, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert t.shape == (5, 32) and t.dtype == torch.float32
    assert torch.equal(t, torch.cat([want.cos(), want.sin()], 1).float())
    for rows, dim in ((0, 32), (4, 0), (4, 24)):
        with pytest.raises(ValueError):
            ob.rope_table(rows, dim, device="cpu")


def test_empty_pools():
    with pytest.raises(ValueError):
        ob.PagedKVCacheQ4.empty_pools(2, 1, 16, 48, device="cpu")
    with pytest.raises(ValueError):
        ob.PagedKVCacheQ4.empty_pools(2, 1, 16, 64, dtype=torch.float32, device="cpu")
    kc, ks, vc, vs = ob.PagedKVCacheQ4.empty_pools(2, 3, 16, 128, device="cpu")
    assert kc.shape == vc.shape == (2, 3, 16, 64) and ks.shape == vs.shape == (2, 3, 16, 4) and ks.dtype == torch.bfloat16
