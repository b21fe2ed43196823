"""Attention operators with the reference's signatures (oasr/functionals/attention.py)."""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib
from .functional import _DTYPE_ID, _check_distinct_rows, _need_cuda, _one_device, _p, _stream

_HALF = (torch.float16, torch.bfloat16)
_Strides = ctypes.c_int64 * 3


@functools.lru_cache(maxsize=4096)
def _stride_array(a: int, b: int, c: int):
    """Three strides as the host array that the entry points read (one for each combination of values)."""
    return _Strides(a, b, c)


def _used_strides(n0: int, n1: int, n2: int, s0: int, s1: int, s2: int):
    """Strides of three dimensions as the kernels use them: that of a dimension of size 1 may be any number, and is none."""
    return s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0


def _strides3(t: torch.Tensor):
    """(batch, head, row) element strides of a (B, H, T, D) view as a host int64[3]; None if the
    view cannot be addressed by the kernel (unit stride along D, the rest multiples of 8)."""
    if t.stride(3) != 1 and t.size(3) > 1:
        return None
    st = [t.stride(0), t.stride(1), t.stride(2)]
    for extent, s in zip(t.shape[:3], st):
        if extent > 1 and (s <= 0 or s % 8):
            return None
    return _Strides(*[s if e > 1 else 8 for e, s in zip(t.shape[:3], st)])


def _canon(t: torch.Tensor):
    st = _strides3(t)
    if st is None or t.data_ptr() % 16:
        t = t.contiguous()
        st = _strides3(t)
    return t, st


def gather_paged_kv(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor):
    """Gather paged K/V into dense ``(B, H_kv, T_kv_logical, D)`` tensors
    (reference: functionals/attention.py:153-178).  Pure data movement: bit-exact."""
    _need_cuda(k_pool, v_pool, block_table)
    if k_pool.dim() != 4 or k_pool.shape != v_pool.shape or block_table.dim() != 2:
        raise ValueError("gather_paged_kv expects pools (num_blocks, block_size, H_kv, D) and a 2-D block table")
    if block_table.dtype != torch.int32:
        block_table = block_table.to(torch.int32)
    block_table = block_table.contiguous()
    k_pool, v_pool = k_pool.contiguous(), v_pool.contiguous()
    B, nblk = block_table.shape
    num_blocks, bs, Hkv, D = k_pool.shape
    k = torch.empty(B, Hkv, nblk * bs, D, device=k_pool.device, dtype=k_pool.dtype)
    v = torch.empty_like(k)
    _lib.call("oasr_b200_paged_kv_gather", _p(k), _p(v), _p(k_pool), _p(v_pool), _p(block_table), B, Hkv, D, nblk, bs,
              num_blocks, k_pool.element_size(), _stream(k_pool))
    return k, v


def fmha(q, k, v, *, softmax_scale: float, attn_bias: Optional[torch.Tensor] = None,
         cache_seqlens: Optional[torch.Tensor] = None, cache_seqstarts: Optional[torch.Tensor] = None,
         block_table: Optional[torch.Tensor] = None, causal: bool = False, out: Optional[torch.Tensor] = None,
         validate: bool = True, token_major: bool = False) -> torch.Tensor:
    """Fused multi-head attention (reference: functionals/attention.py:369-551).

    ``q`` ``(B, H, T_q, D)``; dense ``k``/``v`` ``(B, H_kv, T_k, D)`` or, with
    ``block_table`` ``(B, max_blocks_per_seq)``, page pools
    ``(num_blocks, block_size, H_kv, D)``.  ``attn_bias`` ``(B, H, >=T_q, >=T_k)`` is an
    additive post-scale logit; ``cache_seqlens`` / ``cache_seqstarts`` keep keys in
    ``[start, len)``; ``causal`` masks ``k_col > q_row``.  A fully masked row gives zeros.
    Unlike the reference wrapper no padding of the bias or widening of the block table
    is needed: the kernel predicates its bias reads and clamps page lookups.
    ``token_major=True`` (an extension) returns ``(B, T_q, H, D)``, the layout the output
    projection reads, instead of ``(B, H, T_q, D)``.
    """
    _need_cuda(q, k, v, attn_bias, cache_seqlens, cache_seqstarts, block_table, out)
    if q.dim() != 4:
        raise ValueError(f"q must be (B, H, T_q, D); got {tuple(q.shape)}")
    B, H, T_q, D = q.shape
    paged = block_table is not None
    if paged:
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("paged k/v must be (num_blocks, block_size, H_kv, D)")
        num_blocks, block_size, H_kv = k.size(0), k.size(1), k.size(2)
        T_k = block_table.size(1) * block_size
    else:
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"k and v must match: {tuple(k.shape)} vs {tuple(v.shape)}")
        num_blocks, block_size, H_kv, T_k = 0, 0, k.size(1), k.size(2)
    if validate:
        if q.dtype not in _HALF:
            raise ValueError(f"fmha supports fp16/bf16, got {q.dtype}")
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError("q, k, v must share a dtype")
        if k.size(3) != D:
            raise ValueError("q and k head_dim must match")
        if H % H_kv != 0:
            raise ValueError(f"H ({H}) must be divisible by H_kv ({H_kv})")
        if not paged and k.size(0) != B:
            raise ValueError("q and k batch must match")
        if attn_bias is not None:
            if attn_bias.dim() != 4 or attn_bias.size(0) != B or attn_bias.size(1) != H or \
                    attn_bias.size(2) < T_q or attn_bias.size(3) < (T_k if not paged else 1):
                raise ValueError(f"attn_bias must be (B, H, >=T_q, >=T_k); got {tuple(attn_bias.shape)}")
            if attn_bias.dtype != q.dtype:
                attn_bias = attn_bias.to(q.dtype)
        if cache_seqlens is not None:
            if cache_seqlens.dim() != 1 or cache_seqlens.size(0) != B:
                raise ValueError(f"cache_seqlens must be (B,) = ({B},); got {tuple(cache_seqlens.shape)}")
            if cache_seqlens.dtype != torch.int32:
                cache_seqlens = cache_seqlens.to(torch.int32)
        if cache_seqstarts is not None:
            if cache_seqlens is None:
                raise ValueError("cache_seqstarts requires cache_seqlens (it bounds the window)")
            if cache_seqstarts.dim() != 1 or cache_seqstarts.size(0) != B:
                raise ValueError(f"cache_seqstarts must be (B,) = ({B},); got {tuple(cache_seqstarts.shape)}")
            if cache_seqstarts.dtype != torch.int32:
                cache_seqstarts = cache_seqstarts.to(torch.int32)
        if block_table is not None:
            if block_table.dim() != 2 or block_table.size(0) != B:
                raise ValueError("block_table must be (B, max_blocks_per_seq)")
            if block_table.dtype != torch.int32:
                block_table = block_table.to(torch.int32)
        want = (B, T_q, H, D) if token_major else (B, H, T_q, D)
        if out is not None and (tuple(out.shape) != want or out.dtype != q.dtype or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {want} in q's dtype")
    if out is None:
        out = torch.empty((B, T_q, H, D) if token_major else (B, H, T_q, D), dtype=q.dtype, device=q.device)
    q, qs = _canon(q)
    if paged:
        k, v = k.contiguous(), v.contiguous()
        ks = vs = None
        block_table = block_table.contiguous()
        # a bias narrower than the table's key range is fine as long as it covers the valid keys:
        # the kernel reads bias[..., j] only for j < cache_seqlens[b]
        if attn_bias is not None and attn_bias.size(3) < T_k and cache_seqlens is None:
            raise ValueError("a bias narrower than the block table needs cache_seqlens")
    else:
        k, ks = _canon(k)
        v, vs = _canon(v)
    bsb = bsh = bsq = 0
    if attn_bias is not None:
        if attn_bias.stride(3) != 1 and attn_bias.size(3) > 1:
            attn_bias = attn_bias.contiguous()
        bsb, bsh, bsq = attn_bias.stride(0), attn_bias.stride(1), attn_bias.stride(2)
    _lib.call("oasr_b200_fmha_bthd" if token_major else "oasr_b200_fmha", _p(out), _p(q), _p(k), _p(v), qs, ks, vs,
              _p(attn_bias), bsb, bsh, bsq,
              _p(cache_seqlens), _p(cache_seqstarts), _p(block_table),
              block_table.size(1) if paged else 0, block_size, num_blocks, B, H, H_kv, T_q, T_k, D,
              float(softmax_scale), int(bool(causal)), _DTYPE_ID[q.dtype], _stream(q))
    return out


def fmha_varlen(q, k, v, *, softmax_scale: float, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                max_seqlen_q: int, max_seqlen_k: int, attn_bias: Optional[torch.Tensor] = None,
                bias_offsets: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                validate: bool = True) -> torch.Tensor:
    """Variable-length (sequence-packed) attention (reference: functionals/attention.py:592-693).

    ``q`` ``(total_q, H, D)``, ``k``/``v`` ``(total_k, H_kv, D)``; segment ``s`` spans
    ``[cu[s], cu[s+1])`` and attends only to itself; ``attn_bias`` is the flat packed
    block-diagonal bias whose segment block ``(H, T_q_s, T_k_s)`` starts at ``bias_offsets[s]``.
    No host synchronisation (the reference's sm_100 route loops over ``cu_seqlens.tolist()``).
    """
    _need_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, attn_bias, bias_offsets, out)
    if validate:
        if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
            raise ValueError("varlen q/k/v must be packed 3-D (total, H, D); got "
                             f"{tuple(q.shape)} / {tuple(k.shape)} / {tuple(v.shape)}")
        if k.shape != v.shape:
            raise ValueError(f"k and v must match: {tuple(k.shape)} vs {tuple(v.shape)}")
        if q.size(2) != k.size(2):
            raise ValueError("q and k head_dim must match")
        if q.size(1) % k.size(1) != 0:
            raise ValueError(f"H ({q.size(1)}) must be divisible by H_kv ({k.size(1)})")
        for name, cu in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
            if cu.dim() != 1 or cu.numel() < 2:
                raise ValueError(f"{name} must be 1-D with >= 2 entries")
        if cu_seqlens_q.numel() != cu_seqlens_k.numel():
            raise ValueError("cu_seqlens_q and cu_seqlens_k must have equal length")
        if (attn_bias is None) != (bias_offsets is None):
            raise ValueError("attn_bias and bias_offsets must be provided together")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype):
            raise ValueError("out must match q in shape/dtype")
        if q.dtype not in _HALF or k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError("fmha_varlen supports fp16/bf16 with one dtype for q, k, v")
        if attn_bias is not None and attn_bias.dtype != q.dtype:
            attn_bias = attn_bias.to(q.dtype)
        if cu_seqlens_q.dtype != torch.int32:
            cu_seqlens_q = cu_seqlens_q.to(torch.int32)
        if cu_seqlens_k.dtype != torch.int32:
            cu_seqlens_k = cu_seqlens_k.to(torch.int32)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device, memory_format=torch.contiguous_format)
    elif not out.is_contiguous():
        raise ValueError("out must be contiguous")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    off_i64 = 0
    if bias_offsets is not None:
        if bias_offsets.dtype == torch.int64:
            off_i64 = 1
        elif bias_offsets.dtype != torch.int32:
            bias_offsets = bias_offsets.to(torch.int64)
            off_i64 = 1
        bias_offsets = bias_offsets.contiguous()
        attn_bias = attn_bias.contiguous()
    S = cu_seqlens_q.numel() - 1
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    _lib.call("oasr_b200_fmha_varlen", _p(out), _p(q), _p(k), _p(v), _p(attn_bias), _p(bias_offsets), off_i64,
              _p(cu_seqlens_q), _p(cu_seqlens_k), S, q.size(0), k.size(0),
              int(max_seqlen_q), q.size(1), k.size(1), q.size(2), float(softmax_scale), _DTYPE_ID[q.dtype],
              _stream(q))
    return out


def _narrow(t: torch.Tensor) -> torch.Tensor:
    """As int32; what 32 bits do not hold goes to the nearest number that they do, and not round to one that means something."""
    if t.dtype == torch.int64:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(torch.int32)


def _index32(name: str, t: Optional[torch.Tensor], B: int) -> Optional[torch.Tensor]:
    """A number for each sequence as the kernels take it."""
    if t is None:
        return None
    if t.shape != (B,):
        raise ValueError(f"{name} must be ({B},), got {tuple(t.shape)}")
    if t.dtype != torch.int32:
        t = _narrow(t)
    return t if t.is_contiguous() else t.contiguous()


def _table32(table: torch.Tensor, B: int) -> torch.Tensor:
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError("block_table must be (B, max_blocks_per_seq)")
    if table.dtype != torch.int32:
        table = _narrow(table)
    return table if table.is_contiguous() else table.contiguous()


def _check_q4_pools(k_codes, k_scales, v_codes, v_scales, dtype):
    """``(num_blocks, H_kv, block_size, D)`` of 4-bit pools, or an error."""
    shape = k_codes.shape
    if len(shape) != 4 or k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8 or v_codes.shape != shape:
        raise ValueError("codes must be uint8 (num_blocks, H_kv, block_size, D / 2) and match")
    num_blocks, Hkv, block_size, half = shape
    if half % 16 or half == 0:
        raise ValueError(f"head_dim must be a multiple of 32, got {2 * half}")
    want = (num_blocks, Hkv, block_size, half // 16)
    if k_scales.shape != want or v_scales.shape != want:
        raise ValueError(f"scales must be (num_blocks, H_kv, block_size, D / 32) = {want}, got {tuple(k_scales.shape)}")
    if dtype not in _HALF:
        raise ValueError(f"4-bit pages go with fp16 or bf16, got {dtype}")
    if k_scales.dtype != dtype or v_scales.dtype != dtype:
        raise ValueError(f"scales must have dtype {dtype}, got {k_scales.dtype} / {v_scales.dtype}")
    if not (k_codes.is_contiguous() and k_scales.is_contiguous() and v_codes.is_contiguous() and v_scales.is_contiguous()):
        raise ValueError("pools must be contiguous")
    return num_blocks, Hkv, block_size, 2 * half


def gather_paged_kv_q4(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                       block_table: torch.Tensor, start: Optional[torch.Tensor], length: int):
    """The values of ``length`` positions from ``start[b]`` on (None: from 0) out of 4-bit pages, as dense
    ``(B, H_kv, length, D)`` tensors in the scales' type (exact).  A position without a page gives zeros."""
    num_blocks, Hkv, block_size, D = _check_q4_pools(k_codes, k_scales, v_codes, v_scales, k_scales.dtype)
    length = int(length)
    if block_table.dim() != 2 or length < 0:
        raise ValueError("gather_paged_kv_q4 expects a (B, max_blocks_per_seq) block table and length >= 0")
    B = block_table.shape[0]
    block_table, start = _table32(block_table, B), _index32("start", start, B)
    _one_device(k_codes, k_scales, v_codes, v_scales, block_table, start)
    k = torch.empty(B, Hkv, length, D, device=k_codes.device, dtype=k_scales.dtype)
    v = torch.empty_like(k)
    _lib.call("oasr_b200_paged_kv_gather_q4", k.data_ptr(), v.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
              v_scales.data_ptr(), block_table.data_ptr(), _p(start), B, Hkv, length, D, block_table.shape[1], block_size, num_blocks,
              _DTYPE_ID[k.dtype], _stream(k))
    return k, v


def fmha_q4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor, *,
            softmax_scale: float, block_table: torch.Tensor, cache_seqlens: torch.Tensor,
            cache_seqstarts: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None, causal: bool = False,
            out: Optional[torch.Tensor] = None, token_major: bool = False) -> torch.Tensor:
    """Attention of ``q (B, H, T_q, D)`` over 4-bit pages (``PagedKVCacheQ4``), D 64 or 128, pages of a multiple of 16 rows.

    Row ``t`` of sequence ``b`` sees the keys ``cache_seqstarts[b] <= j < cache_seqlens[b]`` (no start: from 0); with ``causal``
    it stands at position ``cache_seqlens[b] - q_lens[b] + t`` and sees none behind that (``q_lens`` None: T_q), so the same
    call serves a prompt, a chunk and a single token whose keys have been written.  (``fmha``'s ``causal`` counts rows from key
    0.)  Rows ``t >= q_lens[b]`` are padding; those and rows that see nothing are zeros, and so is a sequence of length 0.  Keys
    whose page lies outside the pool are not seen.  ``token_major=True`` returns ``(B, T_q, H, D)``.

    Scores, their maximum and sum and the output are fp32; the weights are rounded to ``q``'s type before they meet the values
    (``fmha`` does the same), and the result once more.  How the work is split goes by the width of ``block_table``, as lengths are
    on the GPU: over a table many times wider than the longest sequence pass ``block_table[:, :blocks]`` of what is in use."""
    if q.dim() != 4:
        raise ValueError(f"q must be (B, H, T_q, D); got {tuple(q.shape)}")
    B, H, T, D = q.shape
    num_blocks, Hkv, block_size, pool_dim = _check_q4_pools(k_codes, k_scales, v_codes, v_scales, q.dtype)
    if pool_dim != D:
        raise ValueError("q and k head_dim must match")
    if Hkv == 0 or H % Hkv:
        raise ValueError(f"H ({H}) must be divisible by H_kv ({Hkv})")
    block_table = _table32(block_table, B)
    lens, starts = _index32("cache_seqlens", cache_seqlens, B), _index32("cache_seqstarts", cache_seqstarts, B)
    q_lens = _index32("q_lens", q_lens, B)
    _one_device(q, k_codes, k_scales, v_codes, v_scales, block_table, lens, starts, q_lens, out)
    qs = q.stride()
    sb, sh, st = _used_strides(B, H, T, *qs[:3])
    if qs[3] != 1 or sb % 8 or sh % 8 or st % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)   # (contiguous() would keep one that is merely misaligned)
        sb, sh, st = H * T * D, T * D, D
    if out is None:
        if token_major:
            out = torch.empty(B, T, H, D, dtype=q.dtype, device=q.device)
            os = _stride_array(T * H * D, D, H * D)
        else:
            out = torch.empty(B, H, T, D, dtype=q.dtype, device=q.device)
            os = _stride_array(H * T * D, T * D, D)
    else:
        want = (B, T, H, D) if token_major else (B, H, T, D)
        if tuple(out.shape) != want or out.dtype != q.dtype or out.stride(3) != 1:
            raise ValueError(f"out must be {want} in q's dtype, with unit stride along D")
        _check_distinct_rows(out=out)
        ob, oh, ot = (out.stride(0), out.stride(2), out.stride(1)) if token_major else out.stride()[:3]
        os = _stride_array(*_used_strides(B, H, T, ob, oh, ot))
    _lib.call("oasr_b200_fmha_q4", out.data_ptr(), os, q.data_ptr(), _stride_array(sb, sh, st), k_codes.data_ptr(), k_scales.data_ptr(),
              v_codes.data_ptr(), v_scales.data_ptr(), block_table.data_ptr(), lens.data_ptr(), _p(starts), _p(q_lens), block_table.shape[1],
              block_size, num_blocks, B, H, Hkv, T, D, softmax_scale, bool(causal), _DTYPE_ID[q.dtype], _stream(q))
    return out
