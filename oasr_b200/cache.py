"""Paged KV-cache data movement with the reference's layout (oasr/cache/paged_kv.py,
oasr/cache/block_pool.py:33-41): per-layer pools ``(num_blocks, block_size, H_kv, D)``,
``block_table (B, max_blocks_per_seq)`` int32, ``cache_seqlens (B,)`` int32."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence, Union

import torch

from . import _lib
from .attention import _HALF, _check_q4_pools, _stride_array, _index32, _narrow, _table32, _used_strides, fmha_q4, fmha_tree, gather_paged_kv, gather_paged_kv_q4  # noqa: F401  (re-exported)
from .functional import _DTYPE_ID, _check_distinct_rows, _check_head_weight, _check_rope_table, _need_cuda, _one_device, _p, _stream


def write_kv_chunk(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, new_k: torch.Tensor,
                   new_v: torch.Tensor, offset: Union[int, torch.Tensor]) -> None:
    """Scatter ``new_k`` / ``new_v`` ``(B, H_kv, T, D)`` into the pools: frame ``t`` of stream ``b``
    lands at logical position ``offset[b] + t`` (reference: PagedKVCache.write_kv_chunk,
    oasr/cache/paged_kv.py:63-137; index rule flat_write_index :23-40).  One kernel, no
    frame-major staging copy; the head-first inputs may be strided views."""
    _need_cuda(k_cache, v_cache, block_table, new_k, new_v)
    if new_k.shape != new_v.shape or new_k.dim() != 4:
        raise ValueError("new_k / new_v must be (B, H_kv, T, D) and match")
    B, Hkv, T, D = new_k.shape
    num_blocks, bs = k_cache.size(0), k_cache.size(1)
    if k_cache.shape != v_cache.shape or k_cache.size(2) != Hkv or k_cache.size(3) != D:
        raise ValueError("pools must be (num_blocks, block_size, H_kv, D) matching the new chunk")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("pools must be contiguous")
    if new_k.dtype != k_cache.dtype or new_v.dtype != v_cache.dtype:
        raise ValueError("chunk and pool dtypes must match")
    if isinstance(offset, int):
        offset = torch.full((B,), offset, dtype=torch.int32, device=new_k.device)
    elif offset.dtype != torch.int32:
        offset = offset.to(torch.int32)
    if block_table.dtype != torch.int32:
        block_table = block_table.to(torch.int32)
    block_table = block_table.contiguous()
    if new_k.stride(3) != 1:
        new_k = new_k.contiguous()
    if new_v.stride() != new_k.stride():
        new_v = new_v.contiguous()
        new_k = new_k.contiguous()
    offset = offset.contiguous()
    _lib.call("oasr_b200_paged_kv_write", _p(k_cache), _p(v_cache), _p(new_k), _p(new_v), _p(block_table), _p(offset),
              B, Hkv, T, D, new_k.stride(0), new_k.stride(1), new_k.stride(2),
              block_table.size(1), bs, num_blocks, k_cache.element_size(), _stream(new_k))


@dataclass
class PagedKVCache:
    """Per-layer pool views plus the shared per-batch paging state; same fields and
    methods as the reference descriptor (oasr/cache/paged_kv.py:43-180)."""

    k_cache: torch.Tensor
    v_cache: torch.Tensor
    block_table: torch.Tensor
    cache_seqlens: torch.Tensor
    block_size: int
    host_seqlen_max: int = 0

    def write_kv_chunk(self, new_k: torch.Tensor, new_v: torch.Tensor, *, offset: Union[int, torch.Tensor]) -> None:
        write_kv_chunk(self.k_cache, self.v_cache, self.block_table, new_k, new_v, offset)

    def fmha_tree(self, q: torch.Tensor, *, softmax_scale: float, **how) -> torch.Tensor:
        return fmha_tree(q, self.k_cache, self.v_cache, softmax_scale=softmax_scale, block_table=self.block_table, cache_seqlens=self.cache_seqlens, **how)

    def commit_drafts(self, offset: Union[int, torch.Tensor], path: torch.Tensor, counts: torch.Tensor) -> None:
        commit_drafts((self.k_cache, self.v_cache), self.block_table, offset, path, counts)

    def gather_full_kv(self, max_total_kv: int):
        B = self.block_table.size(0)
        Hkv, D = self.k_cache.size(2), self.k_cache.size(3)
        if max_total_kv == 0:
            empty = torch.zeros(B, Hkv, 0, D, dtype=self.k_cache.dtype, device=self.k_cache.device)
            return empty, empty.clone()
        nblk = (max_total_kv + self.block_size - 1) // self.block_size
        k, v = gather_paged_kv(self.k_cache, self.v_cache, self.block_table[:, :nblk])
        return k[:, :, :max_total_kv], v[:, :, :max_total_kv]


def _heads(x: torch.Tensor):
    """``x`` with unit stride along D, and its (batch, head, frame) strides."""
    sb, sh, st, unit = x.stride()
    if unit != 1:
        x = x.contiguous()
        sb, sh, st, unit = x.stride()
    return x, _stride_array(*_used_strides(*x.shape[:3], sb, sh, st))


def _write_rope(entry, pools, num_blocks, block_size, pool_heads, pool_dim, block_table, new_k, new_v, offset, cos_sin, q, q_weight,
                k_weight, eps, interleaved, rope_offset, new_lens, q_out):
    if new_k.dim() != 4 or new_k.shape != new_v.shape:
        raise ValueError("new_k / new_v must be (B, H_kv, T, D) and match")
    B, Hkv, T, D = new_k.shape
    dtype = new_k.dtype
    if dtype not in _HALF or new_v.dtype != dtype:
        raise ValueError(f"new_k / new_v must share fp16 or bf16, got {dtype} / {new_v.dtype}")
    if pool_heads != Hkv or pool_dim != D:
        raise ValueError(f"pools hold {pool_heads} heads of {pool_dim}, the chunk has {Hkv} of {D}")
    block_table = _table32(block_table, B)
    if isinstance(offset, int):
        offset = torch.full((B,), offset, dtype=torch.int32, device=new_k.device)
    offset = _index32("offset", offset, B)
    if rope_offset is not None:
        rope_offset = _index32("rope_offset", rope_offset, B)
    if new_lens is not None:
        new_lens = _index32("new_lens", new_lens, B)
    _one_device(new_k, *pools, block_table, new_v, offset, rope_offset, new_lens, cos_sin, q, q_weight, k_weight, q_out)
    rows, rotary = _check_rope_table(cos_sin, D)
    new_k, ks = _heads(new_k)
    new_v, vs = _heads(new_v)
    H, src, dst, qs, qo = 0, None, None, None, None
    if q is not None:
        if q.dim() != 4 or q.dtype != dtype or q.shape[0] != B or q.shape[2:] != (T, D):
            raise ValueError(f"q must be ({B}, H, {T}, {D}) {dtype}, got {tuple(q.shape)} {q.dtype}")
        H = q.shape[1]
        if q_out is None:
            q_out = torch.empty_like(q)
            if q_out.stride(3) != 1:
                q_out = torch.empty(q.shape, dtype=dtype, device=q.device)
        else:
            if q_out.shape != q.shape or q_out.dtype != dtype:
                raise ValueError("q_out must have q's shape and dtype")
            if q_out.stride(3) != 1:
                raise ValueError("q_out needs unit stride along D")
            _check_distinct_rows(q_out=q_out)
        q, qs = _heads(q)
        sb, sh, st, _ = q_out.stride()
        src, dst, qo = q.data_ptr(), q_out.data_ptr(), _stride_array(*_used_strides(B, H, T, sb, sh, st))
    elif q_out is not None or q_weight is not None:
        raise ValueError("q_out and q_weight need q")
    _lib.call(entry, dst, qo, *[p.data_ptr() for p in pools], src, qs, new_k.data_ptr(), ks, new_v.data_ptr(), vs,
              _check_head_weight("q_weight", q_weight, D, dtype), _check_head_weight("k_weight", k_weight, D, dtype), cos_sin.data_ptr(),
              rows, rotary, block_table.data_ptr(), offset.data_ptr(), _p(rope_offset), _p(new_lens), B, H, Hkv, T, D,
              block_table.shape[1], block_size, num_blocks, eps, bool(interleaved), _DTYPE_ID[dtype], _stream(new_k))
    return q_out


def write_kv_rope(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, new_k: torch.Tensor,
                  new_v: torch.Tensor, offset: Union[int, torch.Tensor], cos_sin: torch.Tensor, *,
                  q: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                  k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                  rope_offset: Optional[torch.Tensor] = None, new_lens: Optional[torch.Tensor] = None,
                  q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """``write_kv_chunk`` with the keys' norm (``k_weight``) and rotation on the way, and with ``q (B, H, T, D)`` the queries'
    (``q_weight``) in the same launch; returns the turned queries (None without ``q``).

    Frame ``t`` of stream ``b`` lands at logical position ``offset[b] + t`` and turns by the ``rope_table`` row of
    ``rope_offset[b] + t`` (None: the logical position; streams that have evicted pages pass their own).  Frames ``t >=
    new_lens[b]`` are padding: no page is written and their query rows are zeros.  A position outside the table gives a zero key
    and query.  ``q_out`` may be ``q`` itself.  ``interleaved``, weights and table as in ``qk_norm_rope``."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("pools must be (num_blocks, block_size, H_kv, D) and match")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("pools must be contiguous")
    if k_cache.dtype != new_k.dtype or v_cache.dtype != new_k.dtype:
        raise ValueError("chunk and pool dtypes must match")
    return _write_rope("oasr_b200_write_kv_rope", (k_cache, v_cache), *k_cache.shape, block_table, new_k, new_v, offset, cos_sin, q, q_weight,
                       k_weight, eps, interleaved, rope_offset, new_lens, q_out)


def write_kv_rope_q4(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                     block_table: torch.Tensor, new_k: torch.Tensor, new_v: torch.Tensor, offset: Union[int, torch.Tensor],
                     cos_sin: torch.Tensor, *, q: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                     k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                     rope_offset: Optional[torch.Tensor] = None, new_lens: Optional[torch.Tensor] = None,
                     q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """``write_kv_rope`` into 4-bit pages (``PagedKVCacheQ4`` describes them): the turned keys and the values are rounded to
    codes and scales from fp32."""
    num_blocks, Hkv, block_size, D = _check_q4_pools(k_codes, k_scales, v_codes, v_scales, new_k.dtype)
    return _write_rope("oasr_b200_write_kv_rope_q4", (k_codes, k_scales, v_codes, v_scales), num_blocks, block_size, Hkv, D, block_table,
                       new_k, new_v, offset, cos_sin, q, q_weight, k_weight, eps, interleaved, rope_offset, new_lens, q_out)


@dataclass
class PagedKVCacheQ4:
    """Paged keys and values in 4 bits: 0.28 of the bytes of 16-bit pages.

    Codes are ``(num_blocks, H_kv, block_size, D / 2)`` uint8 and scales ``(num_blocks, H_kv, block_size, D / 32)`` in the
    model's 16-bit type (heads outside the rows, so that a head's rows of a page lie together).  Each 32 dims of a row share the
    scale ``max|x| / 7`` rounded up to five significant bits; a value is ``code * scale`` with a code in [-7, 7], which fp16 and
    bf16 hold exactly.  The row's 32-bit word ``j`` holds dims ``32 (j % G) + 8 (j // G) + i`` (``G = D / 32``) as ``code + 8`` in
    bits ``4 i .. 4 i + 3``.  Logical positions, ``block_table`` and ``cache_seqlens`` are those of ``PagedKVCache``."""

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    block_table: torch.Tensor
    cache_seqlens: torch.Tensor

    @staticmethod
    def empty_pools(num_blocks: int, kv_heads: int, block_size: int, head_dim: int, dtype=torch.bfloat16, device="cuda"):
        """``(k_codes, k_scales, v_codes, v_scales)`` of value 0."""
        if head_dim % 32:
            raise ValueError(f"head_dim must be a multiple of 32, got {head_dim}")
        if dtype not in _HALF:
            raise ValueError(f"4-bit pages have fp16 or bf16 scales, got {dtype}")
        def codes():
            return torch.zeros(num_blocks, kv_heads, block_size, head_dim // 2, dtype=torch.uint8, device=device)
        def scales():
            return torch.zeros(num_blocks, kv_heads, block_size, head_dim // 32, dtype=dtype, device=device)
        return codes(), scales(), codes(), scales()

    @property
    def pools(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales

    def write_kv_rope(self, new_k: torch.Tensor, new_v: torch.Tensor, cos_sin: torch.Tensor, *, offset: Union[int, torch.Tensor],
                      **how) -> Optional[torch.Tensor]:
        return write_kv_rope_q4(*self.pools, self.block_table, new_k, new_v, offset, cos_sin, **how)

    def fmha(self, q: torch.Tensor, *, softmax_scale: float, **how) -> torch.Tensor:
        return fmha_q4(q, *self.pools, softmax_scale=softmax_scale, block_table=self.block_table, cache_seqlens=self.cache_seqlens, **how)

    def commit_drafts(self, offset: Union[int, torch.Tensor], path: torch.Tensor, counts: torch.Tensor) -> None:
        commit_drafts_q4(self.pools, self.block_table, offset, path, counts)

    def gather_full_kv(self, max_total_kv: int):
        return gather_paged_kv_q4(*self.pools, self.block_table, None, max_total_kv)


_WHOLE = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _commit(pools, geometry, block_table, offset, path, counts):
    """``geometry(shape)``: (num_blocks, block_size, outer) of one layer's pages, and which of its dimensions a row has."""
    if path.dim() != 2:
        raise ValueError(f"path must be (B, T), got {tuple(path.shape)}")
    B, T = path.shape
    if len(pools) == 2 and pools[0] is pools[1]:
        pools = pools[:1]                  # keys that are the values too
    table = (_lib.DraftPool * len(pools))()
    shape = None
    for entry, pool in zip(table, pools):
        if pool.dim() not in (4, 5) or not pool.is_contiguous():
            raise ValueError(f"pools must be contiguous pages of one layer or of (layers, ...), got {tuple(pool.shape)}")
        layers = pool.shape[0] if pool.dim() == 5 else 1
        num_blocks, block_size, outer, row = geometry(pool.shape[-4:])
        if shape is None:
            shape = num_blocks, block_size
        elif shape != (num_blocks, block_size):
            raise ValueError(f"pools must have the same pages: {shape} and {(num_blocks, block_size)}")
        entry.data, entry.layers, entry.outer, entry.row_bytes = pool.data_ptr(), layers, outer, row * pool.element_size()
    if shape is None:
        raise ValueError("no pools")
    if isinstance(offset, int):
        offset = torch.full((B,), offset, dtype=torch.int32, device=path.device)
    for name, index in (("block_table", block_table), ("offset", offset), ("path", path), ("counts", counts)):
        if index.dtype not in _WHOLE:      # (rows are moved in place by them: no rounding of something else)
            raise ValueError(f"{name} must be whole numbers, got {index.dtype}")
    block_table = _table32(block_table, B)
    offset, counts = _index32("offset", offset, B), _index32("counts", counts, B)
    path = _narrow(path) if path.dtype != torch.int32 else path
    if not path.is_contiguous():
        path = path.contiguous()
    _one_device(path, *pools, block_table, offset, counts)
    _lib.call("oasr_b200_commit_drafts", table, len(pools), block_table.data_ptr(), offset.data_ptr(), path.data_ptr(), counts.data_ptr(), B, T,
              block_table.shape[1], shape[1], shape[0], _stream(path))


def commit_drafts(pools: Sequence[torch.Tensor], block_table: torch.Tensor, offset: Union[int, torch.Tensor], path: torch.Tensor,
                  counts: torch.Tensor) -> None:
    """Moves the accepted drafts' rows together in the pages, in place: the row of position ``offset[b] + path[b, i]`` goes to ``offset[b] +
    i`` for ``i < counts[b]`` (``verify_drafts`` gives ``path (B, T)`` and ``counts (B,)``; ``offset`` is where the tree's node 0 lies).

    ``pools`` are the keys and values, of any element type, of one layer ``(num_blocks, block_size, H_kv, D)`` or of several
    ``(layers, num_blocks, block_size, H_kv, D)``; all of them are done in one launch (for each 64).  Pools share no memory (one tensor
    as keys and values is one pool).  A path ascends; it ends at the first entry that does not.  Positions without a page move nothing.
    Rows behind the path stay as they are.  The sequences of a call (up to 65535) must not share pages that are written."""
    _commit(pools, lambda s: (s[0], s[1], 1, s[2] * s[3]), block_table, offset, path, counts)


def commit_drafts_q4(pools: Sequence[torch.Tensor], block_table: torch.Tensor, offset: Union[int, torch.Tensor], path: torch.Tensor,
                     counts: torch.Tensor) -> None:
    """``commit_drafts`` in 4-bit pages: codes and scales of ``PagedKVCacheQ4``, ``(num_blocks, H_kv, block_size, ...)`` or with the layers
    before them.  (``fmha_q4`` attends chains, whose accepted rows lie together already; paths of branching trees come from an attention over
    these pages that the caller brings, ``fmha_tree`` reads 16-bit pages.)"""
    _commit(pools, lambda s: (s[0], s[2], s[1], s[3]), block_table, offset, path, counts)


def gather_rows(src: torch.Tensor, index: torch.Tensor, out: torch.Tensor = None) -> torch.Tensor:
    """``out[i] = src[index[i]]`` over the leading dimension (an index outside ``[0, len(src))`` gives a zero row):
    ``pack_hidden`` / gapped-conv gather / ``SlotTensor.gather``
    (oasr/models/conformer/packing.py:222-225, oasr/cache/state.py:88-94)."""
    _need_cuda(src, index, out)
    src = src.contiguous()
    row_bytes = (src.numel() // src.size(0)) * src.element_size() if src.size(0) else 0
    want_shape = (index.numel(),) + tuple(src.shape[1:])
    if out is None:
        out = torch.empty(want_shape, device=src.device, dtype=src.dtype)
    elif tuple(out.shape) != want_shape or out.dtype != src.dtype or not out.is_contiguous() or out.device != src.device:
        raise ValueError(f"out must be a contiguous {src.dtype} tensor of shape {want_shape} on {src.device}")
    if index.dtype != torch.int64:
        index = index.to(torch.int64)
    if index.numel() and row_bytes:
        with torch.cuda.device(src.device):
            _lib.call("oasr_b200_gather_rows", _p(out), _p(src), _p(index.contiguous()), index.numel(), row_bytes,
                      src.size(0), _stream(src))
    return out


def scatter_rows(dst: torch.Tensor, index: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """``dst[index[i]] = src[i]`` (``index_copy_`` along dim 0: unpack_hidden / gapped-conv scatter /
    ``SlotTensor.scatter``); an index outside ``[0, len(dst))`` is skipped."""
    _need_cuda(dst, index, src)
    if not dst.is_contiguous():
        raise ValueError("dst must be contiguous")
    src = src.contiguous()
    if src.dtype != dst.dtype or tuple(src.shape[1:]) != tuple(dst.shape[1:]) or src.size(0) != index.numel():
        raise ValueError("src must hold one row of dst's row shape and dtype per index")
    row_bytes = (src.numel() // src.size(0)) * src.element_size() if src.size(0) else 0
    if index.dtype != torch.int64:
        index = index.to(torch.int64)
    if index.numel() and row_bytes:
        with torch.cuda.device(src.device):
            _lib.call("oasr_b200_scatter_rows", _p(dst), _p(src), _p(index.contiguous()), index.numel(), row_bytes,
                      dst.size(0), _stream(src))
    return dst
