"""The decoding operators where they can go wrong."""
import math

import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import DTYPES, EPS, HALF, attend64, check_scores, chunk, close, form, norm64, pages, pack, quantise64, rand, rope64, score64  # noqa: F401

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


# ---- scores -------------------------------------------------------------------------------------------------------------
LARGE = [1e6, 3e7, 2.0 ** 30, 1e9, 5e9, 1e10, 1e12, 1e15, 1e20, 1e30, 3e37, 9.9e37, 1.1e38, 3e38]
FORMS = [(600, 1000), (5, 2000), (300, 6000), (300, 24001), (3, 9000), (4, 60001)]   # a warp a row, blocks and clusters of four and of sixteen warps


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,V", FORMS)
@pytest.mark.parametrize("sign", [-1, 1])
def test_token_log_probs_of_large_logits(dtype, rows, V, sign):
    """Finite rows of every size: one value alone, neighbours of it, a mask of it with likely tokens left."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(V)
    near = sign * (1 + torch.finfo(dt).eps * torch.randint(0, 5, (V,), generator=g).double())
    left = torch.randperm(V, generator=g)[:40]
    tokens = torch.randint(0, V, (min(rows, 32),), generator=g)
    for size in LARGE:
        x = torch.empty(rows, V, dtype=torch.float64)
        x[0::4] = sign * size
        x[1::4] = (size * near).clamp(-3.3e38, 3.3e38)
        x[2::4] = -size
        x[2::4, left] = 3 * rand(5, 40)
        x[3::4] = sign * size * 0.5
        x[3::4, left[:9]] = sign * size
        # equal rows have equal results: one of each kind is compared with 64 bits, the others with that one
        x = x.to(dt).cuda()
        check_scores(x[:4].contiguous(), tokens[:len(x[:4])].cuda(), 32)
        first, all_ = ob.token_log_probs(x[:4], top_k=32), ob.token_log_probs(x, top_k=32)
        lp, ent, ids = score64(x[:4].cpu().double(), 32)
        tol = (2.0 ** -24 * (V / 32 + 20) + 2.0 ** -20) * (1 + ent.max())      # as in check_scores
        for r in range(len(ids)):
            assert (all_.top_ids[r::4].cpu() == ids[r].int()).all() and (all_.top_ids[r::4] == first.top_ids[r]).all()
            assert ((all_.entropy[r::4].cpu() - ent[r]).abs() <= 2.0 ** -22 * ent[r] + tol).all(), size
            want = lp[r, ids[r]]
            assert ((all_.top_log_probs[r::4].cpu() - want).abs() <= 2.0 ** -22 * want.abs() + tol).all(), size


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V", FORMS + [(3, 8), (700, 8), (2, 1)])
@pytest.mark.parametrize("shift", [0, 1])
def test_token_log_probs_ranks_a_nan_first_wherever_it_is(dtype, rows, V, shift):
    x = (3 * rand(V, rows, V + shift)).to(DTYPES[dtype])[:, shift:]
    x[0, 0] = math.nan                                     # the first token alone
    if rows > 1:
        x[1] = math.nan                                    # nothing else: ids in order
    if rows > 2:
        x[2, 0] = x[2, V - 1] = math.nan
    if rows > 3:
        x[3, 0], x[3, V // 2] = math.inf, math.nan
    tokens = torch.zeros(rows, dtype=torch.int64)
    x = x.cuda() if not shift else torch.empty(rows, V + shift, dtype=x.dtype, device="cuda")[:, shift:].copy_(x)
    for k in {1, min(V, 32)}:
        check_scores(x, tokens.cuda(), k)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V", FORMS + [(2000, 6000), (500, 60001)])
def test_token_log_probs_of_one_token_are_one_number(dtype, rows, V):
    """A token scores the same among the given ones and among the alternatives, and equal logits score the same."""
    x = (3 * rand(V + 9, min(rows, 600), V)).to(DTYPES[dtype]).cuda()
    x = x[torch.arange(rows) % len(x)]
    x[:, -1] = x[:, 0] = x[:, V // 3] = 20.0
    ids = ob.token_log_probs(x, top_k=32).top_ids
    got = ob.token_log_probs(x, ids, top_k=32)
    assert torch.equal(got.top_ids, ids) and torch.equal(got.log_probs, got.top_log_probs)
    assert (got.top_log_probs[:, :3] == got.top_log_probs[:, :1]).all() and got.top_ids[0, :3].tolist() == [0, V // 3, V - 1]


# ---- attention over 4-bit pages -----------------------------------------------------------------------------------------
def attend_bound(q, k, v, scale, lens, partial, dt):
    """``q (B, H, T, D)`` over the first ``lens`` of ``k``, ``v (B, Hkv, N, D)`` in 64 bits: the result, and how far an element may be off.

    A score is a sum of D exact products in steps of 16 on the tensor cores; each of the 17 addends of a step is cut at 2^-23 of the
    largest of them, a product or a partial sum (``partial``: a bound of what that reaches, (B, H, T, N)).  Scores off by at most e
    move weights by a factor within exp(+-2 e), which moves the result by (exp(2 e) - 1) sum p |v - result|.  Weights are rounded to the
    type (their sum is not), and so is the result; 2^-16 is for the exponentials (2^-22 each, their arguments 2^-24 of 126 at most) and sums.
    What a type cannot hold: weights are relative to a maximum that is the row's or up to 2^8 below it, so the largest is 1 or more, and an
    fp16 one below 2^-14 is off by 2^-25 (so is a result); in bf16 exponentials below 2^-126 are zero, relative to a warp's own maximum, whose
    weights may reach 2^8 times that."""
    share = q.shape[1] // k.shape[1]
    k, v = (x.repeat_interleave(share, 1) for x in (k, v))
    seen = torch.arange(k.shape[2]) < torch.tensor(lens)[:, None]
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.softmax(s, -1)
    want = p @ v
    off = 17 * (q.shape[3] // 16) * 2.0 ** -23 * abs(scale) * (partial * seen[:, None, None]).amax(-1, keepdim=True)
    spread = torch.stack([(p[..., j, None] * (v[:, :, None, j] - want).abs()) for j in range(k.shape[2])]).sum(0)
    least = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -118
    tiny = least * (1 + (v.abs() * seen[:, None, :, None]).sum(2, keepdim=True))
    return want, HALF[dt] * want.abs() + (HALF[dt] + 2.0 ** -16) * (p @ v.abs()) + torch.expm1(2 * off) * spread + tiny


def check_attention(q, pools, bt, lens, scale, partial=None):
    """Attention over pools, whose values the gather gives exactly, within the bound above."""
    k, v = (x.cpu().double() for x in ob.gather_paged_kv_q4(*pools, bt.cuda(), None, max(lens)))
    x = q.cpu().double()
    if partial is None:                                    # in whatever order: no partial sum is larger than the sum of magnitudes
        partial = x.abs() @ k.abs().repeat_interleave(x.shape[1] // k.shape[1], 1).transpose(2, 3)
    want, tol = attend_bound(x, k, v, scale, lens, partial, q.dtype)
    got = ob.fmha_q4(q, *pools, softmax_scale=scale, block_table=bt.cuda(), cache_seqlens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, the worst {float((off / tol).max()):.2f} times its bound"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 5, 20, 130])
def test_fmha_q4_scores_of_products_that_cancel(form, dtype, D, T):
    """Queries with a large common offset against keys whose neighbouring dims nearly cancel: moderate scores out of large products."""
    dt, B, H, Hkv, block = DTYPES[dtype], 16, 4, 2, 16
    g = torch.Generator().manual_seed(D + T)
    bt, n = pages(3, B, 1)
    shape = (n, Hkv, block, D // 2)
    even = torch.randint(3, 7, shape, generator=g) * (2 * torch.randint(0, 2, shape, generator=g) - 1)
    few = torch.where(torch.rand(shape, generator=g) < 4 / (D // 2), 2 * torch.randint(0, 2, shape, generator=g) - 1, 0)   # some four pairs of a row
    codes = torch.stack([even, -even + few], -1).flatten(-2)
    v_codes, v_scales = quantise64(rand(4, n, Hkv, block, D), dt)
    k_scales = torch.full((n, Hkv, block, D // 32), 0.375, dtype=dt)
    pools = [pack(codes).cuda(), k_scales.cuda(), pack(v_codes).cuda(), v_scales.to(dt).cuda()]
    q = (256 * 2.0 ** (-6 * torch.rand(B, H, T, D // 2, generator=g, dtype=torch.float64))).repeat_interleave(2, -1).to(dt).cuda()
    lens = torch.randint(2, 7, (B,), generator=g).tolist()
    # a step of 16 holds both dims of a pair in either kernel: partial sums are of pairs, four of which are not zero (or one product)
    k = ob.gather_paged_kv_q4(*pools, bt.cuda(), None, max(lens))[0].cpu().double().repeat_interleave(H // Hkv, 1)
    x = q.cpu().double()
    single = (x[..., None, :] * k[:, :, None]).abs().amax(-1)
    pairs = (x[..., None, :] * k[:, :, None]).unflatten(-1, (-1, 2)).sum(-1).abs().sum(-1)
    check_attention(q, pools, bt, lens, D ** -0.5, torch.maximum(single, pairs))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("size", [300.0, 17.0, 1.0, 1e-3])
def test_fmha_q4_of_scores_of_any_size(form, dtype, D, T, size):
    dt, B, H, Hkv = DTYPES[dtype], 3, 4, 2
    bt, n = pages(5, B, 6)
    pools = []
    for i in range(2):
        codes, scales = quantise64(rand(20 + i, n, Hkv, 16, D), dt)
        pools += [pack(codes).cuda(), scales.to(dt).cuda()]
    check_attention((size * rand(22, B, H, T, D)).to(dt).cuda(), pools, bt, [96, 50, 2], D ** -0.5)


# ---- views --------------------------------------------------------------------------------------------------------------
def odd_view(x, dims):
    """The values of ``x`` behind strides that no kernel may ask for, in dimensions of size 1."""
    buf = torch.empty(x.numel() + 8 * x.dim(), dtype=x.dtype, device=x.device)
    strides = [7 if d in dims else s for d, s in enumerate(x.stride())]
    assert all(x.shape[d] == 1 for d in dims)
    return buf.as_strided(x.shape, strides).copy_(x)


def late(x):
    """The values of ``x``, contiguous, at an address that is a multiple of the element alone."""
    return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape).copy_(x)


def test_fmha_q4_takes_any_query_view():
    bt, n = pages(3, 3, 2)
    codes, scales = quantise64(rand(7, n, 1, 16, 64), torch.bfloat16)
    pools = [pack(codes).cuda(), scales.bfloat16().cuda()] * 2
    for B, H, T in ((1, 1, 1), (3, 2, 1), (1, 4, 5), (3, 1, 2)):
        q = rand(5, B, H, T, 64).bfloat16().cuda()
        how = dict(softmax_scale=0.125, block_table=bt[:B].cuda(), cache_seqlens=torch.full((B,), 20, dtype=torch.int32, device="cuda"))
        want = ob.fmha_q4(q, *pools, **how)
        ones = [d for d in range(3) if q.shape[d] == 1]
        for x in (odd_view(q, ones), late(q), late(q).transpose(1, 2).contiguous().transpose(1, 2)):
            assert torch.equal(ob.fmha_q4(x, *pools, **how), want)
        out = odd_view(torch.empty_like(q), ones)
        assert ob.fmha_q4(q, *pools, out=out, **how) is out and torch.equal(out, want)


@pytest.mark.parametrize("q4", [False, True])
def test_write_kv_rope_takes_any_stride_of_one(q4):
    table = ob.rope_table(64, 64)
    for B, H, T in ((1, 1, 1), (2, 1, 1), (1, 2, 3), (1, 1, 4)):
        q, k, v = (rand(s, B, H, T, 64).bfloat16().cuda() for s in (1, 2, 3))
        bt = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
        ones = [d for d in range(3) if q.shape[d] == 1]
        got = []
        for view in (lambda x: x, lambda x: odd_view(x, ones)):
            pools = ob.PagedKVCacheQ4.empty_pools(B, H, 16, 64) if q4 else [torch.zeros(B, 16, H, 64, device="cuda").bfloat16() for _ in range(2)]
            out = view(torch.empty_like(q))
            write = ob.write_kv_rope_q4 if q4 else ob.write_kv_rope
            assert write(*pools, bt, view(k), view(v), 2, table, q=view(q), q_out=out) is out
            got.append([out, *pools])
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_qk_norm_rope_takes_any_stride_of_one():
    table = ob.rope_table(64, 64)
    for N, H in ((1, 1), (1, 3), (4, 1)):
        q, pos = rand(1, N, H, 64).bfloat16().cuda(), torch.arange(N, device="cuda") + 3
        want = ob.qk_norm_rope(q, q, table, pos)
        ones = [d for d in range(2) if q.shape[d] == 1]
        outs = [odd_view(torch.empty_like(q), ones) for _ in range(2)]
        for how in ({}, dict(q_out=outs[0], k_out=outs[1])):
            got = ob.qk_norm_rope(odd_view(q, ones), odd_view(q, ones), table, pos, **how)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- 4-bit codes, each within its bound ---------------------------------------------------------------------------------
def five_bits(x, dt):
    """The scale of a group whose largest magnitude is ``x``, in 64 bits."""
    m, e = torch.frexp(x / 7)
    lo, hi = (2.0 ** -20, 9216.0) if dt == torch.float16 else (2.0 ** -120, 1.125 * 2.0 ** 125)
    return torch.ldexp(torch.ceil(m * 32) / 32, e).clamp(lo, hi)


def unpacked(codes):
    """(..., D / 2) bytes -> (..., D) codes."""
    D = 2 * codes.shape[-1]
    nib = torch.stack([codes.long() & 15, codes.long() >> 4], -1).flatten(-2) - 8
    d = torch.arange(D)
    return nib[..., ((d % 32) // 8 * (D // 32) + d // 32) * 8 + d % 8].double()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("B,H,Hkv,T,D,R,block,inter", [
    (1, 8, 8, 1, 64, 64, 16, False), (5, 16, 4, 1, 128, 128, 16, False), (3, 4, 1, 17, 64, 32, 16, False), (4, 2, 2, 33, 64, 64, 32, True), (3, 3, 1, 5, 96, 32, 16, False),
    (37, 8, 2, 16, 64, 64, 16, False), (2, 2, 1, 3, 32, 16, 16, False), (2, 1, 1, 9, 256, 128, 16, True), (2, 1, 3, 40, 128, 96, 16, False), (3, 1, 1, 30, 512, 512, 16, False)])
def test_every_code_is_as_near_as_fp32_can_tell(dtype, norm, B, H, Hkv, T, D, R, block, inter):
    dt = DTYPES[dtype]
    _, k, v = chunk(15, B, H, Hkv, T, D, dt, T % 2 == 1)
    kw = (1 + 0.2 * rand(3, D)).to(dt).cuda() if norm else None
    table = ob.rope_table(400, R)
    g = torch.Generator().manual_seed(16)
    off, lens = torch.randint(0, 60, (B,), generator=g), torch.randint((T + 1) // 2, T + 1, (B,), generator=g)
    bt, n = pages(17, B, -(-(60 + T) // block))
    before = [torch.randint(1, 255, p.shape, generator=g, dtype=torch.uint8) if p.dtype == torch.uint8 else rand(9, *p.shape).abs().to(dt)
              for p in ob.PagedKVCacheQ4.empty_pools(n, Hkv, block, D, dt, device="cpu")]
    after = [p.clone().cuda() for p in before]
    ob.write_kv_rope_q4(*after, bt.cuda(), k, v, off.cuda(), table, k_weight=kw, eps=EPS, interleaved=inter, new_lens=lens.cuda())
    after = [p.cpu() for p in after]
    written = torch.zeros(n, block, dtype=torch.bool)
    for b in range(B):
        m = int(lens[b])
        pos = int(off[b]) + torch.arange(m)
        page, slot = bt[b].long()[pos // block], pos % block
        written[page, slot] = True
        kn = norm64(k[b].transpose(0, 1)[:m].cpu().double(), None if kw is None else kw.cpu())
        for i, x, e in ((0, rope64(kn, table.cpu(), pos, inter), None), (2, v[b].transpose(0, 1)[:m].cpu().double(), 0.0)):
            if e is None:
                # in fp32: the sum of squares 16 + 5 steps, mean and eps 3 more, all halved by the root, the root 4, two products; a rotation's
                # two products and sum, each of at most sqrt(2) of the row's largest
                e = (18 + 2) * 2.0 ** -24 * 1.42 * kn.abs().amax(-1, keepdim=True) if norm else 2 * 2.0 ** -24 * 1.42 * kn.abs().amax(-1, keepdim=True)
            e = torch.as_tensor(e, dtype=torch.float64).expand(*x.shape[:-1], 1)
            codes, scales = unpacked(after[i][page, :, slot]), after[i + 1][page, :, slot].double()
            top = x.unflatten(-1, (-1, 32)).abs().amax(-1)
            near = e + 2.0 ** -24 * top if i == 0 else e      # (and its quotient by 7 rounds)
            assert ((scales == five_bits(top - near, dt)) | (scales == five_bits(top + near, dt))).all()
            quotient = x / scales.repeat_interleave(32, -1)
            assert (codes.abs() <= 7).all() and ((codes - quotient.clamp(-7, 7)).abs() <= 0.5 + e / scales.repeat_interleave(32, -1)).all()
    for a, b in zip(after, before):
        assert torch.equal(a.transpose(1, 2)[~written], b.transpose(1, 2)[~written])


# ---- wide indices -------------------------------------------------------------------------------------------------------
def test_64_bit_indices_outside_32_bits_are_outside():
    """int64 tables and numbers: 2^32 more than a page is no page, and what lies beyond 32 bits counts as far."""
    B, H, D = 6, 2, 64
    bt, n = pages(3, B, 2)
    bt = bt.long()
    far = bt.clone()
    far[0, 0] += 2 ** 32
    far[1, 1], far[2, 0], far[2, 1] = -2 ** 63, 2 ** 63 - 1, -2 ** 32
    none = far.where((far >= 0) & (far < n), torch.tensor(-1)).int().cuda()
    far, table = far.cuda(), ob.rope_table(64, D)
    q, k, v = (rand(s, B, H, 3, D).bfloat16().cuda() for s in (1, 2, 3))
    off = torch.tensor([0, 14, 0, 2 ** 32, -2 ** 32, 5], device="cuda")
    off32 = torch.tensor([0, 14, 0, 2 ** 31 - 1, -2 ** 31, 5], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20, 20, 20, 2 ** 32 + 5, 2 ** 33, -2 ** 40], device="cuda")
    lens32 = torch.tensor([20, 20, 20, 2 ** 31 - 1, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 0, 0, -2 ** 40, 2 ** 32, 0], device="cuda")
    start32 = torch.tensor([0, 0, 0, 0, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    got = []
    for t, o, length, s in ((far, off, lens, start), (none, off32, lens32, start32)):
        pools = ob.PagedKVCacheQ4.empty_pools(n, H, 16, D)
        plain = [torch.zeros(n, 16, H, D, device="cuda").bfloat16() for _ in range(2)]
        for p, write in ((pools, ob.write_kv_rope_q4), (plain, ob.write_kv_rope)):
            write(*p, t, k, v, o, table, new_lens=length.clamp(0, 3))
        att = ob.fmha_q4(q, *pools, softmax_scale=0.125, block_table=t, cache_seqlens=length, cache_seqstarts=s)
        got.append([*pools, *plain, att, *ob.gather_paged_kv_q4(*pools, t, o, 9)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ---- tables wider than the sequences, windows ---------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("wide", [1, 4, 32])
@pytest.mark.parametrize("window", [False, True])
def test_fmha_q4_in_a_table_wider_than_its_sequences(form, D, T, wide, window):
    """As a cache of (slots, most pages) hands it out; entries behind the length are of other sequences' pages or none."""
    B, H, Hkv, dt = 3, 4, 2, torch.bfloat16
    lens = [300, 47, 130]
    starts = [250, 0, 129] if window else None
    bt, n = pages(5, B, 19)
    table = torch.randint(-1, n + 1, (B, 19 * wide), generator=torch.Generator().manual_seed(wide)).int()
    table[:, :19] = bt
    pools = []
    for i in range(2):
        codes, scales = quantise64(rand(20 + i, n, Hkv, 16, D), dt)
        pools += [pack(codes).cuda(), scales.to(dt).cuda()]
    q = rand(22, B, H, T, D).to(dt).cuda()
    cuda = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ob.fmha_q4(q, *pools, softmax_scale=D ** -0.5, block_table=table.cuda(), cache_seqlens=cuda(lens), cache_seqstarts=cuda(starts), causal=True)
    k, v = (x.cpu().double() for x in ob.gather_paged_kv_q4(*pools, bt.cuda(), None, max(lens)))
    want = attend64(q.cpu().double(), k, v, D ** -0.5, lens, starts, None, True)
    # half a step of the weights and of the result, and a score's fp32 sum: D products of at most 30 in all, 2^-23 of that for each of D / 16 steps of 17
    close(got, want, HALF[dt], float(v.abs().max()) * (HALF[dt] + 2 * 17 * (D // 16) * 2.0 ** -23 * 30))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("T", [1, 9, 150])
def test_fmha_q4_of_negative_lengths(form, causal, T):
    """A length below zero is one of zero, down to the type's lowest, from which no more can be taken."""
    bt, n = pages(3, 5, 4)
    codes, scales = quantise64(rand(7, n, 1, 16, 64), torch.bfloat16)
    pools = [pack(codes).cuda(), scales.bfloat16().cuda()] * 2
    q = rand(5, 5, 2, T, 64).bfloat16().cuda()
    how = dict(softmax_scale=0.125, block_table=bt.cuda(), causal=causal)
    lens = torch.tensor([-2 ** 31, -2 ** 31 + 3, -1, 0, 60], device="cuda")
    for kind in (torch.int32, torch.int64):
        out = ob.fmha_q4(q, *pools, cache_seqlens=lens.to(kind), **how)
        assert not out[:4].any() and out[4].any()
    assert torch.equal(ob.fmha_q4(q, *pools, cache_seqlens=torch.tensor([-2 ** 40, -2 ** 63, -7, 0, 60], device="cuda"), **how), out)
