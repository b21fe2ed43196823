"""Drafted tokens over paged caches on the GPU, against plain implementations in 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

import oasr_b200 as ob
import oasr_b200.tunables
from tests.test_gpu_decoding import DTYPES, HALF, close, pages, rand

pytestmark = pytest.mark.gpu


def i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- trees --------------------------------------------------------------------------------------------------------------
def random_parents(seed, B, T, width, odd=0.0):
    """Each node continues one of the `width` before it; a share `odd` of them has a parent that is none."""
    r = random.Random(seed)
    return [[r.randint(-2, T + 1) if i == 0 else r.choice((-1, -7, i, T, 2 ** 31 - 1, -2 ** 31)) if r.random() < odd else max(0, i - 1 - r.randrange(min(width, i)))
             for i in range(T)] for _ in range(B)]


def ways(parents):
    out = [[0]]
    for i, p in enumerate(parents[1:], 1):
        out.append(out[p] + [i] if 0 <= p < i and out[p] else [])
    return out


def words_of(rows, T):
    w = np.zeros((len(rows), (T + 31) // 32), np.int64)
    for i, row in enumerate(rows):
        for j in row:
            w[i, j // 32] |= 1 << j % 32
    return torch.from_numpy(w.astype(np.uint32).view(np.int32).copy())


@pytest.mark.parametrize("B,T,width,odd", [(1, 1, 1, 0), (3, 2, 1, 0.3), (2, 32, 3, 0), (5, 33, 4, 0.1), (1, 64, 1, 0), (7, 255, 24, 0.02), (2, 1024, 1, 0), (2, 1000, 9, 0.01), (300, 40, 2, 0.05)])
def test_draft_tree(B, T, width, odd):
    parents = random_parents(B * T, B, T, width, odd)
    got = ob.draft_tree(i32(parents))
    assert got.mask.shape == (B, T, (T + 31) // 32) and got.depth.shape == (B, T) and got.mask.dtype == got.depth.dtype == torch.int32
    for b in range(B):
        w = ways(parents[b])
        assert torch.equal(got.mask[b].cpu(), words_of(w, T)) and got.depth[b].tolist() == [len(x) - 1 for x in w]
    one = ob.draft_tree(torch.tensor(parents[0], device="cuda"))
    assert torch.equal(one.mask, got.mask[0]) and torch.equal(one.depth, got.depth[0])
    strided = torch.stack([i32(parents), i32(parents)], 2)[:, :, 0]
    assert torch.equal(ob.draft_tree(strided).mask, got.mask)


def test_draft_tree_of_nothing():
    for shape in ((0, 5), (3, 0), (0,)):
        t = ob.draft_tree(torch.zeros(shape, dtype=torch.int32, device="cuda"))
        assert t.mask.shape == (*shape, (shape[-1] + 31) // 32) and t.depth.shape == shape


# ---- attention ----------------------------------------------------------------------------------------------------------
@pytest.fixture(params=[0, 1, 2], ids=["by_size", "few_rows", "many_rows"])
def tree_form(request):
    """Both kernels of fmha_tree, and the choice between them."""
    ob.tunables.set("fmha_tree_path", request.param)
    yield request.param
    ob.tunables.set("fmha_tree_path", 0)


def pool16(seed, n, block, Hkv, D, dt):
    return [rand(seed + i, n, block, Hkv, D).to(dt).cuda() for i in range(2)]


def dense16(pools, bt):
    """k, v (B, Hkv, N, D) in 64 bits, and which positions have a page."""
    n = len(pools[0])
    known = (bt >= 0) & (bt < n)
    k, v = (p.cpu()[torch.where(known, bt, 0).long()].flatten(1, 2).transpose(1, 2).double() for p in pools)
    return k, v, known.repeat_interleave(pools[0].shape[1], 1)


def tree64(q, k, v, scale, lens, starts, q_lens, rows, known):
    """``rows[b][t]``: the nodes that row t sees.  -> result, and for each row the sum of weights times |v|."""
    B, H, T, _ = q.shape
    share, out, size = H // k.shape[1], torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        live = T if q_lens is None else min(max(int(q_lens[b]), 0), T)
        n = max(int(lens[b]), 0)
        lo = 0 if starts is None else max(int(starts[b]), 0)
        for t in range(live):
            at = list(range(lo, max(n - live, lo))) + [n - live + u for u in sorted(set(rows[b][t])) if u < live and n - live + u >= lo]
            at = [j for j in at if j < k.shape[2] and known[b, j]]
            if not at:
                continue
            kk, vv = k[b, :, at].repeat_interleave(share, 0), v[b, :, at].repeat_interleave(share, 0)
            p = torch.softmax((kk @ q[b, :, t, :, None])[..., 0] * scale, -1)
            out[b, :, t] = (p[:, None] @ vv)[:, 0]
            size[b, :, t] = (p[:, None] @ vv.abs())[:, 0]
    return out, size


def bound(q, k, scale, size, want, dt):
    """How far a result may be off.  A weight is rounded to the type (half a step, relative; with fp16 2^-25 of the largest at least, with bf16 and in
    fp32 exponentials below 2^-118 of it vanish: of each of N keys, times |v| < 8) and so is the result.  A score is a sum of D exact products in fp32: off by at most D steps of the
    sum of magnitudes, which moves its weight by as much; the exponential and its argument are off by 2^-22 and 2^-24 of 126 (2^-16 for all)."""
    share = q.shape[1] // k.shape[1]
    worst = (q.abs() @ torch.nan_to_num(k.abs(), 0, 0, 0).repeat_interleave(share, 1).transpose(2, 3)).amax() * abs(scale)
    off = 2 * torch.expm1(q.shape[3] * 2.0 ** -23 * worst)
    least = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -118
    return HALF[dt] * want.abs() + (HALF[dt] + 2.0 ** -16 + float(off)) * size + least * 8 * (1 + k.shape[2])


def check(got, want, tol):
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, the worst {float((off / tol).max()):.2f} times its bound"


CASES = [  # B, H, Hkv, T, D, block, lens, starts, q_lens, width
    (1, 8, 8, 1, 64, 16, [300], None, None, 1), (1, 1, 1, 1, 128, 16, [1], None, None, 1), (3, 8, 2, 1, 128, 16, [0, 1, 33], None, None, 1),
    (2, 4, 4, 16, 64, 16, [16, 250], [0, 100], None, 3), (2, 14, 2, 5, 64, 32, [70, 31], None, [5, 2], 2), (2, 8, 1, 17, 128, 48, [96, 17], None, [17, 9], 4),
    (1, 2, 1, 130, 64, 16, [130], None, None, 8), (2, 6, 2, 33, 128, 128, [200, 40], [190, 20], None, 5), (4, 4, 1, 1, 64, 64, [640, 639, 513, 65], [0, 639, 64, 65], None, 1),
    (1, 3, 1, 70, 64, 16, [40], None, None, 6), (2, 32, 8, 3, 128, 16, [1000, 7], None, [3, 0], 2), (1, 1, 1, 300, 128, 16, [333], None, [257], 30),
    (3, 16, 2, 16, 64, 16, [5000, 16, 777], None, None, 4), (1, 14, 2, 16, 128, 128, [9001], None, None, 4), (2, 32, 8, 61, 128, 16, [700, 3001], None, [61, 40], 8),
    (1, 4, 4, 40, 64, 16, [2500], [2470], None, 7), (5, 8, 2, 2, 128, 16, [1, 0, 2, 3, 100], None, [1, 2, 2, 2, 2], 1), (2, 16, 1, 9, 64, 32, [4097, 30], None, None, 3),
    (1, 4, 1, 40, 64, 64, [40000], None, None, 4), (5, 16, 8, 20, 64, 16, [2000, 1500, 20, 700, 1999], None, [20, 7, 20, 0, 19], 3), (3, 16, 8, 9, 128, 32, [3300, 2000, 100], [0, 1990, 99], None, 2),
    (40, 8, 8, 3, 128, 16, [(i * 997) % 2100 // (i % 3 + 1) + 3 for i in range(40)], [i % 5 for i in range(40)], [i % 4 for i in range(40)], 1)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hkv,T,D,block,lens,starts,q_lens,width", CASES)
def test_fmha_tree(tree_form, dtype, B, H, Hkv, T, D, block, lens, starts, q_lens, width):
    dt = DTYPES[dtype]
    bt, n = pages(3, B, -(-max(max(lens), 1) // block) + 1)
    pools = pool16(10, n, block, Hkv, D, dt)
    q = rand(12, B, T, H, D).to(dt).cuda().transpose(1, 2)
    rows = [ways(p) for p in random_parents(T, B, T, width, 0.1 if T > 4 else 0)]
    mask = torch.stack([words_of(r, T) for r in rows]).cuda()
    how = dict(softmax_scale=D ** -0.5, block_table=bt.cuda(), cache_seqlens=i32(lens), cache_seqstarts=i32(starts), q_lens=i32(q_lens))
    got = ob.fmha_tree(q, *pools, tree_mask=mask, **how)
    k, v, known = dense16(pools, bt)
    x = q.cpu().double()
    want, size = tree64(x, k, v, D ** -0.5, lens, starts, q_lens, rows, known)
    check(got, want, bound(x, k, D ** -0.5, size, want, dt))
    assert torch.equal(got, ob.fmha_tree(q, *pools, tree_mask=mask, **how))                       # the same bits again
    major = ob.fmha_tree(q, *pools, tree_mask=mask, token_major=True, **how)
    assert major.shape == (B, T, H, D) and torch.equal(major.transpose(1, 2), got)
    wide = torch.full((B, H, T, 2 * D), 7.0, dtype=dt, device="cuda")
    ob.fmha_tree(q.contiguous(), *pools, tree_mask=mask, out=wide[..., :D], **how)
    assert torch.equal(wide[..., :D], got) and (wide[..., D:] == 7).all()
    # one tree for all, and none
    same = ob.fmha_tree(q, *pools, tree_mask=mask[0], **how)
    assert torch.equal(same, ob.fmha_tree(q, *pools, tree_mask=mask[:1].expand(B, -1, -1), **how)) and torch.equal(same[0], got[0])
    chain = [list(range(t + 1)) for t in range(T)]
    none = ob.fmha_tree(q, *pools, **how)
    assert torch.equal(none, ob.fmha_tree(q, *pools, tree_mask=words_of(chain, T).cuda(), **how))
    want, size = tree64(x, k, v, D ** -0.5, lens, starts, q_lens, [chain] * B, known)
    check(none, want, bound(x, k, D ** -0.5, size, want, dt))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,D,share", [(1, 64, 2), (6, 128, 4), (20, 64, 2), (70, 128, 4)])
def test_fmha_tree_unseen_keys_say_nothing(tree_form, dtype, T, D, share):
    """NaN and infinities behind the length and before the start, pages outside the pool, a table wider than the length, rows that see nothing."""
    dt, block = DTYPES[dtype], 16
    lens, starts = [100 + T, 77 + T, T], [5, 2, 0]
    bt, n = pages(3, 3, 12 + T // 16)
    pools = pool16(10, n, block, 2, D, dt)
    bt[0, 3], bt[1, 0] = -1, n                          # keys 48..63 of one, 0..15 of the other
    k, v, known = dense16(pools, bt)
    for b in range(3):
        for j in list(range(starts[b])) + list(range(lens[b], bt.shape[1] * block)):
            if known[b, j]:
                for p in pools:
                    p[bt[b, j // block], j % block] = (math.nan, math.inf, -math.inf)[j % 3]
    q = rand(12, 3, 2 * share, T, D).to(dt).cuda()
    rows = [[[] if t % 3 == 1 else [u for u in range(T) if (u * 7 + t) % 3] for t in range(T)] for _ in range(3)]
    got = ob.fmha_tree(q, *pools, softmax_scale=0.125, block_table=bt.cuda(), cache_seqlens=i32(lens), cache_seqstarts=i32(starts),
                       tree_mask=torch.stack([words_of(r, T) for r in rows]).cuda())
    x = q.cpu().double()
    want, size = tree64(x, k, v, 0.125, lens, starts, None, rows, known)
    assert not want[2, :, 1::3].any()
    k = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    check(got, want, bound(x, k, 0.125, size, want, dt))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,D,share", [(3, 64, 1), (12, 128, 4), (40, 64, 2), (70, 128, 4)])
def test_fmha_tree_nan_reaches_the_rows_that_see_it_and_no_other(tree_form, dtype, T, D, share):
    dt, block, N = DTYPES[dtype], 16, T + 90
    bt, n = pages(3, 1, -(-N // block))
    pools = pool16(10, n, block, 2, D, dt)
    k, v, known = dense16(pools, bt)
    q = rand(12, 1, 2 * share, T, D).to(dt).cuda()
    q[0, 0, 0] = math.nan
    rows = [sorted({t, t // 2, 0}) for t in range(T)]
    def put(pool, u, head, dim, value):
        pool[bt[0, (N - T + u) // block], (N - T + u) % block, head, dim] = value
    put(pools[0], T - 1, 0, 3, math.nan)                  # a key of head 0: the rows that see node T - 1
    put(pools[1], 1, 1, 5, math.nan)                      # values of head 1
    put(pools[1], 1, 1, D - 1, math.inf)
    put(pools[1], 2, 1, 9, -math.inf)
    got = ob.fmha_tree(q, *pools, softmax_scale=0.125, block_table=bt.cuda(), cache_seqlens=i32([N]), tree_mask=words_of(rows, T).cuda()).cpu().double()
    x = q.nan_to_num(0).cpu().double()
    want, size = tree64(x, k, v, 0.125, [N], None, None, [rows], known)
    tol = bound(x, k, 0.125, size, want, dt)
    for t in range(T):
        if t == T - 1:
            want[0, :share, t] = math.nan
        if 1 in rows[t]:
            want[0, share:, t, 5], want[0, share:, t, D - 1] = math.nan, math.inf
        if 2 in rows[t]:
            want[0, share:, t, 9] = -math.inf
    want[0, 0, 0] = math.nan
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    fine = torch.isfinite(want)
    check(got[fine], want[fine], tol[fine])


@pytest.mark.parametrize("T", [1, 5, 40, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_fmha_tree_of_scores_of_any_size(tree_form, T, D):
    """One key with all the weight, equal weights, a scale of zero and one below it."""
    N = 200 + T
    bt, n = pages(3, 1, 20)
    pools = pool16(10, n, 16, 1, D, torch.bfloat16)
    k, v, known = dense16(pools, bt)
    chain = [list(range(t + 1)) for t in range(T)]
    for size_of, scale in ((1e-3, 1.0), (1.0, 0.0), (1.0, -0.2), (1.0, 1e-40), (30.0, 1.0)):
        q = (size_of * rand(12, 1, 4, T, D)).bfloat16().cuda()
        got = ob.fmha_tree(q, *pools, softmax_scale=scale, block_table=bt.cuda(), cache_seqlens=i32([N]))
        x = q.cpu().double()
        want, size = tree64(x, k, v, scale, [N], None, None, [chain], known)
        check(got, want, bound(x, k, scale, size, want, torch.bfloat16) + size_of * 1e-3 * (size_of > 1) * v.abs().max())


def test_fmha_tree_lengths_outside_the_table(tree_form):
    """Lengths below zero, below the tree's, and of more than the table has; 64-bit tables and lengths."""
    T, D = 4, 64
    bt, n = pages(3, 4, 3)
    pools = pool16(10, n, 16, 2, D, torch.float16)
    k, v, known = dense16(pools, bt)
    q = rand(12, 4, 4, T, D).half().cuda()
    rows = [[[0], [0, 1], [0, 2], [0, 1, 3]]] * 4
    lens = [-5, 2, 49, 2 ** 31 - 1]
    how = dict(softmax_scale=0.2, tree_mask=words_of(rows[0], T).cuda())
    got = ob.fmha_tree(q, *pools, block_table=bt.cuda(), cache_seqlens=i32(lens), **how)
    x = q.cpu().double()
    # (a sequence of 2 whose tree has 4 nodes: nodes 2 and 3 lie at positions 0 and 1)
    ref = torch.zeros_like(x)
    sizes = torch.zeros_like(x)
    for b, n_ in ((1, 2), (2, 49), (3, 2 ** 31 - 1)):
        prefix = n_ - T
        for t in range(T):
            at = [j for j in range(48) if j < min(n_, 48) and (j < prefix or j - prefix in rows[b][t])]
            if at:
                for h in range(4):
                    p = torch.softmax(k[b, h // 2, at] @ x[b, h, t] * 0.2, 0)
                    ref[b, h, t], sizes[b, h, t] = p @ v[b, h // 2, at], p @ v[b, h // 2, at].abs()
    check(got, ref, bound(x, k, 0.2, sizes, ref, torch.float16))
    wide = torch.where(bt == 1, 2 ** 32 + 1, bt.long())           # a page outside 32 bits is no page
    got64 = ob.fmha_tree(q, *pools, block_table=wide.cuda(), cache_seqlens=torch.tensor(lens, device="cuda"), **how)
    same = ~(bt == 1).any(1)
    assert torch.equal(got64[same.cuda()], got[same.cuda()])


def test_fmha_tree_takes_any_query_view(tree_form):
    T, D = 6, 64
    bt, n = pages(3, 2, 8)
    pools = pool16(10, n, 16, 2, D, torch.bfloat16)
    how = dict(softmax_scale=0.125, block_table=bt.cuda(), cache_seqlens=i32([100, 37]))
    q = rand(12, 2, 4, T, D).bfloat16().cuda()
    want = ob.fmha_tree(q, *pools, **how)
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view_as(q).copy_(q)       # 2 bytes off
    last = q.transpose(2, 3).contiguous().transpose(2, 3)                                        # D not innermost
    odd = torch.empty(2, 4, T, D + 3, dtype=q.dtype, device="cuda")[..., :D].copy_(q)
    for view in (flat, last, odd, q.transpose(0, 2).contiguous().transpose(0, 2)):
        assert torch.equal(ob.fmha_tree(view, *pools, **how), want)
    one = q[:1, :, :1]
    assert torch.equal(ob.fmha_tree(one.as_strided((1, 4, 1, D), (3, T * D, 5, 1)), *pools, softmax_scale=0.125, block_table=bt[:1].cuda(), cache_seqlens=i32([50])),
                       ob.fmha_tree(one.contiguous(), *pools, softmax_scale=0.125, block_table=bt[:1].cuda(), cache_seqlens=i32([50])))


def test_fmha_tree_far_pages(tree_form):
    """Rows behind 2^31 elements of a pool."""
    Hkv, D, block, n = 8, 128, 128, 16500                      # 2.16e9 elements a pool
    pools = [torch.zeros(n, block, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    bt = torch.tensor([[n - 1, 3, n - 2]], dtype=torch.int32)
    for i, p in enumerate(pools):
        p[bt[0].long().cuda()] = rand(5 + i, 3, block, Hkv, D).half().cuda()
    small = [p[bt[0].long().cuda()] for p in pools]
    q = rand(9, 1, 16, 5, D).half().cuda()
    how = dict(softmax_scale=0.1, cache_seqlens=i32([300]))
    assert torch.equal(ob.fmha_tree(q, *pools, block_table=bt.cuda(), **how), ob.fmha_tree(q, *small, block_table=i32([[0, 1, 2]]), **how))
    ob.commit_drafts(pools, bt.cuda(), 250, i32([[0, 9, 49]]), i32([3]))
    want = [s.clone() for s in small]
    for s in want:
        rows = s.view(3 * block, Hkv, D)
        rows[251], rows[252] = rows[259].clone(), rows[299].clone()
    assert all(torch.equal(p[bt[0].long().cuda()], w) for p, w in zip(pools, want))


def test_fmha_tree_refusals():
    pool = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    q, bt, lens, mask = pool(2, 4, 3, 64), i32([[0, 1], [2, 3]]), i32([3, 3]), i32([[1], [3], [7]])
    good = dict(q=q, k_cache=pool(4, 16, 2, 64), v_cache=pool(4, 16, 2, 64), softmax_scale=1.0, block_table=bt, cache_seqlens=lens, tree_mask=mask)
    for how in [dict(block_table=bt[:1]), dict(cache_seqlens=lens[:1]), dict(q_lens=lens[:1]), dict(cache_seqstarts=lens[:1]), dict(q=q[:, :3]), dict(q=q.half()), dict(q=q[0]), dict(q=q.float()),
                dict(out=pool(2, 4, 2, 64)), dict(out=q[:, :1].expand_as(q)), dict(v_cache=pool(4, 16, 2, 128)), dict(k_cache=pool(4, 16, 2, 128)[..., :64]), dict(tree_mask=mask[:2]),
                dict(tree_mask=mask.long()), dict(tree_mask=mask[None]), dict(tree_mask=torch.cat([mask, mask], 1)), dict(cache_seqlens=lens.cpu()), dict(tree_mask=mask.cpu()),
                dict(k_cache=pool(4, 8, 2, 64), v_cache=pool(4, 8, 2, 64)), dict(softmax_scale=math.nan), dict(q=pool(2, 4, 3, 96), k_cache=pool(4, 16, 2, 96), v_cache=pool(4, 16, 2, 96))]:
        with pytest.raises((RuntimeError, ValueError)):
            ob.fmha_tree(**(good | how))
    assert not ob.fmha_tree(**(good | dict(q=q + 1, block_table=bt[:, :0]))).any()
    assert ob.fmha_tree(**(good | dict(q=q[:, :, :0], tree_mask=None))).shape == (2, 4, 0, 64)
    assert ob.fmha_tree(**(good | dict(q=q[:0], block_table=bt[:0], cache_seqlens=lens[:0]))).shape == (0, 4, 3, 64)


# ---- verification -------------------------------------------------------------------------------------------------------
def target64(x, temp):
    """Probabilities of a row in 64 bits, or None."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or not np.isfinite(x.max()):
        return None
    if not temp > 0:
        return (np.arange(len(x)) == np.argmax(x)).astype(np.float64)
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp((x - x.max()) / temp)
    return e / e.sum()


def verify64(logits, drafts, parents, u, temps, probs):
    """(tokens, path, counts), and how near the nearest decision was."""
    B, T, V = logits.shape
    tokens, path, counts, near = np.full((B, T), -1), np.full((B, T), -1), np.zeros(B, int), math.inf
    for b in range(B):
        n, m = 0, 0
        while True:
            path[b, m] = n
            p, nxt = target64(logits[b, n], temps[b]), None
            q = None if probs is None else probs[b, n].astype(np.float64)
            for c in range(n + 1, T):
                x = drafts[b, c]
                if p is None or parents[b, c] != n or not 0 <= x < V:
                    continue
                qx = 1.0 if q is None else q[x]
                if temps[b] > 0:
                    near = min(near, abs(u[b, c] * qx - p[x]) / max(p[x], qx, 1e-30))
                if u[b, c] * qx < p[x]:
                    nxt = c
                    break
                if q is None:
                    p[x] = 0.0
                else:
                    p = np.maximum(p - q, 0)
                p = p / p.sum() if p.sum() > 0 else p
            if nxt is not None:
                tokens[b, m] = drafts[b, nxt]
                n, m = nxt, m + 1
                continue
            if p is not None and p.sum() > 0:
                total = np.cumsum(p)
                goal = u[b, 0] * total[-1]
                if temps[b] > 0:
                    near = min(near, float(np.abs(total[p > 0][:-1] - goal).min(initial=math.inf)))
                tokens[b, m] = min(int(np.searchsorted(total, goal, side="right")), int(np.nonzero(p)[0][-1]))
            break
        counts[b] = m + 1
    return tokens, path, counts, near


def check_verify(logits, drafts, parents, u, temps, probs=None, margin=1e-9):
    """``logits`` on the GPU, the others as arrays.  A decision nearer than 1e-9 to its border is a bad input for this test, not a fault."""
    B = len(logits)
    t32 = np.asarray(temps, np.float32)
    tokens, path, counts, near = verify64(logits.float().cpu().numpy(), drafts, parents, u, t32.astype(np.float64), None if probs is None else probs.cpu().numpy())
    assert near > margin, "choose other inputs"
    got = ob.verify_drafts(logits, torch.from_numpy(drafts).cuda(), torch.from_numpy(parents).cuda(), torch.from_numpy(u).cuda(), temperature=torch.from_numpy(t32).cuda(), draft_probs=probs)
    assert got.counts.tolist() == counts.tolist()
    assert got.path.tolist() == path.tolist()
    assert got.tokens.tolist() == tokens.tolist()
    assert got.tokens.dtype == got.path.dtype == got.counts.dtype == torch.int32 and got.counts.shape == (B,)
    return got


def verify_inputs(seed, B, T, V, width, dt, drawn, odd=0.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.RandomState(seed)
    parents = np.array(random_parents(seed, B, T, width, odd), np.int64)
    x = 2.5 * torch.randn(B, T, V + pad, generator=g)
    drafts = rng.randint(0, V, (B, T))
    probs = None
    if drawn:
        probs = torch.softmax(x[..., :V].double() + 0.7 * torch.randn(B, T, V, generator=g).double(), -1).float()
        for b in range(B):
            for i in range(1, T):
                if 0 <= parents[b, i] < i:
                    drafts[b, i] = int(torch.multinomial(probs[b, parents[b, i]], 1, generator=g))
        probs = probs.cuda()
    else:
        for b in range(B):
            for i in range(1, T):
                if 0 <= parents[b, i] < i:
                    x[b, parents[b, i], drafts[b, i]] = math.log(V) + 2 + 2 * rng.rand()
    u = rng.rand(B, T).astype(np.float32)
    return x.to(dt).cuda()[..., :V], drafts, parents, u, probs


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("B,T,V,width,pad,odd", [(1, 1, 1, 1, 0, 0), (3, 5, 7, 1, 0, 0), (2, 9, 100, 3, 1, 0.1), (40, 6, 300, 2, 4, 0), (5, 40, 1000, 6, 0, 0.05), (3, 5, 5002, 1, 6, 0),
                                                 (90, 3, 5002, 2, 0, 0), (7, 12, 40001, 4, 0, 0.1), (2, 8, 131071, 2, 1, 0), (1, 48, 65537, 5, 0, 0), (160, 2, 9000, 1, 0, 0)])
def test_verify_drafts(dtype, drawn, B, T, V, width, pad, odd):
    x, drafts, parents, u, probs = verify_inputs(V + T, B, T, V, width, DTYPES[dtype], drawn, odd, pad)
    temps = 0.5 + np.random.RandomState(3).rand(B)
    temps[1::4] = 0.0
    got = check_verify(x, drafts, parents, u, temps, probs)
    if T > 2 and B > 2 and not odd:
        assert got.counts.max() > 1                         # something was accepted
    # an offset view of everything, the same bits
    wide = torch.empty(B, T + 1, x.shape[2] + 3, dtype=x.dtype, device="cuda")[:, 1:, 3:].copy_(x)
    wide_probs = None if probs is None else torch.empty(B, T, V + 1, device="cuda")[..., 1:].copy_(probs)
    again = ob.verify_drafts(wide, torch.from_numpy(drafts).int().cuda(), torch.from_numpy(parents).int().cuda(), torch.from_numpy(u).cuda(),
                             temperature=torch.from_numpy(temps.astype(np.float32)).cuda(), draft_probs=wide_probs)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [12, 5002, 60001])
def test_verify_drafts_of_odd_rows(dtype, V):
    """Rows far from zero, masked with infinities and the type's lowest value, with nothing, a NaN or an infinity; equal rows; random numbers at the ends."""
    dt = DTYPES[dtype]
    rng = np.random.RandomState(V)
    base = torch.from_numpy(rng.randn(V)).float() * 2
    low = torch.finfo(dt).min
    left = torch.from_numpy(rng.permutation(V)[:3].copy())
    def only(value):
        r = torch.full((V,), value)
        r[left] = base[left]
        return r
    def hole(value, at):
        r = base.clone()
        r[at] = value
        return r
    fine = [base + 300, base - 3000, base * 1e4, only(-math.inf), only(low), only(-1e30), torch.zeros(V), torch.full((V,), low), torch.full((V,), 3e38 if dtype == "fp32" else 3.3e38),
            hole(-math.inf, 0), base * 1e-3]
    none = [torch.full((V,), -math.inf), hole(math.nan, V - 1), hole(math.nan, 0), hole(math.inf, V // 2), torch.full((V,), math.nan)]
    rows = fine + none
    B = len(rows)
    x = torch.stack([torch.stack([r, base, base]) for r in rows]).to(dt).cuda()
    parents = np.array([[-1, 0, 0]] * B)
    for k, temp in enumerate((1.0, 0.0, 0.02, 50.0, 1e-30, 3e38)):
        drafts = rng.randint(0, V, (B, 3))
        drafts[:, 1], drafts[:, 2] = int(left[0]), int(left[k % 3])           # twice the same, once
        u = rng.rand(B, 3).astype(np.float32)
        check_verify(x, drafts, parents, u, [temp] * B)
        u[:, 1:] = 0.999                                                     # mostly refused: the rest without them
        check_verify(x, drafts, parents, u, [temp] * B)
    ends = np.zeros((B, 3), np.float32)                                      # the first possible token
    no_drafts = np.full((B, 3), -1)
    for temp in (1.0, 0.0):                                                  # (without the row that has weights below 2^-300 of its largest)
        some = [r for r in range(B) if r != 2]
        check_verify(x[some], no_drafts[some], parents[some], ends[some], [temp] * len(some), margin=-1)
    for big in (1.0, 2.0):                                                   # not random numbers: the last possible token
        u = np.full((B, 3), big, np.float32)
        got = ob.verify_drafts(x, torch.from_numpy(no_drafts).cuda(), torch.from_numpy(parents).cuda(), torch.from_numpy(u).cuda())
        assert (got.tokens[len(fine):, 0] == -1).all() and (got.counts == 1).all()
        assert got.tokens[3, 0] == left.max() and got.tokens[6, 0] == V - 1
    u = np.full((B, 3), math.nan, np.float32)
    got = ob.verify_drafts(x, torch.from_numpy(drafts).cuda(), torch.from_numpy(parents).cuda(), torch.from_numpy(u).cuda())
    assert (got.counts == 1).all() and ((got.tokens[:, 0] >= -1) & (got.tokens[:, 0] < V)).all()


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("T,V", [(33, 40), (34, 3000), (100, 60), (1024, 200), (1024, 20000)])
def test_verify_drafts_of_many_children(drawn, T, V):
    """All drafts continue node 0, or every second one does and the others its first child: many of the same token, more than a warp's lanes."""
    g, rng = torch.Generator().manual_seed(T + V), np.random.RandomState(T)
    B = 3
    parents = np.zeros((B, T), np.int64)
    parents[1, 2:] = np.arange(T - 2) % 2
    x = 2 * torch.randn(B, 1, V, generator=g).expand(B, T, V).clone()
    x[:, 1] = 2 * torch.randn(B, V, generator=g)
    drafts = rng.randint(0, V, (B, T))
    u = (0.5 + 0.5 * rng.rand(B, T)).astype(np.float32)       # most are refused
    u[:, 0] = rng.rand(B)
    if T > 40:
        u[0, T - 3], x[0, 0, drafts[0, T - 3]] = 1e-4, 6.0       # one of the last stands
    probs = None
    if drawn:
        probs = torch.softmax(x[:, :1].double() + torch.randn(B, 1, V, generator=g).double(), -1).float().expand(B, T, V).contiguous().cuda()
    for temps in ([1.0, 0.8, 1.3], [0.0] * 3):
        check_verify(x.cuda(), drafts, parents, u, temps, probs)


def test_verify_drafts_of_long_rows():
    """A run of more logits than the shorter sums are for, and a vocabulary of one block's."""
    V = 2 ** 20 + 3
    x = (2 * torch.randn(1, 3, V, generator=torch.Generator().manual_seed(1))).half()
    x[0, 0, 77] = x[0, 1, 99] = 14.0
    many = x.expand(150, 3, V)
    u = np.random.RandomState(1).rand(150, 3).astype(np.float32)
    drafts, parents = np.tile([[0, 77, 99]], (150, 1)), np.tile([[0, 0, 1]], (150, 1))
    x = x.cuda()
    one = check_verify(x, drafts[:1], parents[:1], u[:1], [1.0])
    got = ob.verify_drafts(x.expand(150, 3, V), torch.from_numpy(drafts).cuda(), torch.from_numpy(parents).cuda(), torch.from_numpy(u).cuda())
    assert torch.equal(got.tokens[0], one.tokens[0])
    for b in (1, 2, 3, 149):
        assert torch.equal(got.tokens[b], ob.verify_drafts(x, torch.from_numpy(drafts[:1]).cuda(), torch.from_numpy(parents[:1]).cuda(), torch.from_numpy(u[b:b + 1]).cuda()).tokens[0])
    assert many.shape == got.tokens.shape + (V,)


def test_verify_drafts_shapes_and_numbers():
    x = torch.randn(2, 3, 20, device="cuda")
    i, u = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.full((2, 3), 0.5, device="cuda")
    for temperature, tensor in ((0.7, 0.7), (0, 0.0), (-1.0, 0.0), (2, 2.0)):
        a, b = ob.verify_drafts(x, i, i, u, temperature=temperature), ob.verify_drafts(x, i, i[0], u, temperature=torch.full((2,), tensor, device="cuda"))
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    for none in (ob.verify_drafts(x[:0], i[:0], i[:0], u[:0]), ob.verify_drafts(x[:, :0], i[:, :0], i[:, :0], u[:, :0])):
        assert none.tokens.numel() == none.path.numel() == 0 and not none.counts.any()
    with pytest.raises(RuntimeError):
        ob.verify_drafts(x, i, i, u, temperature=math.nan)
    with pytest.raises(RuntimeError):
        ob.verify_drafts(x.double(), i, i, u)


def test_verify_drafts_outside_the_vocabulary_and_the_tree():
    V, T = 50, 6
    x = torch.zeros(1, T, V, device="cuda")
    x[0, 0, 7] = x[0, 2, 9] = 30.0
    drafts = np.array([[0, V, 7, 9, -1, 9]])
    parents = np.array([[0, 0, 0, 2, 2, 7]])               # node 5 hangs on a later one
    u = np.full((1, T), 0.47, np.float32)             # (not on the border between two of the last row's 50 equal tokens)
    got = check_verify(x, drafts, parents, u, [1.0])
    assert got.path.tolist() == [[0, 2, 3, -1, -1, -1]] and got.tokens[0, :2].tolist() == [7, 9]
    wide = ob.verify_drafts(x, torch.tensor([[0, 2 ** 32 + 7, 7, 9, -1, 9]], device="cuda"), torch.from_numpy(parents).cuda(), torch.from_numpy(u).cuda())
    assert torch.equal(wide.tokens, got.tokens)


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_drafts_leave_the_targets_distribution(drawn):
    """However the drafts came about: two tokens of many sequences, against the target's probabilities of pairs."""
    V, B = 4, 200000
    g = torch.Generator(device="cuda").manual_seed(5)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2], device="cuda")
    first, second = 1.2 * torch.randn(V, generator=g, device="cuda"), 1.2 * torch.randn(V, V, generator=g, device="cuda")
    q1, q2 = torch.softmax(1.2 * torch.randn(V, generator=g, device="cuda"), -1), torch.softmax(1.2 * torch.randn(V, V, generator=g, device="cuda"), -1)
    if drawn:
        a = torch.multinomial(q1.expand(B, V), 2, replacement=True, generator=g)
        deep = [torch.multinomial(q2[a[:, i]], 1, generator=g) for i in (0, 0, 1)]
        drafts = torch.cat([a[:, :1], a, *deep], 1)
    else:
        drafts = torch.tensor([0, 2, 1, 3, 0, 2], device="cuda").expand(B, 6)
    logits = second[drafts]                                  # the row behind a token depends on it alone
    logits[:, 0] = first
    probs = q2[drafts] if drawn else None
    if drawn:
        probs[:, 0] = q1
    got = ob.verify_drafts(logits, drafts, parents, torch.rand(B, 6, generator=g, device="cuda"), draft_probs=probs)
    p1, p2 = torch.softmax(first.double(), -1), torch.softmax(second.double(), -1)
    n1 = torch.bincount(got.tokens[:, 0].long(), minlength=V).double()
    assert ((n1 - B * p1).abs() <= 5 * (B * p1 * (1 - p1)).sqrt()).all()
    two = got.counts > 1
    assert two.float().mean() > 0.2
    for x in range(V):                                       # given an accepted first token, the second one
        here = two & (got.tokens[:, 0] == x)
        n = int(here.sum())
        if n:
            n2 = torch.bincount(got.tokens[here, 1].long(), minlength=V).double()
            assert ((n2 - n * p2[x]).abs() <= 5 * (n * p2[x] * (1 - p2[x])).sqrt()).all()


# ---- moving the accepted rows ---------------------------------------------------------------------------------------------
def moved(pool, bt, offset, path, counts, block, outer_dim):
    """The same by hand, on the CPU: pool (layers, n, ...)."""
    old, new, n = pool.clone(), pool.clone(), pool.shape[1]
    for b, row in enumerate(path):
        before = -1
        for i in range(min(counts[b], len(row))):
            p = row[i]
            if p <= before:
                break
            before = p
            a, z = offset[b] + p, offset[b] + i
            if min(a, z) < 0 or max(a, z) // block >= bt.shape[1]:
                continue
            pa, pz = int(bt[b, a // block]), int(bt[b, z // block])
            if 0 <= pa < n and 0 <= pz < n:
                if outer_dim:
                    new[:, pz, :, z % block] = old[:, pa, :, a % block]
                else:
                    new[:, pz, z % block] = old[:, pa, a % block]
    return new


PATHS = [[0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [0, 2, 3, 5, 8, 11, -1, -1, -1, -1, -1, -1], [0, 11] + [-1] * 10, [0, 1, 1, 5] + [7] * 8, [0, 3, 12, 13] + [14] * 8,
         [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12], [0] + [-1] * 11, [2, 4, 5, 6, 7, 8, 9, 10, 11, -1, -1, -1]]
COUNTS = [12, 6, 2, 12, 4, 12, 1, 9]


@pytest.mark.parametrize("kind,layers,Hkv,D", [("bf16", 0, 2, 64), ("bf16", 3, 1, 128), ("fp32", 2, 3, 5), ("int8", 2, 1, 3), ("int8", 1, 1, 6), ("fp16", 70, 1, 8), ("q4", 0, 2, 64),
                                               ("q4", 5, 4, 128), ("q4", 2, 1, 32)])
def test_commit_drafts(kind, layers, Hkv, D):
    block, B, T = 16, 8, 12
    bt, n = pages(7, B, 4)
    bt[4, 1], bt[5, 1] = -1, n
    offset = [0, 3, 20, 60, 13, 10, 63, -2]
    g = torch.Generator().manual_seed(1)
    L = max(layers, 1)
    if kind == "q4":
        shapes, dts = [(L, n, Hkv, block, D // 2), (L, n, Hkv, block, D // 32)] * 2, [torch.uint8, torch.float16] * 2
    else:
        shapes, dts = [(L, n, block, Hkv, D)] * 2, [dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32, int8=torch.uint8)[kind]] * 2
    pools = [torch.randint(0, 255, s, generator=g).to(dt) for s, dt in zip(shapes, dts)]
    want = [moved(p, bt, offset, PATHS, COUNTS, block, kind == "q4") for p in pools]
    dev = [p.cuda() if layers else p[0].cuda() for p in pools]
    if layers == 70:                                       # layer by layer: more pools than one launch takes
        dev = [x for p in pools for x in p.cuda().unbind()]
    entry = ob.commit_drafts_q4 if kind == "q4" else ob.commit_drafts
    assert entry(dev, bt.cuda(), i32(offset), i32(PATHS), i32(COUNTS)) is None
    if layers == 70:
        dev = [torch.stack(dev[:70]), torch.stack(dev[70:])]
    for d, w in zip(dev, want):
        assert torch.equal(d.cpu().view(w.shape), w)


def test_commit_drafts_long_paths():
    """Ascending paths of hundreds of rows, every other one, over page borders; a count beyond the path and one below zero."""
    block, B, T = 32, 3, 700
    bt, n = pages(7, B, 30)
    path = [list(range(0, T, 2)) + [-1] * (T // 2), [0] + list(range(300, T)) + [-1] * 299, list(range(T))]
    counts, offset = [T, 401, -3], [100, 0, 5]
    pool = torch.randint(0, 255, (2, n, block, 2, 24), generator=torch.Generator().manual_seed(1)).to(torch.uint8)
    want = moved(pool, bt, offset, path, [T, 401, 0], block, False)
    dev = pool.cuda()
    ob.commit_drafts((dev,), bt.cuda(), torch.tensor(offset, device="cuda"), torch.tensor(path, device="cuda"), torch.tensor(counts, device="cuda"))
    assert torch.equal(dev.cpu(), want)


def test_the_cache_classes_reach_them():
    bt, n = pages(3, 2, 4)
    k, v = pool16(10, n, 16, 2, 64, torch.bfloat16)
    q, lens = rand(12, 2, 4, 3, 64).bfloat16().cuda(), i32([40, 33])
    cache = ob.PagedKVCache(k, v, bt.cuda(), lens, 16)
    mask = words_of([[0], [0, 1], [0, 2]], 3).cuda()
    assert torch.equal(cache.fmha_tree(q, softmax_scale=0.1, tree_mask=mask), ob.fmha_tree(q, k, v, softmax_scale=0.1, block_table=bt.cuda(), cache_seqlens=lens, tree_mask=mask))
    path, counts = i32([[0, 2, -1], [0, -1, -1]]), i32([2, 1])
    want = [moved(p[None].cpu(), bt, [37, 30], path.tolist(), [2, 1], 16, False)[0] for p in (k, v)]
    cache.commit_drafts(lens - 3, path, counts)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    pools = ob.PagedKVCacheQ4.empty_pools(n, 2, 16, 64)
    for i, p in enumerate(pools):
        p.copy_(torch.randint(0, 200, p.shape, generator=torch.Generator().manual_seed(i)))
    want = [moved(p[None].cpu(), bt, [37, 37], path.tolist(), [2, 1], 16, True)[0] for p in pools]
    ob.PagedKVCacheQ4(*pools, bt.cuda(), lens).commit_drafts(37, path, counts)
    assert all(torch.equal(p.cpu(), w) for p, w in zip(pools, want))
