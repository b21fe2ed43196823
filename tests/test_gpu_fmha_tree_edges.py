"""Attention of trees of drafts where blocks share a cache, or wait for a place: what is not finite, many keys of little weight, and scores of any size, against plain implementations in 64 bits."""
import math

import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import DTYPES, HALF, pages, rand
from tests.test_gpu_drafts import bound, check, dense16, i32, pool16, tree64, tree_form, words_of  # noqa: F401

pytestmark = pytest.mark.gpu

# rows that share a key head, and keys of a sequence: one block, blocks as a cluster or with partial results, many partial results
SPLITS = [(2, 64, 1, 700), (5, 128, 4, 3000), (40, 64, 2, 3000), (70, 128, 4, 3000), (5, 64, 4, 40000), (40, 128, 2, 40000)]


def attend(q, pools, bt, N, rows, scale, start=0):
    return ob.fmha_tree(q, *pools, softmax_scale=scale, block_table=bt.cuda(), cache_seqlens=i32([N]), cache_seqstarts=i32([start]), tree_mask=words_of(rows, q.shape[2]).cuda()).cpu().double()


def plain(q, k, v, scale, N, rows, start=0):
    """One sequence in 64 bits: the result, and for each row the sum of weights times |v|."""
    T, share = q.shape[2], q.shape[1] // k.shape[1]
    seen = torch.arange(k.shape[2])[None].repeat(T, 1) < N - T
    for t, row in enumerate(rows):
        seen[t, torch.tensor(row) + N - T] = True
    seen[:, :start] = False
    k, v = k[0].repeat_interleave(share, 0), v[0].repeat_interleave(share, 0)
    p = torch.softmax((q[0] @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf), -1).nan_to_num(0)
    return (p @ v)[None], (p @ v.abs())[None]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("far", [False, True], ids=["", "no_weight"])
@pytest.mark.parametrize("T,D,share,N", SPLITS)
def test_values_that_are_not_finite_in_split_caches(tree_form, dtype, far, T, D, share, N):
    """A row that sees such a value has it, however little the weight (infinity, or NaN where the weight is zero in fp32); no other row does."""
    dt, block = DTYPES[dtype], 16
    bt, n = pages(3, 1, -(-N // block))
    pools = pool16(10, n, block, 2, D, dt)
    way = torch.sign(rand(20, D))
    q = (way + 0.01 * rand(12, 1, 2 * share, T, D)).to(dt).cuda()
    if far:                                                # the first keys have scores of more than 170 above all others
        for j in range(40):
            pools[0][bt[0, j // block], j % block] = (2048.0 / D * way).to(dt).cuda()
    k, v, _ = dense16(pools, bt)
    rows = [sorted({t, t // 2, 0}) for t in range(T)]
    def put(u, head, dim, value):
        pools[1][bt[0, (N - T + u) // block], (N - T + u) % block, head, dim] = value
    put(1, 1, 5, math.nan)
    put(1, 1, D - 1, math.inf)
    got = attend(q, pools, bt, N, rows, 0.125)
    x = q.cpu().double()
    want, size = plain(x, k, v, 0.125, N, rows)
    tol = bound(x, k, 0.125, size, want, dt)
    for t in range(T):
        if 1 in rows[t]:
            want[0, share:, t, 5], want[0, share:, t, D - 1] = math.nan, math.inf
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    assert torch.isnan(got[torch.isnan(want)]).all()
    if not far:
        assert (got[torch.isinf(want)] == math.inf).all()
    fine = torch.isfinite(want)
    check(got[fine], want[fine], tol[fine])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,D,share,N", SPLITS)
def test_queries_and_keys_that_are_nan_in_split_caches(tree_form, dtype, T, D, share, N):
    """A query that is NaN gives a row of it.  So does a seen key, alone in its tile, in a block of its own: a start leaves few tiles for many blocks."""
    dt, block = DTYPES[dtype], 16
    N = N // 128 * 128 + 1                                 # the last key is the only one of its tile
    bt, n = pages(3, 1, -(-N // block))
    pools = pool16(10, n, block, 2, D, dt)
    k, v, _ = dense16(pools, bt)
    rows = [sorted({t, t // 2, 0}) for t in range(T)]
    q = rand(12, 1, 2 * share, T, D).to(dt).cuda()
    q[0, 0, T - 1] = math.nan
    pools[0][bt[0, (N - 1) // block], (N - 1) % block, 1, 3] = math.nan
    x = q.nan_to_num(0).cpu().double()
    for start in (0, N - 300):
        got = attend(q, pools, bt, N, rows, 0.125, start)
        want, size = plain(x, k, v, 0.125, N, rows, start)
        tol = bound(x, k, 0.125, size, want, dt)
        want[0, 0, T - 1] = math.nan
        for t in range(T):
            if T - 1 in rows[t]:
                want[0, share:, t] = math.nan
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isfinite(got[~torch.isnan(want)]).all()
        fine = torch.isfinite(want)
        check(got[fine], want[fine], tol[fine])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,D,share,N", SPLITS)
def test_many_keys_of_little_weight(tree_form, dtype, T, D, share, N):
    """The first key has nearly all the weight and values of zero; the others, 2^-14 to 2^-25 of it each, are what comes out.  A weight is off by half a
    step, and in fp16 by half a step of its subnormal numbers when it is taken relative to 2^-7 of the largest: 2^-32 of that."""
    dt, block = DTYPES[dtype], 16
    bt, n = pages(3, 1, -(-N // block))
    pools = [torch.zeros(n, block, 1, D, dtype=dt, device="cuda") for _ in range(2)]
    pools[1].copy_((1 + rand(5, n, block, 1, D).abs().clamp(max=6)).to(dt))
    pools[0][bt[0, 0], 0, 0, 0] = 1.0
    pools[1][bt[0, 0], 0] = 0.0
    k, v, _ = dense16(pools, bt)
    q = torch.zeros(1, share, T, D)
    q[0, :, :, 0] = torch.linspace(14.1, 24.9, share * T).view(share, T) * math.log(2)
    q = q.to(dt).cuda()
    rows = [list(range(t + 1)) for t in range(T)]
    got = attend(q, pools, bt, N, rows, 1.0)
    x = q.cpu().double()
    want, size = plain(x, k, v, 1.0, N, rows)
    tol = bound(x, k, 1.0, size, want, dt)
    if dt == torch.float16:
        tol -= (2.0 ** -25 - 2.0 ** -32) * 8 * (1 + k.shape[2])
    check(got, want, tol)


LARGE = {"bf16": (2.0 ** 22, 2.0 ** 26, 2.0 ** 30, 2.0 ** 40, 2.0 ** 80, 2.0 ** 126), "fp16": (2.0 ** 22, 2.0 ** 26, 2.0 ** 29)}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,D,share,N", SPLITS)
def test_scores_of_any_finite_size(tree_form, dtype, T, D, share, N):
    """Scores far from zero, above and below it, that are exact in fp32: all weight to the largest, equal ones in equal parts, and next to them scores that
    differ by small whole numbers."""
    dt, block = DTYPES[dtype], 16
    bt, n = pages(3, 1, -(-N // block))
    rows = [list(range(t + 1)) for t in range(T)]
    g = torch.Generator().manual_seed(N)
    for level in LARGE[dtype]:
        for sign, scale in ((1, 1.0), (-1, 1.0), (-1, 0.7), (1, -1.3)):
            if dtype == "fp16" and level == 2.0 ** 29:
                scale *= 2.0 ** 60
            pools = pool16(10, n, block, 1, D, dt)
            side = 2.0 ** (math.log2(level) // 2)           # a score: level times 1, 1 + 1/8, ..., 1 + 7/8, plus 0 to 3
            pools[0].zero_()
            steps = torch.randint(0, 8, (n, block), generator=g) if level > 2.0 ** 22 else torch.zeros(n, block)
            pools[0][:, :, 0, 0] = (sign * level / side * (1 + steps / 8)).to(dt).cuda()
            pools[0][:, :, 0, D - 1] = torch.randint(0, 4, (n, block), generator=g).to(dt).cuda()
            k, v, _ = dense16(pools, bt)
            q = torch.zeros(1, share, T, D)
            q[..., 0] = side
            q[..., D - 1] = 1.0 if level <= 2.0 ** 22 else 0.0
            got = attend(q.to(dt).cuda(), pools, bt, N, rows, scale)
            want, size = plain(q.double(), k, v, scale, N, rows)
            # (weights are rounded, and off by 2^-16 for their exponents, as in `bound`; the scores are exact)
            least = 2.0 ** -32 if dt == torch.float16 else 2.0 ** -118
            check(got, want, HALF[dt] * want.abs() + (HALF[dt] + 2.0 ** -16) * size + least * 8 * (1 + k.shape[2]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,Hkv", [(64, 8), (128, 4)])
@pytest.mark.parametrize("T,share", [(1, 3), (3, 4), (5, 4), (20, 2)])
def test_more_sequences_than_places(tree_form, dtype, D, Hkv, T, share):
    """Blocks that wait for their turn: 360 groups of 64 dims, 180 of 128, of up to 200 keys, with starts, padding and empty sequences among them."""
    dt, B, block = DTYPES[dtype], 45, 16
    lens = [(i * 67) % 200 + 1 for i in range(B)]
    starts, q_lens = [(i * 13) % 40 for i in range(B)], [(i * 7) % (T + 1) for i in range(B)]
    bt, n = pages(3, B, 13)
    pools = pool16(10, n, block, Hkv, D, dt)
    k, v, known = dense16(pools, bt)
    q = rand(12, B, Hkv * share, T, D).to(dt).cuda()
    rows = [sorted({t, t // 2, 0}) for t in range(T)]
    got = ob.fmha_tree(q, *pools, softmax_scale=0.125, block_table=bt.cuda(), cache_seqlens=i32(lens), cache_seqstarts=i32(starts), q_lens=i32(q_lens), tree_mask=words_of(rows, T).cuda())
    x = q.cpu().double()
    want, size = tree64(x, k, v, 0.125, lens, starts, q_lens, [rows] * B, known)
    check(got, want, bound(x, k, 0.125, size, want, dt))
