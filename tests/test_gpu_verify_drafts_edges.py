"""Verification of drafted tokens where its sums and temperatures can go wrong, against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import DTYPES
from tests.test_gpu_drafts import check_verify

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "fp16", "fp32"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [12, 5002, 60001])
def test_small_temperatures(dtype, V):
    """Rows whose largest logit lies below, at and above zero, alone at the top or not, and rows as small as the temperature itself."""
    dt = DTYPES[dtype]
    rng = np.random.RandomState(V)
    base = torch.from_numpy(rng.randn(V)).float() * 2
    twice = base - base.max() - 1
    twice[[1, V - 2]] = -0.5
    for k, temp in enumerate((1e-3, 1e-6, 2e-7, 1.5e-7, 1e-7, 8e-11, 1e-11, 1e-20, 1e-30, 1e-34, 1.2e-36, 1e-36, 1e-37, 1e-40, 1e-44)):
        rows = [torch.log_softmax(base, -1), base - base.max(), base, base.clamp(max=0.0), twice, base - 60, base + 60, base * temp, -base.abs() * (30 * temp),
                torch.where(base > 1, base, torch.full_like(base, -math.inf)), torch.zeros(V)]
        x = torch.stack([torch.stack([r, base, -base.abs()]) for r in rows]).to(dt).cuda()
        B = len(rows)
        best = x[:, 0].float().argmax(1).cpu().numpy()
        drafts = rng.randint(0, V, (B, 3))
        drafts[::2, 1] = best[::2]                         # the largest, which stands, or one that hardly ever does
        check_verify(x, drafts, np.array([[-1, 0, 1]] * B), rng.rand(B, 3).astype(np.float32), [temp] * B)
        check_verify(x, drafts, np.array([[-1, 0, 0]] * B), rng.rand(B, 3).astype(np.float32), [temp] * B)


def refused_children(x, drafts, parents, B, T):
    """Children that are refused: whatever the kernel makes of it, then the token at the very start of what is left."""
    u = np.full((B, T), 0.999, np.float32)
    u[:, 0] = np.random.RandomState(T).rand(B)
    got = check_verify(x, drafts, parents, u, [1.0] * B)
    assert (got.counts == 1).all()
    u[:, 0] = 0.0
    check_verify(x, drafts, parents, u, [1.0] * B, margin=-1)       # (decisions about children are those that were checked with a margin)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0.0, -900.0])
@pytest.mark.parametrize("V,kids", [(12, 2), (300, 2), (5002, 3), (5002, 40), (60001, 5)])
def test_nothing_is_left_beside_the_refused_children(dtype, shift, V, kids):
    """All that is possible is a few tokens that lie together, all of them refused children, and one far behind them: that one is next."""
    rng = np.random.RandomState(V + kids)
    B, T = 60, kids + 1
    x = torch.full((B, T, V), -math.inf)
    drafts = np.zeros((B, T), np.int64)
    for b in range(B):
        at = rng.choice(min(V - 1, 2 * kids + 3), kids, replace=False)
        x[b, 0, at] = torch.from_numpy(rng.randn(kids)).float()
        x[b, 0, V - 1] = 2.0
        drafts[b, 1:] = at
    refused_children((x + shift).to(DTYPES[dtype]).cuda(), drafts, np.zeros((B, T), np.int64), B, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0.0, -900.0])
@pytest.mark.parametrize("V", [12, 300, 5002, 60001])
def test_little_is_left_beside_the_refused_children(dtype, shift, V):
    """A refused child and, next to it, tokens of e^-20 to e^-100 of its weight; a likely token far behind them."""
    gaps = [20.0, 24.0, 30.0, 36.0, 40.0, 60.0, 100.0]
    B, T = len(gaps), 3
    x = torch.full((B, T, V), -math.inf)
    for b, gap in enumerate(gaps):
        x[b, 0, 1:V // 2] = 1.0 - gap
        x[b, 0, [5, V - 1]] = 1.0
    drafts = np.array([[0, 5, 0]] * B)
    refused_children((x + shift).to(DTYPES[dtype]).cuda(), drafts, np.zeros((B, T), np.int64), B, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [12, 300, 5002, 60001])
def test_weights_down_to_2_to_the_minus_300_count(dtype, V):
    """The first possible token has e^-200 of the weight of one far behind it, wherever the row lies; nothing is drafted, or a token without weight."""
    tops = [0.0, 50.0, 160.0, -60.0, -104.0, -110.0, -126.0, -138.0, -139.0, -200.0]      # (around zero from -110 on)
    B, T = len(tops), 2
    x = torch.full((B, T, V), -math.inf)
    for b, top in enumerate(tops):
        x[b, 0, 1], x[b, 0, V - 1] = top - 200, top
    x = x.to(DTYPES[dtype]).cuda()
    u = np.full((B, T), 0.5, np.float32)
    parents = np.zeros((B, T), np.int64)
    for drafts in (np.full((B, T), -1), np.full((B, T), 2)):
        u[:, 0] = 0.5
        assert check_verify(x, drafts, parents, u, [1.0] * B).tokens[:, 0].tolist() == [V - 1] * B
        u[:, 0] = 0.0
        assert check_verify(x, drafts, parents, u, [1.0] * B, margin=-1).tokens[:, 0].tolist() == [1] * B


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,wrong", [(12, 1), (12, 2), (12, 8), (300, 3), (5002, 4), (5002, 45), (60001, 3)])
def test_refusals_that_leave_little_of_a_distribution(dtype, V, wrong):
    """p and q agree to a few in 10^7 on one token or on two, and other tokens are drafted first: each refusal leaves so little, and of that, divided by its
    sum, the same p.  Then a likely token, which stands, or none, and it is the next token."""
    for likely in ([V - 2], [1, V - 2]):
        B, T = 6, wrong + 2
        x, q = torch.zeros(B, T, V), torch.full((B, T, V), 2.0 ** -26 / V)
        x[:, :, likely] = 80.0
        q[:, :, likely] = (1 - 2.0 ** -22) / len(likely)
        q[1, :, likely[-1]] *= 1 - 2.0 ** -10                # (the second's p goes to one token)
        drafts = np.tile(np.arange(2, wrong + 4) % (V - 4) + 2, (B, 1))[:, :T]
        drafts[::2, T - 1] = likely[0]
        u = np.full((B, T), 0.5, np.float32)
        u[:, 0] = np.random.RandomState(V).rand(B) * 0.4
        for temps in ([1.0] * B, [0.0] * B, [1.0, 0.0, 2.0] * 2):
            got = check_verify(x.to(DTYPES[dtype]).cuda(), drafts, np.zeros((B, T), np.int64), u, temps, q.cuda())
            assert (got.counts[::2] == 2).all() and (got.counts[1::2] == 1).all()


def test_shortened_rows_captured():
    """The second look at the runs of refused children inside a graph: the same answers."""
    V, B, T = 5002, 8, 4
    x = torch.full((B, T, V), -math.inf)
    x[:, 0, 3:6] = torch.randn(B, 3, generator=torch.Generator().manual_seed(2))
    x[:, 0, 4000] = 2.0
    x, drafts = x.cuda(), torch.tensor([[0, 3, 4, 5]] * B, device="cuda", dtype=torch.int32)
    parents, u = torch.zeros(B, T, device="cuda", dtype=torch.int32), torch.full((B, T), 0.999, device="cuda")
    u[:, 0] = 0.0
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    want = ob.verify_drafts(x, drafts, parents, u)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = ob.verify_drafts(x, drafts, parents, u)
    for _ in range(3):
        got.tokens.fill_(-7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got.tokens[:, 0] == 4000).all()
