"""The operators of drafted tokens as a decoder uses them together: trees into pages, attention, verification, commit; eager, captured and on two streams."""
import math

import numpy as np
import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import pages, rand
from tests.test_gpu_drafts import bound, check, i32, random_parents, tree64, verify64, ways

pytestmark = pytest.mark.gpu
H, HKV, D, BLOCK, V = 8, 2, 64, 16, 96


class Decoder:
    """One attention layer and a head over fixed projections of the tokens."""

    def __init__(self, B, longest, dtype):
        bt, n = pages(4, B, -(-longest // BLOCK))
        self.dtype, self.B, self.bt, self.rope = dtype, B, bt.cuda(), ob.rope_table(longest, D)
        self.k, self.v = (torch.zeros(n, BLOCK, HKV, D, device="cuda", dtype=dtype) for _ in range(2))
        self.embed = rand(1, V, (H + 2 * HKV) * D).to(dtype).cuda()
        self.head = (rand(3, V, H * D) / math.sqrt(H * D) * 12).to(dtype).cuda()

    def project(self, tokens, positions):
        """(B, T) -> q (B, T, H, D), k, v (B, T, HKV, D), turned."""
        B, T = tokens.shape
        q, k, v = (x.unflatten(1, (-1, D)) for x in self.embed[tokens.long().flatten()].split([H * D, HKV * D, HKV * D], 1))
        q, k = ob.qk_norm_rope(q, k, self.rope, positions.flatten())
        return q.view(B, T, H, D), k.view(B, T, HKV, D), v.reshape(B, T, HKV, D)

    def step(self, tokens, parents, uniforms, length, temperature):
        """One step over a tree whose node 0 (the last token) is not in the pages yet; ``length`` (B,) moves on."""
        B, T = tokens.shape
        tree = ob.draft_tree(parents)
        q, k, v = self.project(tokens, length[:, None] + tree.depth)
        ob.write_kv_chunk(self.k, self.v, self.bt, k.transpose(1, 2), v.transpose(1, 2), length)
        att = ob.fmha_tree(q.transpose(1, 2), self.k, self.v, softmax_scale=D ** -0.5, block_table=self.bt, cache_seqlens=length + T, tree_mask=tree.mask, token_major=True)
        logits = ob.gemm(att.view(B * T, H * D), self.head).view(B, T, V)
        done = ob.verify_drafts(logits, tokens, parents, uniforms, temperature=temperature)
        ob.commit_drafts((self.k, self.v), self.bt, length, done.path, done.counts)
        length += done.counts
        return q, k, v, att, logits, done

    def rows(self, b, n):
        """The first n rows of a sequence as they lie in the pages."""
        pos = torch.arange(n)
        at = self.bt[b].cpu().long()[pos // BLOCK], pos % BLOCK
        return [p.cpu()[at] for p in (self.k, self.v)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,width", [(7, 2), (40, 5), (1, 1)])
def test_steps_with_trees_of_drafts(dtype, T, width):
    B, steps = 3, 5
    d = Decoder(B, 64 + (steps + 1) * T + T, dtype)
    rng = np.random.RandomState(T)
    length = i32([0, 5, 60])
    ctx = [[], [], []]                                     # the rows that stand: (k, v) of each
    first = torch.from_numpy(rng.randint(0, V, (B, 60))).cuda()
    _, k, v = d.project(first, torch.arange(60, device="cuda").expand(B, -1).contiguous())
    ob.write_kv_chunk(d.k, d.v, d.bt, k.transpose(1, 2), v.transpose(1, 2), 0)
    for b, n in enumerate(length.tolist()):
        ctx[b] = [(k[b, i].cpu(), v[b, i].cpu()) for i in range(n)]
    last = torch.from_numpy(rng.randint(0, V, B)).cuda()
    temps = torch.tensor([1.0, 0.0, 0.7], device="cuda")
    accepted = 0
    for s in range(steps):
        parents = np.array(random_parents(100 * s + T, B, T, width, 0.1 if T > 7 else 0.0))
        tokens = torch.from_numpy(rng.randint(0, V, (B, T))).cuda()
        tokens[:, 0] = last
        uniforms = torch.from_numpy(rng.rand(B, T).astype(np.float32)).cuda()
        uniforms[:, 1:] *= 0.01                            # drafts of little probability stand now and then
        before = length.tolist()
        q, k, v, att, logits, done = d.step(tokens, torch.from_numpy(parents).cuda(), uniforms, length, temps)
        # attention over what stands and the node's own way
        rows = [ways(p) for p in parents.tolist()]
        N = max(before) + T
        dense = [torch.zeros(B, HKV, N, D, dtype=torch.float64) for _ in range(2)]
        for b in range(B):
            for side in (0, 1):
                x = torch.stack([r[side] for r in ctx[b]] + [t for t in ((k, v)[side][b].cpu())]).double()
                dense[side][b, :, :len(x)] = x.transpose(0, 1)
        x = q.transpose(1, 2).cpu().double()
        want, size = tree64(x, *dense, D ** -0.5, [n + T for n in before], None, None, rows, torch.ones(B, N, dtype=torch.bool))
        check(att.transpose(1, 2), want, bound(x, dense[0], D ** -0.5, size, want, dtype))
        # what stands, by these logits
        tok, path, counts, near = verify64(logits.float().cpu().numpy(), tokens.cpu().numpy(), parents, uniforms.cpu().numpy(), temps.double().cpu().numpy(), None)
        assert near > 1e-9 and done.tokens.tolist() == tok.tolist() and done.path.tolist() == path.tolist() and done.counts.tolist() == counts.tolist()
        accepted += int((counts - 1).sum())
        for b in range(B):
            ctx[b] += [(k[b, i].cpu(), v[b, i].cpu()) for i in path[b, :counts[b]]]
            got = d.rows(b, len(ctx[b]))
            assert length[b] == len(ctx[b]) and all(torch.equal(g, torch.stack([r[side] for r in ctx[b]])) for side, g in enumerate(got))
        last = torch.tensor([tok[b, counts[b] - 1] for b in range(B)], device="cuda")
    assert T == 1 or accepted > 0


def test_a_captured_step_is_the_eager_step():
    """Drafts come out of the last token, so that replays go on by themselves; the same tokens, pages and lengths, bit for bit."""
    B, T, steps = 2, 12, 8
    parents = torch.tensor(random_parents(5, B, T, 2), device="cuda")
    temps = torch.tensor([0.0, 0.9], device="cuda")
    numbers = torch.rand(steps, B, T, generator=torch.Generator().manual_seed(3)).cuda()
    numbers[:, :, 1:] *= 0.01                              # drafts of little probability stand now and then

    def run(graphed):
        d = Decoder(B, 40 + steps * T + T, torch.bfloat16)
        length, last = i32([0, 17]), torch.tensor([3, 50], device="cuda")
        uniforms, tokens, out = torch.empty(B, T, device="cuda"), torch.empty(B, T, dtype=torch.int64, device="cuda"), torch.empty(B, T, dtype=torch.int32, device="cuda")

        def one():
            tokens.copy_((last[:, None] + torch.arange(T, device="cuda") * 7) % V)
            done = d.step(tokens, parents, uniforms, length, temps)[-1]
            last.copy_(done.tokens.gather(1, (done.counts - 1).long()[:, None])[:, 0])
            out.copy_(done.tokens)
        saved = [x.clone() for x in (length, last, d.k, d.v)]
        if graphed:
            uniforms.copy_(numbers[0])
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                one()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                one()
            for x, y in zip((length, last, d.k, d.v), saved):
                x.copy_(y)
        seen = []
        for s in range(steps):
            uniforms.copy_(numbers[s])
            graph.replay() if graphed else one()
            seen.append(out.clone())
        return torch.stack(seen), length, d.k, d.v
    eager, graphed = run(False), run(True)
    assert all(torch.equal(a, b) for a, b in zip(eager, graphed))
    assert int(eager[1].sum()) > 17 + 2 * steps             # some drafts stood


@pytest.mark.parametrize("T", [3, 40])
def test_calls_on_two_streams_do_not_meet(T):
    """Two caches that are split over many blocks, and two graphs of them, at once: each has its own partial results."""
    def make(seed):
        bt, n = pages(seed, 1, 400)
        k, v = (rand(seed + i, n, 16, 2, 128).half().cuda() for i in (1, 2))
        q = rand(seed + 3, 1, 8, T, 128).half().cuda()
        return lambda: ob.fmha_tree(q, k, v, softmax_scale=0.1, block_table=bt.cuda(), cache_seqlens=i32([6400]))
    a, b = make(1), make(11)
    want = [a(), b()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, f in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(f())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


def test_graphs_of_split_caches_replayed_at_once():
    made = []
    for seed in (1, 11):
        bt, n = pages(seed, 1, 400)
        args = [rand(seed + 3, 1, 8, 5, 64).half().cuda()] + [rand(seed + i, n, 16, 2, 64).half().cuda() for i in (1, 2)]
        how = dict(softmax_scale=0.1, block_table=bt.cuda(), cache_seqlens=i32([6400]))
        want = ob.fmha_tree(*args, **how)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = ob.fmha_tree(*args, **how)
        made.append((graph, stream, out, want, args, how))     # (a graph reads where its inputs lay: they live on)
    for _ in range(10):
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, _, out, want, _, _ in made)


def test_inputs_of_another_stream_are_waited_for_as_any_torch_operator_does():
    """Inputs made on the caller's stream just before the calls, results read on it just after, many times over."""
    parents = torch.tensor(random_parents(9, 40, 30, 3), device="cuda")
    want = ob.draft_tree(parents)
    x = rand(5, 40, 30, 300).float().cuda()
    drafts, u = torch.randint(0, 300, (40, 30), device="cuda", dtype=torch.int32), torch.rand(40, 30, device="cuda")
    done = ob.verify_drafts(x, drafts, parents, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(30):
            t = ob.draft_tree(parents + 0)
            y = ob.verify_drafts(x * 1, drafts + 0, parents + 0, u * 1)
            assert torch.equal(t.mask, want.mask) and torch.equal(t.depth, want.depth) and torch.equal(y.tokens, done.tokens) and torch.equal(y.path, done.path)
