"""The decoding operators as a decoder uses them together: prompts into pages, then token by token, eager and as a captured graph."""
import math

import pytest
import torch

import oasr_b200 as ob
from tests.test_gpu_decoding import HALF, attend64, check_scores, close, dense64, pages, rand

pytestmark = pytest.mark.gpu
H, HKV, D, BLOCK, V = 8, 2, 64, 16, 1000


class Layer:
    """One attention layer and a head over fixed projections: what stands between the products of a decoder."""

    def __init__(self, kind, B, longest, dtype=torch.bfloat16):
        self.kind, self.dtype, self.B = kind, dtype, B
        bt, n = pages(4, B, -(-longest // BLOCK))
        self.bt, self.table = bt.cuda(), ob.rope_table(longest, D)
        self.pools = ob.PagedKVCacheQ4.empty_pools(n, HKV, BLOCK, D, dtype) if kind == "q4" else tuple(torch.zeros(n, BLOCK, HKV, D, device="cuda", dtype=dtype) for _ in range(2))
        self.qw, self.kw = ((1 + 0.1 * rand(s, D)).to(dtype).cuda() for s in (1, 2))
        self.head = (rand(3, V, H * D) / math.sqrt(H * D) * 8).to(dtype).cuda()

    def step(self, fused, offset, lens, new_lens=None):
        """fused (B, T, (H + 2 Hkv) D) -> (attention (B, T, H D), scores of the last row)."""
        q, k, v = (x.unflatten(2, (-1, D)).transpose(1, 2) for x in fused.split([H * D, HKV * D, HKV * D], 2))
        how = dict(q=q, q_weight=self.qw, k_weight=self.kw, new_lens=new_lens)
        write = ob.write_kv_rope_q4 if self.kind == "q4" else ob.write_kv_rope
        q = write(*self.pools, self.bt, k, v, offset, self.table, **how)
        if self.kind == "q4":
            att = ob.fmha_q4(q, *self.pools, softmax_scale=D ** -0.5, block_table=self.bt, cache_seqlens=lens, q_lens=new_lens, causal=True, token_major=True)
        else:
            att = ob.fmha(q, *self.pools, softmax_scale=D ** -0.5, block_table=self.bt, cache_seqlens=lens, token_major=True)
        att = att.flatten(2)
        logits = ob.gemm(att[:, -1].contiguous(), self.head)
        return att, logits, ob.token_log_probs(logits, top_k=5)


@pytest.mark.parametrize("prompt", [7, 90])
def test_prompts_then_tokens_over_4_bit_pages(prompt):
    B, tokens = 3, 12
    fused = rand(7, B, prompt + tokens, (H + 2 * HKV) * D).bfloat16().cuda()
    first = torch.tensor([prompt, max(prompt // 2, 1), 1], dtype=torch.int32, device="cuda")       # a padded batch of prompts
    layer, whole = Layer("q4", B, prompt + tokens), Layer("q4", B, prompt + tokens)
    att = [layer.step(fused[:, :prompt], torch.zeros_like(first), first, first)[0]]
    rows = [fused[b, :int(first[b])] for b in range(B)]
    pos = first.clone()
    for t in range(tokens):
        new = fused[:, prompt + t:prompt + t + 1]
        out, logits, scores = layer.step(new, pos, pos + 1)
        check_scores(logits, scores.top_ids, 5)
        assert torch.equal(scores.top_ids[:, 0].long(), logits.float().argmax(-1)) or (logits == logits.amax(-1, keepdim=True)).sum() > B
        att.append(out)
        rows = [torch.cat([r, new[b]]) for b, r in enumerate(rows)]
        pos = pos + 1
    # the same tokens in one call of unequal lengths: the same pages, bit for bit, and the same rows of attention
    lens = torch.tensor([len(r) for r in rows], dtype=torch.int32, device="cuda")
    packed = torch.zeros(B, int(lens.max()), fused.shape[2], device="cuda", dtype=torch.bfloat16)
    for b, r in enumerate(rows):
        packed[b, :len(r)] = r
    once = whole.step(packed, torch.zeros_like(lens), lens, lens)[0]
    for a, b in zip(layer.pools, whole.pools):
        assert torch.equal(a, b)
    k, v, _ = dense64(layer.pools, layer.bt.cpu())
    top = float(v.abs().max())
    for b in range(B):
        n = int(first[b])
        both = torch.cat([att[0][b, :n]] + [a[b] for a in att[1:]])
        # either is within half a step of the weights and half a step of the result of the exact one
        close(both, once[b, :len(both)].cpu(), 2 * HALF[torch.bfloat16], 2 * top * (2.0 ** -8 + 20 * D * 2.0 ** -24))
        assert not once[b, len(both):].any()


@pytest.mark.parametrize("kind", ["q4", "16"])
def test_a_captured_step_follows_its_buffers(kind):
    B, steps = 5, 40
    eager, captured = Layer(kind, B, 64), Layer(kind, B, 64)
    fused = rand(9, steps, B, 1, (H + 2 * HKV) * D).bfloat16().cuda()
    x, pos = fused[0].clone(), torch.zeros(B, dtype=torch.int32, device="cuda")
    lens = pos + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step(x, pos, lens)                       # its writes are overwritten by the first replay
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step(x, pos, lens)
    for t in range(steps):
        x.copy_(fused[t])
        pos.fill_(t)
        lens.fill_(t + 1)
        graph.replay()
        want = eager.step(fused[t], torch.full_like(pos, t), torch.full_like(pos, t + 1))
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        for a, b in zip(out[2][1:], want[2][1:]):
            assert torch.equal(a, b)
    for a, b in zip(eager.pools, captured.pools):
        assert torch.equal(a, b)


def test_steps_on_two_streams_do_not_touch_each_other():
    B = 4
    fused = [rand(s, 30, B, 1, (H + 2 * HKV) * D).bfloat16().cuda() for s in (1, 2)]
    alone = []
    for f in fused:
        layer = Layer("q4", B, 64)
        alone.append([layer.step(f[t], torch.full((B,), t, dtype=torch.int32, device="cuda"), torch.full((B,), t + 1, dtype=torch.int32, device="cuda"))[0] for t in range(30)])
    layers, streams, got = [Layer("q4", B, 64) for _ in fused], [torch.cuda.Stream() for _ in fused], [[], []]
    torch.cuda.synchronize()
    for t in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                p = torch.full((B,), t, dtype=torch.int32, device="cuda")
                got[i].append(layers[i].step(fused[i][t], p, p + 1)[0])
    torch.cuda.synchronize()
    for a, g in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, g))


def test_pages_behind_four_gigabytes():
    """Page numbers whose byte offsets pass 32 bits, in every operator of the 4-bit pages and both forms of attention."""
    n = 2 ** 32 // (HKV * BLOCK * D // 2) + 40           # codes of 4.3 GB each
    pools = ob.PagedKVCacheQ4.empty_pools(n, HKV, BLOCK, D)
    bt = torch.tensor([[n - 1, n - 7, 3, n - 20]], dtype=torch.int32, device="cuda")
    small = ob.PagedKVCacheQ4.empty_pools(4, HKV, BLOCK, D)
    bs = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    fused = rand(5, 1, 60, (H + 2 * HKV) * D).bfloat16().cuda()
    q, k, v = (x.unflatten(2, (-1, D)).transpose(1, 2) for x in fused.split([H * D, HKV * D, HKV * D], 2))
    table, lens = ob.rope_table(64, D), torch.tensor([60], dtype=torch.int32, device="cuda")
    for p, t in ((pools, bt), (small, bs)):
        ob.write_kv_rope_q4(*p, t, k, v, 0, table)
    assert all(torch.equal(a, b) for a, b in zip(ob.gather_paged_kv_q4(*pools, bt, None, 64), ob.gather_paged_kv_q4(*small, bs, None, 64)))
    for form in (1, 2):
        ob.tunables.set("fmha_q4_path", form)
        try:
            a, b = (ob.fmha_q4(q, *p, softmax_scale=0.125, block_table=t, cache_seqlens=lens, causal=True) for p, t in ((pools, bt), (small, bs)))
        finally:
            ob.tunables.set("fmha_q4_path", 0)
        assert torch.equal(a, b)
    del pools
    wide = [torch.zeros(2 ** 31 // (BLOCK * HKV * D) + 9, BLOCK, HKV, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]   # more than 2^31 values
    last = torch.tensor([[wide[0].shape[0] - 1, 2, wide[0].shape[0] - 3, 5]], dtype=torch.int32, device="cuda")
    near = [torch.zeros(4, BLOCK, HKV, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    ob.write_kv_rope(*wide, last, k, v, 0, table)
    ob.write_kv_rope(*near, bs, k, v, 0, table)
    assert all(torch.equal(w[last[0].long()], x) for w, x in zip(wide, near))


def test_logits_behind_two_to_the_31():
    rows, vocab = 22000, 100000
    x = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    x[-1] = (3 * rand(1, vocab)).bfloat16().cuda()
    r = ob.token_log_probs(x, torch.full((rows,), 17, device="cuda"), top_k=4)
    one = ob.token_log_probs(x[-1:], torch.tensor([17], device="cuda"), top_k=4)
    assert torch.equal(r.top_ids[-1], one.top_ids[0]) and torch.equal(r.top_ids[0].cpu(), torch.arange(4, dtype=torch.int32))
    close(r.log_probs[-1:], one.log_probs.cpu().double(), 2.0 ** -20, 2.0 ** -18)
    close(r.entropy[:1], torch.tensor([math.log(vocab)], dtype=torch.float64), 2.0 ** -20, 2.0 ** -18)


def test_the_cache_object():
    pools = ob.PagedKVCacheQ4.empty_pools(6, HKV, BLOCK, D)
    lens = torch.tensor([20, 3], dtype=torch.int32, device="cuda")
    cache = ob.PagedKVCacheQ4(*pools, torch.tensor([[4, 0], [2, 5]], dtype=torch.int32, device="cuda"), lens)
    fused = rand(5, 2, 20, (H + 2 * HKV) * D).bfloat16().cuda()
    q, k, v = (x.unflatten(2, (-1, D)).transpose(1, 2) for x in fused.split([H * D, HKV * D, HKV * D], 2))
    table = ob.rope_table(32, D)
    turned = cache.write_kv_rope(k, v, table, offset=0, q=q, new_lens=lens)
    got = cache.fmha(turned, softmax_scale=0.125, causal=True, q_lens=lens)
    kk, vv = cache.gather_full_kv(20)
    want = attend64(turned.cpu().double(), kk.cpu().double(), vv.cpu().double(), 0.125, lens.tolist(), None, lens.tolist(), True)
    close(got, want, 2.0 ** -8, float(vv.abs().max()) * (2.0 ** -8 + 20 * D * 2.0 ** -24))
    assert cache.gather_full_kv(0)[0].shape == (2, HKV, 0, D)
