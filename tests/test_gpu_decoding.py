"""The operators of a decoding step on the GPU, against plain implementations in 64 bits."""
import math

import pytest
import torch

import oasr_b200 as ob
import oasr_b200.tunables

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative
EPS = 1e-6


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


# ---- plain forms --------------------------------------------------------------------------------------------------------
def norm64(x, w):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()


def rope64(x, table, pos, inter):
    """x (..., heads, D), pos (...): rows outside the table are zero."""
    R = table.shape[1]
    ok = (pos >= 0) & (pos < len(table))
    rows = table[pos.clamp(0, len(table) - 1)].double()[..., None, :]
    c, s = rows[..., :R // 2], rows[..., R // 2:]
    y = x.clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if inter else (slice(0, R // 2), slice(R // 2, R))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return torch.where(ok[..., None, None], y, torch.zeros_like(y))


def quantise64(x, dtype):
    """(..., D) -> (codes, scales (..., D / 32)), both 64-bit."""
    g = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(g.abs().amax(-1) / 7)
    lo, hi = (2.0 ** -20, 9216.0) if dtype == torch.float16 else (2.0 ** -120, 1.125 * 2.0 ** 125)
    s = torch.ldexp(torch.ceil(m * 32) / 32, e).clamp(lo, hi)
    return torch.round(g / s[..., None]).clamp(-7, 7).flatten(-2), s


def pack(codes):
    """(..., D) codes -> (..., D / 2) bytes in the pages' order."""
    D = codes.shape[-1]
    G = D // 32
    out = torch.zeros(*codes.shape[:-1], D // 2, dtype=torch.int64)
    for d in range(D):
        word, i = (d % 32) // 8 * G + d // 32, d % 8
        out[..., word * 4 + i // 2] |= (codes[..., d].long() + 8) << (4 * (i % 2))
    return out.to(torch.uint8)


def attend64(q, k, v, scale, lens, starts, q_lens, causal, known=None):
    """q (B, H, T, D), k / v (B, Hkv, N, D) 64-bit."""
    B, H, T, _ = q.shape
    share = H // k.shape[1]
    out = torch.zeros_like(q)
    for b in range(B):
        n, ql = min(int(lens[b]), k.shape[2]), T if q_lens is None else min(int(q_lens[b]), T)
        for t in range(ql):
            lo, hi = 0 if starts is None else max(int(starts[b]), 0), n
            if causal:
                hi = min(hi, int(lens[b]) - ql + t + 1)
            at = [j for j in range(lo, hi) if known is None or known[b, j]]
            if not at:
                continue
            for h in range(H):
                s = (k[b, h // share, at] @ q[b, h, t]) * scale
                out[b, h, t] = torch.softmax(s, 0) @ v[b, h // share, at]
    return out


def close(got, want, rel, floor):
    """|got - want| <= rel |want| + floor, elementwise, with the same infinities."""
    got, want = got.detach().cpu().double(), want.double()
    off = (got - want).abs()
    bad = off > rel * want.abs() + floor
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {off.max():.3e} at {want.flatten()[off.argmax()]:.3e}"


# ---- norms and rotation -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,H,Hkv,D,R,inter,norm", [
    (1, 8, 8, 64, 64, False, True), (7, 16, 4, 64, 32, True, True), (129, 4, 1, 128, 128, False, True), (33, 3, 2, 80, 32, False, False),
    (40, 5, 1, 96, 96, True, False), (3, 2, 1, 256, 256, False, True), (2, 1, 1, 512, 64, False, True), (5, 2, 2, 16, 16, False, True),
    (4099, 8, 2, 64, 64, False, True), (9, 2, 1, 48, 32, False, True), (9, 2, 1, 32, 16, True, True)])
def test_qk_norm_rope(dtype, N, H, Hkv, D, R, inter, norm):
    dt = DTYPES[dtype]
    fused = rand(1, N, (H + 2 * Hkv) * D).to(dt).cuda()
    q, k = fused[:, :H * D].unflatten(1, (H, D)), fused[:, H * D:(H + Hkv) * D].unflatten(1, (Hkv, D))
    qw, kw = ((1 + 0.2 * rand(s, D)).to(dt).cuda() if norm else None for s in (2, 3))
    table = ob.rope_table(300, R)
    pos = torch.randint(0, 300, (N,), generator=torch.Generator().manual_seed(4))
    if N > 2:
        pos[1], pos[2] = -1, 300                      # no such position: zero rows
    for positions in (pos.cuda(), pos.int().cuda()):
        got = ob.qk_norm_rope(q, k, table, positions, qw, kw, eps=EPS, interleaved=inter)
        for g, x, w in zip(got, (q, k), (qw, kw)):
            n = norm64(x.cpu().double(), None if w is None else w.cpu())
            want = rope64(n, table.cpu(), pos, inter)
            # fp32 steps: norm 6 roundings, two products and a sum (of values up to the pair's length), then one to the type
            pair = n.abs().amax(-1, keepdim=True) * 1.42
            close(g, want, HALF[dt], (12 * 2.0 ** -24 * pair).expand_as(want))
    assert got[0].is_contiguous() and got[1].is_contiguous()
    ob.qk_norm_rope(q, k, table, pos.cuda(), qw, kw, eps=EPS, interleaved=inter, q_out=q, k_out=k)     # in place, beside the values
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])
    assert torch.equal(fused[:, (H + Hkv) * D:].cpu(), rand(1, N, (H + 2 * Hkv) * D).to(dt)[:, (H + Hkv) * D:])


def test_qk_norm_rope_of_queries_alone_and_of_one_weight():
    q, k, w = rand(1, 5, 4, 64).bfloat16().cuda(), rand(2, 5, 2, 64).bfloat16().cuda(), (1 + 0.1 * rand(3, 64)).bfloat16().cuda()
    table, pos = ob.rope_table(64, 64), torch.arange(5, device="cuda") * 7
    alone, none = ob.qk_norm_rope(q, None, table, pos, w)
    both = ob.qk_norm_rope(q, k, table, pos, w)
    plain = ob.qk_norm_rope(q, k, table, pos)
    assert none is None and torch.equal(alone, both[0]) and torch.equal(both[1], plain[1]) and not torch.equal(both[0], plain[0])
    empty = ob.qk_norm_rope(q[:0], k[:0], table, pos[:0], w, w)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 2, 64)


def test_rope_table_of_far_positions():
    t = ob.rope_table(100001, 32)
    ang = 100000 * 10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    close(t[-1], torch.cat([ang.cos(), ang.sin()]), 2.0 ** -24, 1e-10)


def test_qk_norm_rope_refusals():
    q, k = torch.zeros(4, 2, 64, device="cuda").bfloat16(), torch.zeros(4, 1, 64, device="cuda").bfloat16()
    table, pos = ob.rope_table(8, 64), torch.arange(4, device="cuda")
    bad = [dict(q=q.cpu()), dict(k=k.half()), dict(k=k[:3]), dict(cos_sin=table.double()), dict(cos_sin=ob.rope_table(8, 128)), dict(positions=pos[:3]),
           dict(positions=pos.float()), dict(q_weight=torch.ones(64, device="cuda")), dict(k_weight=k[0, 0, :32]), dict(q=q.transpose(1, 2)),
           dict(q_out=torch.empty(4, 2, 32, device="cuda").bfloat16()), dict(q_out=q[:1].expand(4, 2, 64)), dict(q=q.double(), k=k.double()),
           dict(q=torch.zeros(4, 2, 72, device="cuda").bfloat16(), k=None), dict(q=torch.zeros(4 * 130 + 1, device="cuda").bfloat16()[1:].view(4, 130)[:, :128].view(4, 2, 64)),
           dict(k=None, k_weight=k[0, 0])]
    for how in bad:
        args = dict(q=q, k=k, cos_sin=table, positions=pos, q_weight=None, k_weight=None) | how
        out = args.pop("q_out", None)
        with pytest.raises(RuntimeError):
            ob.qk_norm_rope(*args.values(), q_out=out)


# ---- pages --------------------------------------------------------------------------------------------------------------
def chunk(seed, B, H, Hkv, T, D, dt, flat):
    """q, k, v (B, heads, T, D): views of one token-major projection, or head-major tensors of their own."""
    if flat:
        f = rand(seed, B, T, (H + 2 * Hkv) * D).to(dt).cuda()
        return [x.unflatten(2, (-1, D)).transpose(1, 2) for x in f.split([H * D, Hkv * D, Hkv * D], 2)]
    return [rand(seed + i, B, n, T, D).to(dt).cuda() for i, n in enumerate((H, Hkv, Hkv))]


def pages(seed, B, per, spare=2):
    order = torch.randperm(B * per + spare, generator=torch.Generator().manual_seed(seed))
    return order[:B * per].view(B, per).int(), B * per + spare


WRITES = [  # B, H, Hkv, T, D, R, block, interleaved, norm, flat
    (1, 8, 8, 1, 64, 64, 16, False, True, True), (5, 16, 4, 1, 128, 128, 16, False, True, True), (3, 4, 1, 17, 64, 32, 16, False, False, False),
    (4, 2, 2, 33, 64, 64, 32, True, False, True), (2, 12, 12, 70, 128, 64, 48, False, True, False), (3, 3, 1, 5, 96, 32, 16, False, False, True),
    (37, 8, 2, 16, 64, 64, 16, False, False, True), (2, 2, 1, 3, 32, 16, 16, False, True, True), (2, 1, 1, 9, 256, 128, 16, True, True, False)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hkv,T,D,R,block,inter,norm,flat", WRITES)
def test_write_kv_rope_into_16_bit_pages(dtype, B, H, Hkv, T, D, R, block, inter, norm, flat):
    """What qk_norm_rope computes, where write_kv_chunk puts it, bit for bit."""
    dt = DTYPES[dtype]
    q, k, v = chunk(5, B, H, Hkv, T, D, dt, flat)
    qw, kw = ((1 + 0.2 * rand(s, D)).to(dt).cuda() if norm else None for s in (2, 3))
    table = ob.rope_table(400, R)
    g = torch.Generator().manual_seed(6)
    off, lens = torch.randint(0, 60, (B,), generator=g), torch.randint(0, T + 1, (B,), generator=g)
    rope = torch.randint(0, 300, (B,), generator=g)
    bt, n = pages(7, B, -(-(60 + T) // block))
    bt[0, -1] = n + 5                                  # outside the pool: dropped
    pools = [rand(8 + i, n, block, Hkv, D).to(dt).cuda() for i in range(2)]
    for rope_offset, new_lens in ((None, None), (rope, lens)):
        start = off if rope_offset is None else rope_offset
        pos = (start[:, None] + torch.arange(T)).flatten().cuda()
        qf, kf = (x.transpose(1, 2).flatten(0, 1) for x in (q, k))
        tq, tk = (x.unflatten(0, (B, T)).transpose(1, 2).contiguous() for x in ob.qk_norm_rope(qf, kf, table, pos, qw, kw, eps=EPS, interleaved=inter))
        got, want = [p.clone() for p in pools], [p.clone() for p in pools]
        if new_lens is None:
            ob.write_kv_chunk(*want, bt.cuda(), tk, v.contiguous(), off.cuda())
        else:
            for b in range(B):
                m = int(new_lens[b])
                tq[b, :, m:] = 0
                if m:
                    ob.write_kv_chunk(*want, bt[b:b + 1].cuda(), tk[b:b + 1, :, :m], v[b:b + 1, :, :m].contiguous(), off[b:b + 1].cuda())
        cuda = lambda x: None if x is None else x.cuda()  # noqa: E731
        how = dict(q_weight=qw, k_weight=kw, eps=EPS, interleaved=inter, rope_offset=cuda(rope_offset), new_lens=cuda(new_lens))
        out = ob.write_kv_rope(*got, bt.cuda(), k, v, off.cuda(), table, q=q, **how)
        assert torch.equal(out, tq) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        again = [p.clone() for p in pools]
        how.pop("q_weight")
        assert ob.write_kv_rope(*again, bt.cuda(), k, v, off.cuda(), table, **how) is None    # keys and values alone
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hkv,T,D,R,block,inter,norm,flat", WRITES)
def test_write_kv_rope_into_4_bit_pages(dtype, B, H, Hkv, T, D, R, block, inter, norm, flat):
    dt = DTYPES[dtype]
    q, k, v = chunk(5, B, H, Hkv, T, D, dt, flat)
    qw, kw = ((1 + 0.2 * rand(s, D)).to(dt).cuda() if norm else None for s in (2, 3))
    table = ob.rope_table(400, R)
    g = torch.Generator().manual_seed(6)
    off, lens = torch.randint(0, 60, (B,), generator=g), torch.randint(0, T + 1, (B,), generator=g)
    bt, n = pages(7, B, -(-(60 + T) // block))
    pools = ob.PagedKVCacheQ4.empty_pools(n, Hkv, block, D, dt)
    before = [torch.randint(1, 255, p.shape, generator=g, dtype=torch.uint8).cuda() if p.dtype == torch.uint8 else rand(9, *p.shape).abs().to(dt).cuda() for p in pools]
    after = [p.clone() for p in before]
    out = ob.write_kv_rope_q4(*after, bt.cuda(), k, v, off.cuda(), table, q=q, q_weight=qw, k_weight=kw, eps=EPS, interleaved=inter, new_lens=lens.cuda())
    whole = [torch.zeros(n, block, Hkv, D, device="cuda", dtype=dt) for _ in range(2)]
    assert torch.equal(out, ob.write_kv_rope(*whole, bt.cuda(), k, v, off.cuda(), table, q=q, q_weight=qw, k_weight=kw, eps=EPS, interleaved=inter, new_lens=lens.cuda()))
    want = [p.cpu().clone() for p in before]
    for b in range(B):
        m = int(lens[b])
        pos = int(off[b]) + torch.arange(m)
        page, slot = bt[b].long()[pos // block], pos % block
        kx = rope64(norm64(k[b].transpose(0, 1)[:m].cpu().double(), None if kw is None else kw.cpu()), table.cpu(), pos, inter)
        for i, x in ((0, kx), (2, v[b].transpose(0, 1)[:m].cpu().double())):
            codes, scales = quantise64(x, dt)
            want[i][page, :, slot] = pack(codes)
            want[i + 1][page, :, slot] = scales.to(dt)
    for name, got, w in zip(("k codes", "k scales", "v codes", "v scales"), after, want):
        got = got.cpu()
        if name[0] == "v":
            assert torch.equal(got, w), name           # not turned: exact
        elif name == "k scales":
            # the largest magnitude carries fp32 roundings: a scale on the edge may fall to the next of the five-bit numbers
            assert (got != w).float().mean() < 1e-3 and ((got.float() - w.float()).abs() <= w.float() / 15).all()
        else:
            # a code on the edge between two may fall to either side: an fp32 rounding of the value against a step of at most 7
            diff = sum(((got >> s) & 15).int() - ((w >> s) & 15).int() != 0 for s in (0, 4)).float().mean()
            assert diff < 2e-3, diff
    # the values come back at the row's own place; pages that nobody wrote hold scales of more than five bits here, whose
    # products (15 bits at most: exact in fp32) are rounded once
    length = 60 + T
    kv = ob.gather_paged_kv_q4(*after, bt.cuda(), None, length)
    for i, got in ((0, kv[0]), (2, kv[1])):
        codes, scales = after[i].cpu().long(), after[i + 1].cpu().double()
        nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - 8
        G = D // 32
        d = torch.arange(D)
        x = nib[..., ((d % 32) // 8 * G + d // 32) * 8 + d % 8] * scales[..., d // 32]          # (n, Hkv, block, D)
        dense = x[bt.long()].transpose(2, 3).flatten(1, 2).transpose(1, 2)[:, :, :length]
        assert torch.equal(got.cpu(), dense.to(dt))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_4_bit_rounding_of_odd_values(dtype):
    dt = DTYPES[dtype]
    rows = rand(3, 16, 64).to(dt)
    top = torch.finfo(dt).max
    rows[0] = 0
    rows[1, :32], rows[1, 32:] = top, -top
    rows[2, 5] = math.inf
    rows[3, 40] = math.nan
    rows[4] = torch.finfo(dt).tiny / 4
    rows[5, :32] = torch.arange(32) - 16.0             # halves of steps: ties to even
    rows[6] = rows[6] * 1e4
    rows[7] = rows[7] * 1e-4
    pools = ob.PagedKVCacheQ4.empty_pools(1, 1, 16, 64, dt)
    x = rows.view(1, 1, 16, 64).cuda()
    ob.write_kv_rope_q4(*pools, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), x, x, 0, torch.cat([torch.ones(16, 32), torch.zeros(16, 32)], 1).cuda())
    k, v = (t.cpu().view(16, 64) for t in ob.gather_paged_kv_q4(*pools, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), None, 16))
    assert torch.isnan(v[3, 32:]).all() and torch.isfinite(v[3, :32]).all()
    fine = [i for i in range(16) if i not in (2, 3)]
    codes, scales = quantise64(rows[fine].double(), dt)
    want = codes * scales.repeat_interleave(32, -1)
    assert torch.equal(v[fine].double(), want) and torch.equal(k[fine], v[fine])   # turned by nothing: the same
    assert torch.isfinite(v[2]).all() and v[2, 5] == 7 * (9216.0 if dtype == "fp16" else 1.125 * 2.0 ** 125)
    # the step is at most 17 / 16 of amax / 7, and a value at most half a step off
    g = rows[fine].double().unflatten(-1, (-1, 32))
    step = (g.abs().amax(-1) / 7 * 17 / 16).clamp(min=2.0 ** -20 if dtype == "fp16" else 2.0 ** -120)
    assert ((want.unflatten(-1, (-1, 32)) - g).abs() <= step[..., None] / 2 + g.abs().amax(-1, keepdim=True) / 64).all()


def test_write_kv_rope_refusals():
    B, H, Hkv, T, D = 2, 4, 2, 3, 64
    q, k, v = chunk(1, B, H, Hkv, T, D, torch.bfloat16, True)
    bt, table = torch.zeros(B, 2, dtype=torch.int32, device="cuda"), ob.rope_table(64, 64)
    off = torch.zeros(B, dtype=torch.int32, device="cuda")
    pool = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    good = dict(k_cache=pool(4, 16, Hkv, D), v_cache=pool(4, 16, Hkv, D), block_table=bt, new_k=k, new_v=v, offset=off, cos_sin=table)
    for how in [dict(new_v=v[:, :, :2]), dict(new_k=k.half(), new_v=v.half()), dict(k_cache=pool(4, 16, 3, D), v_cache=pool(4, 16, 3, D)),
                dict(block_table=bt[:1]), dict(offset=off[:1]), dict(cos_sin=ob.rope_table(64, 128)), dict(q=q[:, :, :2]), dict(q=q.half()),
                dict(q_weight=q[0, 0, 0]), dict(k_weight=k[0, 0, 0, :32]), dict(new_lens=off[:1]), dict(rope_offset=off[:1]), dict(q_out=q),
                dict(q=q, q_out=q[:, :1].expand_as(q)), dict(k_cache=pool(4, 16, Hkv, 2 * D)[..., :D], v_cache=pool(4, 16, Hkv, 2 * D)[..., :D])]:
        args = good | how
        with pytest.raises((RuntimeError, ValueError)):
            ob.write_kv_rope(**args)
    good = dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), ob.PagedKVCacheQ4.empty_pools(4, Hkv, 16, D)), block_table=bt, new_k=k, new_v=v, offset=off, cos_sin=table)
    for how in [dict(k_codes=pool(4, Hkv, 16, D)), dict(k_scales=pool(4, Hkv, 16, 2, dt=torch.float16)), dict(v_scales=pool(4, Hkv, 16, 4)),
                dict(v_codes=pool(4, Hkv, 16, 16, dt=torch.uint8))]:
        with pytest.raises((RuntimeError, ValueError)):
            ob.write_kv_rope_q4(**(good | how))


@pytest.fixture(params=[0, 1, 2], ids=["by_size", "few_rows", "prompt"])
def form(request):
    """Both kernels of fmha_q4, and the choice between them."""
    ob.tunables.set("fmha_q4_path", request.param)
    yield request.param
    ob.tunables.set("fmha_q4_path", 0)


# ---- attention over 4-bit pages -----------------------------------------------------------------------------------------
def q4_pool(seed, n, Hkv, block, D, dt):
    out = []
    for i in range(2):
        codes, scales = quantise64(rand(seed + i, n, Hkv, block, D).to(dt).double(), dt)
        out += [pack(codes).cuda(), scales.to(dt).cuda()]
    return out


def dense64(pools, bt):
    n, Hkv, block, half = pools[0].shape
    known = (bt >= 0) & (bt < n)
    k, v = ob.gather_paged_kv_q4(*pools, bt.cuda(), None, bt.shape[1] * block)
    return k.cpu().double(), v.cpu().double(), known.repeat_interleave(block, 1)


ATTEND = [  # B, H, Hkv, T, D, block, lens, starts, q_lens, causal
    (1, 8, 8, 1, 64, 16, [300], None, None, True), (1, 1, 1, 1, 128, 16, [1], None, None, False), (3, 8, 2, 1, 128, 16, [0, 1, 33], None, None, True),
    (2, 4, 4, 16, 64, 16, [16, 250], [0, 100], None, False), (2, 14, 2, 5, 64, 32, [70, 31], None, [5, 2], True),
    (2, 8, 1, 17, 128, 48, [96, 17], None, [17, 9], True), (1, 2, 1, 130, 64, 16, [130], None, None, True), (2, 6, 2, 33, 128, 128, [200, 40], [190, 50], None, True),
    (4, 4, 1, 1, 64, 64, [640, 639, 513, 65], [0, 639, 64, 65], None, False), (1, 3, 1, 70, 64, 16, [40], None, None, True),
    (2, 32, 8, 3, 128, 16, [1000, 7], None, [3, 0], True), (1, 1, 1, 300, 128, 16, [333], None, [257], True), (3, 16, 2, 16, 64, 16, [5000, 16, 777], None, None, True)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hkv,T,D,block,lens,starts,q_lens,causal", ATTEND)
def test_fmha_q4(form, dtype, B, H, Hkv, T, D, block, lens, starts, q_lens, causal):
    dt = DTYPES[dtype]
    bt, n = pages(3, B, -(-max(max(lens), 1) // block) + 1)
    pools = q4_pool(10, n, Hkv, block, D, dt)
    q = rand(12, B, T, H, D).to(dt).cuda().transpose(1, 2)
    cuda = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    how = dict(softmax_scale=D ** -0.5, block_table=bt.cuda(), cache_seqlens=cuda(lens), cache_seqstarts=cuda(starts), q_lens=cuda(q_lens), causal=causal)
    got = ob.fmha_q4(q, *pools, **how)
    k, v, _ = dense64(pools, bt)
    want = attend64(q.cpu().double(), k, v, D ** -0.5, lens, starts, q_lens, causal)
    # one rounding of each weight and of the result to the type (weights of one row: their errors add up to half a step of the
    # largest |v| at most), and fp32 steps of the scores: |s| up to 20, each 2^-24 * D of that off before the exponential
    top = v.abs().amax()
    close(got, want, HALF[dt], float(top * (HALF[dt] + 20 * D * 2.0 ** -24)))
    assert torch.equal(got, ob.fmha_q4(q, *pools, **how))                                     # the same bits again
    major = ob.fmha_q4(q, *pools, token_major=True, **how)
    assert major.shape == (B, T, H, D) and torch.equal(major.transpose(1, 2), got)
    wide = torch.full((B, H, T, 2 * D), 7.0, dtype=dt, device="cuda")
    ob.fmha_q4(q.contiguous(), *pools, out=wide[..., :D], **how)
    assert torch.equal(wide[..., :D], got) and (wide[..., D:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [1, 20, 200])
def test_fmha_q4_unseen_keys_say_nothing(form, dtype, T):
    """NaN scales behind the length and before the start, pages outside the pool, and a table wider than the length."""
    dt, block, D = DTYPES[dtype], 16, 64
    bt, n = pages(3, 2, 8)
    pools = q4_pool(10, n, 2, block, D, dt)
    bt[0, 3], bt[1, 0] = -1, n                          # keys 48..63 of one, 0..15 of the other
    lens, starts = [100, 77], [5, 2]
    known = torch.ones(2, 128, dtype=torch.bool)
    known[0, 48:64] = known[1, :16] = False
    k, v, there = dense64(pools, bt)
    assert torch.equal(there, known)
    for b in range(2):
        for j in list(range(starts[b])) + list(range(lens[b], 128)):
            if known[b, j]:
                for p in (1, 3):
                    pools[p][bt[b, j // block], :, j % block] = math.nan
    q = rand(12, 2, 4, T, D).to(dt).cuda()
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ob.fmha_q4(q, *pools, softmax_scale=0.125, block_table=bt.cuda(), cache_seqlens=cuda(lens), cache_seqstarts=cuda(starts))
    want = attend64(q.cpu().double(), k, v, 0.125, lens, starts, None, False, known)
    top = v[known[:, None].expand(2, 2, 128)].abs().max()
    close(got, want, HALF[dt], float(top * (HALF[dt] + 20 * D * 2.0 ** -24)))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [3, 40, 200])
def test_fmha_q4_nan_reaches_the_rows_that_see_it_and_no_other(form, T, D):
    """NaN keys and values inside the length, seen by the later rows of a causal chunk only, and a NaN query."""
    block, N = 16, T + 70
    bt, n = pages(3, 1, -(-N // block))
    pools = q4_pool(10, n, 2, block, D, torch.bfloat16)
    k, v, _ = dense64(pools, bt)
    q = rand(12, 1, 4, T, D).bfloat16().cuda()
    q[0, 1, 0] = math.nan
    at = N - 2                                           # the last row and the one before it see this key
    pools[3][bt[0, at // block], 1, at % block, 1] = math.nan     # values of key head 1: dims 32..63
    pools[1][bt[0, at // block], 0, at % block, 0] = math.nan     # keys of key head 0
    got = ob.fmha_q4(q, *pools, softmax_scale=0.125, block_table=bt.cuda(), cache_seqlens=torch.tensor([N], device="cuda"), causal=True).cpu().double()
    want = attend64(q.nan_to_num(0).cpu().double(), k, v, 0.125, [N], None, None, True)
    want[0, 1, 0] = math.nan
    want[0, :2, T - 2:] = math.nan
    want[0, 2:, T - 2:, 32:64] = math.nan
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    close(got.nan_to_num(0), want.nan_to_num(0), 2.0 ** -8, float(v.abs().max() * (2.0 ** -8 + 20 * D * 2.0 ** -24)))


@pytest.mark.parametrize("T", [1, 40])
def test_fmha_q4_of_large_and_small_scores(form, T):
    """Scores of thousands (one key has all the weight) and of nothing (all have the same)."""
    D, N = 64, 96
    bt, n = pages(3, 1, 6)
    pools = q4_pool(10, n, 1, 16, D, torch.bfloat16)
    k, v, _ = dense64(pools, bt)
    for size in (300.0, 1e-3):
        q = (size * rand(12, 1, 1, T, D)).bfloat16().cuda()
        got = ob.fmha_q4(q, *pools, softmax_scale=1.0, block_table=bt.cuda(), cache_seqlens=torch.tensor([N], device="cuda"))
        want = attend64(q.cpu().double(), k, v, 1.0, [N], None, None, False)
        # scores up to 64 * 300 * 10: their fp32 error 2^-24 * 2e5 * 8 is 0.1 in the exponent between near ties
        close(got, want, 2.0 ** -8, float(v.abs().max()) * (0.1 if size > 1 else 2.0 ** -8 + 1e-4))


def test_fmha_q4_refusals():
    pools = ob.PagedKVCacheQ4.empty_pools(4, 2, 16, 64)
    q, bt, lens = torch.zeros(2, 4, 1, 64, device="cuda").bfloat16(), torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    good = dict(softmax_scale=1.0, block_table=bt, cache_seqlens=lens)
    for how in [dict(block_table=bt[:1]), dict(cache_seqlens=lens[:1]), dict(q_lens=lens[:1]), dict(cache_seqstarts=lens[:1]), dict(q=q[:, :3]), dict(q=q.half()), dict(q=q[0]),
                dict(q=q.float()), dict(out=torch.empty(2, 4, 2, 64, device="cuda").bfloat16()), dict(out=q[:, :1].expand_as(q)),
                dict(pools=ob.PagedKVCacheQ4.empty_pools(4, 2, 8, 64)), dict(pools=ob.PagedKVCacheQ4.empty_pools(4, 2, 16, 128)),
                dict(q=torch.zeros(2, 4, 1, 96, device="cuda").bfloat16(), pools=ob.PagedKVCacheQ4.empty_pools(4, 2, 16, 96)), dict(cache_seqlens=lens.cpu())]:
        args = good | how
        x, p = args.pop("q", q), args.pop("pools", pools)
        with pytest.raises((RuntimeError, ValueError)):
            ob.fmha_q4(x, *p, **args)
    packed = torch.zeros(2 * 4 * 64 + 64, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):                     # heads one row apart, sequences two: some rows are the same memory
        ob.fmha_q4(q, *pools, out=packed.as_strided((2, 4, 1, 64), (128, 64, 64, 1)), **good)
    for form in (1, 2):                                   # no pages at all
        ob.tunables.set("fmha_q4_path", form)
        assert not ob.fmha_q4(q + 1, *pools, softmax_scale=1.0, block_table=bt[:, :0], cache_seqlens=lens).any()
    ob.tunables.set("fmha_q4_path", 0)
    assert not any(x.any() for x in ob.gather_paged_kv_q4(*pools, bt[:, :0], None, 3))
    assert ob.fmha_q4(q[:, :, :0], *pools, **good).shape == (2, 4, 0, 64)
    assert ob.fmha_q4(q[:0], *pools, softmax_scale=1.0, block_table=bt[:0], cache_seqlens=lens[:0]).shape == (0, 4, 1, 64)


# ---- scores -------------------------------------------------------------------------------------------------------------
def score64(x, k):
    """lse, log-probs, entropy and the top ids of (rows, V); NaN ranks first."""
    lp = torch.log_softmax(x, -1)
    none = (x == -math.inf).all(-1)
    lp[none] = -math.inf
    ent = -(lp.exp() * torch.where(lp == -math.inf, torch.zeros_like(lp), lp)).sum(-1)
    rank = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)
    ids = torch.sort(torch.stack([torch.isnan(x).double(), rank], 0)[1] + 0.0, descending=True, stable=True, dim=-1).indices
    for r in torch.isnan(x).any(-1).nonzero().flatten().tolist():      # NaN before +inf
        ids[r] = torch.tensor(sorted(range(x.shape[1]), key=lambda i: (not math.isnan(x[r, i]), -rank[r, i].item(), i)))
    return lp, ent, ids[:, :k]


def check_scores(logits, tokens, k):
    got = ob.token_log_probs(logits, tokens, top_k=k)
    x = logits.detach().cpu().double()
    lp, ent, ids = score64(x, k)
    assert torch.equal(got.top_ids.cpu().long(), ids)
    rows = torch.arange(len(x))[:, None]
    t = tokens.cpu().long().view(len(x), -1)
    want = torch.where((t >= 0) & (t < x.shape[1]), lp.gather(1, t.clamp(0, x.shape[1] - 1)), torch.zeros(t.shape, dtype=torch.float64)).view(tokens.shape)
    # x - m rounds to half a step of itself; the sum's relative error (V terms in a tree of at most V / 32 + 20 steps, each
    # exponential 2^-21 for |d| up to 32) is an absolute one of the logarithm
    tol = 2.0 ** -24 * (x.shape[1] / 32 + 20) + 2.0 ** -20
    for g, w in ((got.log_probs, want), (got.top_log_probs, lp[rows, ids]), (got.entropy, ent)):
        g = g.cpu().double()
        same = torch.where(torch.isnan(w), torch.isnan(g), torch.where(torch.isinf(w), g == w, (g - w).abs() <= 2.0 ** -22 * w.abs() + tol * (1 + ent.abs().nan_to_num(0).max())))
        assert same.all(), (g[~same][:4], w[~same][:4])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V,pad,k", [(1, 1, 0, 1), (3, 2, 1, 2), (5, 31, 0, 8), (2, 1024, 0, 32), (700, 40, 3, 4), (600, 1000, 0, 16), (1300, 2001, 7, 8),
                                          (601, 5002, 6, 8), (17, 5002, 0, 30), (4, 20011, 1, 16), (2, 65537, 7, 32), (1, 262144, 0, 5), (300, 9001, 0, 8), (310, 11000, 8, 1)])
def test_token_log_probs(dtype, rows, V, pad, k):
    x = (3 * rand(rows + V, rows, V + pad)).to(DTYPES[dtype]).cuda()[:, :V]
    g = torch.Generator().manual_seed(V)
    check_scores(x, torch.randint(0, V, (rows,), generator=g).cuda(), k)
    tokens = torch.randint(-1, V + 1, (rows, 3), generator=g).int().cuda()      # with padding on both sides
    check_scores(x, tokens, k)
    again = [ob.token_log_probs(x, tokens, top_k=k) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*again))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V", [(3, 300), (700, 300), (2, 5002), (700, 5002), (2, 40000)])
def test_token_log_probs_of_odd_rows(dtype, rows, V):
    dt = DTYPES[dtype]
    x = (3 * rand(V, rows, V)).to(dt)
    low = torch.finfo(dt).min
    x[0] = -math.inf                                   # nothing possible
    x[0, 7 if rows > 2 else 0] = 1.5 if rows > 2 else -math.inf
    x[1] = low                                          # the type's lowest value everywhere: uniform
    if rows > 2:
        x[2] = 0.25                                     # all equal
    if rows > 600:
        x[3] = -math.inf                                # nothing at all
        x[4, :] = low
        x[4, 100:105] = torch.tensor([1.0, 2.0, 2.0, -1.0, 2.0]).to(dt)
        x[5, 17] = math.nan
        x[6, 11] = math.inf
        x[7] = torch.arange(V).to(dt) * (1 if dtype == "fp32" else 0.01)
        x[8, ::2] = 5.0                                 # half of the row ties for the lead
        x[9] = torch.finfo(dt).max
        x[10, 1:] = low
        x[11, 1:] = -math.inf
        x[12, 3], x[12, 200] = math.nan, math.inf
        x[13] = -0.0
        x[13, 5] = 0.0
        x[14] = torch.finfo(dt).max * (0.5 + 0.5 * torch.rand(V, generator=torch.Generator().manual_seed(1)))
    tokens = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(2))
    check_scores(x.cuda(), tokens.cuda(), min(V, 32))
    check_scores(x.cuda(), tokens.cuda(), 3)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V,k", [(300, 7001, 32), (303, 24001, 30), (297, 52345, 32), (298, 81923, 16), (620, 5002, 30)])
def test_token_log_probs_of_many_long_rows(dtype, rows, V, k):
    test_token_log_probs(dtype, rows, V, 3, k)                 # clusters of other than a power of two among them


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_token_log_probs_of_many_long_odd_rows(dtype):
    test_token_log_probs_of_odd_rows(dtype, 601, 23999)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V", [(601, 4000), (300, 6000), (4, 6000), (4, 60000)])
def test_token_log_probs_of_values_in_one_place(dtype, rows, V):
    """Likely tokens all next to one another, more of them than parts of a row hold a maximum of, and many equal ones."""
    x = 0.1 * rand(V, rows, V)
    x[:, 100:260] += 8 + 4 * rand(V + 1, rows, 160)
    x[1, 300:1500] = 30.0
    x[2, 300:492] = 30.0                                       # as many as are listed, and one more
    x[3, 300:493] = 30.0
    check_scores(x.to(DTYPES[dtype]).cuda(), torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(3)).cuda(), 32)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,V", [(601, 4001), (600, 77), (3, 999), (300, 24001), (4, 60001), (2, 200003)])
def test_token_log_probs_of_masked_rows(dtype, rows, V):
    """Masks that leave fewer tokens than alternatives are asked for: the rest are the lowest masked ids."""
    dt = DTYPES[dtype]
    x = rand(V + 2, rows, V).to(dt)
    g = torch.Generator().manual_seed(V)
    for r in range(min(rows, 40)):
        left = torch.randperm(V, generator=g)[:r % 34]
        if r % 3 == 0:
            left = torch.cat([left, torch.tensor([0, 1, 5, V - 1])])
        y = torch.full((V,), (-math.inf, torch.finfo(dt).min, 0.0, math.inf)[r % 4], dtype=dt)
        y[left] = x[r, left]
        x[r] = y
    tokens = torch.randint(0, V, (rows,), generator=g)
    for k in (1, 32):
        check_scores(x.cuda(), tokens.cuda(), k)


def test_token_log_probs_shapes_and_refusals():
    x = rand(1, 2, 3, 50).cuda()
    x32 = x.float()
    tokens = torch.zeros(2, 3, 4, dtype=torch.int64, device="cuda")
    r = ob.token_log_probs(x32, tokens, top_k=2)
    assert r.log_probs.shape == (2, 3, 4) and r.entropy.shape == (2, 3) and r.top_ids.shape == (2, 3, 2) and r.top_ids.dtype == torch.int32
    only = ob.token_log_probs(x32, top_k=2, entropy=False)
    assert only.log_probs is None and only.entropy is None and torch.equal(only.top_ids, r.top_ids)
    none = ob.token_log_probs(x32[:0], tokens[:0], top_k=2)
    assert none.log_probs.shape == (0, 3, 4) and none.top_ids.shape == (0, 3, 2)
    columns = rand(2, 50, 7).float().cuda()
    assert torch.equal(ob.token_log_probs(columns.t(), top_k=3).top_ids, ob.token_log_probs(columns.t().contiguous(), top_k=3).top_ids)
    for args, how in [((x,), {}), ((x32.cpu(),), {}), ((x32, tokens.float()), {}), ((x32, tokens[:1]), {}), ((x32,), dict(top_k=51)), ((x32,), dict(top_k=33)), ((x32,), dict(top_k=-1)),
                      ((torch.zeros(1, 262145, device="cuda"),), {}), ((x32, tokens.cpu()), {})]:
        with pytest.raises((RuntimeError, ValueError)):
            ob.token_log_probs(*args, **how)
