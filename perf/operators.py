"""The operators of a decoding step over paged keys and values, as a user's program calls them, beside their plain forms.

``qk``     ``qk_norm_rope``: RMS norms of the queries and keys of each head and their rotation, out of one fused projection.
``write``  ``write_kv_rope``: a chunk's keys and values appended to their pages, keys and queries normed and rotated on the
           way.  16-bit pages come back whole; of 4-bit pages the values of the chunk's rows come back (``gather_paged_kv_q4``).
``attend`` ``fmha_q4``: attention over 4-bit pages, from single tokens over long caches to whole prompts.
``score``  ``token_log_probs``: log-probs of given tokens, entropy and top alternatives out of a head's logits.

Every case is a dict of plain values; ``listed()`` names the standing ones, ``draw(rng)`` gives another of the same ranges.

4-bit pages: codes ``(num_blocks, H_kv, block_size, D / 2)`` uint8 and scales ``(num_blocks, H_kv, block_size, D / 32)`` in the
keys' type.  A row's 32-bit word ``j`` holds the eight dims ``32 * (j % G) + 8 * (j // G) + i`` (``G = D / 32``), dim ``i`` in bits
``4 i .. 4 i + 3`` as ``code + 8``; the value is ``code * scale``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6
_BASE = 10000.0


def listed():
    return [
        # one token of eight live sequences, between two layers' products: latency is all there is
        {"name": "qk_step", "kind": "qk", "tokens": 8, "heads": 16, "kv_heads": 4, "dim": 64, "rotary": 64, "interleaved": False,
         "norm": True, "table": 8192, "dtype": "bf16"},
        # a pack of odd length, half of each head rotated in neighbouring pairs, no norms
        {"name": "qk_pack_partial", "kind": "qk", "tokens": 5003, "heads": 8, "kv_heads": 8, "dim": 64, "rotary": 32, "interleaved": True,
         "norm": False, "table": 8192, "dtype": "fp16"},
        # the prompts of a full batch
        {"name": "qk_prompts", "kind": "qk", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False,
         "norm": True, "table": 32768, "dtype": "bf16"},
        # one token of 37 sequences into 16-bit pages, with norms
        {"name": "write_step", "kind": "write", "streams": 37, "chunk": 1, "longest": 1000, "ragged": False, "page": 16, "heads": 16,
         "kv_heads": 4, "dim": 64, "rotary": 64, "interleaved": False, "norm": True, "pages": "16", "dtype": "bf16"},
        # a 16-frame chunk of 256 live streams into 4-bit pages
        {"name": "write_chunk_q4", "kind": "write", "streams": 256, "chunk": 16, "longest": 256, "ragged": False, "page": 16, "heads": 8,
         "kv_heads": 8, "dim": 64, "rotary": 64, "interleaved": False, "norm": False, "pages": "q4", "dtype": "fp16"},
        # a padded batch of prompts of odd lengths into 4-bit pages
        {"name": "write_prompts_q4", "kind": "write", "streams": 48, "chunk": 417, "longest": 100, "ragged": True, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "norm": False, "pages": "q4", "dtype": "bf16"},
        # the next token of one sequence with a short history
        {"name": "attend_single", "kind": "attend", "streams": 1, "rows": 1, "shortest": 300, "longest": 300, "page": 16, "heads": 8,
         "kv_heads": 8, "dim": 64, "causal": True, "ragged": False, "dtype": "bf16"},
        # a 16-frame chunk of 256 live streams over their cached frames
        {"name": "attend_chunk", "kind": "attend", "streams": 256, "rows": 16, "shortest": 16, "longest": 1001, "page": 16, "heads": 8,
         "kv_heads": 8, "dim": 64, "causal": False, "ragged": False, "dtype": "fp16"},
        # the next token of a full batch with long and unequal histories, four query heads to a key head
        {"name": "attend_tokens", "kind": "attend", "streams": 128, "rows": 1, "shortest": 500, "longest": 8191, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True, "ragged": False, "dtype": "bf16"},
        # a long prompt over pages that already hold its own keys and a short prefix
        {"name": "attend_prompt", "kind": "attend", "streams": 1, "rows": 4001, "shortest": 4098, "longest": 4098, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True, "ragged": False, "dtype": "bf16"},
        # the next token of five sequences over a large vocabulary
        {"name": "score_step", "kind": "score", "rows": 5, "vocab": 65537, "stride": 65544, "top": 16, "dtype": "bf16"},
        # every frame of a full CTC batch: the transcript's tokens, confidence and alternatives
        {"name": "score_frames", "kind": "score", "rows": 16722, "vocab": 5002, "stride": 5008, "top": 8, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice(((8, 8), (16, 4), (32, 8), (12, 12), (16, 2), (8, 1), (14, 2)))


def draw(rng: random.Random):
    kind = rng.choice(("qk", "write", "attend", "score"))
    if kind == "qk":
        heads, kv = _heads(rng)
        dim = rng.choice((64, 128, 80, 96, 256))
        most = max(2, min(16384, 16384 * 40 * 128 // ((heads + kv) * dim)))
        rotary = rng.choice((dim, dim, 32))
        return {"kind": kind, "tokens": _log_int(rng, 1, most), "heads": heads, "kv_heads": kv, "dim": dim, "rotary": rotary,
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.7, "table": 32768, "dtype": rng.choice(("bf16", "fp16"))}
    if kind == "write":
        heads, kv = _heads(rng)
        dim = rng.choice((64, 128))
        q4 = rng.random() < 0.6
        chunk = rng.choice((1, 16, _log_int(rng, 1, 512)))
        most = max(1, min(512, 48 * 417 * 48 * 128 // (chunk * (heads + 2 * kv) * dim)))
        return {"kind": kind, "streams": _log_int(rng, 1, most), "chunk": chunk, "longest": _log_int(rng, 1, 1000),
                "ragged": chunk > 1 and rng.random() < 0.5, "page": rng.choice((16, 32, 64, 128)), "heads": heads, "kv_heads": kv, "dim": dim,
                "rotary": rng.choice((dim, dim, 32)), "interleaved": rng.random() < 0.3, "norm": not q4 and rng.random() < 0.7,
                "pages": "q4" if q4 else "16", "dtype": rng.choice(("bf16", "fp16"))}
    if kind == "attend":
        heads, kv = _heads(rng)
        dim = rng.choice((64, 128))
        rows = rng.choice((1, 1, 16, _log_int(rng, 2, 1024)))
        longest = max(_log_int(rng, 1, 8192), rows)
        most = min(128, 10 ** 8 // (longest * kv * dim) + 1, 25 * 10 ** 7 // (heads * rows * longest) + 1)
        return {"kind": kind, "streams": _log_int(rng, 1, most), "rows": rows, "shortest": max(rows, longest // 8), "longest": longest,
                "page": rng.choice((16, 32, 64, 128)), "heads": heads, "kv_heads": kv, "dim": dim, "causal": rng.random() < 0.6,
                "ragged": rows > 1 and rng.random() < 0.4, "dtype": rng.choice(("bf16", "fp16"))}
    vocab = _log_int(rng, 300, 131071)
    rows = _log_int(rng, 1, max(1, min(16384, 80 * 10 ** 6 // vocab)))
    return {"kind": kind, "rows": rows, "vocab": vocab, "stride": vocab + rng.choice((0, 0, 1, 8 - vocab % 8)), "top": rng.choice((1, 4, 8, 16, 30)),
            "dtype": rng.choice(("bf16", "fp16", "fp32"))}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _table(rows, rotary, device):
    """cos | sin of every position, angles in 64 bits (far positions)."""
    inv = _BASE ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    ang = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _pages(case, gen, longest):
    """A block table whose pages lie in random order, with a few pages that nobody owns."""
    per = -(-longest // case["page"])
    blocks = case["streams"] * per + 3
    order = torch.randperm(blocks, generator=gen, device="cuda")
    return order[:case["streams"] * per].to(torch.int32).view(case["streams"], per), blocks


def _codes(x):
    """(..., D) values -> codes and scales in the pages' order (any float type in, 32-bit arithmetic)."""
    dtype, x = x.dtype, x.float()
    groups = x.unflatten(-1, (-1, 32))
    scale = _scale(groups.abs().amax(-1), dtype)
    codes = torch.round(groups / scale[..., None]).clamp(-7, 7).to(torch.int16) + 8
    octets = codes.unflatten(-1, (4, 8)).transpose(-3, -2)          # (..., octet, group, 8): the order of the words
    return (octets[..., 0::2] | (octets[..., 1::2] << 4)).to(torch.uint8).flatten(-3), scale.to(dtype)


def _scale(amax, dtype):
    """amax / 7 rounded up to five significant bits, within what 7 * scale can be in the type."""
    bits = (amax / torch.full_like(amax, 7.0)).view(torch.int32)     # a divisor that is a number would become a product by 1 / 7
    up = ((bits + 0x7FFFF) & ~0x7FFFF).view(torch.float32)
    low, high = (2.0 ** -20, 9216.0) if dtype == torch.float16 else (2.0 ** -120, 1.125 * 2.0 ** 125)
    return up.clamp(low, high)


def _values(codes, scales):
    """What codes and scales stand for, in 32 bits: (..., D)."""
    groups = scales.shape[-1]
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    rows = nibbles.unflatten(-1, (4, groups, 8)).transpose(-3, -2).flatten(-2)        # (..., group, 32)
    return (rows * scales.float()[..., None]).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def between(lo, hi, n):                                          # whole numbers in [lo, hi], int32
        return torch.randint(lo, hi + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)

    if kind == "score":
        # a trained head: most of the mass on a few tokens, a long tail, 16-bit ties among it
        buf = normal(case["rows"], case["stride"]).mul_(2.5)
        tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda")
        buf.scatter_add_(1, tokens[:, None], 6.0 + 4.0 * normal(case["rows"], 1).abs())
        return {"case": case, "logits": buf.to(dtype)[:, :case["vocab"]], "tokens": tokens}
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    if kind == "qk":
        fused = normal(case["tokens"], (H + 2 * Hkv) * D).to(dtype)  # one product gives queries, keys and values
        weights = [(1.0 + 0.1 * normal(D)).to(dtype) if case["norm"] else None for _ in range(2)]
        return {"case": case, "q": fused[:, :H * D].unflatten(1, (H, D)), "k": fused[:, H * D:(H + Hkv) * D].unflatten(1, (Hkv, D)),
                "q_weight": weights[0], "k_weight": weights[1], "table": _table(case["table"], case["rotary"], "cuda"),
                "positions": between(0, case["table"] - 1, case["tokens"])}
    B = case["streams"]
    if kind == "write":
        T = case["chunk"]
        offset = between(0, case["longest"], B)
        table, blocks = _pages(case, gen, case["longest"] + T)
        fused = normal(B, T, (H + 2 * Hkv) * D).to(dtype)
        q, k, v = (x.unflatten(2, (-1, D)).transpose(1, 2) for x in fused.split([H * D, Hkv * D, Hkv * D], 2))
        weights = [(1.0 + 0.1 * normal(D)).to(dtype) if case["norm"] else None for _ in range(2)]
        state = {"case": case, "q": q, "k": k, "v": v, "offset": offset, "block_table": table, "q_weight": weights[0], "k_weight": weights[1],
                 "table": _table(case["longest"] + T, case["rotary"], "cuda"), "new_lens": between(1, T, B) if case["ragged"] else None}
        if case["pages"] == "16":
            state["k_cache"], state["v_cache"] = (normal(blocks, case["page"], Hkv, D).to(dtype) for _ in range(2))
        else:
            for name in ("k", "v"):
                state[name + "_codes"], state[name + "_scales"] = _codes(normal(blocks, Hkv, case["page"], D).to(dtype))
        return state
    lens = between(case["shortest"], case["longest"], B)
    lens[0] = case["longest"]
    table, blocks = _pages(case, gen, case["longest"])
    state = {"case": case, "lens": lens, "block_table": table, "q": normal(B, case["rows"], H, D).to(dtype).transpose(1, 2),
             "q_lens": between(1, case["rows"], B) if case["ragged"] else None}
    for name in ("k", "v"):
        state[name + "_codes"], state[name + "_scales"] = _codes(normal(blocks, Hkv, case["page"], D).to(dtype))
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return _OWN[state["case"]["kind"]](state) if own else _PLAIN[state["case"]["kind"]](state)


def _own_qk(s):
    import oasr_b200 as ob

    return ob.qk_norm_rope(s["q"], s["k"], s["table"], s["positions"], s["q_weight"], s["k_weight"], eps=_EPS,
                           interleaved=s["case"]["interleaved"])


def _own_write(s):
    import oasr_b200 as ob

    c = s["case"]
    how = dict(q=s["q"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS, interleaved=c["interleaved"], new_lens=s["new_lens"])
    if c["pages"] == "16":
        q = ob.write_kv_rope(s["k_cache"], s["v_cache"], s["block_table"], s["k"], s["v"], s["offset"], s["table"], **how)
        return q, s["k_cache"], s["v_cache"]
    pools = s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]
    q = ob.write_kv_rope_q4(*pools, s["block_table"], s["k"], s["v"], s["offset"], s["table"], **how)
    return (q, *ob.gather_paged_kv_q4(*pools, s["block_table"], s["offset"], c["chunk"]))


def _own_attend(s):
    import oasr_b200 as ob

    c = s["case"]
    return ob.fmha_q4(s["q"], s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], softmax_scale=c["dim"] ** -0.5,
                      block_table=s["block_table"], cache_seqlens=s["lens"], q_lens=s["q_lens"], causal=c["causal"])


def _own_score(s):
    import oasr_b200 as ob

    r = ob.token_log_probs(s["logits"], s["tokens"], top_k=s["case"]["top"])
    return r.log_probs, r.entropy, r.top_log_probs, r.top_ids


def _norm(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()


def _rotate(x, cos, sin, interleaved):
    """x (..., D) in 32 bits; cos / sin (..., R / 2)."""
    rotary = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rotary:]], -1)


def _plain_qk(s):
    c = s["case"]
    cos, sin = s["table"][s["positions"].long()][:, None].chunk(2, -1)
    return tuple(_rotate(_norm(x.float(), w), cos, sin, c["interleaved"]).to(x.dtype)
                 for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _rows_of(s, T):
    """Pages and slots of a chunk's rows (B, T)."""
    page = s["case"]["page"]
    at = s["offset"].long()[:, None] + torch.arange(T, device="cuda")
    return at, s["block_table"].long().gather(1, at // page), at % page


def _plain_write(s):
    c, T, dtype = s["case"], s["case"]["chunk"], s["k"].dtype
    at, block, slot = _rows_of(s, T)
    cos, sin = s["table"][at][:, None].chunk(2, -1)
    q = _rotate(_norm(s["q"].float(), s["q_weight"]), cos, sin, c["interleaved"]).to(dtype)
    k = _rotate(_norm(s["k"].float(), s["k_weight"]), cos, sin, c["interleaved"])
    keep = torch.ones_like(at, dtype=torch.bool)
    if s["new_lens"] is not None:
        keep = torch.arange(T, device="cuda") < s["new_lens"][:, None]
        q = torch.where(keep[:, None, :, None], q, torch.zeros_like(q))
    b, t = block[keep], slot[keep]
    k, v = k.transpose(1, 2)[keep], s["v"].transpose(1, 2)[keep]      # (rows, H_kv, D)
    if c["pages"] == "16":
        s["k_cache"][b, t] = k.to(dtype)
        s["v_cache"][b, t] = v
        return q, s["k_cache"], s["v_cache"]
    for name, x in (("k", k), ("v", v.float())):
        groups = x.unflatten(-1, (-1, 32))
        scale = _scale(groups.abs().amax(-1), dtype)
        codes = torch.round(groups / scale[..., None]).clamp(-7, 7).to(torch.int16) + 8
        octets = codes.unflatten(-1, (4, 8)).transpose(-3, -2)
        s[name + "_codes"][b, :, t] = (octets[..., 0::2] | (octets[..., 1::2] << 4)).to(torch.uint8).flatten(-3)
        s[name + "_scales"][b, :, t] = scale.to(dtype)
    return (q, *(_values(s[n + "_codes"][block, :, slot], s[n + "_scales"][block, :, slot]).transpose(1, 2).to(dtype) for n in ("k", "v")))


def _plain_attend(s):
    c, q = s["case"], s["q"]
    B, H, T, D = q.shape
    share = H // c["kv_heads"]
    longest = s["block_table"].shape[1] * c["page"]
    k, v = (_values(s[n + "_codes"][s["block_table"].long()], s[n + "_scales"][s["block_table"].long()]).transpose(1, 2).flatten(2, 3)
            for n in ("k", "v"))                                     # (B, H_kv, keys, D)
    rows = q.float().unflatten(1, (-1, share)).flatten(2, 3)          # (B, H_kv, share * T, D)
    scores = (rows @ k.transpose(-1, -2)).mul_(D ** -0.5).unflatten(2, (share, T))
    lens, key = s["lens"].long()[:, None, None], torch.arange(longest, device="cuda")
    row = torch.arange(T, device="cuda")[:, None]
    last = s["q_lens"].long()[:, None, None] if s["q_lens"] is not None else T
    seen = (key < lens) & (row < last)
    if c["causal"]:
        seen = seen & (key <= lens - last + row)
    seen = seen[:, None, None]                                       # (B, 1, 1, T, keys)
    top = scores.masked_fill_(~seen, -math.inf).amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (share, T)) / torch.where(total == 0, torch.ones_like(total), total)
    return out.flatten(1, 2).to(q.dtype)


def _plain_score(s):
    x = s["logits"].float()
    low = x - x.amax(-1, keepdim=True)
    e = low.exp()
    total = e.sum(-1, keepdim=True)
    logp = low - total.log()
    entropy = (total.log() - (low * e).sum(-1, keepdim=True) / total)[:, 0]
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    ids = ids[:, :s["case"]["top"]]
    return logp.gather(1, s["tokens"][:, None])[:, 0], entropy, logp.gather(1, ids), ids.int()


_PLAIN = {"qk": _plain_qk, "write": _plain_write, "attend": _plain_attend, "score": _plain_score}
_OWN = {"qk": _own_qk, "write": _own_write, "attend": _own_attend, "score": _own_score}


# ---- the same in 64 bits, from the definitions ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "write": _exact_write, "attend": _exact_attend, "score": _exact_score}[case["kind"]](s)


def _exact_turn(x, weight, table, position, interleaved):
    """x (rows, heads, D), position (rows,): complex rotation of the pairs."""
    x = x.double()
    if weight is not None:
        x = x * weight.double() / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS)
    half = table.shape[1] // 2
    turn = torch.complex(table[position, :half].double(), table[position, half:].double())[:, None]
    lead = x[..., :2 * half]
    pairs = lead.reshape(*lead.shape[:-1], half, 2) if interleaved else lead.reshape(*lead.shape[:-1], 2, half).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    lead = turned.reshape(lead.shape) if interleaved else turned.transpose(-1, -2).reshape(lead.shape)
    return torch.cat([lead, x[..., 2 * half:]], -1)


def _exact_qk(s):
    at = s["positions"].long()
    return tuple(_exact_turn(x, w, s["table"], at, s["case"]["interleaved"]) for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _exact_q4(x, dtype):
    """The values that 64-bit (rows, heads, D) stand for after the 4-bit rounding."""
    groups = x.reshape(*x.shape[:-1], -1, 32)
    part, power = torch.frexp(groups.abs().max(-1, keepdim=True).values / 7)
    low, high = (2.0 ** -20, 9216.0) if dtype == torch.float16 else (2.0 ** -120, 1.125 * 2.0 ** 125)
    scale = torch.ldexp(torch.ceil(part * 32) / 32, power).clamp(low, high)
    return (torch.round(groups / scale).clamp(-7, 7) * scale).reshape(x.shape)


def _exact_old(s, name, b, at):
    """What the 4-bit pages of stream b hold at positions `at`: (positions, H_kv, D), by nibble."""
    page = s["case"]["page"]
    block, slot = s["block_table"][b].long()[at // page], at % page
    codes, scales = s[name + "_codes"][block, :, slot].int(), s[name + "_scales"][block, :, slot].double()
    D, G = codes.shape[-1] * 2, scales.shape[-1]
    d = torch.arange(D, device="cuda")
    word, i = (d % 32) // 8 * G + d // 32, d % 8
    nibble = (codes[..., word * 4 + i // 2] >> (4 * (i % 2))) & 15
    return (nibble.double() - 8) * scales[..., d // 32]


def _exact_write(s):
    c, T, dtype = s["case"], s["case"]["chunk"], s["k"].dtype
    B, page = c["streams"], c["page"]
    q_out, k_out, v_out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), [], []
    if c["pages"] == "16":
        k_out, v_out = s["k_cache"].double(), s["v_cache"].double()
    for b in range(B):
        n = T if s["new_lens"] is None else int(s["new_lens"][b])
        at = int(s["offset"][b]) + torch.arange(T, device="cuda")
        q_out[b, :, :n] = _exact_turn(s["q"][b].transpose(0, 1)[:n], s["q_weight"], s["table"], at[:n], c["interleaved"]).transpose(0, 1)
        k = _exact_turn(s["k"][b].transpose(0, 1)[:n], s["k_weight"], s["table"], at[:n], c["interleaved"])
        v = s["v"][b].transpose(0, 1)[:n].double()
        if c["pages"] == "16":
            block, slot = s["block_table"][b].long()[at[:n] // page], at[:n] % page
            k_out[block, slot], v_out[block, slot] = k, v
        else:
            for name, new, out in (("k", k, k_out), ("v", v, v_out)):
                out.append(torch.cat([_exact_q4(new, dtype), _exact_old(s, name, b, at[n:])]).transpose(0, 1))
    if c["pages"] == "16":
        return q_out, k_out, v_out
    return q_out, torch.stack(k_out), torch.stack(v_out)


def _exact_attend(s):
    c, q = s["case"], s["q"]
    share = c["heads"] // c["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(c["streams"]):
        n = int(s["lens"][b])
        rows = c["rows"] if s["q_lens"] is None else int(s["q_lens"][b])
        at = torch.arange(n, device="cuda")
        k, v = (_exact_old(s, name, b, at).transpose(0, 1).repeat_interleave(share, 0) for name in ("k", "v"))
        scores = torch.einsum("htd,hnd->htn", q[b, :, :rows].double(), k) / math.sqrt(c["dim"])
        if c["causal"]:
            scores = scores.masked_fill(at > n - rows + torch.arange(rows, device="cuda")[:, None], -math.inf)
        out[b, :, :rows] = torch.nan_to_num(torch.softmax(scores, -1), nan=0.0) @ v
    return out


def _exact_score(s):
    x, k = s["logits"], s["case"]["top"]
    logp, entropy, top = [], [], []
    for part, tokens in zip(x.split(2048), s["tokens"].split(2048)):
        lp = torch.log_softmax(part.double(), -1)
        logp.append(lp[torch.arange(len(lp), device="cuda"), tokens])
        entropy.append(-(lp.exp() * lp).sum(-1))
        top.append(lp.topk(k, -1).values)
    return torch.cat(logp), torch.cat(entropy), torch.cat(top), None


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    kind, e = case["kind"], _BYTES[case["dtype"]]
    if kind == "score":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * e + case["rows"] * (8 + 8 + 8 * case["top"]), "flops": 6.0 * cells}
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    if kind == "qk":
        n = case["tokens"]
        table = min(n, case["table"]) * case["rotary"] * 4
        return {"bytes": n * (2 * (H + Hkv) * D * e + 4) + table, "flops": float(n * (H + Hkv) * (3 * case["rotary"] + (4 * D if case["norm"] else 0)))}
    B = case["streams"]
    if kind == "write":
        rows = B * case["chunk"]
        new = rows // 2 if case["ragged"] else rows
        row = D // 2 + D // 16
        kept = 2 * new * Hkv * D * e if case["pages"] == "16" else 2 * rows * Hkv * (row + D * e) + 2 * new * Hkv * row
        table = min(new, case["longest"] + case["chunk"]) * case["rotary"] * 4
        return {"bytes": new * (H + 2 * Hkv) * D * e + rows * H * D * e + kept + table, "flops": float(new * (H + Hkv) * 7 * D)}
    keys = (case["shortest"] + case["longest"]) / 2
    rows = case["rows"] / (2 if case["ragged"] else 1)
    seen = keys - (rows - 1) / 2 if case["causal"] else keys
    return {"bytes": B * (keys * Hkv * 2 * (D // 2 + D // 16) + 2 * case["rows"] * H * D * e), "flops": 4.0 * B * H * D * rows * seen}
