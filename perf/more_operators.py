"""The operators of a decoding step with drafted tokens over paged keys and values, as a user's program calls them, beside their plain forms.

``tree``    ``draft_tree``: from the parents of each sequence's drafted tokens, who sees whom (bit masks) and how deep everyone stands.
``attend``  ``fmha_tree``: attention of the drafted tokens over 16-bit pages; a single token is a tree of one node.
``verify``  ``verify_drafts``: which drafts stand against the target's logits, from given random numbers, and the token behind them.
``commit``  ``commit_drafts`` / ``commit_drafts_q4``: the accepted tokens' rows moved together in the pages of every layer.

Every case is a dict of plain values; ``listed()`` names the standing ones, ``draw(rng)`` gives another of the same ranges.

A tree's node 0 is the last token that stands already; ``parents[b, i] < i`` for the drafts, anything else is padding.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the trees of a few live sequences, drafted this step
        {"name": "tree_step", "kind": "tree", "streams": 4, "nodes": 33, "width": 4, "ragged": True},
        # a full server's trees, wide and of many nodes
        {"name": "tree_many", "kind": "tree", "streams": 256, "nodes": 255, "width": 24, "ragged": True},
        # one sequence, no drafts: the plain next token, where latency is all there is
        {"name": "attend_single", "kind": "attend", "streams": 1, "nodes": 1, "width": 1, "shortest": 300, "longest": 300, "page": 16,
         "heads": 16, "kv_heads": 4, "dim": 64, "ragged": False, "dtype": "bf16"},
        # small trees of 37 live transcriptions over at most 1001 keys, of different sizes
        {"name": "attend_ragged", "kind": "attend", "streams": 37, "nodes": 21, "width": 3, "shortest": 100, "longest": 1001, "page": 32,
         "heads": 8, "kv_heads": 8, "dim": 64, "ragged": True, "dtype": "fp16"},
        # four drafts in a row and the token before them, 64 sequences: the cache is read once for all five
        {"name": "attend_chain", "kind": "attend", "streams": 64, "nodes": 5, "width": 1, "shortest": 500, "longest": 6000, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "ragged": False, "dtype": "bf16"},
        # wide trees of a few sequences: the products count as much as the cache
        {"name": "attend_tree", "kind": "attend", "streams": 8, "nodes": 61, "width": 8, "shortest": 4000, "longest": 8191, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "ragged": False, "dtype": "bf16"},
        # one sequence with a very long cache
        {"name": "attend_long", "kind": "attend", "streams": 1, "nodes": 16, "width": 4, "shortest": 100003, "longest": 100003, "page": 128,
         "heads": 14, "kv_heads": 2, "dim": 128, "ragged": False, "dtype": "fp16"},
        # three transcriptions with four drafts each, over a recogniser's vocabulary
        {"name": "verify_step", "kind": "verify", "streams": 3, "nodes": 5, "width": 1, "vocab": 5002, "stride": 5008, "drawn": False,
         "greedy": False, "ragged": False, "dtype": "bf16"},
        # trees over a large vocabulary, some sequences greedy
        {"name": "verify_tree", "kind": "verify", "streams": 16, "nodes": 48, "width": 6, "vocab": 131071, "stride": 131072, "drawn": False,
         "greedy": True, "ragged": True, "dtype": "bf16"},
        # chains that a small model drew: accepted by the ratio of both models' probabilities
        {"name": "verify_drawn", "kind": "verify", "streams": 32, "nodes": 8, "width": 1, "vocab": 65537, "stride": 65537, "drawn": True,
         "greedy": False, "ragged": False, "dtype": "fp32"},
        # the accepted rows of four sequences in the pages of 24 layers
        {"name": "commit_step", "kind": "commit", "streams": 4, "nodes": 33, "width": 4, "layers": 24, "longest": 1000, "page": 16, "kv_heads": 4,
         "dim": 64, "pages": "16", "dtype": "bf16"},
        # a full server's accepted rows in 4-bit pages
        {"name": "commit_q4", "kind": "commit", "streams": 96, "nodes": 48, "width": 3, "layers": 16, "longest": 300, "page": 64, "kv_heads": 8,
         "dim": 128, "pages": "q4", "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(("tree", "attend", "attend", "verify", "verify", "commit"))
    nodes = rng.choice((1, _log_int(rng, 2, 8), _log_int(rng, 2, 64), _log_int(rng, 2, 64)))
    width = rng.choice((1, rng.randint(2, 8)))
    if kind == "tree":
        nodes = _log_int(rng, 1, 256)
        return {"kind": kind, "streams": _log_int(rng, 1, 256), "nodes": nodes, "width": rng.randint(1, 24), "ragged": rng.random() < 0.7}
    if kind == "attend":
        heads, kv = rng.choice(((8, 8), (16, 4), (32, 8), (12, 12), (16, 2), (8, 1), (14, 2)))
        dim = rng.choice((64, 128))
        longest = max(_log_int(rng, 1, 30000), nodes)
        most = max(1, min(64, 2 * 10 ** 8 // (longest * kv * dim), 125 * 10 ** 6 // (heads * nodes * longest)))
        return {"kind": kind, "streams": _log_int(rng, 1, most), "nodes": nodes, "width": width, "shortest": max(nodes, longest // 8),
                "longest": longest, "page": rng.choice((16, 32, 64, 128)), "heads": heads, "kv_heads": kv, "dim": dim,
                "ragged": nodes > 1 and rng.random() < 0.4, "dtype": rng.choice(("bf16", "fp16"))}
    if kind == "verify":
        vocab = _log_int(rng, 300, 131071)
        drawn = rng.random() < 0.4
        most = max(1, min(64, (2 * 10 ** 7 if drawn else 10 ** 8) // (vocab * nodes)))
        return {"kind": kind, "streams": _log_int(rng, 1, most), "nodes": nodes, "width": width, "vocab": vocab,
                "stride": vocab + rng.choice((0, 0, 1, 8 - vocab % 8)), "drawn": drawn, "greedy": rng.random() < 0.4,
                "ragged": rng.random() < 0.5, "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    q4 = rng.random() < 0.5
    kv, dim, longest, layers = rng.choice((1, 2, 4, 8)), rng.choice((64, 128)), _log_int(rng, 1, 1000), rng.randint(1, 32)
    most = max(1, min(96, 10 ** 9 // (layers * (longest + nodes + 128) * kv * dim)))
    return {"kind": kind, "streams": _log_int(rng, 1, most), "nodes": nodes, "width": width, "layers": layers, "longest": longest,
            "page": rng.choice((16, 32, 64, 128)), "kv_heads": kv, "dim": dim, "pages": "q4" if q4 else "16", "dtype": rng.choice(("bf16", "fp16"))}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _trees(case, gen):
    """parents (B, T) int32: each draft continues one of the `width` nodes before it, late ones more often; padding at the end of ragged ones."""
    B, T = case["streams"], case["nodes"]
    i = torch.arange(T, device="cuda")
    back = (torch.rand(B, T, generator=gen, device="cuda").square() * i.clamp(max=case["width"])).long()
    parents = (i - 1 - back).clamp(min=-1)
    if case.get("ragged"):
        sizes = torch.randint(1, T + 1, (B, 1), generator=gen, device="cuda")
        sizes[0] = T
        parents = torch.where(i < sizes, parents, -1)
    return parents.int()


def _ancestors(parents):
    """(B, T, T) truth values: column j is row i's node itself or one before it on its way from node 0; and the depths (-1: not in the tree)."""
    B, T = parents.shape
    i = torch.arange(T, device=parents.device)
    p = parents.long()
    step = ((p[..., None] == i) & (p >= 0)[..., None] & (p < i)[..., None]).float()
    reach = step + torch.eye(T, device=parents.device)
    for _ in range(max(1, (T - 1).bit_length())):                    # ways of up to 1, 2, 4, ... steps
        reach = (reach @ reach > 0).float()
    inside = reach[..., :1] > 0                                      # connected with node 0
    seen = (reach > 0) & inside
    return seen, seen.sum(-1, dtype=torch.int32) - 1


def _words(seen):
    """Truth values (B, T, T) -> bits of int32 words (B, T, ceil(T / 32))."""
    T = seen.shape[-1]
    bits = torch.nn.functional.pad(seen, (0, -T % 32)).unflatten(-1, (-1, 32)).long()
    words = (bits << torch.arange(32, device=seen.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def _pages(case, gen, longest):
    """A block table whose pages lie in random order, with a few pages that nobody owns."""
    per = -(-longest // case["page"])
    blocks = case["streams"] * per + 3
    order = torch.randperm(blocks, generator=gen, device="cuda")
    return order[:case["streams"] * per].to(torch.int32).view(case["streams"], per), blocks


def _at(parents, i):
    """parents of node i as indexes (B, 1, 1) of rows; padding points at row 0."""
    return parents[:, i].long().clamp(min=0)[:, None, None]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, B, T = case["kind"], case["streams"], case["nodes"]
    parents = _trees(case, gen)
    state = {"case": case, "parents": parents}
    if kind == "tree":
        return state

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def between(lo, hi, n):                                          # whole numbers in [lo, hi], int32
        return torch.randint(lo, hi + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)

    dtype = _DTYPES[case["dtype"]]
    if kind == "attend":
        H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
        lens = between(case["shortest"], case["longest"], B)         # with the tree's own rows
        lens[0] = case["longest"]
        table, blocks = _pages(case, gen, case["longest"])
        q_lens = None
        if case["ragged"]:
            q_lens = ((parents >= 0).sum(1) + 1).int()               # node 0 and the drafts; padding stands behind them
            lens = torch.maximum(lens, q_lens)
        return state | {"q": normal(B, T, H, D).to(dtype).transpose(1, 2), "k": normal(blocks, case["page"], Hkv, D).to(dtype),
                        "v": normal(blocks, case["page"], Hkv, D).to(dtype), "lens": lens, "block_table": table, "q_lens": q_lens,
                        "mask": _words(_ancestors(parents)[0])}
    if kind == "verify":
        V, N = case["vocab"], case["stride"]
        logits = normal(B, T, N).mul_(2.5)
        uniforms = torch.rand(B, T, generator=gen, device="cuda")
        drafts = torch.randint(0, V, (B, T), generator=gen, device="cuda", dtype=torch.int32)
        probs = None
        if case["drawn"]:
            # the draft model's logits lie near the target's; its children of a node are drawn from one row, one by one
            logits.mul_(1.6)
            probs = torch.softmax(logits[..., :V] + 0.8 * normal(B, T, V), -1)
            for i in range(1, T):
                rows = probs.gather(1, _at(parents, i).expand(-1, 1, V))[:, 0]
                drafts[:, i] = torch.multinomial(rows, 1, generator=gen)[:, 0]
        else:
            # a draft usually has a good part of the target's mass
            level = math.log(V) + 2.5 ** 2 / 2
            for i in range(1, T):
                row = logits.gather(1, _at(parents, i).expand(-1, 1, N))
                row.scatter_(2, drafts[:, i].long()[:, None, None], level - 1.0 + 3.0 * torch.rand(B, 1, 1, generator=gen, device="cuda"))
                logits.scatter_(1, _at(parents, i).expand(-1, 1, N), row)
        temperature = 0.6 + 0.8 * torch.rand(B, generator=gen, device="cuda")
        if case["greedy"]:
            temperature[::3] = 0.0
        return state | {"logits": logits.to(dtype)[..., :V], "drafts": drafts, "uniforms": uniforms, "probs": probs, "temperature": temperature}
    # commit: an ascending path through each tree, as a verification leaves it, of none to all of its drafts
    Hkv, D, L = case["kv_heads"], case["dim"], case["layers"]
    keep = torch.rand(B, T, generator=gen, device="cuda") < torch.rand(B, 1, generator=gen, device="cuda")
    keep[:, 0] = True
    i = torch.arange(T, device="cuda")
    path = torch.where(keep, i, T).sort(1).values.int()
    counts = keep.sum(1, dtype=torch.int32)
    path = torch.where(i < counts[:, None], path, -1)
    offset = between(0, case["longest"], B)
    table, blocks = _pages(case, gen, case["longest"] + T)
    state |= {"path": path, "counts": counts, "offset": offset, "block_table": table}
    if case["pages"] == "16":
        state["pools"] = [normal(L, blocks, case["page"], Hkv, D).to(dtype) for _ in range(2)]
    else:
        codes = [torch.randint(0, 256, (L, blocks, Hkv, case["page"], D // 2), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
        scales = [normal(L, blocks, Hkv, case["page"], D // 32).abs().to(dtype) for _ in range(2)]
        state["pools"] = [codes[0], scales[0], codes[1], scales[1]]
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return _OWN[state["case"]["kind"]](state) if own else _PLAIN[state["case"]["kind"]](state)


def _own_tree(s):
    import oasr_b200 as ob

    t = ob.draft_tree(s["parents"])
    return t.mask, t.depth


def _own_attend(s):
    import oasr_b200 as ob

    return ob.fmha_tree(s["q"], s["k"], s["v"], softmax_scale=s["case"]["dim"] ** -0.5, block_table=s["block_table"], cache_seqlens=s["lens"],
                        tree_mask=s["mask"], q_lens=s["q_lens"])


def _own_verify(s):
    import oasr_b200 as ob

    r = ob.verify_drafts(s["logits"], s["drafts"], s["parents"], s["uniforms"], temperature=s["temperature"], draft_probs=s["probs"])
    return r.tokens, r.path, r.counts


def _own_commit(s):
    import oasr_b200 as ob

    (ob.commit_drafts if s["case"]["pages"] == "16" else ob.commit_drafts_q4)(s["pools"], s["block_table"], s["offset"], s["path"], s["counts"])
    return s["pools"]


def _plain_tree(s):
    seen, depth = _ancestors(s["parents"])
    return _words(seen), depth


def _plain_attend(s):
    c, q = s["case"], s["q"]
    B, H, T, D = q.shape
    Hkv = c["kv_heads"]
    k, v = (s[n][s["block_table"].long()].flatten(1, 2).transpose(1, 2).float() for n in ("k", "v"))       # (B, H_kv, keys, D)
    rows = q.float().unflatten(1, (Hkv, H // Hkv)).flatten(2, 3)                                           # (B, H_kv, share T, D)
    scores = (rows @ k.transpose(2, 3)).unflatten(2, (H // Hkv, T)) * D ** -0.5
    live = torch.full_like(s["lens"], T) if s["q_lens"] is None else s["q_lens"]
    prefix = (s["lens"] - live)[:, None, None]
    j = torch.arange(k.shape[2], device="cuda")
    node = (j - prefix).expand(-1, T, -1)                                                                  # (B, T, keys)
    inside = (node >= 0) & (node < live[:, None, None])
    node = node.clamp(0, T - 1)
    bit = s["mask"].gather(2, node // 32) >> (node % 32) & 1
    seen = (j < prefix) | (inside & (bit == 1))
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weights = torch.exp(scores - top)
    out = (weights.flatten(2, 3) @ v).unflatten(2, (H // Hkv, T)) / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.where((torch.arange(T, device="cuda") < live[:, None])[:, None, None, :, None], out, 0.0)
    return out.flatten(1, 2).to(q.dtype)


def _softmax64(logits, temperature):
    """Rows (B, V) -> probabilities in 64 bits; temperature 0: all on the first maximum."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    ids = torch.arange(x.shape[-1], device=x.device)
    first = torch.where(x == top, ids, x.shape[-1]).amin(-1, keepdim=True)
    warm = temperature.double()[:, None]
    e = torch.exp((x - top) / torch.where(warm > 0, warm, 1.0))
    return torch.where(warm > 0, e / e.sum(-1, keepdim=True), (ids == first).double())


def _plain_verify(s):
    """All sequences at once: `at` is the node that each has come to, `p` what is left of the distribution behind it."""
    logits, drafts, parents, u = s["logits"], s["drafts"].long(), s["parents"].long(), s["uniforms"].double()
    B, T, V = logits.shape
    b = torch.arange(B, device="cuda")
    at = torch.zeros(B, dtype=torch.int64, device="cuda")
    p = _softmax64(logits[:, 0], s["temperature"])
    path = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    tokens = path.clone()
    counts = torch.ones(B, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    for i in range(1, T):
        tried = parents[:, i] == at
        x = drafts[:, i:i + 1]
        q = torch.zeros_like(p).scatter_(1, x, 1.0) if s["probs"] is None else s["probs"][b, at].double()
        good = tried & (u[:, i] * q.gather(1, x)[:, 0] < p.gather(1, x)[:, 0])
        rest = (p - q).clamp(min=0)
        rest = rest / rest.sum(-1, keepdim=True).clamp(min=1e-300)
        p = torch.where(good[:, None], _softmax64(logits[:, i], s["temperature"]), torch.where(tried[:, None], rest, p))
        at = torch.where(good, i, at)
        old = counts.clamp(max=T - 1)
        path[b, old] = torch.where(good, i, path[b, old]).int()
        tokens[b, counts - 1] = torch.where(good, x[:, 0], tokens[b, counts - 1]).int()
        counts = counts + good
    total = p.cumsum(-1)
    last = torch.where(p > 0, torch.arange(V, device="cuda"), -1).amax(-1)
    behind = (total <= u[:, :1] * total[:, -1:]).sum(-1)
    tokens[b, counts - 1] = torch.minimum(behind, last).int()
    return tokens, path, counts.int()


def _plain_commit(s):
    c, T = s["case"], s["case"]["nodes"]
    i = torch.arange(T, device="cuda")
    keep = i < s["counts"][:, None]
    to = s["offset"].long()[:, None] + i
    frm = s["offset"].long()[:, None] + torch.where(keep, s["path"], 0)
    table, page = s["block_table"].long(), c["page"]
    tb, ts = table.gather(1, to // page)[keep], (to % page)[keep]
    fb, fs = table.gather(1, frm // page)[keep], (frm % page)[keep]
    for pool in s["pools"]:                                          # (layers, blocks, page, ...), 4-bit: heads before the page's rows
        if c["pages"] == "16":
            pool[:, tb, ts] = pool[:, fb, fs]
        else:
            rows = pool.transpose(2, 3)
            rows[:, tb, ts] = rows[:, fb, fs]
    return s["pools"]


_OWN = {"tree": _own_tree, "attend": _own_attend, "verify": _own_verify, "commit": _own_commit}
_PLAIN = {"tree": _plain_tree, "attend": _plain_attend, "verify": _plain_verify, "commit": _plain_commit}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    kind, B, T = case["kind"], case["streams"], case["nodes"]
    if kind == "tree":
        return {"bytes": 4 * B * T * (2 + -(-T // 32)), "flops": 0}
    if kind == "attend":
        H, Hkv, D, size = case["heads"], case["kv_heads"], case["dim"], 2
        keys = (case["shortest"] + case["longest"]) / 2 if B > 1 else case["longest"]
        return {"bytes": int(B * (2 * keys * Hkv * D * size + 2 * T * H * D * size + 4 * T * -(-T // 32))),
                "flops": int(4 * B * T * H * D * keys)}
    if kind == "verify":
        # which rows are needed depends on the numbers: the root's in any case, and here one more on average for a tree with drafts
        rows = 1 if T == 1 else 2
        return {"bytes": int(B * (rows * case["vocab"] * _BYTES[case["dtype"]] + (4 * case["vocab"] if case["drawn"] else 0) + 24 * T)),
                "flops": 2 * B * rows * case["vocab"]}
    row = case["kv_heads"] * case["dim"] * 2 if case["pages"] == "16" else case["kv_heads"] * (case["dim"] // 2 + case["dim"] // 16)
    return {"bytes": int(B * (T + 1) / 2 * 2 * case["layers"] * 2 * row + 8 * B * T), "flops": 0}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "attend": _exact_attend, "verify": _exact_verify, "commit": _exact_commit}[case["kind"]](s)


def _ways(parents):
    """For each node of one tree the nodes on its way from node 0, itself the last; none where it is not in the tree."""
    ways = [[0]]
    for i, p in enumerate(parents[1:], 1):
        ways.append(ways[p] + [i] if 0 <= p < i and ways[p] else [])
    return ways


def _exact_tree(s):
    parents = s["parents"].tolist()
    T = len(parents[0])
    mask, depth = np.zeros((len(parents), T, -(-T // 32)), np.int64), np.zeros((len(parents), T), np.int32)
    for b, row in enumerate(parents):
        for i, way in enumerate(_ways(row)):
            depth[b, i] = len(way) - 1
            for j in way:
                mask[b, i, j // 32] |= 1 << (j % 32)
    return mask.astype(np.uint32).view(np.int32), depth


def _exact_attend(s):
    c, q = s["case"], s["q"].double()
    B, H, T, D = q.shape
    share, out = H // c["kv_heads"], torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, (n, parents) in enumerate(zip(s["lens"].tolist(), s["parents"].tolist())):
        ways = _ways(parents)
        live = T if s["q_lens"] is None else int(s["q_lens"][b])
        pages = s["block_table"][b, :-(-n // c["page"])].long()
        k, v = (s[name][pages].flatten(0, 1)[:n].double() for name in ("k", "v"))
        hidden = torch.ones(live, n, dtype=torch.bool, device="cuda")
        hidden[:, :n - live] = False
        for t in range(live):
            hidden[t, [n - live + u for u in ways[t] if u < live]] = False
        for h in range(H):
            x = (q[b, h, :live] @ k[:, h // share].T) / math.sqrt(D)
            out[b, h, :live] = torch.nan_to_num(torch.softmax(x.masked_fill(hidden, -math.inf), -1)) @ v[:, h // share]
    return out


def _exact_verify(s):
    B, T, V = s["logits"].shape
    drafts, parents, u = (s[n].cpu().numpy().astype(np.float64 if n == "uniforms" else np.int64) for n in ("drafts", "parents", "uniforms"))
    tokens, path, counts = np.full((B, T), -1, np.int32), np.full((B, T), -1, np.int32), np.zeros(B, np.int32)
    for b, temp in enumerate(s["temperature"].double().tolist()):
        def target(n):
            x = s["logits"][b, n].double().cpu().numpy()
            if temp == 0:
                return (np.arange(V) == np.argmax(x)).astype(np.float64)
            e = np.exp((x - x.max()) / temp)
            return e / e.sum()
        n, p = 0, target(0)
        path[b, 0] = 0
        while True:
            m = counts[b]
            counts[b] += 1
            q = None if s["probs"] is None else s["probs"][b, n].double().cpu().numpy()
            for i in np.nonzero(parents[b] == n)[0]:
                if i == 0 or i <= n:
                    continue
                x = drafts[b, i]
                if u[b, i] * (1.0 if q is None else q[x]) < p[x]:
                    break
                if q is None:
                    p[x] = 0.0
                else:
                    p = np.maximum(p - q, 0.0)
                p /= max(p.sum(), 1e-300)
            else:
                total = np.cumsum(p)
                tokens[b, m] = min(int(np.searchsorted(total, u[b, 0] * total[-1], side="right")), int(np.nonzero(p)[0][-1]))
                break
            tokens[b, m], n, p = x, i, target(i)
            path[b, m + 1] = i
    return tokens, path, counts


def _exact_commit(s):
    return None                                                      # rows are moved: nothing is computed
