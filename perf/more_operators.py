"""What the operators of a 4-bit paged cache and the verification of drafted tokens are measured on: calls that a serving
program makes through `iron_amd.operators`.

Each case is one operator at one size. `listed()` holds sizes of this repository's configurations, tests and benchmark
(32/8 heads of 64, 16 layers, 2048 and 3968 positions, 128256 tokens) and generic ones; `draw(rng)` gives other sizes of
the same ranges, odd and ragged ones among them.

Kinds:
  tree    TreeAttentionInt4: queries of drafted trees (one node: an ordinary decode step) against 4-bit caches
  append  PagedAppendInt4: rows of accepted tokens or of prompts are quantized into the pages of all layers, and
          PagedGatherInt4 reads the new positions back (the values that the cache now holds for them)
  gather  PagedGatherInt4: positions of sequences come back as 16-bit rows, in all layers
  verify  DraftVerify: which drafted tokens the target accepts, the rows to append, and the next tokens

A row of a 4-bit cache is D/2 bytes of codes and four fp16 pairs (s, b), one for each quarter of its D values; a value is
b + s (16 + code). The append changes tables and counts in place, so a pass first puts back the ones it started from: one
copy of one small buffer, the same for the plain form and for the kernels.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One token of one conversation: the smallest attention call, where launches and latency count.
        {"name": "tree4_decode_2047", "kind": "tree", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 1, "nodes": 1, "lo": 2047, "hi": 2047},
        # A batch of decode steps behind contexts of very different lengths: bound by the cache's bytes.
        {"name": "tree4_decode_batch", "kind": "tree", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 64, "nodes": 1, "lo": 150, "hi": 16384},
        # Drafted trees of ordinary size for a few conversations.
        {"name": "tree4_drafts", "kind": "tree", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 8, "nodes": 26, "lo": 37, "hi": 3968},
        # Wide trees behind long documents, the wider heads, fp16: the most arithmetic.
        {"name": "tree4_long_wide", "kind": "tree", "dtype": "fp16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "seqs": 2, "nodes": 64, "lo": 20011, "hi": 32768},
        # The tokens that a verification step accepted, for every layer.
        {"name": "append4_accepted", "kind": "append", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 8, "lo": 100, "hi": 4000, "rows_lo": 1, "rows_hi": 6},
        # Prompts enter the cache.
        {"name": "append4_prompts", "kind": "append", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 4, "lo": 1, "hi": 40, "rows_lo": 512, "rows_hi": 3968},
        # The last turn of a conversation read back.
        {"name": "gather4_turn", "kind": "gather", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 1, "lo": 700, "hi": 3968, "rows_lo": 77, "rows_hi": 77},
        # Whole conversations move to a cache of 16 bits.
        {"name": "gather4_move", "kind": "gather", "dtype": "fp16", "layers": 16, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "seqs": 6, "lo": 900, "hi": 8000, "rows_lo": 900, "rows_hi": 8000},
        # One conversation's chain of four drafted tokens: the smallest verification.
        {"name": "verify_chain", "kind": "verify", "dtype": "bf16", "vocab": 128256, "seqs": 1, "nodes": 5, "children": 1,
         "draft": True, "greedy": 0.0},
        # Sampled trees with several children to a node.
        {"name": "verify_trees", "kind": "verify", "dtype": "bf16", "vocab": 128256, "seqs": 8, "nodes": 26, "children": 3,
         "draft": True, "greedy": 0.0},
        # A batch of chains that a lookup proposed (no probabilities of their own), a quarter of the requests greedy.
        {"name": "verify_lookup_batch", "kind": "verify", "dtype": "fp32", "vocab": 32001, "seqs": 64, "nodes": 6, "children": 1,
         "draft": False, "greedy": 0.25},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "append", "gather", "verify", "verify"])
    if kind == "verify":
        vocab, nodes = _log(rng, 500, 131072), _log(rng, 2, 64)
        seqs = _log(rng, 1, max(1, min(64, 8 * 26 * 128256 // (nodes * vocab))))
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "vocab": vocab, "seqs": seqs, "nodes": nodes,
                "children": rng.choice([1, 1, 2, 3, 4]), "draft": rng.random() < 0.6, "greedy": rng.choice([0.0, 0.0, 0.3, 1.0])}
    c = {"kind": kind, "page_size": rng.choice([16, 16, 32, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "tree":
        heads, kv = rng.choice([(32, 8), (32, 8), (16, 16), (64, 8), (8, 2), (24, 8), (10, 2), (12, 1)])
        c |= {"heads": heads, "kv_heads": kv, "head_dim": rng.choice([64, 64, 128]), "nodes": rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 200)])}
        seqs = _log(rng, 1, 64)
        most = min(32768, 64 * 8192 // seqs, 2 * 64 * 32768 * 32 // (seqs * c["nodes"] * heads))
        hi = _log(rng, 16, max(64, most))
        return {**c, "seqs": seqs, "lo": _log(rng, 1, hi), "hi": hi}
    c |= {"layers": rng.choice([1, 2, 4, 16]), "kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 128])}
    room = 16 * 8 * 64 / (c["layers"] * c["kv_heads"] * c["head_dim"])  # how many of this case's positions make one of the largest one's
    seqs = _log(rng, 1, 32)
    hi = _log(rng, 40, int(min(16384, 30000 * room / seqs)))
    lo = _log(rng, 1, hi)
    rows = _log(rng, 1, int(min(4000, 9000 * room / seqs)))
    if kind == "gather":  # of sequences that have that many positions
        rows = min(rows, hi)
        lo = max(lo, rows)
    return {**c, "seqs": seqs, "lo": lo, "hi": hi, "rows_lo": rng.randint(1, rows), "rows_hi": rows}


# ------------------------------------------------------------------ sizes ----
def _spread(lo, hi, count):
    """`count` lengths of [lo, hi], ragged, the same for every seed (the golden ratio's multiples)."""
    return [min(hi, max(lo, round(lo * (hi / lo) ** ((i * 0.6180339887 + 0.31) % 1.0)))) for i in range(count)]


def _pages(n, ps):
    return -(-n // ps)


def _tree(nodes, most):
    """Parents of a tree: a node of the tree before it with fewer than `most` children (most == 1: a chain)."""
    parents, free = [-1], [0]
    count = [0] * nodes
    for i in range(1, nodes):
        p = free[int(len(free) * ((i * 0.6180339887) % 1.0))] if most > 1 else i - 1
        parents.append(p)
        count[p] += 1
        if count[p] == most:
            free.remove(p)
        free.append(i)
    return parents


def _sizes(c):
    """Lengths and counts that the case fixes."""
    S, kind = c["seqs"], c["kind"]
    if kind == "verify":
        nodes = _spread(max(1, c["nodes"] // 2), c["nodes"], S)
        nodes[0] = c["nodes"]
        return {"nodes": nodes, "parents": [_tree(n, c["children"]) for n in nodes]}
    ps = c["page_size"]
    z = {"lens": _spread(c["lo"], c["hi"], S)}
    grown = z["lens"]
    if kind == "tree":
        z["nodes"] = _spread(max(1, c["nodes"] // 2), c["nodes"], S)
        z["nodes"][0], z["lens"][-1] = c["nodes"], c["hi"]
    else:
        z["rows"] = _spread(c["rows_lo"], c["rows_hi"], S)
    if kind == "append":
        grown = [n + r for n, r in zip(grown, z["rows"])]
    if kind == "gather":
        z["rows"] = [min(r, n) for r, n in zip(z["rows"], z["lens"])]
    z["max_pages"] = max(_pages(n, ps) for n in grown) + 1
    live = sum(_pages(n, ps) for n in grown)
    z["num_pages"] = live + live // 8 + 2
    return z


# ------------------------------------------------------------- 4-bit rows ----
def _quantize(x):
    """Rows of values -> (codes, s, b) of their quarters: the nearest code, of two equally near ones the upper."""
    g = x.double().clamp(-20480, 20480).unflatten(-1, (4, -1))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).to(torch.float16)
    b = (lo - 16 * s.double()).to(torch.float16)
    code = torch.where(s > 0, torch.floor((g - b.double()) / s.double() - 15.5), 0.0).clamp_(0, 15)
    return code.to(torch.uint8), s, b


def _pack(x):
    """Rows of D values -> rows of D/2 + 16 bytes. Eight codes make a word: the even ones in its low half, the odd ones in its high half."""
    code, s, b = _quantize(x)
    c = code.flatten(-2).unflatten(-1, (-1, 8))
    word = torch.stack([c[..., 0] | c[..., 2] << 4, c[..., 4] | c[..., 6] << 4, c[..., 1] | c[..., 3] << 4, c[..., 5] | c[..., 7] << 4], -1)
    pairs = torch.cat([s, b], -1).contiguous().view(torch.uint8).flatten(-2)
    return torch.cat([word.flatten(-2), pairs], -1)


def _codes(rows, head_dim):
    word = rows[..., :head_dim // 2].unflatten(-1, (-1, 4))
    low, high = word & 15, word >> 4
    pick = [low[..., 0], low[..., 2], high[..., 0], high[..., 2], low[..., 1], low[..., 3], high[..., 1], high[..., 3]]
    return torch.stack(pick, -1).flatten(-2)


def _unpack(rows, head_dim):
    """Rows of bytes -> rows of values."""
    pairs = rows[..., head_dim // 2:].contiguous().view(torch.float16).unflatten(-1, (4, 2)).float()
    code = _codes(rows, head_dim).unflatten(-1, (4, -1)).float()
    return (pairs[..., 1:] + pairs[..., :1] * (16 + code)).flatten(-2)


# ----------------------------------------------------------------- inputs ----
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _starts(counts):
    return torch.tensor([0] + counts, device=DEV).cumsum(0).to(torch.int32)


def _meta(parts):
    """Tables and counts in one buffer (each part on a multiple of 16 bytes), and their values before the call."""
    at, sizes = [], [p.numel() for p in parts]
    total = 0
    for n in sizes:
        at.append(total)
        total += -(-n // 4) * 4
    start = torch.zeros(total, dtype=torch.int32, device=DEV)
    now = torch.zeros(total, dtype=torch.int32, device=DEV)
    views = []
    for o, n, p in zip(at, sizes, parts):
        start[o:o + n] = p.reshape(-1).to(torch.int32)
        views.append(now[o:o + n].view(p.shape))
    now.copy_(start)
    return start, now, views


def _tables(c, z, g):
    """A page table whose sequences lie scattered over the pool, and how often each page is in use."""
    ps, P, MP = c["page_size"], z["num_pages"], z["max_pages"]
    lens = torch.tensor(z["lens"], device=DEV)
    used = (lens + ps - 1) // ps
    base = torch.cumsum(used, 0) - used
    e = torch.arange(MP, device=DEV)
    live = e[None] < used[:, None]
    ids = torch.randperm(P, generator=g, device=DEV)
    table = torch.where(live, ids[torch.where(live, base[:, None] + e[None], 0)], -1)
    refs = torch.zeros(P, dtype=torch.int64, device=DEV)
    refs.index_add_(0, table.clamp(min=0).reshape(-1), live.reshape(-1).to(torch.int64))
    return table.to(torch.int32), lens.to(torch.int32), refs.to(torch.int32)


def _masks(c, g):
    """Random trees: each node's parent is one of the nodes before it; a node sees itself and those above it, as bits."""
    S, T = c["seqs"], c["nodes"]
    parent = (torch.rand(S, T, generator=g, device=DEV) * torch.arange(T, device=DEV)).long()
    sees = torch.eye(T, dtype=torch.bool, device=DEV).repeat(S, 1, 1)
    for i in range(1, T):
        sees[:, i] |= sees[torch.arange(S, device=DEV), parent[:, i]]
    W = (T + 31) // 32
    bits = torch.nn.functional.pad(sees, (0, 32 * W - T)).view(S, T, W, 32).long()
    words = (bits << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _prepare_verify(c, z, g):
    """Logits with a few likely tokens to a row (some 40 % of the probability), a drafter that is near the target, and
    drafted tokens drawn from the drafter's row at their parent."""
    V, N, dt = c["vocab"], sum(z["nodes"]), DTYPES[c["dtype"]]
    tall = min(64, V)
    draft = torch.randn(N, V, generator=g, device=DEV).mul_(1.5)
    at = torch.randint(0, V, (N, tall), generator=g, device=DEV)
    draft.scatter_(1, at, torch.linspace(math.log(V) + 1, 4, tall, device=DEV).expand(N, -1))
    target = torch.randn(N, V, generator=g, device=DEV).mul_(0.5).add_(draft).to(dt)
    draft = draft.to(dt)
    first = [sum(z["nodes"][:s]) for s in range(c["seqs"])]
    up = torch.tensor([f + max(p, 0) for f, parents in zip(first, z["parents"]) for p in parents], device=DEV)
    heat = torch.rand(c["seqs"], generator=g, device=DEV) * 0.8 + 0.4
    greedy = round(c["greedy"] * c["seqs"])
    heat[torch.randperm(c["seqs"], generator=g, device=DEV)[:greedy]] = 0
    seq = torch.tensor([s for s, n in enumerate(z["nodes"]) for _ in range(n)], device=DEV)
    tokens = torch.empty(N, dtype=torch.int32, device=DEV)
    for i in range(0, N, 64):  # the largest of logits and Gumbel noise is a draw from their softmax
        noise = torch.rand(min(64, N - i), V, generator=g, device=DEV).clamp_(min=1e-30).log_().neg_().log_().neg_()
        tokens[i:i + 64] = (draft[up[i:i + 64]].float() + noise * heat[seq[i:i + 64], None]).argmax(1).to(torch.int32)
    st = {"logits": target, "tokens": tokens, "parents": torch.tensor(sum(z["parents"], []), dtype=torch.int32, device=DEV),
          "starts": _starts(z["nodes"]), "heat": heat, "accept": torch.rand(N, generator=g, device=DEV),
          "sample": torch.rand(c["seqs"], generator=g, device=DEV), "rows": torch.zeros(N, dtype=torch.int32, device=DEV),
          "row_starts": torch.zeros(c["seqs"] + 1, dtype=torch.int32, device=DEV), "next": torch.zeros(c["seqs"], dtype=torch.int32, device=DEV)}
    if c["draft"]:
        st["draft"] = draft
    return st


def prepare(case, seed):
    c, z, g = dict(case), _sizes(case), _generator(seed)
    st = {"c": c, "z": z}
    if c["kind"] == "verify":
        return st | _prepare_verify(c, z, g)
    table, lens, refs = _tables(c, z, g)
    Hkv, D, ps, dt = c["kv_heads"], c["head_dim"], c["page_size"], DTYPES[c["dtype"]]

    def noise(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dt).mul_(scale)

    def pool(layers):
        """Pages of quantized values, a slice at a time."""
        rows = layers * z["num_pages"] * Hkv * ps
        out = torch.empty(rows, D // 2 + 16, dtype=torch.uint8, device=DEV)
        for i in range(0, rows, 1 << 20):
            out[i:i + (1 << 20)] = _pack(torch.randn(min(1 << 20, rows - i), D, generator=g, device=DEV))
        return out.view(layers, z["num_pages"], Hkv, ps, D // 2 + 16)

    if c["kind"] == "tree":
        H, T, N = c["heads"], c["nodes"], sum(z["nodes"])
        words = _masks(c, g)
        mask = torch.zeros(N, words.shape[-1], dtype=torch.int32, device=DEV)
        for s, n in enumerate(z["nodes"]):
            mask[sum(z["nodes"][:s]):sum(z["nodes"][:s]) + n] = words[s, :n]
        # queries of twice the unit size: some keys stand out, as they do in a trained model
        return st | {"q": noise(N, H, D, scale=2.0), "k_new": noise(N, Hkv, D), "v_new": noise(N, Hkv, D),
                     "k_pages": pool(1)[0], "v_pages": pool(1)[0], "table": table, "lens": lens, "starts": _starts(z["nodes"]),
                     "mask": mask, "out": torch.zeros(N, H, D, dtype=dt, device=DEV)}
    L, M = c["layers"], sum(z["rows"])
    st |= {"row_starts": _starts(z["rows"]), "k_out": torch.zeros(L, M, Hkv, D, dtype=dt, device=DEV),
           "v_out": torch.zeros(L, M, Hkv, D, dtype=dt, device=DEV)}
    if c["kind"] == "gather":  # the last positions of each sequence
        return st | {"k_pages": pool(L), "v_pages": pool(L), "table": table, "lens": lens,
                     "begins": lens - torch.tensor(z["rows"], dtype=torch.int32, device=DEV)}
    st["start"], st["now"], (st["table"], st["lens"], st["refs"]) = _meta([table, lens, refs])
    N = M + M // 2 + 1  # the accepted ones are some of the rows that the step computed
    shape = (L, z["num_pages"], Hkv, ps, D // 2 + 16)
    return st | {"k_pages": torch.zeros(shape, dtype=torch.uint8, device=DEV), "v_pages": torch.zeros(shape, dtype=torch.uint8, device=DEV),
                 "k_new": noise(L, N, Hkv, D), "v_new": noise(L, N, Hkv, D), "begins": lens.clone(),
                 "rows": torch.randperm(N, generator=g, device=DEV)[:M].to(torch.int32),
                 "told": torch.zeros(c["seqs"], dtype=torch.int32, device=DEV)}


# ------------------------------------------------------------ plain forms ----
def _plain_tree(s):
    c = s["c"]
    S, H, Hkv, D, T, ps = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], c["nodes"], c["page_size"]
    G, table = H // Hkv, s["table"].long()
    cap = table.shape[1] * ps
    starts = s["starts"].long()
    counts = starts[1:] - starts[:-1]
    node = torch.arange(T, device=DEV)
    real = node[None] < counts[:, None]
    at = torch.where(real, starts[:-1, None] + node[None], 0)
    q = s["q"].float()[at].view(S, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, T * G, D)
    keys = _unpack(s["k_pages"][table.clamp(min=0)], D).transpose(1, 2).reshape(S, Hkv, cap, D)
    values = _unpack(s["v_pages"][table.clamp(min=0)], D).transpose(1, 2).reshape(S, Hkv, cap, D)
    scale = 1.0 / math.sqrt(D)
    old = torch.matmul(q, keys.transpose(-1, -2).contiguous()).mul_(scale)
    new = torch.matmul(q, s["k_new"].float()[at].permute(0, 2, 3, 1).contiguous()).mul_(scale)
    cached = (torch.arange(cap, device=DEV)[None] < s["lens"][:, None]) & (table >= 0).repeat_interleave(ps, 1)
    old.masked_fill_(~cached[:, None, None], -math.inf)
    seen = ((s["mask"][at][..., node // 32] >> (node % 32)) & 1).bool() & real[:, None]
    new.masked_fill_(~seen.repeat_interleave(G, 1)[:, None], -math.inf)
    top = torch.maximum(old.amax(-1, keepdim=True), new.amax(-1, keepdim=True)).clamp(min=-1e30)
    old, new = old.sub_(top).exp_(), new.sub_(top).exp_()
    total = old.sum(-1, keepdim=True) + new.sum(-1, keepdim=True)
    values.masked_fill_(~cached[:, None, :, None], 0.0)
    o = torch.matmul(old, values) + torch.matmul(new, s["v_new"].float()[at].permute(0, 2, 1, 3).contiguous())
    o = torch.where(total > 0, o / total, 0.0).view(S, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(S, T, H, D)
    s["out"][at[real]] = o[real].to(s["out"].dtype)


def _plain_append(s):
    """Free pages go out lowest first; the quantizing is in 64 bits, as values lie next to the border of two codes."""
    ps, table, lens, refs = s["c"]["page_size"], s["table"], s["lens"].long(), s["refs"]
    starts = s["row_starts"].long()
    grown = lens + starts[1:] - starts[:-1]
    have, want = (lens + ps - 1) // ps, (grown + ps - 1) // ps
    base = torch.cumsum(want - have, 0) - (want - have)
    e = torch.arange(table.shape[1], device=DEV)
    fresh = (e[None] >= have[:, None]) & (e[None] < want[:, None])
    order = torch.sort((refs != 0).to(torch.int8), stable=True).indices
    given = order[torch.where(fresh, base[:, None] + e[None] - have[:, None], 0)]
    table.copy_(torch.where(fresh, given, table))
    refs.index_add_(0, given.reshape(-1), fresh.reshape(-1).to(torch.int32))
    r = torch.arange(s["rows"].numel(), device=DEV)
    seq = torch.searchsorted(starts, r, right=True) - 1
    pos = lens[seq] + r - starts[seq]
    page = table[seq, pos // ps].long()
    for l in range(s["c"]["layers"]):
        s["k_pages"][l, page, :, pos % ps] = _pack(s["k_new"][l, s["rows"].long()])
        s["v_pages"][l, page, :, pos % ps] = _pack(s["v_new"][l, s["rows"].long()])
    s["lens"].copy_(grown)
    s["told"].zero_()


def _plain_gather(s):
    ps, D, starts = s["c"]["page_size"], s["c"]["head_dim"], s["row_starts"].long()
    r = torch.arange(s["k_out"].shape[1], device=DEV)
    seq = torch.searchsorted(starts, r, right=True) - 1
    pos = s["begins"].long()[seq] + r - starts[seq]
    page = s["table"][seq, pos // ps].long()
    for l in range(s["c"]["layers"]):
        s["k_out"][l] = _unpack(s["k_pages"][l, page, :, pos % ps], D).to(s["k_out"].dtype)
        s["v_out"][l] = _unpack(s["v_pages"][l, page, :, pos % ps], D).to(s["v_out"].dtype)


def _plain_verify(s):
    """All nodes at once, in 64 bits: which drafted token is taken can hang on the last of them."""
    c, z = s["c"], s["z"]
    parents = sum(z["parents"], [])
    first = [f for f, n in zip(_starts_list(z["nodes"]), z["nodes"]) for _ in range(n)]
    seq = torch.tensor([i for i, n in enumerate(z["nodes"]) for _ in range(n)], device=DEV)
    up = [f + p if p >= 0 else -1 for f, p in zip(first, parents)]
    kids = [[] for _ in up]
    for i, p in enumerate(up):
        if p >= 0:
            kids[p].append(i)
    heat = s["heat"].double()[seq][:, None]
    greedy, T = (heat <= 0)[:, 0], torch.where(heat > 0, heat, 1.0)

    def softmax(x):
        x = x.double()
        e = torch.exp((x - x.amax(1, keepdim=True)) / T)
        return e / e.sum(1, keepdim=True)

    w = softmax(s["logits"])
    best = s["logits"].float().argmax(1)
    q = softmax(s["draft"]) if c["draft"] else None
    total = torch.ones(len(up), dtype=torch.float64, device=DEV)
    taken = torch.zeros(len(up), dtype=torch.bool, device=DEV)  # this child, if its parent is reached
    over = torch.zeros(len(up), dtype=torch.bool, device=DEV)  # by parent: one of its children is taken
    tokens = s["tokens"].long()
    for j in range(c["children"]):
        at = torch.tensor([i for i, k in enumerate(kids) if len(k) > j], dtype=torch.long, device=DEV)
        if not at.numel():
            break
        kid = torch.tensor([k[j] for k in kids if len(k) > j], device=DEV)
        x = tokens[kid]
        rival = q[at, x] if c["draft"] else 1.0
        passes = torch.where(greedy[at], best[at] == x, s["accept"][kid].double() * rival < w[at, x] / total[at]) & ~over[at]
        taken[kid] = passes
        over[at] = over[at] | passes
        rest = w[at] / total[at][:, None]
        if c["draft"]:
            rest = (rest - q[at]).clamp_(min=0)
        else:
            rest[torch.arange(at.numel(), device=DEV), x] = 0
        w[at] = rest  # a node that takes a child has no use for it
        total[at] = rest.sum(1)
    reached = torch.tensor([p < 0 for p in up], device=DEV)
    depth = [0] * len(up)
    for i, p in enumerate(up):
        depth[i] = depth[p] + 1 if p >= 0 else 0
    for d in range(1, max(depth) + 1):
        level = torch.tensor([i for i, k in enumerate(depth) if k == d], device=DEV)
        reached[level] = reached[torch.tensor([up[i] for i in level.tolist()], device=DEV)] & taken[level]
    ends = reached & ~over
    run = torch.cumsum(w, 1)
    drawn = (run <= (s["sample"].double()[seq] * run[:, -1])[:, None]).sum(1)
    drawn = torch.where(greedy, best, drawn)
    s["next"].zero_().index_add_(0, seq, torch.where(ends, drawn, 0).to(torch.int32))
    order = torch.sort((~reached).to(torch.int8), stable=True).indices
    count = torch.zeros(c["seqs"], dtype=torch.int64, device=DEV).index_add_(0, seq, reached.long())
    s["rows"].copy_(torch.where(torch.arange(len(up), device=DEV) < count.sum(), order, -1))
    s["row_starts"][1:] = torch.cumsum(count, 0)


def _starts_list(counts):
    at, out = 0, []
    for n in counts:
        out.append(at)
        at += n
    return out


# ------------------------------------------------------------ the kernels ----
def _calls(s):
    """The operators that a program builds once for its cache and its batch."""
    from iron_amd import operators as ops

    c, z, kind = s["c"], s["z"], s["c"]["kind"]
    if kind == "verify":
        return [ops.DraftVerify(vocab=c["vocab"], num_seqs=c["seqs"], num_nodes=sum(z["nodes"]), max_nodes=c["nodes"],
                                max_children=c["children"], draft=c["draft"], dtype=DTYPES[c["dtype"]]).get_callable()]
    pool = dict(num_pages=z["num_pages"], page_size=c["page_size"], num_seqs=c["seqs"], max_pages=z["max_pages"],
                num_kv_heads=c["kv_heads"], head_dim=c["head_dim"], dtype=DTYPES[c["dtype"]])
    if kind == "tree":
        return [ops.TreeAttentionInt4(num_heads=c["heads"], num_nodes=sum(z["nodes"]), max_nodes=c["nodes"], **pool).get_callable()]
    pool["num_layers"] = c["layers"]
    calls = [ops.PagedGatherInt4(num_rows=sum(z["rows"]), **pool).get_callable()]
    if kind == "append":
        calls.insert(0, ops.PagedAppendInt4(num_nodes=s["k_new"].shape[1], num_rows=s["rows"].numel(), **pool).get_callable())
    return calls


GATHER = ("begins", "row_starts", "k_pages", "v_pages", "table", "lens", "k_out", "v_out")
ARGS = {
    "tree": [("q", "k_new", "v_new", "k_pages", "v_pages", "table", "lens", "starts", "mask", "out")],
    "append": [("k_new", "v_new", "rows", "row_starts", "k_pages", "v_pages", "table", "lens", "refs", "told"), GATHER],
    "gather": [GATHER],
    "verify": [("logits", "draft", "tokens", "parents", "starts", "heat", "accept", "sample", "rows", "row_starts", "next")],
}
PLAIN = {"tree": [_plain_tree], "append": [_plain_append, _plain_gather], "gather": [_plain_gather], "verify": [_plain_verify]}
OUT = {"tree": ("out",), "append": ("table", "lens", "refs", "told", "k_out", "v_out"), "gather": ("k_out", "v_out"),
       "verify": ("rows", "row_starts", "next")}


def run(state):
    kind = state["c"]["kind"]
    if kind == "append":
        state["now"].copy_(state["start"])
    if own:
        if "calls" not in state:
            state["calls"] = _calls(state)
        for call, names in zip(state["calls"], ARGS[kind]):
            call(*(state[a] for a in names if a in state))
    else:
        for step in PLAIN[kind]:
            step(state)
    return {k: state[k] for k in OUT[kind]}


# ------------------------------------------------------ work and 64 bits ----
def work(case):
    c, z = case, _sizes(case)
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "verify":
        N = sum(z["nodes"])
        inner = sum(len({p for p in up if p >= 0}) for up in z["parents"]) if c["draft"] else 0
        rows = (N + inner) * c["vocab"]
        return {"bytes": float(rows * size + 16 * N + 16 * c["seqs"]), "flops": 4.0 * rows}
    D, row16, row4 = c["head_dim"], c["kv_heads"] * c["head_dim"] * 4, c["kv_heads"] * (c["head_dim"] // 2 + 16) * 2  # K and V of a position
    if c["kind"] == "tree":
        N, lens = sum(z["nodes"]), z["lens"]
        nbytes = sum(lens) * row4 + N * row16 + 2 * N * c["heads"] * D * 2 + 4 * sum(_pages(n, c["page_size"]) for n in lens)
        seen = sum(t * (n + 1) for t, n in zip(z["nodes"], lens))
        return {"bytes": float(nbytes), "flops": 4.0 * D * c["heads"] * seen}
    moved = float(sum(z["rows"]) * c["layers"] * (row16 + row4))
    return {"bytes": moved * (2 if c["kind"] == "append" else 1), "flops": 0}


def _exact_rows(s, source, layer, row):
    """What the cache holds for these rows, in 64 bits: a value's code is how many of the 15 borders lie at or below it."""
    g = s[source][layer, row].double().unflatten(-1, (4, -1))
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    step = torch.true_divide(hi - lo, 15.0).float().half().double()
    base = (lo - 16 * step).float().half().double()
    code = torch.zeros_like(g)
    for k in range(15):
        code += ((g >= base + (k + 16.5) * step) & (step > 0)).double()
    return (base + step * (16 + code)).flatten(-2)


def _exact_values(raw, D):
    """The values that rows of bytes stand for, in 64 bits."""
    word = raw[..., :D // 2].contiguous().view(torch.int32)
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=DEV)
    code = ((word[..., None] >> shifts) & 15).flatten(-2).unflatten(-1, (4, -1)).double()
    pair = raw[..., D // 2:].contiguous().view(torch.float16).double().unflatten(-1, (4, 2))
    return (pair[..., 1:] + pair[..., :1] * (code + 16)).flatten(-2)


def _exact_tree(s):
    """Sequence by sequence and position by position."""
    c, z = s["c"], s["z"]
    H, Hkv, D, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    out, first = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV), 0
    for b, (n, t) in enumerate(zip(z["lens"], z["nodes"])):
        pos = torch.arange(n, device=DEV)
        page = s["table"][b, pos // ps].long()
        mine = slice(first, first + t)
        j = torch.arange(t, device=DEV)
        sees = (s["mask"][mine].long()[:, j // 32] >> (j % 32)) & 1 == 1
        hidden = torch.cat([torch.zeros(t, n, dtype=torch.bool, device=DEV), ~sees], 1)
        for h in range(Hkv):
            k = torch.cat([_exact_values(s["k_pages"][page, h, pos % ps], D), s["k_new"][mine, h].double()])
            v = torch.cat([_exact_values(s["v_pages"][page, h, pos % ps], D), s["v_new"][mine, h].double()])
            for x in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                w = (s["q"][mine, x].double() @ k.t().contiguous() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[mine, x] = torch.softmax(w, -1) @ v
        first += t
    return out


def _exact_verify(s):
    """The walk down each tree, one node after the other."""
    c, z = s["c"], s["z"]
    rows, starts, drawn, first = [], [0], [], 0
    heat, accept, sample = s["heat"].tolist(), s["accept"].tolist(), s["sample"].tolist()
    tokens = s["tokens"].tolist()
    for b, up in enumerate(z["parents"]):
        node = 0
        while True:
            rows.append(first + node)
            row = s["logits"][first + node].double()
            if heat[b] <= 0:
                best = int((row == row.max()).nonzero()[0])
                after = [i for i, p in enumerate(up) if p == node and i and tokens[first + i] == best][:1]
            else:
                p = torch.softmax(row / heat[b], 0)
                q = torch.softmax(s["draft"][first + node].double() / heat[b], 0) if c["draft"] else None
                after = []
                for i in (i for i, u in enumerate(up) if u == node and i):
                    x = tokens[first + i]
                    rival = q if c["draft"] else torch.zeros_like(p).index_fill_(0, torch.tensor([x], device=DEV), 1.0)
                    if accept[first + i] * float(rival[x]) < float(p[x]):
                        after = [i]
                        break
                    p = (p - rival).clamp(min=0)
                    p = p / p.sum()
                if not after:
                    run = torch.cumsum(p, 0)
                    best = int((run > sample[b] * run[-1]).nonzero()[0])
            if not after:
                break
            node = after[0]
        drawn.append(best)
        starts.append(len(rows))
        first += len(up)
    rows += [-1] * (first - len(rows))
    return {k: torch.tensor(v, dtype=torch.int32, device=DEV) for k, v in (("rows", rows), ("row_starts", starts), ("next", drawn))}


def exact(case, seed):
    """The attention, the values behind the codes and the walk in 64 bits; tables and counts have no such value."""
    s = prepare(case, seed)
    if case["kind"] == "tree":
        return {"out": _exact_tree(s)}
    if case["kind"] == "verify":
        return _exact_verify(s)
    D, got = case["head_dim"], dict.fromkeys(OUT[case["kind"]])
    if case["kind"] == "append":
        for k in ("k", "v"):
            got[k + "_out"] = torch.stack([_exact_rows(s, k + "_new", l, s["rows"].long()) for l in range(case["layers"])])
        return got
    pos = torch.cat([torch.arange(n - r, n) for n, r in zip(s["z"]["lens"], s["z"]["rows"])]).to(DEV)
    seq = torch.tensor([b for b, r in enumerate(s["z"]["rows"]) for _ in range(r)], device=DEV)
    page = s["table"][seq, pos // case["page_size"]].long()
    for k in ("k", "v"):
        got[k + "_out"] = _exact_values(s[k + "_pages"][:, page, :, pos % case["page_size"]].transpose(0, 1), D)
    return got
