"""What the operators of the paged cache are measured on: calls that a serving program makes through `iron_amd.operators`.

Each case is one operator at one size. `listed()` holds sizes of this repository's configurations, tests and benchmark
(32/8 heads of 64, 16 layers, 2048 and 3968 positions) and generic ones; `draw(rng)` gives other sizes of the same
ranges, odd and ragged ones among them.

Kinds:
  tree     TreeAttention: queries of drafted trees (one node: an ordinary decode step) against paged caches
  append   PagedAppend: rows of accepted tokens or of prompts go to the ends of their sequences, in all layers
  fork     PageFork: children share their parents' whole pages and get a copy of the last, partly filled one
  copy     PageFork(share=False): children get pages of their own with everything in them
  compact  PageCompact: pages in use move down into the holes, the tables follow
  free     PageFree: sequences give their pages back

The page operators change tables and counts in place, so a pass first puts back the ones it started from: one copy of
one small buffer, the same for the plain form and for the kernels.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One token of one conversation: the smallest call, where launches and latency count.
        {"name": "tree_decode_2047", "kind": "tree", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 1, "nodes": 1, "lo": 2047, "hi": 2047},
        # A batch of decode steps behind contexts of very different lengths: bound by the cache's bytes.
        {"name": "tree_decode_batch", "kind": "tree", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 64, "nodes": 1, "lo": 150, "hi": 16384},
        # Drafted trees of ordinary size for a few conversations.
        {"name": "tree_drafts", "kind": "tree", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 8, "nodes": 26, "lo": 37, "hi": 3968},
        # Wide trees behind long documents, the wider heads, fp16: the most arithmetic.
        {"name": "tree_long_wide", "kind": "tree", "dtype": "fp16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "seqs": 2, "nodes": 64, "lo": 20011, "hi": 32768},
        # The tokens that a verification step accepted, for every layer.
        {"name": "append_accepted", "kind": "append", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 8, "lo": 100, "hi": 4000, "rows_lo": 1, "rows_hi": 6},
        # Prompts enter the cache.
        {"name": "append_prompts", "kind": "append", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 4, "lo": 1, "hi": 40, "rows_lo": 512, "rows_hi": 3968},
        # Several continuations of each of a few conversations.
        {"name": "fork_samples", "kind": "fork", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 24, "children": 16, "lo": 700, "hi": 3968},
        # Sequences copied whole, so that their copies can be changed.
        {"name": "copy_sequences", "kind": "copy", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 8, "children": 4, "lo": 1000, "hi": 3968},
        # A pool that is a third holes, packed before it is cut smaller.
        {"name": "compact_third", "kind": "compact", "dtype": "bf16", "layers": 16, "kv_heads": 8, "head_dim": 64,
         "page_size": 16, "seqs": 24, "lo": 500, "hi": 3968, "holes": 0.33, "shared": 8},
        # Tidying up a nearly dense pool: few moves, so the search for them counts.
        {"name": "compact_tidy", "kind": "compact", "dtype": "bf16", "layers": 4, "kv_heads": 2, "head_dim": 64,
         "page_size": 16, "seqs": 64, "lo": 3000, "hi": 16000, "holes": 0.002, "shared": 3},
        # A step's finished conversations.
        {"name": "free_finished", "kind": "free", "page_size": 16, "seqs": 256, "ends": 16, "lo": 100, "hi": 3968, "shared": 4},
        # A server that lets go of long documents, many of their pages shared.
        {"name": "free_long", "kind": "free", "page_size": 16, "seqs": 128, "ends": 96, "lo": 20000, "hi": 131072, "shared": 600},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "append", "fork", "copy", "compact", "free"])
    c = {"kind": kind, "page_size": rng.choice([16, 16, 32, 64, 128])}
    if kind == "free":
        seqs = _log(rng, 2, 256)
        hi = _log(rng, 200, 131072 * 64 // max(64, seqs))
        return {**c, "seqs": seqs, "ends": rng.randint(1, seqs), "lo": _log(rng, 1, hi), "hi": hi, "shared": rng.randint(0, 40)}
    c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "tree":
        heads, kv = rng.choice([(32, 8), (32, 8), (16, 16), (64, 8), (8, 2), (24, 8), (10, 2), (12, 1)])
        c |= {"heads": heads, "kv_heads": kv, "head_dim": rng.choice([64, 64, 128]), "nodes": rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 200)])}
        seqs = _log(rng, 1, 64)
        most = min(32768, 64 * 8192 // seqs, 2 * 64 * 32768 * 32 // (seqs * c["nodes"] * heads))
        hi = _log(rng, 16, max(64, most))
        return {**c, "seqs": seqs, "lo": _log(rng, 1, hi), "hi": hi}
    c |= {"layers": rng.choice([1, 2, 4, 16]), "kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 128])}
    room = 16 * 8 * 64 / (c["layers"] * c["kv_heads"] * c["head_dim"])  # how many of this case's positions make one of the largest one's
    seqs = _log(rng, 2, 32)
    hi = _log(rng, 40, int(min(16384, 60000 * room / seqs)))
    c |= {"seqs": seqs, "lo": _log(rng, 1, hi), "hi": hi}
    if kind == "append":
        rows = _log(rng, 1, int(min(4000, 16000 * room / seqs)))
        return {**c, "rows_lo": rng.randint(1, rows), "rows_hi": rows}
    if kind == "compact":
        return {**c, "holes": rng.choice([0.003, 0.05, 0.3, 0.6]), "shared": rng.randint(0, 4)}
    children = rng.randint(1, seqs - 1 if kind == "copy" else max(1, seqs // 2))
    return {**c, "seqs": seqs, "children": children}


# ------------------------------------------------------------------ sizes ----
def _spread(lo, hi, count):
    """`count` lengths of [lo, hi], ragged, the same for every seed (the golden ratio's multiples)."""
    return [min(hi, max(lo, round(lo * (hi / lo) ** ((i * 0.6180339887 + 0.31) % 1.0)))) for i in range(count)]


def _pages(n, ps):
    return -(-n // ps)


def _sizes(c):
    """Lengths and counts that the case fixes."""
    ps, S, kind = c["page_size"], c["seqs"], c["kind"]
    z = {"lens": _spread(c["lo"], c["hi"], S)}
    if kind == "tree":
        z["nodes"] = _spread(max(1, c["nodes"] // 2), c["nodes"], S)
        z["nodes"][0], z["lens"][-1] = c["nodes"], c["hi"]
    if kind in ("fork", "copy"):  # the last slots are the children, empty before the call
        z["parents"] = S - c["children"]
        z["lens"][z["parents"]:] = [0] * c["children"]
        z["from"] = [(5 * i + 1) % z["parents"] for i in range(c["children"])]
    grown = list(z["lens"])
    if kind == "append":
        z["rows"] = _spread(c["rows_lo"], c["rows_hi"], S)
        grown = [n + r for n, r in zip(grown, z["rows"])]
    z["max_pages"] = max(_pages(n, ps) for n in grown) + 1
    z["shared"] = [min(c.get("shared", 0), n // ps) for n in z["lens"]]  # leading pages shared by neighbouring sequences
    z["distinct"] = sum(_pages(n, ps) for n in grown)
    live = z["distinct"]
    if kind in ("fork", "copy"):
        live += sum(_pages(z["lens"][p], ps) for p in z["from"])
    z["num_pages"] = int(live / (1 - c["holes"])) + 1 if kind == "compact" else live + live // 8 + 2
    return z


# ----------------------------------------------------------------- inputs ----
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


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
    ps, S, P, MP = c["page_size"], c["seqs"], z["num_pages"], z["max_pages"]
    lens = torch.tensor(z["lens"], device=DEV)
    used = (lens + ps - 1) // ps
    base = torch.cumsum(used, 0) - used
    e = torch.arange(MP, device=DEV)
    live = e[None] < used[:, None]
    ids = torch.randperm(P, generator=g, device=DEV)
    first = torch.arange(S, device=DEV) // 4 * 4  # the first of four neighbours lends its leading pages
    shared = torch.minimum(torch.tensor(z["shared"], device=DEV), torch.tensor(z["shared"], device=DEV)[first])
    owner = torch.where(e[None] < shared[:, None], base[first][:, None], base[:, None])
    table = torch.where(live, ids[torch.where(live, owner + e[None], 0)], -1)
    refs = torch.zeros(P, dtype=torch.int64, device=DEV)
    refs.index_add_(0, table.clamp(min=0).reshape(-1), live.reshape(-1).to(torch.int64))
    return table.to(torch.int32), lens.to(torch.int32), refs.to(torch.int32)


def _masks(c, z, g):
    """Random trees: each node's parent is one of the nodes before it; a node sees itself and those above it, as bits."""
    S, T = c["seqs"], c["nodes"]
    parent = (torch.rand(S, T, generator=g, device=DEV) * torch.arange(T, device=DEV)).long()
    sees = torch.eye(T, dtype=torch.bool, device=DEV).repeat(S, 1, 1)
    for i in range(1, T):
        sees[:, i] |= sees[torch.arange(S, device=DEV), parent[:, i]]
    W = (T + 31) // 32
    bits = torch.nn.functional.pad(sees, (0, 32 * W - T)).view(S, T, W, 32).long()
    words = (bits << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32), sees


def prepare(case, seed):
    c, z, g = dict(case), _sizes(case), _generator(seed)
    st = {"c": c, "z": z}
    table, lens, refs = _tables(c, z, g)

    def noise(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=DTYPES[c["dtype"]]).mul_(scale)

    if c["kind"] == "tree":
        S, H, Hkv, D, T = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], c["nodes"]
        N = sum(z["nodes"])
        starts = torch.tensor([0] + z["nodes"], device=DEV).cumsum(0).to(torch.int32)
        words, _ = _masks(c, z, g)
        mask = torch.zeros(N, words.shape[-1], dtype=torch.int32, device=DEV)
        for s, n in enumerate(z["nodes"]):
            mask[sum(z["nodes"][:s]):sum(z["nodes"][:s]) + n] = words[s, :n]
        # queries of twice the unit size: some keys stand out, as they do in a trained model
        return st | {"q": noise(N, H, D, scale=2.0), "k_new": noise(N, Hkv, D), "v_new": noise(N, Hkv, D),
                     "k_pages": noise(z["num_pages"], Hkv, c["page_size"], D), "v_pages": noise(z["num_pages"], Hkv, c["page_size"], D),
                     "table": table, "lens": lens, "starts": starts, "mask": mask,
                     "out": torch.zeros(N, H, D, dtype=DTYPES[c["dtype"]], device=DEV)}
    st["start"], st["now"], (st["table"], st["lens"], st["refs"]) = _meta([table, lens, refs])
    # what each request came to (0: done), and of the packing the number of pages moved
    told = {"append": c["seqs"], "fork": c.get("children"), "copy": c.get("children"), "compact": 1, "free": c.get("ends")}[c["kind"]]
    st["told"] = torch.zeros(told, dtype=torch.int32, device=DEV)
    if c["kind"] == "free":
        return st | {"slots": torch.randperm(c["seqs"], generator=g, device=DEV)[:c["ends"]].to(torch.int32)}
    L, Hkv, D = c["layers"], c["kv_heads"], c["head_dim"]
    st |= {"k_pages": noise(L, z["num_pages"], Hkv, c["page_size"], D), "v_pages": noise(L, z["num_pages"], Hkv, c["page_size"], D)}
    if c["kind"] == "append":
        M = sum(z["rows"])
        # the accepted ones are some of the rows that the step computed
        N = M + M // 2 + 1
        st |= {"k_new": noise(L, N, Hkv, D), "v_new": noise(L, N, Hkv, D),
               "rows": torch.randperm(N, generator=g, device=DEV)[:M].to(torch.int32),
               "row_starts": torch.tensor([0] + z["rows"], device=DEV).cumsum(0).to(torch.int32)}
    if c["kind"] in ("fork", "copy"):
        to = z["parents"] + torch.randperm(c["children"], generator=g, device=DEV)
        st["forks"] = torch.stack([torch.tensor(z["from"], device=DEV), to], 1).to(torch.int32).contiguous()
    return st


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
    keys = s["k_pages"][table.clamp(min=0)].float().transpose(1, 2).reshape(S, Hkv, cap, D)
    values = s["v_pages"][table.clamp(min=0)].float().transpose(1, 2).reshape(S, Hkv, cap, D)
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
    return s["out"]


def _lowest_free(refs):
    """The pages in the order in which they are given out: free ones first, each kind by its number."""
    return torch.sort((refs != 0).to(torch.int8), stable=True).indices


def _plain_append(s):
    ps, table, lens, refs = s["c"]["page_size"], s["table"], s["lens"].long(), s["refs"]
    starts = s["row_starts"].long()
    grown = lens + starts[1:] - starts[:-1]
    have, want = (lens + ps - 1) // ps, (grown + ps - 1) // ps
    base = torch.cumsum(want - have, 0) - (want - have)
    e = torch.arange(table.shape[1], device=DEV)
    fresh = (e[None] >= have[:, None]) & (e[None] < want[:, None])
    order = _lowest_free(refs)
    given = order[torch.where(fresh, base[:, None] + e[None] - have[:, None], 0)]
    table.copy_(torch.where(fresh, given, table))
    refs.index_add_(0, given.reshape(-1), fresh.reshape(-1).to(torch.int32))
    r = torch.arange(s["rows"].numel(), device=DEV)
    seq = torch.searchsorted(starts, r, right=True) - 1
    pos = lens[seq] + r - starts[seq]
    page = table[seq, pos // ps].long()
    s["k_pages"][:, page, :, pos % ps] = s["k_new"][:, s["rows"].long()].transpose(0, 1)
    s["v_pages"][:, page, :, pos % ps] = s["v_new"][:, s["rows"].long()].transpose(0, 1)
    s["lens"].copy_(grown)


def _plain_fork(s):
    """Both ways: `own_from` is the first page of a child that is its own and not its parent's."""
    ps, table, refs = s["c"]["page_size"], s["table"], s["refs"]
    parent, child = s["forks"].long().unbind(1)
    n = s["lens"].long()[parent]
    own_from = n // ps if s["c"]["kind"] == "fork" else torch.zeros_like(n)
    pages = (n + ps - 1) // ps
    base = torch.cumsum(pages - own_from, 0) - (pages - own_from)
    e = torch.arange(table.shape[1], device=DEV)
    live, copied = e[None] < pages[:, None], (e[None] < pages[:, None]) & (e[None] >= own_from[:, None])
    order = _lowest_free(refs)
    was = table.long()[parent]
    now = torch.where(copied, order[torch.where(copied, base[:, None] + e[None] - own_from[:, None], 0)], was)
    refs.index_add_(0, torch.where(live, now, 0).reshape(-1), live.reshape(-1).to(torch.int32))
    table[child] = torch.where(live, now, table.long()[child]).to(torch.int32)
    src, dst = was[copied], now[copied]
    rows = (n[:, None] - e[None] * ps).clamp(max=ps)[copied]
    inside = (torch.arange(ps, device=DEV)[None] < rows[:, None])[None, :, None, :, None]
    s["k_pages"][:, dst] = torch.where(inside, s["k_pages"][:, src], s["k_pages"][:, dst])
    s["v_pages"][:, dst] = torch.where(inside, s["v_pages"][:, src], s["v_pages"][:, dst])
    s["lens"][child] = s["lens"][parent]


def _plain_compact(s):
    ps, table, refs = s["c"]["page_size"], s["table"], s["refs"]
    live, page = refs > 0, torch.arange(refs.numel(), device=DEV)
    kept = page < live.sum()
    src, dst = page[live & ~kept], page[~live & kept]
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    page[src] = dst
    used = torch.arange(table.shape[1], device=DEV)[None] < ((s["lens"].long() + ps - 1) // ps)[:, None]
    table.copy_(torch.where(used & (table >= 0), page[table.long().clamp(min=0)], table))
    refs[dst] = refs[src]
    refs[src] = 0
    s["told"].fill_(src.numel())


def _plain_free(s):
    ps, table, slots = s["c"]["page_size"], s["table"], s["slots"].long()
    rows = table[slots].long()
    used = torch.arange(table.shape[1], device=DEV)[None] < ((s["lens"].long()[slots] + ps - 1) // ps)[:, None]
    s["refs"].index_add_(0, rows.clamp(min=0).reshape(-1), -(used & (rows >= 0)).reshape(-1).to(torch.int32))
    table[slots] = torch.where(used, -1, rows).to(torch.int32)
    s["lens"][slots] = 0


PLAIN = {"append": _plain_append, "fork": _plain_fork, "copy": _plain_fork, "compact": _plain_compact, "free": _plain_free}


# ------------------------------------------------------------ the kernels ----
def _callable(s):
    """The operator that a program builds once for its cache."""
    from iron_amd import operators as ops

    c, z, kind = s["c"], s["z"], s["c"]["kind"]
    pool = dict(num_pages=z["num_pages"], page_size=c["page_size"], num_seqs=c["seqs"], max_pages=z["max_pages"])
    if kind == "free":
        return ops.PageFree(**pool, num_slots=c["ends"]).get_callable()
    pool |= dict(num_kv_heads=c["kv_heads"], head_dim=c["head_dim"], dtype=DTYPES[c["dtype"]])
    if kind == "tree":
        return ops.TreeAttention(num_heads=c["heads"], num_nodes=sum(z["nodes"]), max_nodes=c["nodes"], **pool).get_callable()
    pool["num_layers"] = c["layers"]
    if kind == "append":
        return ops.PagedAppend(num_nodes=s["k_new"].shape[1], num_rows=s["rows"].numel(), **pool).get_callable()
    if kind == "compact":
        return ops.PageCompact(**pool).get_callable()
    return ops.PageFork(num_forks=c["children"], share=kind == "fork", **pool).get_callable()


ARGS = {
    "tree": ("q", "k_new", "v_new", "k_pages", "v_pages", "table", "lens", "starts", "mask", "out"),
    "append": ("k_new", "v_new", "rows", "row_starts", "k_pages", "v_pages", "table", "lens", "refs", "told"),
    "fork": ("forks", "k_pages", "v_pages", "table", "lens", "refs", "told"),
    "copy": ("forks", "k_pages", "v_pages", "table", "lens", "refs", "told"),
    "compact": ("k_pages", "v_pages", "table", "lens", "refs", "told"),
    "free": ("slots", "table", "lens", "refs", "told"),
}


def run(state):
    kind = state["c"]["kind"]
    if kind != "tree":
        state["now"].copy_(state["start"])
    if own:
        if "call" not in state:
            state["call"] = _callable(state)
        state["call"](*(state[a] for a in ARGS[kind]))
    elif kind == "tree":
        _plain_tree(state)
    else:
        PLAIN[kind](state)
    if kind == "tree":
        return state["out"]
    got = {k: state[k] for k in ("table", "lens", "refs", "told")}
    if kind != "free":
        got |= {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    return got


# ------------------------------------------------------ work and 64 bits ----
def work(case):
    c, z = case, _sizes(case)
    ps, lens = c["page_size"], z["lens"]
    pages = [_pages(n, ps) for n in lens]
    if c["kind"] == "free":
        share = c["ends"] / c["seqs"]
        return {"bytes": 16.0 * sum(pages) * share, "flops": 0}  # an entry read and cleared, a count read and written
    row = c["kv_heads"] * c["head_dim"] * 2 * 2  # a position's K and V in one layer
    if c["kind"] == "tree":
        N = sum(z["nodes"])
        nbytes = (sum(lens) + N) * row + 2 * N * c["heads"] * c["head_dim"] * 2 + 4 * sum(pages)
        seen = sum(t * (n + 1) for t, n in zip(z["nodes"], lens))
        return {"bytes": nbytes, "flops": 4.0 * c["head_dim"] * c["heads"] * seen}
    row *= c["layers"]
    if c["kind"] == "append":
        return {"bytes": 2.0 * sum(z["rows"]) * row, "flops": 0}
    if c["kind"] == "compact":
        distinct = sum(pages) - sum(min(a, z["shared"][i // 4 * 4]) for i, a in enumerate(z["shared"]) if i % 4)
        moved = distinct * (z["num_pages"] - distinct) / z["num_pages"]  # of the pages in use, those behind the last kept one
        return {"bytes": 2.0 * moved * ps * row + 4.0 * z["num_pages"] + 4.0 * sum(pages), "flops": 0}
    total = sum(lens[p] % ps if c["kind"] == "fork" else lens[p] for p in z["from"])
    return {"bytes": 2.0 * total * row + 8.0 * sum(pages[p] for p in z["from"]), "flops": 0}


def exact(case, seed):
    """The attention in 64 bits, sequence by sequence and position by position; the other operators only move values."""
    if case["kind"] != "tree":
        return None
    s = prepare(case, seed)
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
            k = torch.cat([s["k_pages"][page, h, pos % ps], s["k_new"][mine, h]]).double()
            v = torch.cat([s["v_pages"][page, h, pos % ps], s["v_new"][mine, h]]).double()
            for x in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                w = (s["q"][mine, x].double() @ k.t().contiguous() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[mine, x] = torch.softmax(w, -1) @ v
        first += t
    return out
