"""Plain implementations of the 4-bit cache's operators and of the verification of drafted tokens for the tests, in 64
bits and as loops, written from the operators' documentation."""

import math

import numpy as np
import torch

MOST = 20480.0


def row_bytes(D):
    return D // 2 + 16


def quantize(x):
    """Rows of values (any leading shape, D) -> (codes uint8 (.., D), s and b fp16 (.., 4)): every code by its definition,
    the number of borders at or below the value."""
    g = x.double().reshape(*x.shape[:-1], 4, -1)
    nan = torch.isnan(g).any(-1)
    g = torch.where(nan[..., None], 0.0, g).clamp(-MOST, MOST)
    lo, hi = g.amin(-1), g.amax(-1)
    s = torch.from_numpy(((hi - lo) / 15).numpy().astype(np.float16))
    b = torch.from_numpy((lo - 16 * s.double() + 0.0).numpy().astype(np.float16))
    code = torch.zeros(g.shape, dtype=torch.uint8)
    for k in range(15):
        border = b.double() + (k + 16.5) * s.double()
        code += ((g >= border[..., None]) & (s > 0)[..., None]).to(torch.uint8)
    b = torch.where(nan, torch.tensor(float("nan"), dtype=torch.float16), b)
    return code.reshape(x.shape), s, b


def pack(code, s, b):
    c = code.reshape(*code.shape[:-1], -1, 8).numpy().astype(np.uint32)
    word = sum(c[..., i] << (4 * (i // 2) + 16 * (i % 2)) for i in range(8)).astype("<u4")
    pairs = np.stack([s.numpy().view(np.uint16), np.where(np.isnan(b.numpy()), 0x7e00, b.numpy().view(np.uint16))], -1).astype("<u2")
    flat = lambda a, n: np.ascontiguousarray(a).view(np.uint8).reshape(*code.shape[:-1], n)
    return torch.from_numpy(np.concatenate([flat(word, code.shape[-1] // 2), flat(pairs, 16)], -1))


def to_rows(x):
    return pack(*quantize(x))


def values(rows, D):
    """Rows of bytes (any leading shape) -> their values in 64 bits, on the rows' device."""
    word = rows[..., :D // 2].contiguous().view(torch.int32)
    shifts = torch.tensor([4 * (i // 2) + 16 * (i % 2) for i in range(8)], device=rows.device)
    code = ((word[..., None] >> shifts) & 15).flatten(-2).unflatten(-1, (4, -1)).double()
    pair = rows[..., D // 2:].contiguous().view(torch.float16).double().unflatten(-1, (4, 2))
    return (pair[..., 1:] + pair[..., :1] * (16 + code)).flatten(-2)


def attention(q, k_new, v_new, k_pages, v_pages, table, lens, starts, sees, scale, prior, max_nodes):
    """TreeAttentionInt4 in 64 bits, with the bound of its rounding: (out, tolerance), both float64, on q's device.

    Roundings, each relative: a cached value to fp16, h = 2^-11 (2^-25 where it is subnormal); a score's sum of D terms in
    fp32, (D + 2) 2^-24 of the terms' sizes; its product with log2(e) and the subtraction of a maximum, 2^-22 of the largest
    score; the exponential, 2^-22. A weight is rounded before the second product: a cached position's to fp16, h; a tree
    node's 2^-16 in two parts, or half a step of dtype where a KV head has more than 32 rows. Each shows in the sum of the
    weights too, hence twice. Weights may lie under fp16's normal range: 2^-30 of the largest each (2^-24 for the lower of two
    fp16 parts). Sums of n terms in fp32 add n 2^-24. All of it is relative to sum(p |v|). The result is rounded once.
    """
    dev = q.device
    out, tol = prior.double().clone(), torch.zeros(prior.shape, dtype=torch.float64, device=dev)
    D, ps, h = q.shape[-1], k_pages.shape[2], 2.0 ** -11
    G, half = q.shape[1] // k_new.shape[1], torch.finfo(prior.dtype).eps / 2
    node_weight = half if max_nodes * G > 32 else 2.0 ** -16
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        if b == a:
            continue
        t = torch.arange(n, device=dev)
        page = table[s].to(dev).long()[t // ps]
        t = t[(page >= 0) & (page < k_pages.shape[0])]
        page = table[s].to(dev).long()[t // ps]
        hidden = ~sees[a:b, :b - a].to(dev)
        for hk in range(k_new.shape[1]):
            kc, vc = values(k_pages[page, hk, t % ps], D), values(v_pages[page, hk, t % ps], D)
            kn, vn = k_new[a:b, hk].double(), v_new[a:b, hk].double()
            for x in range(hk * G, (hk + 1) * G):
                w = torch.cat([q[a:b, x].double() @ kc.t().contiguous(), (q[a:b, x].double() @ kn.t().contiguous()).masked_fill(hidden, -math.inf)], 1) * scale
                none = (w == -math.inf).all(1)
                p = torch.where(none[:, None], 0.0, torch.softmax(torch.where(none[:, None], 0.0, w), 1))
                v = torch.cat([vc, vn])
                out[a:b, x] = p @ v
                size = q[a:b, x].double().abs() @ torch.cat([kc, kn]).abs().t().contiguous() * scale
                size = size.masked_fill(w == -math.inf, 0).amax(1)
                top = w.masked_fill(w == -math.inf, 0).abs().amax(1)
                each = (h + (D + 2) * 2.0 ** -24) * size + 2.0 ** -22 * (1 + 1.5 * top) + D * 2.0 ** -25 * q[a:b, x].double().abs().amax(1) * scale
                keys = w.shape[1]
                rel = 2 * (each + max(h, node_weight)) + h + (keys + 8) * 2.0 ** -24
                tol[a:b, x] = half * out[a:b, x].abs() + rel[:, None] * (p @ v.abs()) * (1 + half)
                floor = 2.0 ** -30 * len(kc) + (2.0 ** -24 * (b - a) if prior.dtype == torch.float16 else 0)
                tol[a:b, x] += floor * float(v.abs().max()) + 2.0 ** -25
    return out, tol


def gather(k_pages, v_pages, table, lens, begins, starts, prior_k, prior_v, D):
    """PagedGatherInt4 on CPU tensors: what k_out and v_out hold afterwards."""
    ps, out = k_pages.shape[3], (prior_k.clone(), prior_v.clone())
    for r in range(prior_k.shape[1]):
        owner = [s for s in range(len(lens)) if starts[s] <= r < starts[s + 1]]
        if not owner:
            continue
        s = owner[0]
        pos = begins[s] + r - starts[s]
        page = int(table[s][pos // ps]) if 0 <= pos < min(lens[s], table.shape[1] * ps) else -1
        for o, pages in zip(out, (k_pages, v_pages)):
            o[:, r] = values(pages[:, page, :, pos % ps], D).to(o.dtype) if 0 <= page < k_pages.shape[1] else 0
    return out


def softmax(row, temp):
    """Probabilities of a row of logits in 64 bits; all zero for a row without any."""
    x = row.double().numpy().copy()
    x[np.isnan(x)] = -math.inf
    x = np.minimum(x, float(np.finfo(np.float32).max))
    none = x == -math.inf
    if none.all():
        return np.zeros_like(x)
    e = np.where(none, 0.0, np.exp(np.where(none, 0.0, x - x.max()) * (1.0 / float(temp))))
    return e / e.sum()


def verify(logits, draft, tokens, parents, starts, temps, accept, sample, max_children):
    """DraftVerify on CPU tensors: (rows, row_starts, next_tokens) as lists, and the smallest distance of a decision from
    its border, relative to what is compared (a test that rounding can turn tells nothing)."""
    rows, row_starts, nexts, margin = [], [0], [], math.inf
    V = logits.shape[1]
    for s in range(len(starts) - 1):
        a, n = starts[s], starts[s + 1] - starts[s]
        row_starts.append(row_starts[-1])
        if n == 0:
            nexts.append(-1)
            continue
        temp = float(temps[s])
        node, i = 0, 0
        while True:
            rows.append(a + node)
            row_starts[-1] += 1
            kids = [c for c in range(node + 1, n) if parents[a + c] == node][:max_children]
            taken = None
            if not temp > 0:
                x = logits[a + node].double().numpy().copy()
                x[np.isnan(x)] = -math.inf
                x = np.minimum(x, float(np.finfo(np.float32).max))
                best = int(np.argmax(x)) if x.max() > -math.inf else -1
                taken = next((c for c in kids if best >= 0 and tokens[a + c] == best), None)
            else:
                p0 = softmax(logits[a + node], temp)
                q = softmax(draft[a + node], temp) if draft is not None else None
                p = p0.copy()
                for c in kids:
                    if p.sum() == 0:
                        break
                    x, u = int(tokens[a + c]), float(accept[a + c])
                    if draft is None:
                        q = np.zeros(V)
                        if 0 <= x < V:
                            q[x] = 1.0
                    px, qx = (p[x], q[x]) if 0 <= x < V else (0.0, 0.0 if draft is not None else 1.0)
                    if px or qx * u:
                        margin = min(margin, abs(u * qx - px) / max(px, u * qx))
                    if u * qx < px:
                        taken = c
                        break
                    p = np.maximum(p - q, 0.0)
                    if p.sum() > 0:
                        p = p / p.sum()
                if taken is None:
                    if p.sum() == 0:
                        p = p0
                    if p.sum() == 0:
                        best = -1
                    else:
                        run = np.cumsum(p)
                        goal = float(sample[s]) * run[-1]
                        hits = np.nonzero((run > goal) & (p > 0))[0]  # none without probability, whatever the number
                        best = int(hits[0]) if len(hits) else int(np.nonzero(p)[0][-1])
                        if 0 < goal < run[-1]:
                            margin = min(margin, float(np.abs(run - goal).min() / run[-1]))
            if taken is None:
                nexts.append(best)
                break
            node = taken
    return rows + [-1] * (len(tokens) - len(rows)), row_starts, nexts, margin
