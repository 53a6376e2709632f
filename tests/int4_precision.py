"""How far a result of TreeAttentionInt4 may be off, key by key, and what other roundings of the cache would make of it: the
kernels are held to the documented ones, not to any that a wide bound lets through."""

import math

import torch

from tests import int4_reference as ref

H16, H32 = 2.0 ** -11, 2.0 ** -24  # half a step of fp16, of fp32


def keep(x):
    return x


def fp16(x):
    return x.half().double()


def bf16(x):
    return x.to(torch.bfloat16).double()


def sequences(c):
    """Of each sequence and KV head of a case: its rows, queries (rows, G, D), keys and values (cached ones first) in 64 bits,
    the pairs of the cached keys, what each row sees, and how many positions are cached."""
    q, D, ps = c["q"], c["q"].shape[-1], c["k"].shape[2]
    Hkv = c["k_new"].shape[1]
    G = q.shape[1] // Hkv
    for s, n in enumerate(c["lens"]):
        a, b = c["starts"][s], c["starts"][s + 1]
        if a == b:
            continue
        t = torch.arange(n, device=q.device)
        page = c["table"][s].to(q.device).long()[t // ps]
        seen = torch.cat([torch.ones(b - a, n, dtype=torch.bool, device=q.device), c["sees"][a:b, :b - a].to(q.device)], 1)
        for h in range(Hkv):
            raw = c["k"][page, h, t % ps]
            k = torch.cat([ref.values(raw, D), c["k_new"][a:b, h].double()])
            v = torch.cat([ref.values(c["v"][page, h, t % ps], D), c["v_new"][a:b, h].double()])
            pair = raw[:, D // 2:].contiguous().view(torch.float16).double().unflatten(-1, (4, 2)).repeat_interleave(D // 4, 1)
            yield slice(a, b), slice(h * G, (h + 1) * G), q[a:b, h * G:(h + 1) * G].double(), k, v, pair, seen, n


def attention(c, scale, keys=keep, values=keep, weights=keep):
    """The attention in 64 bits, with cached keys and values and all weights (the largest of a row is 64) as the given functions
    round them; the sum of a row's weights is of the rounded ones."""
    out = torch.zeros(c["q"].shape, dtype=torch.float64, device=c["q"].device)
    for rows, heads, q, k, v, _, seen, n in sequences(c):
        k, v = torch.cat([keys(k[:n]), k[n:]]), torch.cat([values(v[:n]), v[n:]])
        for g in range(q.shape[1]):
            w = (q[:, g] @ k.t().contiguous() * scale).masked_fill(~seen, -math.inf)
            p = weights(64 * torch.exp(w - w.amax(1, keepdim=True)))
            out[rows, heads.start + g] = p @ v / p.sum(1, keepdim=True)
    return out


def bound(c, scale, exact_scores=False):
    """(result, how far it may be off) in 64 bits. A weight's relative error is what its own score is off by, and its rounding:

    - sums of n terms in fp32, 2^-23 of the terms' sizes each, with D terms; in fp16 calls 2 D + 8, of b + s (16 + code) apart
      (nothing, nor the next but one, where fp32 holds them: `exact_scores`);
    - bf16: a cached key's rounding to fp16, and q's elements far under the row's largest (2^-39 of that);
    - fp16: the lower part of s (2^-24 of a code's value), b by sums of q in two parts: 2^-22 of the sum, D / 4 roundings of it,
      and like q's small elements 2^-33 of the row's largest;
    - the score times log2(e) less the maximum, 2^-22 of the largest score, the exponential and the parts' joining, 2^-21;
    - its rounding for the second product: fp16 (bf16 calls, cached), 2^-20 in two parts, half a step of dtype for nodes where a
      KV head has more than 32 rows; 2^-30 of a row's largest for weights under fp16's normal range.
    A cached value is rounded to fp16 (nothing where fp16 holds it). Sums of n terms add n 2^-23. The result is rounded once."""
    dtype, D = c["prior"].dtype, c["q"].shape[-1]
    out, tol = (torch.zeros(c["q"].shape, dtype=torch.float64, device=c["q"].device) for _ in range(2))
    half, two = torch.finfo(dtype).eps / 2, 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -16
    node = half if c["T"] * (c["q"].shape[1] // c["k_new"].shape[1]) > 32 else two
    for rows, heads, q, k, v, pair, seen, n in sequences(c):
        kr = torch.full((len(k),), node, dtype=torch.float64, device=q.device)
        kr[:n] = H16 if dtype == torch.bfloat16 else two
        vr = torch.where(fp16(v) == v, 0.0, H16 * v.abs() + 2.0 ** -25)
        vr[n:] = 0
        for g in range(q.shape[1]):
            x, w = q[:, g], (q[:, g] @ k.t().contiguous() * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(w, 1)
            size = x.abs() @ k.abs().t().contiguous() * scale
            off = torch.zeros_like(w) if exact_scores else 2 * (D + 2) * H32 * size
            if dtype == torch.bfloat16:
                off[:, :n] += H16 * size[:, :n] + scale * (2.0 ** -25 * x.abs().sum(1)[:, None] + 2.0 ** -39 * x.abs().amax(1)[:, None] * k[:n].abs().sum(1)[None])
            elif not exact_scores:
                b = pair[..., 1].abs()
                apart = x.abs() @ (b + (k[:n] - pair[..., 1]).abs()).t().contiguous()
                sums = x.unflatten(1, (4, -1)).sum(2).abs().repeat_interleave(D // 4, 1) / (D // 4)
                least = 2.0 ** -33 * x.abs().amax(1, keepdim=True)
                off[:, :n] = scale * (2 * (2 * D + 10) * H32 * apart + 2.0 ** -24 * x.abs().sum(1)[:, None] + least * (k[:n] - pair[..., 1]).abs().sum(1)[None]
                                      + (2.0 ** -22 * sums + D / 4 * H32 * x.abs() + least) @ b.t().contiguous())
            top = w.masked_fill(~seen, 0).abs().amax(1, keepdim=True)
            each = off + 2.0 ** -21 * (1 + 1.5 * top) + kr
            o, m = p @ v, p @ v.abs()
            err = (p * each) @ v.abs() + (p * each).sum(1, keepdim=True) * o.abs() + p @ vr + 4 * (len(k) + 8) * H32 * m + 2.0 ** -30 * len(k) * v.abs().amax()
            out[rows, heads.start + g] = o
            tol[rows, heads.start + g] = half * o.abs() + 1.01 * err + 2.0 ** -25
    return out, tol


def rms(x):
    return float(x.double().pow(2).mean().sqrt())


def ratio(got, want):
    """The error over that of rounding `want` once, both as root mean squares."""
    return rms(got.double() - want) / rms(want.to(got.dtype).double() - want)


def with_pairs(pages, D, s, b):
    pages = pages.clone()
    pages[..., D // 2:] = torch.stack([s, b], -1).half().view(torch.uint8).flatten(-2)
    return pages


def exact_values(c, seed):
    """The case with cached values that fp16 holds: whole eighths."""
    g = torch.Generator(device=c["v"].device).manual_seed(seed)
    b = -(23 + torch.randint(-8, 9, (*c["v"].shape[:-1], 4), generator=g, device=c["v"].device)) / 8
    return {**c, "v": with_pairs(c["v"], c["q"].shape[-1], torch.full_like(b, 0.125), b)}


def exact_scores(c, seed):
    """The case with queries of +-1 and keys whose sums fp32 holds: multiples of 2^-13 below 2^10 (D 64, 2^11 with 128), b and
    the trees' keys of 2^-6. Cached keys have up to 16 bits, so fp16 does not hold them."""
    g = torch.Generator(device=c["k"].device).manual_seed(seed)
    draw = lambda shape, lo, hi: torch.randint(lo, hi, shape, generator=g, device=c["k"].device)
    shape = (*c["k"].shape[:-1], 4)
    s = draw(shape, 1024, 2048) / 2.0 ** 12
    b = -torch.round(s * 23.5 * 64) / 64 + draw(shape, -32, 33) / 64
    return {**c, "k": with_pairs(c["k"], c["q"].shape[-1], s, b), "q": (draw(c["q"].shape, 0, 2) * 2 - 1).to(c["q"].dtype),
            "k_new": (draw(c["k_new"].shape, -128, 129) / 64).to(c["q"].dtype)}
