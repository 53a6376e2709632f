"""DraftVerify where one token has nearly all of the probability of both rows and the drafted ones next to none: what is left
after a child is 10^-8 and less, and what is left of that after the next one hangs on how it is computed. The oracle here works with
60 digits; a case counts where 64 bits with errors of 2^-46 in the exponentials decide it."""

import math
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

from tests import int4_reference as ref
from tests import test_draft_verify_gpu as calls


def softmax60(row, temp):
    getcontext().prec = 60
    x = row.double().tolist()
    top = max(x)
    if top == -math.inf:
        return [Decimal(0)] * len(x)
    e = [Decimal(0) if v == -math.inf else ((Decimal(v) - Decimal(top)) / Decimal(temp)).exp() for v in x]
    total = sum(e)
    return [v / total for v in e]


def softmax64(row, temp, g):
    """In 64 bits, each exponential off by up to 2^-46."""
    e = ref.softmax(row, temp)
    e = e * (1 + 2.0 ** -46 * g.uniform(-1, 1, len(e)) * (e < 0.5)) if g is not None else e
    return e / e.sum() if e.sum() > 0 else e


def walk(c, most, rows_of, unrolled=False):
    """(rows, next tokens) with the probabilities that `rows_of(row, temp)` gives: what is left is scaled to 1 child by child,
    or, unrolled, kept as a p - b q with two numbers a and b."""
    rows, nexts, starts = [], [], c["starts"].tolist()
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        temp, node = float(c["temps"][s]), a
        while True:
            rows.append(node)
            p = rows_of(c["logits"][node], temp)
            one = p[0] * 0 + 1
            q = rows_of(c["draft"][node], temp) if c["draft"] is not None else [one] * len(p)  # of the drafted token; others are not taken off
            left, at, bt, total, taken = p, one, one * 0, one, None
            for k in [i for i in range(node + 1, b) if int(c["parents"][i]) == node - a][:most]:
                x = int(c["tokens"][k])
                if type(one)(float(c["accept"][k])) * q[x] < left[x] / total:
                    taken = k
                    break
                at, bt = at / total, bt / total + 1
                if c["draft"] is None:
                    left = [one * 0 if i == x else u / total for i, u in enumerate(left)]
                elif unrolled:
                    left = [max(at * u - bt * v, one * 0) for u, v in zip(p, q)]
                else:
                    left = [max(u / total - v, one * 0) for u, v in zip(left, q)]
                total = sum(left)
                if total == 0:
                    break
            if taken is None:
                if total == 0:
                    left = p
                run, goal = one * 0, type(one)(float(c["sample"][s])) * sum(left)
                nexts.append(-1)
                for i, v in enumerate(left):
                    run += v
                    if v > 0 and (nexts[-1] < 0 or run - v <= goal):
                        nexts[-1] = i
                break
            node = taken
    return rows, nexts


def cases(dtype, want):
    """Cases that 64 bits decide, with what they come to."""
    seed = 0
    while want:
        seed += 1
        g = torch.Generator().manual_seed(seed)
        V = int(torch.randint(2, 12, (1,), generator=g))
        most = int(torch.randint(2, 6, (1,), generator=g))
        c = calls.make(V, [6, 4, 9], most, dtype, True, seed=seed, near=(0.01, 0.05, 0.5)[seed % 3])
        c["temps"] = c["temps"] * (0.3, 0.1, 0.05)[seed // 3 % 3]
        c["accept"] = c["accept"] * 0.1 + 0.9
        for name in ("logits", "draft"):
            c[name][torch.rand(c[name].shape, generator=g) < 0.3] = -math.inf
        if seed % 2:
            c["tokens"] = torch.randint(0, V, c["tokens"].shape, generator=g).to(torch.int32)
        if bool((c["logits"] == -math.inf).all(1).any()):  # the walk above has no row without any
            continue
        exact = walk(c, most, softmax60)
        noise = np.random.default_rng(seed)
        if all(walk(c, most, lambda row, temp: softmax64(row, temp, r)) == exact for r in (None, *[noise] * 6)):
            want -= 1
            yield c, most, exact


def test_unrolled_weights_would_not_do():
    """Of the cases below: 64 bits go wrong in some where what is left after two children and more is a p - b q."""
    wrong = [walk(c, most, lambda row, temp: softmax64(row, temp, None), unrolled=True) != exact for c, most, exact in cases(torch.float32, 150)]
    assert 0 < sum(wrong) < 20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sharp_rows(gpu, dtype):
    for c, most, (rows, nexts) in cases(dtype, 150):
        got = calls.call(gpu, c, 9, most)
        assert [r for r in got[0] if r >= 0] == rows and got[2] == nexts


def lookups(dtype, V, want):
    """Stars without draft logits: the likeliest tokens in order, or any, tried with numbers near 1, so that little is left."""
    seed = 0
    while want:
        seed += 1
        g = torch.Generator().manual_seed(seed)
        pick = lambda values: values[int(torch.randint(0, len(values), (1,), generator=g))]
        S, kids = 8, pick([2, 3, 5])
        logits = (torch.randn(S * (kids + 1), V, generator=g) * pick([1, 3, 10])).to(dtype)
        c = dict(logits=logits, draft=None, temps=torch.full((S,), pick([1.0, 0.5, 0.2, 0.05])), sample=torch.rand(S, generator=g),
                 starts=torch.arange(0, S * (kids + 1) + 1, kids + 1, dtype=torch.int32), parents=torch.tensor(([-1] + [0] * kids) * S, dtype=torch.int32),
                 tokens=torch.randint(0, V, (S * (kids + 1),), generator=g).to(torch.int32),
                 accept=1 - 2.0 ** -torch.tensor([24.0, 23, 20, 10, 3])[torch.randint(0, 5, (S * (kids + 1),), generator=g)])
        for s in range(0, S, 2):
            top = torch.argsort(logits[s * (kids + 1)].float(), descending=True, stable=True)[:kids]
            c["tokens"][s * (kids + 1) + 1:(s + 1) * (kids + 1)][:len(top)] = top.to(torch.int32)
        exact = walk(c, kids, softmax60)
        noise = np.random.default_rng(seed)
        if all(walk(c, kids, lambda row, temp: softmax64(row, temp, r)) == exact for r in (None, *[noise] * 3)):
            want -= 1
            yield c, kids, exact


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,want", [(2, 50), (9, 200), (2200, 4)])
def test_sharp_rows_of_lookups(gpu, dtype, V, want):
    """1 less the probabilities of the tokens tried has none of the digits of what they leave."""
    for c, kids, (rows, nexts) in lookups(dtype, V, want):
        got = calls.call(gpu, c, kids + 1, kids)
        assert [r for r in got[0] if r >= 0] == rows and got[2] == nexts
