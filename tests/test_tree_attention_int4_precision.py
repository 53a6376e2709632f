"""TreeAttentionInt4 keeps the roundings that it documents: bf16 calls round cached keys, values and weights once to fp16,
fp16 calls round cached values only. On the CPU: that coarser ones would show."""

import math

import pytest
import torch

from tests import int4_precision as precise
from tests import test_tree_attention_int4_gpu as shapes

BF16, FP16 = torch.bfloat16, torch.float16
CPU = torch.device("cpu")

# A result whose error is one rounding and others of a part r of it each is off by sqrt(1 + sum r^2) of one rounding. Against
# the documented roundings of keys and values nothing is left but, in bf16, that of the weights to fp16: r = 1/8, 1.008.
LEFT = 1.05
# Against 64 bits: cached values in fp16 calls have r = 1 (1.41); in bf16 calls values and weights have 1/8 each and keys
# 1/4 (queries of size 2): 1.046.
ALL = {FP16: 1.5, BF16: 1.1}

# Times 1 / sqrt(D): scores of an ordinary size, where keys count most and a few weights have all the sum; flat ones, where
# many weights of like size do.
SCALES = (1.0, 0.25)


def documented(c, scale):
    dtype = c["prior"].dtype
    return precise.attention(c, scale, keys=precise.fp16 if dtype == BF16 else precise.keep, values=precise.fp16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv,lens,counts,ps", [
    (32, 8, [2047], [1], 16),
    (16, 2, [700, 90, 1033], [2, 1, 3], 16),
    (8, 8, [350, 800], [12, 30], 32),
    (8, 2, [3000, 2500], [40, 33], 64),
    (4, 4, [2100], [130], 16),
])
def test_error_is_that_of_the_documented_roundings(gpu, dtype, D, H, Hkv, lens, counts, ps):
    c = shapes.case(gpu, H, Hkv, D, dtype, lens, counts, ps, seed=D + H)
    for scale in (x / math.sqrt(D) for x in SCALES):
        got = shapes.run(gpu, c, scale)
        assert precise.ratio(got, documented(c, scale)) < LEFT
        assert precise.ratio(got, precise.attention(c, scale)) < ALL[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv,lens,counts", [(8, 2, [0, 1, 2, 15], [1, 2, 1, 3]), (16, 2, [64, 129], [2, 1]), (8, 2, [5, 40], [40, 33]), (8, 8, [700], [30])])
def test_every_element_is_within_its_own_bound(gpu, dtype, D, H, Hkv, lens, counts):
    """With any keys and values; with values that fp16 holds; with scores, too, that fp32 sums hold."""
    any_values = shapes.case(gpu, H, Hkv, D, dtype, lens, counts, seed=D + len(lens))
    values = precise.exact_values(any_values, D)
    for c, exact_scores in ((any_values, False), (values, False), (precise.exact_scores(values, D), True)):
        for scale in (x / math.sqrt(D) for x in SCALES):
            want, tol = precise.bound(c, scale, exact_scores)
            off = (shapes.run(gpu, c, scale).double() - want).abs()
            assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_coarser_roundings_show(dtype, D):
    """Of the tests above: the documented roundings pass both; each coarser one fails the first at one of the scales, and
    fp16 calls' keys or weights that are rounded once fail the second too."""
    both = dict(keys=precise.fp16, weights=precise.fp16, values=precise.fp16) if dtype == BF16 else dict(values=precise.fp16)
    step = precise.bf16 if dtype == BF16 else precise.fp16
    coarser = [dict(keys=step), dict(weights=step), dict(keys=precise.bf16), dict(weights=precise.bf16), dict(values=precise.bf16)]
    scales = [x / math.sqrt(D) for x in SCALES]

    def result(c, scale, **roundings):
        return precise.attention(c, scale, **{**both, **roundings}).to(dtype)

    c = shapes.case(CPU, 8, 2, D, dtype, [700, 90], [4, 2], seed=D)
    worst = [0.0] * len(coarser)
    for scale in scales:
        want, exact, fine = documented(c, scale), precise.attention(c, scale), result(c, scale)
        assert precise.ratio(fine, want) < LEFT and precise.ratio(fine, exact) < ALL[dtype]
        worst = [max(x, precise.ratio(result(c, scale, **r), want) / LEFT) for x, r in zip(worst, coarser)]
    assert min(worst) > 1.1, worst
    c = precise.exact_scores(precise.exact_values(shapes.case(CPU, 8, 2, D, dtype, [64, 15, 2], [1, 2, 1], seed=D), D), D)
    for scale in scales:
        near, tol = precise.bound(c, scale, True)
        assert bool(((result(c, scale).double() - near).abs() <= tol).all())
        if dtype == FP16:
            for r in coarser[:2]:
                assert bool(((result(c, scale, **r).double() - near).abs() > tol).any()), r
