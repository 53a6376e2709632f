"""GPU: TreeAttentionInt4 against 64 bits, with the bound of its rounding (int4_reference.attention says from what)."""

import math

import pytest
import torch

import iron_amd.operators as ops
from iron_amd.common.paging import int4_row_bytes
from tests import int4_reference as ref

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def pages_of(P, H, ps, D, gpu, seed, size=1.0):
    """Pages of quantized values, made on the GPU: random codes, steps and offsets as rows of that size have them."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    rows = torch.randint(0, 256, (P, H, ps, int4_row_bytes(D)), generator=g, device=gpu, dtype=torch.uint8)
    s = (torch.rand(P, H, ps, 4, generator=g, device=gpu) * 0.2 + 0.2) * size
    b = -s * (23.5 + torch.randn(P, H, ps, 4, generator=g, device=gpu))
    rows[..., D // 2:] = torch.stack([s, b], -1).half().view(torch.uint8).flatten(-2)
    return rows


def case(gpu, H, Hkv, D, dtype, lens, counts, ps=16, seed=0, max_nodes=None, sees=None, spare=0, kind="tree", size=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    S, N, T = len(lens), sum(counts) + spare, max_nodes or max(counts)
    used = [-(-n // ps) for n in lens]
    MP, P = max(max(used), 1) + 1, sum(used) + 3
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed))
    table = torch.full((S, MP), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    if sees is None:
        sees = torch.zeros(N, T, dtype=torch.bool)
        up = torch.Generator().manual_seed(seed)
        for a, b in zip(starts, starts[1:]):
            for i in range(a, b):
                if i > a:
                    p = i - 1 if kind == "chain" else a + int(torch.randint(0, i - a, (1,), generator=up))
                    sees[i] = sees[p]
                sees[i, i - a] = True
    noise = lambda *shape: torch.randn(*shape, generator=g, device=gpu).to(dtype)
    return dict(q=noise(N, H, D) * 2, k_new=noise(N, Hkv, D), v_new=noise(N, Hkv, D), k=pages_of(P, Hkv, ps, D, gpu, seed + 1, size),
                v=pages_of(P, Hkv, ps, D, gpu, seed + 2, size), table=table, lens=lens, starts=starts, sees=sees, T=T, prior=noise(N, H, D))


def op_of(c, scale=None):
    S, MP = c["table"].shape
    N, H, D = c["q"].shape
    P, Hkv, ps, _ = c["k"].shape
    return ops.TreeAttentionInt4(num_heads=H, num_kv_heads=Hkv, head_dim=D, num_pages=P, page_size=ps, num_seqs=S, max_pages=MP,
                                 num_nodes=N, max_nodes=c["T"], dtype=c["q"].dtype, scale=scale)


def args_of(c, gpu, op):
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(gpu)
    return [c["q"], c["k_new"], c["v_new"], c["k"], c["v"], i32(c["table"]), i32(c["lens"]), i32(c["starts"]),
            op.pack_mask(c["sees"]).to(gpu), c["prior"].clone()]


def check(c, got, scale=None):
    want, tol = ref.attention(c["q"], c["k_new"], c["v_new"], c["k"], c["v"], c["table"], c["lens"], c["starts"], c["sees"],
                              scale or 1 / math.sqrt(c["q"].shape[-1]), c["prior"], c["T"])
    tol[c["starts"][-1]:] = 0  # rows behind the last tree are left as they were
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float(((got.double() - want).abs() / tol.clamp(min=1e-30))[bad].max()):.3g} times the bound"


def run(gpu, c, scale=None):
    op = op_of(c, scale)
    args = args_of(c, gpu, op)
    op.get_callable()(*args)
    return args[-1]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv,lens,counts,ps", [
    (4, 2, [0, 1, 15, 16, 17], [1, 1, 1, 1, 1], 16),
    (8, 2, [63, 64, 65, 127, 129], [1, 2, 1, 3, 4], 16),
    (32, 8, [2047], [1], 16),
    (5, 5, [40, 0, 300], [9, 16, 1], 32),
    (12, 1, [333, 1000], [1, 2], 64),
    (6, 2, [500, 31], [8, 10], 128),
    (64, 8, [70, 260], [4, 3], 16),
    (4, 4, [100, 0, 37], [32, 20, 0], 16),
    (8, 2, [100, 700, 0], [26, 13, 40], 16),
    (8, 1, [33, 5], [64, 63], 64),
    (2, 1, [1029, 0, 31, 32], [130, 65, 1, 200], 16),
    (10, 2, [513], [33], 1024),
])
def test_against_64_bits(gpu, dtype, D, H, Hkv, lens, counts, ps):
    c = case(gpu, H, Hkv, D, dtype, lens, counts, ps, seed=len(lens) + H, spare=2)
    check(c, run(gpu, c))


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 128)])
def test_long_contexts(gpu, dtype, D):
    c = case(gpu, 8, 2, D, dtype, [30011, 3, 7777], [1, 1, 2], seed=3)
    check(c, run(gpu, c))
    c = case(gpu, 8, 2, D, dtype, [9001, 20000], [60, 33], 64, seed=4)
    check(c, run(gpu, c))


@pytest.mark.parametrize("D", [64, 128])
def test_chunk_of_a_prompt(gpu, D):
    """1024 nodes in a chain behind cached positions, and a sequence of fewer."""
    c = case(gpu, 4, 2, D, BF16, [100, 45], [1024, 300], seed=5, kind="chain")
    check(c, run(gpu, c))


@pytest.mark.parametrize("counts", [[3, 2], [40, 50]])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_that_see_nothing(gpu, dtype, counts):
    """Masks without a bit: only the cache is seen, or (no cache) nothing: zeros."""
    c = case(gpu, 4, 2, 64, dtype, [0, 20], counts, seed=6)
    c["sees"][::2] = False
    got = run(gpu, c)
    check(c, got)
    assert not got[0].any() and got[counts[0]].any()


@pytest.mark.parametrize("counts", [[2, 1, 1], [40, 1, 1]])
def test_holes(gpu, counts):
    """Table entries outside the pool: their positions are not seen, whole sequences of them are empty."""
    c = case(gpu, 4, 2, 64, BF16, [200, 90, 64], counts, seed=7)
    c["table"][0, 2], c["table"][0, 5], c["table"][1, 5] = -1, c["k"].shape[0], -7
    c["table"][2, :] = 1 << 30
    check(c, run(gpu, c))


@pytest.mark.parametrize("counts", [[2, 1], [40, 3]])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_what_is_not_seen_does_not_matter(gpu, dtype, counts):
    """NaN and infinities behind the last position, in holes' pages, in unseen nodes."""
    c = case(gpu, 4, 2, 64, dtype, [37, 70], counts, seed=8)
    c["sees"][:, 1] = False
    c["table"][1, 1] = -1
    clean = {**c, **{k: c[k].clone() for k in ("k", "v", "k_new", "v_new")}}
    check(clean, run(gpu, clean))
    nan_row = torch.full((int4_row_bytes(64),), 0xff, dtype=torch.uint8, device=gpu)  # s and b are NaN
    inf_row = nan_row.clone()
    inf_row[32:] = torch.tensor([0x00, 0x7c] * 8, dtype=torch.uint8, device=gpu)
    for row in (nan_row, inf_row):
        for s, n in enumerate(c["lens"]):
            page = int(c["table"][s, n // 16])
            c["k"][page, :, n % 16:] = row
            c["v"][page, :, n % 16:] = row
        unused = [p for p in range(c["k"].shape[0]) if p not in c["table"].flatten().tolist()]
        c["k"][unused] = row
        c["v"][unused] = row
        c["k_new"][1] = math.nan
        c["v_new"][1] = math.inf
        check(clean, run(gpu, c))  # rows may be done over for it, with other roundings


@pytest.mark.parametrize("counts", [[2, 1], [40, 3]])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_and_infinite_rows_of_the_cache(gpu, counts, D):
    """What a row sees does reach it: a NaN key makes the row NaN, a NaN or infinite value its dims, a score of -inf nothing."""
    c = case(gpu, 4, 2, D, BF16, [40, 70], counts, seed=9)
    base = run(gpu, c).clone()
    page, q4 = int(c["table"][0, 1]), D // 4
    v = c["v"].clone()
    pair = lambda rows, quarter: rows[..., D // 2 + 4 * quarter:D // 2 + 4 * quarter + 4].view(torch.float16)
    pair(c["v"][page, 0, 3], 1)[1] = math.nan
    got = run(gpu, c)
    n = counts[0]
    assert torch.isnan(got[:n, :2, q4:2 * q4]).all() and torch.equal(got[:n, 2:], base[:n, 2:]) and torch.equal(got[n:], base[n:])
    tol = base[:n, :2, 2 * q4:].abs() * 2.0 ** -6 + 2.0 ** -6  # the other dims of that head were computed another way
    assert ((got[:n, :2, 2 * q4:] - base[:n, :2, 2 * q4:]).abs() <= tol).all()
    c["v"] = v.clone()
    pair(c["v"][page, 1, 3], 0)[1] = -math.inf
    got = run(gpu, c)
    assert (got[:n, 2:, :q4] == -math.inf).all() and torch.isfinite(got[:n, 2:, q4:]).all()
    c["v"] = v
    k = c["k"].clone()
    pair(c["k"][page, 0, 5], 2)[1] = math.nan
    got = run(gpu, c)
    assert torch.isnan(got[:n, :2]).all() and torch.equal(got[:n, 2:], base[:n, 2:])
    c["k"] = k
    c["q"][:n, 2:] = c["q"][:n, 2:].abs() + 1
    pair(c["k"][page, 1, 5], 3)[1] = -math.inf  # every score of that key is -inf for the second head
    got = run(gpu, c)
    c["k"] = k
    hidden = {**c, "k": k}
    want = []
    for i in range(2, 4):
        kv = ref.values(torch.cat([k[c["table"][0, t // 16].item(), 1, t % 16][None] for t in range(40) if t != 21]), D)
        vv = ref.values(torch.cat([v[c["table"][0, t // 16].item(), 1, t % 16][None] for t in range(40) if t != 21]), D)
        x = torch.cat([kv, c["k_new"][:1, 1].double()]) @ c["q"][0, i].double() / math.sqrt(D)
        want.append(torch.softmax(x, 0) @ torch.cat([vv, c["v_new"][:1, 1].double()]))
    want = torch.stack(want)
    assert ((got[0, 2:].double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -7).all()


@pytest.mark.parametrize("counts", [[1, 2], [40, 3]])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_and_small_numbers(gpu, dtype, counts):
    """Queries, keys and values near the ends of their types; scales from 1e-30 up."""
    for q_size, kv_size, scale in ((1e-4, 1.0, 1e4), (3e4, 1.0, 1e-5), (1.0, 800.0, 1e-3), (0.0, 1.0, 1.0), (2.0, 1e-3, 1.0), (1.0, 1.0, 1e-30)):
        c = case(gpu, 4, 2, 64, dtype, [50, 100], counts, seed=10, size=kv_size)
        c["q"] = c["q"].float().clamp(-2, 2).mul(q_size).to(dtype)
        check(c, run(gpu, c, scale), scale)
    if dtype == BF16:  # a query that fp16 does not hold, and one under its smallest
        for q_size, scale in ((1e30, 1e-30), (1e-30, 1e30), (1e-38, 1.0)):
            c = case(gpu, 4, 2, 64, dtype, [50, 100], counts, seed=11)
            c["q"] = c["q"].float().mul(q_size).to(dtype)
            check(c, run(gpu, c, scale), scale)
        c = case(gpu, 4, 2, 64, dtype, [50, 100], counts, seed=12)
        c["q"][:, :, 3] *= 1e6  # one dim far above the others
        c["k_new"][0] *= 1e6
        check(c, run(gpu, c, 1e-6), 1e-6)
        c["v_new"][0] *= 1e8
        check(c, run(gpu, c, 1e-6), 1e-6)


@pytest.mark.parametrize("counts", [[1, 2], [40, 3]])
def test_scores_far_out(gpu, counts):
    """Scores past 2^24: one key has all the weight."""
    c = case(gpu, 4, 2, 64, BF16, [50, 100], counts, seed=13)
    got = run(gpu, c, 1e8)
    for s, a in enumerate(c["starts"][:-1]):
        t = torch.arange(c["lens"][s])
        page = c["table"][s].long()[t // 16].to(gpu)
        for h in range(4):
            k = torch.cat([ref.values(c["k"][page, h // 2, t.to(gpu) % 16], 64), c["k_new"][a:a + 1, h // 2].double()])
            v = torch.cat([ref.values(c["v"][page, h // 2, t.to(gpu) % 16], 64), c["v_new"][a:a + 1, h // 2].double()])
            w = k @ c["q"][a, h].double()
            top2 = torch.topk(w, 2)
            if float(top2.values[0] - top2.values[1]) > 0.05:
                want = v[top2.indices[0]]
                assert ((got[a, h].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * want.abs() + 1e-6).all()
    assert torch.isfinite(got).all()


def test_infinite_queries(gpu):
    """An infinite or NaN query makes NaN of its row and of no other."""
    for counts in ([3, 1], [40, 1]):
        c = case(gpu, 4, 2, 64, BF16, [30, 60], counts, seed=14)
        base = run(gpu, c).clone()
        c["q"][1, 2, 5], c["q"][2, 0, 0] = math.inf, math.nan
        got = run(gpu, c)
        assert torch.isnan(got[2, 0]).all()
        rest = torch.ones(got.shape[:2], dtype=torch.bool, device=gpu)
        rest[1, 2] = rest[2, 0] = False
        assert torch.equal(got[rest], base[rest])


def test_past_4_gib(gpu):
    """Pages whose bytes lie past 2^32 of the pools, for few rows and many."""
    H, D, ps = 4, 64, 64
    P = (1 << 32) // (H * ps * int4_row_bytes(D)) + 200
    pools = []
    for seed in (15, 16):
        pool = torch.zeros(P, H, ps, int4_row_bytes(D), dtype=torch.uint8, device=gpu)
        pool[-200:] = pages_of(200, H, ps, D, gpu, seed)
        pools.append(pool)
    for counts in ([1, 2], [40, 30]):
        c = case(gpu, 8, H, D, BF16, [6000, 5001], counts, ps, seed=17)
        c["k"], c["v"] = pools
        c["table"] = torch.where(c["table"] >= 0, c["table"] + P - 200, c["table"])
        assert int(c["table"].max()) >= P - 30
        check(c, run(gpu, c))


def test_many_sequences(gpu):
    S = 8192
    lens = [(37 * i) % 90 for i in range(S)]
    c = case(gpu, 2, 1, 64, BF16, lens, [1] * S, seed=18)
    got = run(gpu, c)
    some = list(range(0, S, 173))
    part = {**c, "lens": [lens[s] for s in some], "starts": list(range(len(some) + 1)), "table": c["table"][some]}
    part |= {k: c[k][some] for k in ("q", "k_new", "v_new", "sees", "prior")}
    check(part, got[some])


def test_same_result_every_time_and_on_any_stream(gpu):
    side = torch.cuda.Stream()
    for counts in ([1, 4, 2], [40, 9, 33]):
        c = case(gpu, 8, 2, 64, BF16, [3000, 17, 900], counts, seed=19)
        first = run(gpu, c)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            again = run(gpu, c)
        side.synchronize()
        assert torch.equal(first, again) and torch.equal(first, run(gpu, c))


def test_graphs(gpu):
    """Two captured calls share nothing: replays in turn, with lengths that change and eager calls between."""
    graphs = []
    for counts in ([1, 1], [40, 20]):
        c = case(gpu, 8, 2, 128, FP16, [2000, 900], counts, seed=20)
        op = op_of(c)
        fn, args = op.get_callable(), args_of(c, gpu, op)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fn(*args)
        graphs.append((graph, c, fn, args))
    for lens in ([1999, 900], [0, 1], [64, 512], [2000, 3]):
        for graph, c, fn, args in graphs:
            c["lens"] = lens
            args[6].copy_(torch.tensor(lens, dtype=torch.int32))
            args[-1].copy_(c["prior"])
            graph.replay()
            eager = [*args[:-1], c["prior"].clone()]
            fn(*eager)
            torch.cuda.synchronize()
            assert torch.equal(args[-1], eager[-1])
            check(c, args[-1])


def test_refusals(gpu):
    c = case(gpu, 4, 2, 64, BF16, [20], [1], seed=21)
    op = op_of(c)
    args = args_of(c, gpu, op)
    with pytest.raises(ValueError, match="expected torch.uint8"):
        op.get_callable()(*args[:3], args[3].view(torch.int8), *args[4:])
    with pytest.raises(ValueError, match="elements"):
        op.get_callable()(*args[:3], args[3][1:], *args[4:])


@pytest.mark.parametrize("counts", [[1, 2], [40, 3]])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_queries_at_the_ends_of_fp16(gpu, dtype, D, counts):
    """Subnormal queries of fp16 with scales that make ordinary scores of them, and its largest ones."""
    for q_size, scale in ((1e-6, 2e5), (1e-5, 2e4), (2.0 ** -24, 1e6), (3e4, 3e-6)):
        c = case(gpu, 4, 2, D, dtype, [50, 100], counts, seed=31)
        c["q"] = c["q"].float().clamp(-2, 2).mul(q_size).to(dtype)
        check(c, run(gpu, c, scale), scale)
    c["q"] = torch.full_like(c["q"], 6e4)  # sums of a quarter past fp16
    check(c, run(gpu, c, 1e-6), 1e-6)
