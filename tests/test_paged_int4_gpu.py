"""GPU: PagedAppendInt4 and PagedGatherInt4 against loops, bit for bit; the page operators on 4-bit pages; a serving loop
of attention, verification and append."""

import math

import numpy as np
import pytest
import torch

import iron_amd.operators as ops
from iron_amd.common.paging import int4_row_bytes
from tests import int4_reference as ref
from tests import paged_reference as paged

pytestmark = pytest.mark.gpu


def cache_of(L, P, H, ps, D, S, MP, seed=0):
    """A paged cache of 4-bit rows on the CPU, its pages full of random bytes."""
    c = paged.Cache(L, P, H, ps, int4_row_bytes(D), S, MP, seed=seed, dtype=torch.float32)
    g = torch.Generator().manual_seed(seed)
    c.k, c.v = (torch.randint(0, 256, c.k.shape, generator=g, dtype=torch.uint8) for _ in range(2))
    c.dtype = torch.uint8
    return c


def append_want(c, k_new, v_new, rows, starts):
    return paged.append(c, ref.to_rows(k_new), ref.to_rows(v_new), rows, starts)


def append_op(c, D, N, M, dtype):
    return ops.PagedAppendInt4(num_layers=c.k.shape[0], num_kv_heads=c.k.shape[2], head_dim=D, num_pages=c.pages, page_size=c.ps,
                               num_seqs=len(c.lens), max_pages=c.max_pages, num_nodes=N, num_rows=M, dtype=dtype)


def i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def do_append(gpu, c, D, k_new, v_new, rows, starts):
    dev = c.to(gpu)
    status = torch.full((len(c.lens),), 9, dtype=torch.int32, device=gpu)
    append_op(c, D, k_new.shape[1], len(rows), k_new.dtype).get_callable()(k_new.to(gpu), v_new.to(gpu), i32(rows, gpu), i32(starts, gpu), *dev, status)
    return dev, status.tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,ps,L", [(64, 2, 16, 3), (128, 3, 32, 1), (64, 8, 64, 1), (128, 1, 16, 2)])
def test_append(gpu, dtype, D, H, ps, L):
    g = torch.Generator().manual_seed(D + H)
    c = cache_of(L, 40, H, ps, D, 5, 8)
    ids = list(range(39, -1, -2))
    for s, n in enumerate([0, 1, ps - 1, ps, 2 * ps + 5]):
        c.hold(s, n, [ids.pop() for _ in range(4)])
    counts = [3, 0, ps + 2, 1, 2 * ps - 5]
    starts = [0, *np.cumsum(counts).tolist()]
    N, M = 4 * ps + 9, starts[-1] + 2
    scale = torch.logspace(-4, 3, N)[None, :, None, None]
    k, v = ((torch.randn(L, N, H, D, generator=g) * scale).to(dtype) for _ in range(2))
    rows = torch.randint(0, N, (M,), generator=g).tolist()
    rows[1], rows[4] = -1, N  # no such row: zeros
    want = c.copy()
    status = append_want(want, k, v, rows, starts)
    dev, got = do_append(gpu, c, D, k, v, rows, starts)
    assert got == status == [0] * 5 and all(want.same(dev))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_values_at_the_edges(gpu, D, dtype):
    """Constant quarters, ties, values past the cut, infinities, NaN, subnormal ranges, signed zeros, one outlier."""
    q, top = D // 4, torch.finfo(dtype).max
    rows = torch.zeros(16, D)
    rows[0] = 3.25
    rows[1] = torch.arange(D) % 16 * 0.5  # codes exactly, and
    rows[2] = torch.arange(D) % 31 * 0.25  # values half way between two
    rows[3, 3], rows[3, q + 1] = top, -top
    rows[4, 0], rows[4, q] = math.inf, -math.inf
    rows[5, 7], rows[5, 3 * q] = math.nan, 2.0
    rows[6] = torch.arange(D) * 1e-7
    rows[7] = torch.arange(D) * -3e-39
    rows[8, ::2], rows[8, 1::2] = -0.0, 0.0
    rows[9], rows[9, 5] = 0.01 * torch.randn(D, generator=torch.Generator().manual_seed(1)), 500.0
    rows[10] = 20480.0 - torch.arange(D) * 16
    rows[11] = 1000 + torch.arange(D) % 2
    rows[12] = -rows[2]
    rows[13, :q] = torch.nan
    rows[14] = torch.linspace(-1, 1, D)
    rows[15] = torch.arange(D) * 6e-8
    k = rows.to(dtype).reshape(1, 16, 1, D)
    v = k.flip(3).contiguous()
    c = cache_of(1, 3, 1, 16, D, 1, 2)
    want = c.copy()
    append_want(want, k, v, list(range(16)), [0, 16])
    dev, status = do_append(gpu, c, D, k, v, list(range(16)), [0, 16])
    assert status == [0] and all(want.same(dev)), [(i, (a[0, 0, 0, i].cpu() != b[0, 0, 0, i]).nonzero().flatten().tolist())
                                                   for a, b in ((dev[0], want.k), (dev[1], want.v)) for i in range(16)]


def test_append_every_pair_of_sixteen_bits(gpu):
    """Many scales, offsets and ties: 2^15 rows of random bit patterns and of small whole numbers, byte for byte."""
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.bfloat16, torch.float16):
        bits = torch.randint(-32768, 32768, (1, 4096, 4, 64), generator=g).to(torch.int16).view(dtype)
        bits = torch.where(torch.isnan(bits), 0, bits)  # NaN of any bits is tested on its own
        whole = torch.randint(-9, 10, (1, 4096, 4, 64), generator=g).to(dtype)
        small = whole * torch.tensor(0.125, dtype=dtype) + 7
        for k, v in ((bits, whole), (small, whole + 96)):
            c = cache_of(1, 258, 4, 16, 64, 1, 257)
            want = c.copy()
            append_want(want, k, v, list(range(4096)), [0, 4096])
            dev, status = do_append(gpu, c, 64, k, v, list(range(4096)), [0, 4096])
            assert status == [0] and all(want.same(dev))


def test_append_refuses_as_the_16_bit_one(gpu):
    """No room, a shared last page, a hole, ranges that leave the rows or overlap: nothing changes."""
    D, H, ps = 64, 2, 16
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1, 30, H, D, generator=g).to(torch.bfloat16) for _ in range(2))
    for starts in ([0, 4, 9, 12, 30, 31], [0, 20, 5, 12, 14, 20], [0, 40, 40, 40, 41, 42], [-1, 3, 3, 6, 8, 9]):
        c = cache_of(1, 7, H, ps, D, 5, 2)
        c.hold(0, 5, [3])
        c.hold(1, 7, [3])  # shared with the first
        c.hold(2, 3, [-1])
        c.hold(3, 20, [0, 5])
        c.hold(4, 31, [1, 2])
        want = c.copy()
        rows = list(range(30))
        status = append_want(want, k, v, rows, starts)
        dev, got = do_append(gpu, c, D, k, v, rows, starts)
        assert got == status and any(status) and all(want.same(dev))


def gather_op(c, D, M, dtype):
    return ops.PagedGatherInt4(num_layers=c.k.shape[0], num_kv_heads=c.k.shape[2], head_dim=D, num_pages=c.pages, page_size=c.ps,
                               num_seqs=len(c.lens), max_pages=c.max_pages, num_rows=M, dtype=dtype)


def sane(c, D, seed=0):
    """Rows with finite values: pages are random bytes otherwise."""
    g = torch.Generator().manual_seed(seed)
    for pages in (c.k, c.v):
        pages[:] = ref.to_rows(torch.randn(*pages.shape[:-1], D, generator=g) * 2)
    return c


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,ps,L", [(64, 2, 16, 3), (128, 3, 32, 1), (64, 8, 64, 2)])
def test_gather(gpu, dtype, D, H, ps, L):
    c = sane(cache_of(L, 30, H, ps, D, 6, 5), D)
    for s, n in enumerate([0, 1, ps, 3 * ps + 7, 2 * ps, 5 * ps]):
        c.hold(s, n, [(7 * s + 11 * e) % 30 for e in range(5)])
    c.table[4, 1] = -1
    c.table[5, 2] = 30
    begins = [0, 0, 3, ps - 2, -4, 5 * ps - 3]
    counts = [2, 1, ps + 4, 2 * ps + 9, ps + 20, 9]
    starts = [2, *(2 + np.cumsum(counts)).tolist()]
    M = starts[-1] + 3
    g = torch.Generator().manual_seed(3)
    prior = [torch.randn(L, M, H, D, generator=g).to(dtype) for _ in range(2)]
    want = ref.gather(c.k, c.v, c.table, c.lens, begins, starts, *prior, D)
    dev = c.to(gpu)
    out = [p.to(gpu) for p in prior]
    gather_op(c, D, M, dtype).get_callable()(i32(begins, gpu), i32(starts, gpu), *dev[:4], *out)
    for o, w in zip(out, want):
        assert torch.equal(o.cpu().view(torch.int16), w.view(torch.int16))


def test_gather_of_odd_ranges(gpu):
    """Ranges that overlap (the first sequence's rows), decrease, leave the rows, begin near 2^31; lengths that do not fit."""
    D, H, ps = 64, 1, 16
    c = sane(cache_of(1, 12, H, ps, D, 4, 3), D)
    for s in range(4):
        c.hold(s, 40, [3 * s, 3 * s + 1, 3 * s + 2])
    c.lens[3] = 10 ** 9
    for starts, begins in (([0, 10, 5, 20, 21], [0, 1, 2, 3]), ([-7, 40, 40, 3, 9], [10, 0, 0, 45]), ([0, 4, 8, 12, 16], [2 ** 31 - 2, -2 ** 31, 39, 47])):
        prior = [torch.full((1, 20, H, D), 5.0, dtype=torch.bfloat16) for _ in range(2)]
        want = ref.gather(c.k, c.v, c.table, c.lens, begins, starts, *prior, D)
        dev, out = c.to(gpu), [p.to(gpu) for p in prior]
        gather_op(c, D, 20, torch.bfloat16).get_callable()(i32(begins, gpu), i32(starts, gpu), *dev[:4], *out)
        for o, w in zip(out, want):
            assert torch.equal(o.cpu().view(torch.int16), w.view(torch.int16))


def test_page_operators_take_the_pages(gpu):
    """Fork, copy, pack and free of a 4-bit cache: dtype uint8, head_dim the bytes of a row."""
    for D in (64, 128):
        c = cache_of(2, 20, 2, 16, D, 6, 4)
        c.hold(0, 37, [3, 9, 14])
        c.hold(1, 16, [17])
        pool = dict(num_pages=20, page_size=16, num_seqs=6, max_pages=4)
        data = dict(num_layers=2, num_kv_heads=2, head_dim=int4_row_bytes(D), dtype=torch.uint8, **pool)
        want, dev = c.copy(), c.to(gpu)
        status = torch.zeros(2, dtype=torch.int32, device=gpu)
        for share, pairs in ((True, [(0, 2), (1, 3)]), (False, [(0, 4), (2, 5)])):
            expect = paged.fork(want, pairs, share)
            ops.PageFork(num_forks=2, share=share, **data).get_callable()(i32(pairs, gpu), *dev, status)
            assert status.tolist() == expect and all(want.same(dev))
        expect = paged.free(want, [0, 1])
        ops.PageFree(num_slots=2, **pool).get_callable()(i32([0, 1], gpu), *dev[2:], status)
        assert status.tolist() == expect and all(want.same(dev))
        moved = torch.zeros(1, dtype=torch.int32, device=gpu)
        expect = paged.compact(want)
        ops.PageCompact(**data).get_callable()(*dev, moved)
        assert moved.tolist() == [expect] and all(want.same(dev))


def test_append_past_4_gib(gpu):
    """Byte offsets past 2^32 in both pools, and many rows at once."""
    D, H, ps, L = 128, 8, 128, 1
    P = (1 << 32) // (H * ps * int4_row_bytes(D)) + 40
    pages = [torch.zeros(L, P, H, ps, int4_row_bytes(D), dtype=torch.uint8, device=gpu) for _ in range(2)]
    refs = torch.ones(P, dtype=torch.int32, device=gpu)
    refs[-40:] = 0
    table, lens = i32([[-1] * 33], gpu), i32([0], gpu)
    M = 33 * ps - 5
    g = torch.Generator(device=gpu).manual_seed(4)
    k, v = (torch.randn(L, M, H, D, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2))
    shape = dict(num_layers=L, num_kv_heads=H, head_dim=D, num_pages=P, page_size=ps, num_seqs=1, max_pages=33, num_rows=M)
    status = torch.ones(1, dtype=torch.int32, device=gpu)
    ops.PagedAppendInt4(num_nodes=M, **shape).get_callable()(k, v, torch.arange(M, dtype=torch.int32, device=gpu), i32([0, M], gpu), *pages, table, lens, refs, status)
    assert status.item() == 0 and lens.item() == M and table.tolist() == [list(range(P - 40, P - 7))]
    out = [torch.zeros_like(k) for _ in range(2)]
    ops.PagedGatherInt4(**shape).get_callable()(i32([0], gpu), i32([0, M], gpu), *pages, table, lens, *out)
    for o, x in zip(out, (k, v)):
        some = torch.arange(0, M, 509)
        want = ref.values(ref.to_rows(x[0, some.to(gpu)].cpu()), D).to(torch.bfloat16)
        assert torch.equal(o[0, some.to(gpu)].cpu(), want)
    for p in pages:
        assert not p[:, :P - 40].any()


def test_append_and_gather_in_a_graph(gpu):
    """Captured together; every replay works on the tables as they are then. On a side stream too."""
    D, H, ps, L, S = 64, 2, 16, 2, 3
    c = cache_of(L, 24, H, ps, D, S, 2)
    g = torch.Generator().manual_seed(6)
    N, M = 20, 12
    k, v = (torch.randn(L, N, H, D, generator=g).to(torch.float16) for _ in range(2))
    rows, starts = torch.randint(0, N, (M,), generator=g).tolist(), [0, 5, 6, 12]
    put, read = append_op(c, D, N, M, torch.float16).get_callable(), gather_op(c, D, M, torch.float16).get_callable()
    dev = c.to(gpu)
    args = [k.to(gpu), v.to(gpu), i32(rows, gpu), i32(starts, gpu)]
    status, begins = torch.zeros(S, dtype=torch.int32, device=gpu), torch.zeros(S, dtype=torch.int32, device=gpu)
    out = [torch.zeros(L, M, H, D, dtype=torch.float16, device=gpu) for _ in range(2)]

    def step():
        begins.copy_(dev[3])
        put(*args, *dev, status)
        read(begins, args[3], *dev[:4], *out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    want = c.copy()
    assert append_want(want, k, v, rows, starts) == status.tolist() and all(want.same(dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(6):
        was = want.lens.copy()
        graph.replay()
        expect = append_want(want, k, v, rows, starts)
        torch.cuda.synchronize()
        assert expect == status.tolist() and all(want.same(dev))
        zero = [torch.zeros(L, M, H, D, dtype=torch.float16) for _ in range(2)]
        for o, w in zip(out, ref.gather(want.k, want.v, want.table, want.lens, was.tolist(), starts, *zero, D)):
            assert torch.equal(o.cpu(), w)
    assert 0 in expect and 2 in expect  # the last turns run out of table entries


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_serving_steps(gpu, D, dtype):
    """A few steps as a program takes them: attention of drafted trees per layer, logits, verification, and the accepted rows
    into the cache, all from device memory and without reading anything back; checked against the plain forms."""
    L, H, Hkv, ps, S, P, MP, V, T, most = 2, 4, 2, 16, 3, 40, 12, 200, 6, 2
    g = torch.Generator().manual_seed(D)
    c = sane(cache_of(L, P, Hkv, ps, D, S, MP), D)
    for s, n in enumerate([0, 31, 70]):
        c.hold(s, n, [(5 * s + e) for e in range(5)])
    counts = [6, 1, 5]
    starts = [0, 6, 7, 12]
    parents = [-1, 0, 0, 1, 1, 3] + [-1] + [-1, 0, 1, 2, 0]
    N = 12
    pool = dict(num_pages=P, page_size=ps, num_seqs=S, max_pages=MP)
    attend = ops.TreeAttentionInt4(num_heads=H, num_kv_heads=Hkv, head_dim=D, num_nodes=N, max_nodes=T, dtype=dtype, **pool)
    check = ops.DraftVerify(vocab=V, num_seqs=S, num_nodes=N, max_nodes=T, max_children=most, dtype=torch.float32)
    put = append_op(c, D, N, N, dtype)
    mask = attend.mask_of_parents(torch.tensor(parents), torch.tensor(starts)).to(gpu)
    sees = torch.zeros(N, T, dtype=torch.bool)
    for s in range(S):
        for i in range(starts[s], starts[s + 1]):
            j = i - starts[s]
            while j >= 0:
                sees[i, j] = True
                j = parents[starts[s] + j]
    head = torch.randn(H * D, V, generator=g)
    dev, want = c.to(gpu), c.copy()
    calls = [op.get_callable() for op in (attend, check, put)]
    for step in range(4):
        x = [torch.randn(L, N, n, D, generator=g).to(dtype) for n in (H, Hkv, Hkv)]
        draft = torch.randn(N, V, generator=g)
        tokens = torch.randint(0, V, (N,), generator=g).to(torch.int32)
        temps, accept, sample = torch.tensor([0.7, 1.0, 0.0]), torch.rand(N, generator=g) * 0.2, torch.rand(S, generator=g)
        q, k, v = (t.to(gpu) for t in x)
        out = torch.zeros(L, N, H, D, dtype=dtype, device=gpu)
        for l in range(L):
            calls[0](q[l].contiguous(), k[l].contiguous(), v[l].contiguous(), dev[0][l], dev[1][l], dev[2], dev[3], i32(starts, gpu), mask, out[l])
        logits = out[-1].reshape(N, -1).float() @ head.to(gpu)
        rows, row_starts, nexts = (torch.zeros(n, dtype=torch.int32, device=gpu) for n in (N, S + 1, S))
        calls[1](logits, draft.to(gpu), tokens.to(gpu), i32(parents, gpu), i32(starts, gpu), temps.to(gpu), accept.to(gpu), sample.to(gpu), rows, row_starts, nexts)
        status = torch.ones(S, dtype=torch.int32, device=gpu)
        calls[2](k, v, rows, row_starts, *dev, status)
        for l in range(L):
            o, tol = ref.attention(x[0][l], x[1][l], x[2][l], want.k[l], want.v[l], torch.from_numpy(want.table), want.lens.tolist(), starts, sees, 1 / math.sqrt(D), torch.zeros(N, H, D, dtype=dtype), T)
            assert bool(((out[l].cpu().double() - o).abs() <= tol).all())
        r, rs, nx, margin = ref.verify(logits.cpu(), draft, tokens, parents, starts, temps, accept, sample, most)
        assert margin > 1e-12 and [rows.tolist(), row_starts.tolist(), nexts.tolist()] == [r, rs, nx]
        assert append_want(want, x[1], x[2], r, rs) == status.tolist() and all(want.same(dev))
    assert want.lens.sum() >= 4 * S + 101


@pytest.mark.parametrize("dispatch", ["fused", "separate"])
def test_in_an_operator_sequence(gpu, dispatch):
    """Attention, verification, append and reading back as one runlist, called three times: the cache that a call leaves is
    the next one's."""
    from iron_amd.common import OperatorSequence

    D, H, Hkv, ps, S, P, MP, V, N = 64, 4, 2, 16, 2, 12, 4, 50, 5
    g = torch.Generator().manual_seed(31)
    c = sane(cache_of(1, P, Hkv, ps, D, S, MP), D)
    c.hold(0, 30, [7, 2])
    c.hold(1, 5, [9])
    starts, parents, begins = [0, 3, 5], [-1, 0, 1, -1, 0], [20, 0]
    pool = dict(num_kv_heads=Hkv, head_dim=D, num_pages=P, page_size=ps, num_seqs=S, max_pages=MP)
    attend = ops.TreeAttentionInt4(num_heads=H, num_nodes=N, max_nodes=3, **pool)
    check = ops.DraftVerify(vocab=V, num_seqs=S, num_nodes=N, max_nodes=3, dtype=torch.float32)
    put = ops.PagedAppendInt4(num_layers=1, num_nodes=N, num_rows=N, **pool)
    read = ops.PagedGatherInt4(num_layers=1, num_rows=12, **pool)
    cache = ("k_pages", "v_pages", "table", "lens")
    numbers = ("tokens", "parents", "starts", "temps", "accept", "sample")
    seq = OperatorSequence(name="int4_step", dispatch=dispatch,
                           runlist=[(attend, "q", "k", "v", *cache, "starts", "mask", "out"),
                                    (check, "logits", "draft", *numbers, "rows", "row_starts", "next"),
                                    (put, "k", "v", "rows", "row_starts", *cache, "refs", "status"),
                                    (read, "begins", "ranges", *cache, "k_out", "v_out")],
                           input_args=["q", "k", "v", "mask", "logits", "draft", *numbers, "begins", "ranges", *cache, "refs"],
                           output_args=["out", "rows", "row_starts", "next", "status", "k_out", "v_out"]).compile()
    fn = seq.get_callable()
    x = [torch.randn(N, n, D, generator=g).to(torch.bfloat16) for n in (H, Hkv, Hkv)]
    sees = torch.tensor([[1, 0, 0], [1, 1, 0], [1, 1, 1], [1, 0, 0], [1, 1, 0]], dtype=torch.bool)
    i32 = lambda v: torch.as_tensor(np.asarray(v), dtype=torch.int32)
    step = dict(logits=torch.randn(N, V, generator=g), draft=torch.randn(N, V, generator=g), tokens=i32([0, 3, 5, 0, 9]), parents=i32(parents),
                starts=i32(starts), temps=torch.tensor([0.8, 1.1]), accept=torch.rand(N, generator=g) * 0.1, sample=torch.rand(S, generator=g))
    ranges = [0, 8, 12]
    for name, value in dict(q=x[0], k=x[1], v=x[2], mask=attend.pack_mask(sees), begins=i32(begins), ranges=i32(ranges),
                            k_pages=c.k, v_pages=c.v, table=i32(c.table), lens=i32(c.lens), refs=i32(c.refs), **step).items():
        fn.get_buffer(name).torch_view(torch.uint8).copy_(value.contiguous().view(-1).view(torch.uint8))
    want = c.copy()
    rows, row_starts, nexts, margin = ref.verify(step["logits"], step["draft"], step["tokens"], parents, starts, step["temps"], step["accept"], step["sample"], 1)
    assert margin > 1e-12 and max(row_starts) > 2
    got = lambda name, dtype: fn.get_buffer(name).torch_view(dtype).cpu()
    for _ in range(3):
        fn()
        torch.cuda.synchronize()
        o, tol = ref.attention(*x, want.k[0], want.v[0], torch.from_numpy(want.table), want.lens.tolist(), starts, sees, 1 / math.sqrt(D), torch.zeros(N, H, D, dtype=torch.bfloat16), 3)
        assert bool(((got("out", torch.bfloat16).view(N, H, D).double() - o).abs() <= tol).all())
        assert [got(n, torch.int32).tolist() for n in ("rows", "row_starts", "next")] == [rows, row_starts, nexts]
        assert append_want(want, x[1][None], x[2][None], rows, row_starts) == got("status", torch.int32).tolist()
        zero = [torch.zeros(1, 12, Hkv, D, dtype=torch.bfloat16) for _ in range(2)]
        for name, w in zip(("k_out", "v_out"), ref.gather(want.k, want.v, want.table, want.lens, begins, ranges, *zero, D)):
            assert torch.equal(got(name, torch.bfloat16).view(w.shape), w)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0x7f81), (torch.float16, 0x7c01)])
def test_append_signalling_nan(gpu, D, dtype, bits):
    """NaN whose quiet bit is not set make their quarter NaN too, and no other, at any place of it."""
    k = torch.randn(1, D, 1, D, generator=torch.Generator().manual_seed(7)).to(dtype)
    v = k.flip(3).contiguous()
    for i in range(D):
        k.view(torch.int16)[0, i, 0, i] = v.view(torch.int16)[0, i, 0, (7 * i) % D] = bits
    c = cache_of(1, 9, 1, 16, D, 1, 8)
    want = c.copy()
    append_want(want, k, v, list(range(D)), [0, D])
    dev, status = do_append(gpu, c, D, k, v, list(range(D)), [0, D])
    assert status == [0] and all(want.same(dev))
