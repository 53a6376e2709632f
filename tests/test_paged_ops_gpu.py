"""GPU: the page operators (PagedAppend, PageFork, PageCompact, PageFree) against loops over Python integers, bit for bit,
with requests that cannot be met and tables that hold nonsense among them; the state around what they may write stays."""

import numpy as np
import pytest
import torch

import iron_amd.operators as ops
from iron_amd.common.graph import capture_graph
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def _pool(c):
    return dict(num_pages=c.pages, page_size=c.ps, num_seqs=len(c.lens), max_pages=c.max_pages)


def _data(c):
    L, _, Hkv, _, D = c.k.shape
    return dict(num_layers=L, num_kv_heads=Hkv, head_dim=D, dtype=c.dtype, **_pool(c))


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _filled(seed, pages=60, ps=16, seqs=8, max_pages=9, layers=2, kv_heads=2, dim=64, lens=None, dtype=torch.bfloat16, spare=0.2):
    """A cache whose sequences lie scattered over the pool; some free pages are left."""
    rng = np.random.default_rng(seed)
    c = ref.Cache(layers, pages, kv_heads, ps, dim, seqs, max_pages, seed, dtype)
    ids = list(rng.permutation(pages)[: int(pages * (1 - spare))])
    for s, n in enumerate(lens if lens is not None else rng.integers(0, max_pages * ps // 2, seqs)):
        need = c.used(int(n))
        if need <= len(ids):
            c.hold(s, int(n), [ids.pop() for _ in range(need)])
    return c


def _run(op, tensors, n):
    status = torch.full((n,), -7, dtype=torch.int32, device=tensors[-1].device)
    op.get_callable()(*tensors, status)
    torch.cuda.synchronize()
    return status.cpu().tolist()


def _append(gpu, c, counts, seed=0, rows=None, starts=None):
    M = max(1, sum(counts))
    N = M + 3
    g = torch.Generator().manual_seed(seed + 100)
    L, _, Hkv, _, D = c.k.shape
    kn, vn = (torch.randn(L, N, Hkv, D, generator=g).to(c.dtype) for _ in range(2))
    rows = torch.randperm(N, generator=g)[:M].tolist() if rows is None else rows
    starts = [0] + list(np.cumsum(counts)) if starts is None else starts
    op = ops.PagedAppend(num_nodes=N, num_rows=M, **_data(c))
    state = c.to(gpu)
    got = _run(op, [kn.to(gpu), vn.to(gpu), _ints(rows, gpu), _ints(starts, gpu), *state], len(c.lens))
    return got, state, (kn, vn, rows, [int(x) for x in starts])


@pytest.mark.parametrize("seed,ps,counts,layers,kv_heads,dim,dtype", [
    (0, 16, [1, 0, 3, 16, 17, 2, 0, 5], 2, 2, 64, torch.bfloat16),
    (1, 16, [1] * 8, 16, 8, 64, torch.bfloat16),
    (2, 32, [40, 1, 0, 0, 0, 0, 0, 33], 1, 1, 128, torch.float16),
    (3, 64, [0, 0, 0, 200, 0, 0, 0, 1], 3, 3, 64, torch.bfloat16),
    (4, 16, [0, 0, 0, 0, 0, 0, 0, 1], 1, 1, 16, torch.uint8),
    (5, 128, [5, 300, 2, 0, 1, 1, 1, 1], 2, 2, 24, torch.float32),
])
def test_append(gpu, seed, ps, counts, layers, kv_heads, dim, dtype):
    print(f"append seed {seed}", flush=True)
    c = _filled(seed, ps=ps, layers=layers, kv_heads=kv_heads, dim=dim, dtype=dtype)
    got, state, (kn, vn, rows, starts) = _append(gpu, c, counts, seed)
    want = ref.append(c, kn, vn, rows, starts)
    assert got == want and all(c.same(state))


def test_append_requests_that_cannot_be_met(gpu):
    """Short of pages, of table entries, on shared and missing last pages, with bad lengths; a row number outside appends zeros."""
    c = _filled(3, pages=30, seqs=8, max_pages=4, lens=[5, 20, 33, 40, 16, 0, 63, 10], spare=0.4)
    c.refs[c.table[1, 1]] = 2          # shared: not its own
    c.table[2, 2] = -1                 # a hole
    c.lens[3] = 65                     # longer than the table
    for counts in ([1, 1, 1, 1, 1, 1, 1, 1], [0, 1, 1, 0, 40, 30, 2, 30], [59, 0, 0, 0, 48, 64, 1, 54], [60, 0, 0, 0, 48, 64, 0, 1]):
        print(f"append {counts}", flush=True)
        case = c.copy()
        M = sum(counts)
        rows = [(-1 if i % 5 == 2 else i if i % 5 else M + 3) for i in range(M)]
        got, state, (kn, vn, rows, starts) = _append(gpu, case, counts, 3, rows=rows)
        want = ref.append(case, kn, vn, rows, starts)
        assert got == want and all(case.same(state)), counts
    assert set(got) >= {ref.DONE, ref.NO_ROOM, ref.INVALID}


@pytest.mark.parametrize("counts,taken,status", [
    ([16, 1, 120, 2, 1, 0], 0, [0, 0, 2, 0, 0, 0]),   # 136 positions do not fit the third's table row: it takes no pages from the others
    ([16, 1, 100, 2, 1, 0], 8, [0, 0, 2, 0, 2, 0]),   # 5 free pages, the third needs 7
    ([16, 1, 100, 2, 1, 0], 13, [2, 0, 2, 0, 2, 0]),  # none free
    ([16, 1, 100, 2, 1, 0], 4, [0, 0, 0, 0, 0, 0]),
])
def test_append_when_the_pages_run_out(gpu, counts, taken, status):
    """The first that does not fit and all later ones that need pages stay; those that need none go on."""
    c = _filled(4, pages=20, seqs=6, max_pages=8, lens=[16, 30, 16, 3, 16, 16], spare=0.1)
    c.refs[np.flatnonzero(c.refs == 0)[:taken]] = 1
    got, state, (kn, vn, rows, starts) = _append(gpu, c, counts, 4)
    want = ref.append(c, kn, vn, rows, starts)
    assert got == want == status and all(c.same(state))


def test_append_with_row_starts_that_decrease_or_leave_the_rows(gpu):
    """Undefined for the sequences concerned, but nothing outside the arrays is touched: lengths stay within the table."""
    c = _filled(5, pages=40, seqs=4, max_pages=6, lens=[5, 20, 33, 0])
    for starts in ([0, 9, 4, 12, 7], [-5, 3, 100, 1 << 30, -(1 << 30)], [12, 0, 0, 0, 0]):
        got, state, _ = _append(gpu, c.copy(), [3, 3, 3, 3], 5, starts=starts)
        assert set(got) <= {0, 1, 2, 3} and 0 <= state[3].min() and state[3].max() <= 6 * 16, starts


@pytest.mark.parametrize("seqs,max_pages,pages,n", [(1, 1, 1, 16), (1, 3, 4, 1), (300, 5, 1600, 1), (1100, 2, 40000, 3)])
def test_append_batch_sizes(gpu, seqs, max_pages, pages, n):
    c = _filled(6, pages=pages, seqs=seqs, max_pages=max_pages, layers=1, kv_heads=1, dim=8, lens=[(7 * s) % (max_pages * 16 - n + 1) for s in range(seqs)])
    got, state, (kn, vn, rows, starts) = _append(gpu, c, [n] * seqs, 6)
    want = ref.append(c, kn, vn, rows, starts)
    assert got == want and all(c.same(state))


@pytest.mark.parametrize("pages", [2, 3, 4095, 4097, 4099, 20482, 36871])
def test_free_pages_are_found_wherever_they_are(gpu, pages):
    """A nearly full pool: the free pages lie around the edges of what the search looks at together, and at its end."""
    edges = sorted({e + d for e in (0, 4, 4096, 8192, 20480, 24576, 36864, pages) for d in (-2, -1, 0, 1)} & set(range(pages)))
    for held in (0, 1, len(edges) // 2, len(edges) - 1, len(edges)):
        c = ref.Cache(1, pages, 1, 16, 8, 3, 64)
        c.refs[:] = 1
        c.refs[edges[held:]] = 0
        free = len(edges) - held
        for counts in ([16 * free, 0, 0], [0, 16, 16 * max(0, free - 1)], [16 * (free + 1), 0, 0]):
            print(f"{pages} pages, {free} free, rows {counts}", flush=True)
            case = c.copy()
            got, state, (kn, vn, rows, starts) = _append(gpu, case, counts, pages)
            assert got == ref.append(case, kn, vn, rows, starts) and all(case.same(state))


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("seed,ps,layers,kv_heads,dim,dtype,forks", [
    (0, 16, 2, 2, 64, torch.bfloat16, [(0, 5), (1, 6), (0, 7)]),
    (1, 32, 16, 8, 64, torch.bfloat16, [(2, 5)]),
    (2, 64, 1, 1, 128, torch.float16, [(3, 6), (3, 7), (2, 5)]),
    (3, 16, 3, 1, 16, torch.uint8, [(0, 5), (5, 6), (6, 7)]),  # from sequences that are empty before the call
    (4, 16, 1, 3, 8, torch.int16, [(0, 5), (1, 5), (8, 6), (0, -1), (5, 5), (0, 1), (4, 7), (-3, 6)]),
])
def test_fork(gpu, share, seed, ps, layers, kv_heads, dim, dtype, forks):
    print(f"fork seed {seed} share {share}", flush=True)
    c = _filled(seed, pages=80, ps=ps, layers=layers, kv_heads=kv_heads, dim=dim, dtype=dtype, spare=0.5,
                lens=[3 * ps, 4 * ps + 1, 3, 5 * ps - 1, 0, 0, 0, 0])
    c.table[1, 2] = 77777  # a hole in the middle
    state = c.to(gpu)
    got = _run(ops.PageFork(num_forks=len(forks), share=share, **_data(c)), [_ints(forks, gpu), *state], len(forks))
    want = ref.fork(c, forks, share)
    assert got == want and all(c.same(state))


@pytest.mark.parametrize("share", [True, False])
def test_fork_when_the_pages_run_out(gpu, share):
    """Pairs that need no page go on after one that got none."""
    c = _filled(7, pages=14, seqs=9, lens=[33, 32, 20, 5, 0, 0, 0, 0, 0], spare=0.0)
    c.refs[[p for p in range(14) if c.refs[p] == 0]] = 0
    forks = [(0, 4), (2, 5), (0, 6), (1, 7), (3, 8)]
    free = int((c.refs == 0).sum())
    for drop in range(free + 1):
        case = c.copy()
        case.refs[np.flatnonzero(case.refs == 0)[:drop]] = 1
        state = case.to(gpu)
        got = _run(ops.PageFork(num_forks=5, share=share, **_data(case)), [_ints(forks, gpu), *state], 5)
        want = ref.fork(case, forks, share)
        assert got == want and all(case.same(state)), drop


def test_fork_many(gpu):
    """More pairs than threads of the planning workgroup, long table rows."""
    c = _filled(8, pages=9000, seqs=2400, max_pages=1500, layers=1, kv_heads=1, dim=8, lens=[1200 * 16 + 5, 17] + [0] * 2398)
    forks = [(i % 2, 2 + (i * 7) % 1300) for i in range(1400)]
    state = c.to(gpu)
    got = _run(ops.PageFork(num_forks=len(forks), **_data(c)), [_ints(forks, gpu), *state], len(forks))
    want = ref.fork(c, forks, True)
    assert got == want and all(c.same(state))


@pytest.mark.parametrize("seed,pages,ps,layers,kv_heads,dim,dtype", [
    (0, 60, 16, 2, 2, 64, torch.bfloat16), (1, 1, 16, 1, 1, 64, torch.bfloat16), (2, 4096, 16, 1, 1, 8, torch.int16),
    (3, 4097, 16, 1, 1, 8, torch.int16), (4, 12289, 16, 1, 1, 8, torch.int16), (5, 33, 64, 16, 8, 64, torch.float16),
    (6, 40, 128, 1, 2, 256, torch.float32), (7, 16384, 16, 1, 1, 8, torch.int16), (8, 16385, 16, 1, 1, 8, torch.int16),
    (9, 40001, 16, 1, 1, 8, torch.int16),
])
@pytest.mark.parametrize("spare", [0.0, 0.02, 0.4, 0.9, 1.0])
def test_compact(gpu, seed, pages, ps, layers, kv_heads, dim, dtype, spare):
    print(f"compact seed {seed} spare {spare}", flush=True)
    rng = np.random.default_rng(seed + 50)
    seqs, max_pages = 7, max(2, pages // 5)
    c = ref.Cache(layers, pages, kv_heads, ps, dim, seqs, max_pages, seed, dtype)
    ids = list(rng.permutation(pages)[: round(pages * (1 - spare))])
    shared = ids[:2]
    for s in range(seqs):
        own = [ids.pop() for _ in range(min(len(ids), max_pages - 2))] if s else []
        pages_of = (shared if s % 2 else []) + own
        c.hold(s, max(0, len(pages_of) * ps - s), pages_of)
        c.table[s, len(pages_of):] = rng.integers(-3, pages + 3, max_pages - len(pages_of))  # behind the last page: anything
    if len(ids):
        c.refs[ids] = 1  # held by nobody in the table: moved all the same
    c.lens[0] = -4
    state = c.to(gpu)
    got = _run(ops.PageCompact(**_data(c)), state, 1)
    want = ref.compact(c)
    assert got == [want] and all(c.same(state))
    assert (c.refs[int((c.refs != 0).sum()):] == 0).all()


def test_free(gpu):
    c = _filled(9, pages=400, seqs=12, max_pages=30, layers=1, kv_heads=1, dim=8, lens=[16 * 30, 0, 1, 16, 17, 100, 200, 31, 33, 64, 5, 6])
    for s in (6, 7, 8):  # shared first pages
        c.refs[c.table[s, 0]] -= 1
        c.table[s, 0] = c.table[5, 0]
        c.refs[c.table[5, 0]] += 1
    c.table[6, 3] = 1 << 30  # a hole
    c.refs[c.table[9, 1]] = 0  # a count that is already zero
    c.lens[10] = 16 * 30 + 1
    for slots in ([0], [5, 6], [8, 8, 7, 8], [3, -1, 12, 3, 1, 10, 9, 0, 2], list(range(12)), [11] * 2000):
        print(f"free {slots[:9]}", flush=True)
        case = c.copy()
        state = case.to(gpu)
        got = _run(ops.PageFree(num_slots=len(slots), **_pool(case)), [_ints(slots, gpu), *state[2:]], len(slots))
        want = ref.free(case, slots)
        assert got == want and all(case.same(state)), slots


def test_free_of_pages_counted_too_low(gpu):
    """More entries hold a page than its count says: it ends at 0, free, and never below."""
    c = _filled(29, pages=64, seqs=12, max_pages=4, layers=1, kv_heads=1, dim=8, lens=[64] * 12)
    for s in range(1, 12):
        c.refs[c.table[s, :2]] = 0
        c.table[s, :2] = c.table[0, :2]
    c.refs[c.table[0, 0]], c.refs[c.table[0, 1]] = 2, 11
    state = c.to(gpu)
    assert _run(ops.PageFree(num_slots=12, **_pool(c)), [_ints(list(range(12)), gpu), *state[2:]], 12) == ref.free(c, list(range(12)))
    assert all(c.same(state)) and (c.refs == 0).all()


def test_large_pools_by_64_bit_offsets(gpu):
    """A pool past 4 GiB: the last pages are written and copied where they are, not 2^32 bytes before."""
    L, P, Hkv, ps, D = 2, 66000, 8, 32, 64  # 2.2 GB of K in each layer
    k, v = (torch.empty(L, P, Hkv, ps, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    k[:, P - 40:] = 1.0
    v[:, P - 40:] = 2.0
    data = dict(num_layers=L, num_kv_heads=Hkv, head_dim=D, num_pages=P, page_size=ps, num_seqs=2, max_pages=4)
    table = torch.full((2, 4), -1, dtype=torch.int32, device=gpu)
    lens, refs = torch.zeros(2, dtype=torch.int32, device=gpu), torch.ones(P, dtype=torch.int32, device=gpu)
    refs[[P - 1, P - 7]] = 0
    new = torch.randn(L, 5, Hkv, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    tables = (table, lens, refs)
    got = _run(ops.PagedAppend(num_nodes=5, num_rows=5, **data),
               [new.to(gpu), (new + 1).to(gpu), _ints([4, 3, 2, 1, 0], gpu), _ints([0, 5, 5], gpu), k, v, *tables], 2)
    assert got == [0, 0] and table[0].tolist() == [P - 7, -1, -1, -1]
    assert torch.equal(k[:, P - 7, :, :5].cpu(), new.flip(1).transpose(1, 2))
    got = _run(ops.PageFork(num_forks=1, **data), [_ints([[0, 1]], gpu), k, v, *tables], 1)
    assert got == [0] and table[1, 0].item() == P - 1
    assert torch.equal(k[:, P - 1, :, :5].cpu(), new.flip(1).transpose(1, 2))
    assert (v[:, P - 1, :, 5:] == 2).all() and (k[:, P - 40:P - 7] == 1).all() and (k[:, P - 6:P - 1] == 1).all()
    refs[:40] = 0  # room at the front: the last 40 pages move there
    got = _run(ops.PageCompact(**data), [k, v, *tables], 1)
    assert got == [40] and table[:, 0].tolist() == [33, 39]
    assert torch.equal(k[:, 33, :, :5].cpu(), new.flip(1).transpose(1, 2)) and (k[:, :33] == 1).all() and (v[:, 34:39] == 2).all()


def test_a_captured_step_is_replayed(gpu):
    """Append, fork and free in one graph, replayed with eager work between: each replay equals the loops over integers."""
    c = _filled(11, pages=200, seqs=6, max_pages=12, lens=[5, 20, 16, 0, 0, 0])
    L, _, Hkv, _, D = c.k.shape
    kn, vn = (torch.randn(L, 4, Hkv, D, generator=torch.Generator().manual_seed(s)).to(c.dtype) for s in (1, 2))
    rows, starts, forks, slots = [3, 0, 1], [0, 1, 1, 3, 3, 3, 3], [(0, 3), (2, 4)], [3, 4]
    state = c.to(gpu)
    told = [torch.empty(n, dtype=torch.int32, device=gpu) for n in (6, 2, 2)]
    calls = (ops.PagedAppend(num_nodes=4, num_rows=3, **_data(c)).get_callable(),
             ops.PageFork(num_forks=2, **_data(c)).get_callable(), ops.PageFree(num_slots=2, **_pool(c)).get_callable())
    new = (kn.to(gpu), vn.to(gpu), _ints(rows, gpu), _ints(starts, gpu))
    pairs, ends = _ints(forks, gpu), _ints(slots, gpu)

    def step():
        calls[0](*new, *state, told[0])
        calls[1](pairs, *state, told[1])
        calls[2](ends, *state[2:], told[2])

    def want():
        return ref.append(c, kn, vn, rows, starts), ref.fork(c, forks, True), ref.free(c, slots)

    step()
    torch.cuda.synchronize()
    want()
    graph = capture_graph(step, gpu)
    for _ in range(5):
        scratch = torch.randn(1 << 20, device=gpu).sum()  # the program's own work between replays
        graph.replay()
        torch.cuda.synchronize()
        assert tuple(t.tolist() for t in told) == want() and all(c.same(state))


def test_other_streams(gpu):
    """Two caches on two streams, one operator: nothing is shared between the calls."""
    cases = [_filled(20 + i, pages=300, seqs=8, max_pages=20, lens=[10 * i + 3 * s + 1 for s in range(8)]) for i in range(2)]
    op = ops.PageFork(num_forks=2, share=False, **_data(cases[0])).get_callable()
    streams, states, told = [torch.cuda.Stream(gpu) for _ in cases], [c.to(gpu) for c in cases], []
    for c, st in zip(cases, states):
        for s in (6, 7):
            ref.free(c, [s])
        for t, w in zip(st[2:], (c.table, c.lens, c.refs)):
            t.copy_(torch.from_numpy(w))
    pairs = _ints([(0, 6), (3, 7)], gpu)
    torch.cuda.synchronize()
    for stream, st in zip(streams, states):
        with torch.cuda.stream(stream):
            told.append(torch.empty(2, dtype=torch.int32, device=gpu))
            op(pairs, *st, told[-1])
    torch.cuda.synchronize()
    for c, st, t in zip(cases, states, told):
        assert t.tolist() == ref.fork(c, [(0, 6), (3, 7)], False) and all(c.same(st))


@pytest.mark.parametrize("starts,status", [
    ([0, 3, 8, 13, 13, 13], [0, 0, 1, 0, 0]),                    # one row more than there are: the sequence stays whole as it was
    ([0, 3, 1 << 30, 1 << 30, 1 << 30, 1 << 30], [0, 1, 0, 0, 0]),  # and those that have no rows are done wherever they lie
    ([-1, 3, 8, 12, 12, 12], [1, 0, 0, 0, 0]),
    ([2, 3, 8, 8, 8, 12], [0, 0, 0, 0, 0]),                      # rows before the first range are nobody's
    ([0, 8, 4, 10, 10, 12], [0, 1, 1, 0, 0]),                    # a range that ends before its start, and one on an earlier one's rows
    ([0, 10, 2, 6, 8, 12], [0, 1, 1, 1, 1]),
    ([0, 4, 4, 4, 3, 7], [0, 0, 0, 1, 1]),
    ([9, 5, 5, 7, 12, 12], [1, 0, 1, 1, 0]),
    ([-(1 << 31), (1 << 31) - 1, 0, 12, 12, 12], [1, 1, 1, 0, 0]),
    ([12, 0, 0, 0, 0, 0], [1, 0, 0, 0, 0]),
])
def test_append_ranges_that_are_none(gpu, starts, status):
    """A sequence gets all rows of its range or none: ranges that leave the rows, decrease or overlap change nothing, and
    rows that two ranges name are the first one's."""
    print(f"append row_starts {starts}", flush=True)
    c = _filled(31, pages=60, seqs=5, max_pages=6, lens=[5, 20, 33, 0, 16])
    got, state, (kn, vn, rows, starts) = _append(gpu, c, [3, 3, 3, 2, 1], 31, starts=starts)
    assert got == status == ref.append(c, kn, vn, rows, starts) and all(c.same(state))


def test_append_ranges_of_many_sequences(gpu):
    """More sequences than threads of the planning workgroup: a range far behind one that it overlaps."""
    c = _filled(32, pages=3000, seqs=2600, max_pages=2, layers=1, kv_heads=1, dim=8, lens=[s % 17 for s in range(2600)])
    starts = [0] + list(np.cumsum([1] * 2600))
    starts[1030] = 1035                   # the ranges after it start before its end, up to that of row 1035
    starts[2100:2200] = [900] * 100       # one that decreases, then empty ones, then one over all rows from 900 on
    got, state, (kn, vn, rows, starts) = _append(gpu, c, [1] * 2600, 32, starts=starts)
    want = ref.append(c, kn, vn, rows, starts)
    assert got == want and all(c.same(state))
    assert [s for s in range(2600) if got[s]] == [*range(1030, 1035), 2099, 2199]


@pytest.mark.parametrize("max_pages", [2048, 2049, 5000])
def test_free_of_long_table_rows(gpu, max_pages):
    """Several workgroups to a slot: lengths around multiples of a workgroup's 2048 entries and the whole table row, shared
    pages and holes in every part, one that is short of a count, slots named twice and slots that are none."""
    ps, at = 16, [2047, 2048, 2049, 4095, 4096, 4097]
    lens = [max_pages * ps] * 2 + [0, 1] + [min(e, max_pages) * ps - d for e in at for d in (0, 15)] + [max_pages * ps + 1, -1]
    c = _filled(33, pages=max_pages * 17, ps=ps, seqs=len(lens), max_pages=max_pages, layers=1, kv_heads=1, dim=8, lens=lens[:-2], spare=0.0)
    c.lens[:] = lens
    for s in (1, 5, 6, 9, 14):  # entries all along the row are those of sequence 0
        e = np.arange(s % 3, c.used(int(c.lens[s])), 3)
        c.refs[c.table[s, e]] -= 1
        c.table[s, e] = c.table[0, e]
        c.refs[c.table[0, e]] += 1
    c.table[1, 2::500] = -1
    c.table[7, [0, 2047]] = 1 << 30
    c.refs[c.table[8, [3, 2040]]] = 0
    S = len(lens)
    for slots in ([0], [1, 0], [6, 6, 0, 6, S, -1], list(range(S)), [S - 1, S - 2, 14, 3, 2, 14, 1]):
        print(f"free {slots[:9]} of {max_pages} entries", flush=True)
        case = c.copy()
        state = case.to(gpu)
        got = _run(ops.PageFree(num_slots=len(slots), **_pool(case)), [_ints(slots, gpu), *state[2:]], len(slots))
        want = ref.free(case, slots)
        assert got == want and all(case.same(state)), slots


@pytest.mark.parametrize("ps", [256, 512, 1024])
@pytest.mark.parametrize("layers,kv_heads,dim,dtype", [(1, 8, 128, torch.bfloat16), (3, 2, 64, torch.float16), (2, 1, 24, torch.float32)])
def test_large_pages(gpu, ps, layers, kv_heads, dim, dtype):
    """Pages of hundreds of positions: rows appended up to, onto and across their ends, last pages of one row and of all but
    one forked and copied, a pool packed."""
    print(f"pages of {ps} {dtype}", flush=True)
    c = _filled(34, pages=26, ps=ps, seqs=9, max_pages=4, layers=layers, kv_heads=kv_heads, dim=dim, dtype=dtype,
                lens=[2 * ps - 3, ps, 1, 3 * ps - 1, 5, 0, 0, 0, 0], spare=0.0)
    got, state, (kn, vn, rows, starts) = _append(gpu, c, [2, 1, ps, 2, 0, ps + 1, 0, 0, 0], 34)
    assert got == ref.append(c, kn, vn, rows, starts) == [0] * 9 and all(c.same(state))
    for forks, share in (([(0, 6), (3, 7)], True), ([(2, 8)], False)):
        got = _run(ops.PageFork(num_forks=len(forks), share=share, **_data(c)), [_ints(forks, gpu), *state], len(forks))
        assert got == ref.fork(c, forks, share) == [0] * len(forks) and all(c.same(state))
    got = _run(ops.PageFree(num_slots=2, **_pool(c)), [_ints([0, 1], gpu), *state[2:]], 2)
    assert got == ref.free(c, [0, 1]) == [0, 0] and all(c.same(state))
    got = _run(ops.PageCompact(**_data(c)), state, 1)
    assert got == [ref.compact(c)] and got[0] > 0 and all(c.same(state))


def test_the_largest_batches(gpu):
    """8192 sequences and requests, of which a request in ten cannot be met."""
    S = 8192
    c = _filled(40, pages=40000, seqs=S, max_pages=3, layers=1, kv_heads=1, dim=8, lens=[(5 * s) % 33 if s < S // 2 else 0 for s in range(S)])
    c.lens[9:S // 2:10] = 49
    got, state, (kn, vn, rows, starts) = _append(gpu, c, [s % 3 if s < S // 2 else 0 for s in range(S)], 40)
    assert got == ref.append(c, kn, vn, rows, starts) and all(c.same(state))
    forks = [(i % (S // 2), S // 2 + i % (S // 2 - 5)) for i in range(S)]  # the last 4101 name children that earlier pairs name
    firsts = set(b for _, b in forks)
    got = _run(ops.PageFork(num_forks=S, **_data(c)), [_ints(forks, gpu), *state], S)
    assert got == ref.fork(c, forks, True) and all(c.same(state)) and got.count(ref.DONE) > 0.85 * len(firsts)
    slots = [(i * 7) % S for i in range(S)]
    got = _run(ops.PageFree(num_slots=S, **_pool(c)), [_ints(slots, gpu), *state[2:]], S)
    assert got == ref.free(c, slots) and all(c.same(state))


def test_the_longest_append(gpu):
    """2^20 rows to one sequence in one call, copied whole, freed: the pages in order, the rows in their places."""
    n, ps, MP = 1 << 20, 16, 1 << 16
    P = 2 * MP + 100
    pool = dict(num_pages=P, page_size=ps, num_seqs=3, max_pages=MP)
    data = dict(num_layers=1, num_kv_heads=1, head_dim=8, **pool)
    i32 = lambda n, v: torch.full((n,), v, dtype=torch.int32, device=gpu)
    kn = torch.randn(1, n, 1, 8, generator=torch.Generator(gpu).manual_seed(41), device=gpu).to(torch.bfloat16)
    k, v = (torch.zeros(1, P, 1, ps, 8, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    table, lens, refs = i32(3 * MP, -1).view(3, MP), i32(3, 0), i32(P, 0)
    refs[:100] = 1
    rows = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=gpu)
    got = _run(ops.PagedAppend(num_nodes=n, num_rows=n, **data), [kn, kn + 1, rows, _ints([0, 0, n, n], gpu), k, v, table, lens, refs], 3)
    assert got == [0, 0, 0] and lens.tolist() == [0, n, 0]
    assert torch.equal(table[1], torch.arange(100, 100 + MP, dtype=torch.int32, device=gpu)) and (refs[:100 + MP] == 1).all()
    assert torch.equal(k[0, 100:100 + MP].reshape(n, 8), kn[0, :, 0].flip(0)) and torch.equal(v[0, 100:100 + MP].reshape(n, 8), (kn + 1)[0, :, 0].flip(0))
    got = _run(ops.PageFork(num_forks=1, share=False, **data), [_ints([[1, 2]], gpu), k, v, table, lens, refs], 1)
    assert got == [0] and lens.tolist() == [0, n, n] and (refs == 1).all()
    assert torch.equal(table[2], table[1] + MP) and torch.equal(k[0, 100 + MP:], k[0, 100:100 + MP]) and torch.equal(v[0, 100 + MP:], v[0, 100:100 + MP])
    got = _run(ops.PageFree(num_slots=1, **pool), [_ints([1], gpu), table, lens, refs], 1)
    assert got == [0] and lens.tolist() == [0, 0, n] and (table[1] == -1).all() and int((refs == 0).sum()) == MP
    got = _run(ops.PageCompact(**data), [k, v, table, lens, refs], 1)
    assert got == [MP] and torch.equal(table[2], torch.arange(100, 100 + MP, dtype=torch.int32, device=gpu)) and int(refs.sum()) == 100 + MP
    assert torch.equal(k[0, 100:100 + MP].reshape(n, 8), kn[0, :, 0].flip(0))
