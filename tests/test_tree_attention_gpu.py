"""GPU: TreeAttention against the attention in 64 bits, within the bound of its own rounding (paged_reference.attention)."""

import math

import numpy as np
import pytest
import torch

import iron_amd.operators as ops
from iron_amd import _lib
from iron_amd.common.graph import capture_graph
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


class Case:
    """Random trees over a scattered cache. `spare` rows of out stand behind the last tree."""

    def __init__(self, H, Hkv, D, ps, lens, nodes, dtype=BF16, seed=0, mask="tree", max_nodes=None, spare=2, scale=None, q_scale=2.0):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        S = len(lens)
        self.H, self.Hkv, self.D, self.ps, self.lens, self.nodes = H, Hkv, D, ps, list(lens), list(nodes)
        self.N, self.T = sum(nodes) + spare, max_nodes or max(1, max(nodes))
        self.starts = [0] + [int(x) for x in np.cumsum(nodes)]
        self.MP = max(1, max(-(-n // ps) for n in lens)) + 1
        used = sum(-(-n // ps) for n in lens)
        self.P = used + 5
        ids = rng.permutation(self.P)
        self.table = rng.integers(0, self.P, (S, self.MP)).astype(np.int32)  # behind the last page: any page
        at = 0
        for s, n in enumerate(lens):
            c = -(-n // ps)
            self.table[s, :c] = ids[at:at + c]
            at += c
        r = lambda *shape: torch.randn(*shape, generator=g).to(dtype)
        self.q, self.kn, self.vn = (r(self.N, H, D) * q_scale).to(dtype), r(self.N, Hkv, D), r(self.N, Hkv, D)
        self.kp, self.vp = r(self.P, Hkv, ps, D), r(self.P, Hkv, ps, D)
        self.sees = np.zeros((self.N, self.T), bool)
        for s, t in enumerate(nodes):
            a = self.starts[s]
            for i in range(t):
                if mask == "tree":
                    if i:
                        self.sees[a + i] = self.sees[a + rng.integers(0, i)]
                    self.sees[a + i, i] = True
                elif mask == "chain":
                    self.sees[a + i, :i + 1] = True
                elif mask == "random":
                    self.sees[a + i, :t] = rng.random(t) < 0.3
        self.prior = torch.full((self.N, H, D), 7.0).to(dtype)
        self.scale = scale if scale is not None else 1 / math.sqrt(D)
        self.op = ops.TreeAttention(num_heads=H, num_kv_heads=Hkv, head_dim=D, num_pages=self.P, page_size=ps, num_seqs=S,
                                    max_pages=self.MP, num_nodes=self.N, max_nodes=self.T, dtype=dtype, scale=scale)

    def tensors(self, gpu):
        i = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)
        words = self.op.pack_mask(torch.from_numpy(self.sees))
        return [*(t.to(gpu) for t in (self.q, self.kn, self.vn, self.kp, self.vp)), i(self.table), i(self.lens), i(self.starts),
                words.to(gpu), self.prior.to(gpu)]

    def want(self):
        return ref.attention(self.q, self.kn, self.vn, self.kp, self.vp, self.table, self.lens, self.starts, self.sees, self.scale, self.prior,
                             self.op.max_nodes)

    def check(self, gpu, got=None):
        if got is None:
            t = self.tensors(gpu)
            self.op.get_callable()(*t)
            torch.cuda.synchronize()
            got = t[-1]
        got = got.cpu().double()
        want, tol = self.want()
        assert torch.isfinite(got).all()
        bad = (got - want).abs() > tol
        assert not bad.any(), (int(bad.sum()), (got - want).abs().max().item(), bad.nonzero()[:3].tolist())
        return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv,ps,lens,nodes", [
    (32, 8, 16, [2047], [1]),                                   # one decode step
    (4, 2, 16, [0, 1, 15, 16, 17, 63, 64, 65, 300], [1] * 9),   # lengths around pages and tiles, none at all
    (4, 4, 32, [100, 0, 31], [5, 3, 7]),                        # one head to a KV head
    (8, 1, 64, [129, 500], [13, 26]),                           # eight heads to one
    (6, 2, 16, [77, 200, 1, 40], [2, 0, 17, 1]),                # three heads, a sequence without nodes
    (10, 2, 128, [1000, 3], [7, 33]),                           # five heads
    (4, 2, 16, [250], [70]),                                    # a tree of more than 64 nodes
    (2, 1, 1024, [1500], [3]),
])
def test_trees(gpu, H, Hkv, ps, lens, nodes, D, dtype):
    print(f"tree H {H}/{Hkv} D {D} lens {lens} nodes {nodes} {dtype}", flush=True)
    Case(H, Hkv, D, ps, lens, nodes, dtype).check(gpu)


@pytest.mark.parametrize("nodes,G", [(1, 16), (1, 17), (16, 1), (33, 1), (8, 8), (16, 8), (64, 2), (65, 2), (129, 1), (200, 4)])
def test_row_counts(gpu, nodes, G):
    """Rows of a KV head (nodes times heads) around the sizes of the kernels' tiles."""
    print(f"rows {nodes} x {G}", flush=True)
    Case(G, 1, 64, 16, [90, 200], [nodes, max(1, nodes // 3)], seed=nodes).check(gpu)
    Case(2 * G, 2, 128, 32, [70], [nodes], FP16, seed=nodes).check(gpu)


@pytest.mark.parametrize("mask", ["none", "random", "chain"])
@pytest.mark.parametrize("lens", [[0, 0, 0], [5, 0, 200]])
def test_masks_and_empty_rows(gpu, mask, lens):
    """Rows that see nothing are zeros (no context and no node); a random mask leaves some; a chain is causal attention."""
    c = Case(4, 2, 64, 16, lens, [9, 40, 3], mask=mask, seed=3)
    got = c.check(gpu)
    if mask == "none":
        assert (got[9:49] == 0).all()
    assert (got[-2:] == 7).all()  # behind the last tree: as it was


def test_mask_bits_behind_the_tree_do_not_count(gpu):
    c = Case(4, 2, 64, 16, [20, 30], [5, 4], max_nodes=40, seed=4)
    t = c.tensors(gpu)
    t[8] |= torch.tensor([-(1 << 5), -1], dtype=torch.int32, device=gpu)  # all bits from 5 on; the second tree has 4 nodes
    t[8][5:] &= ~(1 << 4)
    t[8][5:, 0] |= -(1 << 5)
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    c.check(gpu, t[-1])


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("nodes", [(12, 20), (4, 8), (4, 4)])  # 80, 32 and 16 rows to a KV head
def test_what_is_not_seen_does_not_count(gpu, value, D, dtype, nodes):
    """Rows of a page behind the length, other pages, holes, and nodes that a row does not see hold what they like."""
    c = Case(8, 2, D, 16, [37, 100], nodes, dtype, seed=5, mask="chain")
    c.sees[:] = False
    for s, t in enumerate(nodes):
        for i in range(t):
            c.sees[c.starts[s] + i, : i + 1] = True
            c.sees[c.starts[s] + i, 3] = False
    c.table[1, 2] = -1
    c.table[1, 4] = c.P
    held = {int(p) for p in c.table[0, :3]} | {int(c.table[1, e]) for e in (0, 1, 3, 5, 6)}
    for p in range(c.P):
        if p not in held:
            c.kp[p], c.vp[p] = value, value
    c.kp[c.table[0, 2], :, 5:], c.vp[c.table[0, 2], :, 5:] = value, value
    c.kp[c.table[1, 6], :, 4:], c.vp[c.table[1, 6], :, 4:] = value, value
    for s in (0, 1):
        c.kn[c.starts[s] + 3], c.vn[c.starts[s] + 3] = value, value
    c.kn[sum(nodes):], c.vn[sum(nodes):] = value, value
    c.check(gpu)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_is_seen_counts(gpu, value, D, dtype):
    """A value that is not finite reaches the rows that see its node, in its dimension, and no other."""
    c = Case(8, 2, D, 16, [37, 100], [12, 40], dtype, seed=6)
    node, dim = c.starts[1] + 2, 5
    c.vn[node, 1, dim] = value
    t = c.tensors(gpu)
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    got = t[-1].cpu().double()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    for i in range(12, 52):
        hit[i, 4:, dim] = bool(c.sees[i, 2])
    assert hit.any() and not hit[12:52, 4:, dim].all()
    assert torch.equal(torch.isnan(got[hit]) | torch.isinf(got[hit]), torch.ones_like(got[hit], dtype=torch.bool))
    if value == value:
        assert (got[hit] == value).all()
    c.vn[node, 1, dim] = 0.0
    want, tol = c.want()
    assert ((got - want).abs() <= tol)[~hit].all()


def test_cached_values_that_are_not_finite(gpu):
    """The same for a cached position, which every row of its sequence sees."""
    c = Case(4, 2, 64, 16, [37, 100], [3, 4], seed=7)
    c.vp[c.table[1, 1], 1, 3, 9] = float("inf")
    t = c.tensors(gpu)
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    got = t[-1].cpu().double()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[3:7, 2:, 9] = True
    assert (got[hit] == float("inf")).all()
    c.vp[c.table[1, 1], 1, 3, 9] = 0.0
    want, tol = c.want()
    assert ((got - want).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("nodes", [3, 30])  # 12 and 120 rows to a KV head
@pytest.mark.parametrize("behind", [0.0, float("nan"), float("inf")])
def test_scores_of_minus_infinity(gpu, behind, nodes):
    """Such a key has no weight, whatever its value; a row that sees no other is a row that sees nothing."""
    c = Case(4, 1, 64, 16, [37, 100], [nodes, 1], seed=28)
    c.q[:] = c.q.abs() + 0.125
    n = c.starts[1]
    for p in c.table[0, :3]:
        c.kp[p] = -float("inf")
    c.kn[:n] = -float("inf")
    c.vp[c.table[0, 2], :, 5:] = behind  # behind the last position
    c.kp[c.table[1, 0], :, 3], c.vp[c.table[1, 0], :, 3] = -float("inf"), behind
    c.vn[:n, :, 7] = behind
    t = c.tensors(gpu)
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    got = t[-1].cpu().double()
    assert (got[:n] == 0).all()
    c.kp[c.table[1, 0], :, 3] = c.q[n:n + 1].mean(1) * -1e4  # a weight of zero in 64 bits too
    c.kp[c.table[0, :3]], c.kn[:n], c.vn[:n] = 0.0, 0.0, 0.0
    c.vp[c.table[0, 2]], c.vp[c.table[1, 0], :, 3] = 0.0, 0.0
    want, tol = c.want()
    assert ((got - want).abs() <= tol)[n].all()


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (128, FP16)])
@pytest.mark.parametrize("nodes", [3, 30])
def test_the_largest_values(gpu, nodes, D, dtype):
    """A mean of values at the end of the type's range is one: no sum on the way overflows."""
    c = Case(4, 1, D, 16, [70, 5], [nodes, 1], dtype, seed=30)
    most = torch.finfo(dtype).max
    c.vp[:], c.vn[:] = most, -most
    c.check(gpu)
    c.vn[:] = most
    c.q[:] = 0.0
    assert (c.check(gpu)[:nodes + 1] >= most * (1 - 2 * torch.finfo(dtype).eps)).all()


@pytest.mark.parametrize("nodes", [3, 30])
@pytest.mark.parametrize("others", [0.0, -float("inf")])
def test_a_score_of_nan(gpu, others, nodes):
    """It makes its rows NaN, whatever the other scores are; a score of plus infinity does too."""
    c = Case(4, 1, 64, 16, [37, 20, 20], [nodes, nodes, 1], seed=29)
    c.q[:] = c.q.abs() + 0.125
    for s, value in ((0, float("nan")), (1, float("inf"))):
        c.kp[c.table[s, :-(-c.lens[s] // 16)]] = others
        c.kn[c.starts[s]:c.starts[s + 1]] = others
        c.kp[c.table[s, 1], :, 2] = value
    t = c.tensors(gpu)
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    got = t[-1].cpu().double()
    assert got[:2 * nodes].isnan().all() and got[2 * nodes:].isfinite().all()


@pytest.mark.parametrize("q_scale", [0.0, 1e-3, 60.0])
def test_flat_and_peaked_softmax(gpu, q_scale):
    """Equal weights, and rows that one key decides; scores of many hundreds."""
    Case(8, 2, 64, 16, [333, 64], [10, 1], seed=8, q_scale=q_scale).check(gpu)
    Case(8, 2, 128, 16, [333, 64], [10, 1], FP16, seed=9, q_scale=q_scale).check(gpu)


def test_growing_scores(gpu):
    """The maximum rises from key to key all the way, and the weights before it fade."""
    c = Case(4, 2, 64, 16, [400], [5], seed=10)
    c.q[:] = 1.0
    for t in range(400):
        c.kp[c.table[0, t // 16], :, t % 16] = 0.01 * t
    c.check(gpu)


def test_scale(gpu):
    Case(4, 2, 64, 16, [100, 7], [5, 6], seed=11, scale=0.5, q_scale=0.5).check(gpu)


def test_lengths_outside_the_table_and_starts_that_lead_out(gpu):
    """A length is cut to the table's range; node_starts cannot lead out of the rows."""
    c = Case(4, 2, 64, 16, [100, 40], [5, 6], seed=12)
    t = c.tensors(gpu)
    t[6].copy_(torch.tensor([1 << 30, -3]))
    c.lens = [c.MP * 16, 0]
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    c.check(gpu, t[-1])
    for starts in ([-7, 5, 1 << 30], [5, 2, 20], [1 << 30, -(1 << 30), 3], [0, 0, 0]):
        t[7].copy_(torch.tensor(starts))
        c.op.get_callable()(*t)
        torch.cuda.synchronize()
        assert torch.isfinite(t[-1].float()).all()


def test_trees_cut_to_max_nodes(gpu):
    """Nodes behind max_nodes of a tree are no part of it: their rows stay."""
    c = Case(4, 2, 64, 16, [50], [9], max_nodes=9, seed=13)
    t = c.tensors(gpu)
    op = ops.TreeAttention(num_heads=4, num_kv_heads=2, head_dim=64, num_pages=c.P, page_size=16, num_seqs=1, max_pages=c.MP,
                           num_nodes=c.N, max_nodes=6)
    op.get_callable()(*t)
    torch.cuda.synchronize()
    c.starts, c.sees = [0, 6], c.sees[:, :6]
    got = c.check(gpu, t[-1])
    assert (got[6:] == 7).all()


def test_many_sequences(gpu):
    """More sequences than a wave, ragged, some empty: the split of the work over the chip."""
    rng = np.random.default_rng(14)
    lens = [int(x) for x in rng.integers(0, 260, 150)]
    Case(4, 2, 64, 16, lens, [int(x) for x in rng.integers(0, 4, 150)], seed=14).check(gpu)
    lens[40] = 5000
    Case(8, 4, 128, 64, lens[:70], [1] * 70, FP16, seed=15).check(gpu)


def test_a_thousand_sequences(gpu):
    """Several sequences to a lane of the wave that shares out the work; most of them without nodes in this call."""
    rng = np.random.default_rng(23)
    lens, nodes = [int(x) for x in rng.integers(0, 70, 1000)], [0] * 1000
    for s in rng.choice(1000, 90, replace=False):
        nodes[s] = int(rng.integers(1, 4))
    Case(2, 1, 64, 16, lens, nodes, seed=23).check(gpu)


def test_the_largest_trees(gpu):
    Case(2, 2, 64, 16, [40], [1024], seed=24, mask="random").check(gpu)
    Case(2, 1, 128, 16, [0, 300], [1000, 24], FP16, seed=25).check(gpu)


def test_more_blocks_than_can_be_counted_are_refused(gpu):
    op = ops.TreeAttention(num_heads=1024, num_kv_heads=1024, head_dim=64, num_pages=1, page_size=16, num_seqs=64, max_pages=8192,
                           num_nodes=1, max_nodes=1024)
    args = [torch.zeros(s.shape, dtype=s.dtype, device=gpu) for s in op.get_arg_spec()]
    with pytest.raises(_lib.IronHipError, match="must count below 2\\^31"):
        op.get_callable()(*args)


def test_long_context(gpu):
    """Many pieces of one sequence's keys, joined."""
    Case(8, 2, 64, 16, [20011], [3], seed=16).check(gpu)
    Case(4, 2, 128, 32, [9001, 17], [20, 2], FP16, seed=17).check(gpu)


def test_cache_past_32_bits(gpu):
    """Pages whose byte offsets pass 2^32."""
    P, Hkv, ps, D = 70000, 8, 64, 64  # 4.6 GB each of K and V
    c = Case(16, 8, 64, 64, [300], [4], seed=18)
    kp, vp = (torch.empty(P, Hkv, ps, D, dtype=BF16, device=gpu) for _ in range(2))
    t = c.tensors(gpu)
    ids = [P - 1 - 3 * e for e in range(5)]
    kp[ids], vp[ids] = t[3][t[5][0, :5].long()], t[4][t[5][0, :5].long()]
    t[3], t[4], t[5][0, :5] = kp, vp, torch.tensor(ids, dtype=torch.int32, device=gpu)
    ops.TreeAttention(num_heads=16, num_kv_heads=8, head_dim=64, num_pages=P, page_size=64, num_seqs=1, max_pages=c.MP, num_nodes=c.N,
                      max_nodes=c.T).get_callable()(*t)
    torch.cuda.synchronize()
    c.check(gpu, t[-1])


def test_same_bits_every_time(gpu):
    c = Case(32, 8, 64, 16, [3000, 100, 777], [26, 10, 1], seed=19)
    t = c.tensors(gpu)
    fn = c.op.get_callable()
    fn(*t)
    torch.cuda.synchronize()
    first = t[-1].clone()
    for _ in range(5):
        t[-1].fill_(7.0)
        fn(*t)
        torch.cuda.synchronize()
        assert torch.equal(first, t[-1])


def test_captured_and_replayed_with_other_lengths(gpu):
    """One graph serves every step: lengths, trees and tables are read when it runs."""
    c = Case(8, 2, 64, 16, [150, 20, 90], [6, 9, 1], seed=20, max_nodes=12, spare=8)
    t = c.tensors(gpu)
    fn = c.op.get_callable()
    fn(*t)
    torch.cuda.synchronize()
    graph = capture_graph(lambda: fn(*t), gpu)
    for lens, nodes in (([150, 20, 90], [6, 9, 1]), ([0, 1, 60], [1, 1, 1]), ([17, 16, 15], [0, 12, 4]), ([158, 32, 96], [12, 0, 12])):
        o = Case(8, 2, 64, 16, lens, nodes, seed=21, max_nodes=12, spare=24 - sum(nodes))
        o.table = c.table
        for n in ("q", "kn", "vn", "kp", "vp"):
            setattr(o, n, getattr(c, n))
        o.sees, o.prior = o.sees[:24], c.prior
        words = c.op.pack_mask(torch.from_numpy(o.sees))
        for dst, src in ((t[6], torch.tensor(lens)), (t[7], torch.tensor(o.starts)), (t[8], words)):
            dst.copy_(src)
        for _ in range(2):
            t[-1].fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            o.check(gpu, t[-1])


def test_two_graphs_and_two_streams_at_once(gpu):
    """One operator captured into two graphs that run at the same time on two streams: each has its own workspace."""
    cases = [Case(32, 8, 64, 16, [3000 - 700 * i, 100], [20, 6], seed=22 + i) for i in range(2)]
    P, MP = max(c.P for c in cases), max(c.MP for c in cases)
    op = ops.TreeAttention(num_heads=32, num_kv_heads=8, head_dim=64, num_pages=P, page_size=16, num_seqs=2, max_pages=MP,
                           num_nodes=cases[0].N, max_nodes=20)
    fn, graphs, sets = op.get_callable(), [], []
    for c in cases:
        t = c.tensors(gpu)
        for i in (3, 4):
            t[i] = torch.cat([t[i], torch.zeros(P - c.P, *t[i].shape[1:], dtype=BF16, device=gpu)])
        t[5] = torch.nn.functional.pad(t[5], (0, MP - c.MP), value=-1).contiguous()
        fn(*t)
        torch.cuda.synchronize()
        graphs.append(capture_graph(lambda t=t: fn(*t), gpu))
        sets.append(t)
    streams = [torch.cuda.Stream(gpu) for _ in cases]
    for _ in range(4):
        for t in sets:
            t[-1].fill_(7.0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, t in zip(cases, sets):
            c.check(gpu, t[-1])


@pytest.mark.parametrize("dispatch", ["fused", "separate"])
def test_in_an_operator_sequence(gpu, dispatch):
    """Attention and append as one runlist, called three times: the cache that a call leaves is the next one's."""
    from iron_amd.common import OperatorSequence

    c = Case(8, 2, 64, 16, [30, 5], [3, 2], seed=26, spare=0, max_nodes=4)
    c.P, c.MP = 16, 6
    c.table = np.full((2, 6), -1, np.int32)
    c.table[0, :2], c.table[1, 0] = (3, 9), 4
    g = torch.Generator().manual_seed(27)
    c.kp, c.vp = (torch.randn(16, 2, 16, 64, generator=g).to(BF16) for _ in range(2))
    pool = dict(num_kv_heads=2, head_dim=64, num_pages=16, page_size=16, num_seqs=2, max_pages=6)
    tree = ops.TreeAttention(num_heads=8, num_nodes=5, max_nodes=4, **pool)
    append = ops.PagedAppend(num_layers=1, num_nodes=5, num_rows=4, **pool)
    cache = ("k_pages", "v_pages", "table", "lens")
    seq = OperatorSequence(name="paged_step", dispatch=dispatch,
                           runlist=[(tree, "q", "k", "v", *cache, "starts", "mask", "out"),
                                    (append, "k", "v", "rows", "row_starts", *cache, "refs", "status")],
                           input_args=["q", "k", "v", "starts", "mask", "rows", "row_starts", *cache, "refs"],
                           output_args=["out", "status"]).compile()
    fn = seq.get_callable()
    refs = torch.zeros(16, dtype=torch.int32)
    refs[[3, 9, 4]] = 1
    rows, row_starts = [0, 2, 3, 4], [0, 2, 4]
    words = tree.pack_mask(torch.from_numpy(c.sees))
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32)
    for name, value in dict(q=c.q, k=c.kn, v=c.vn, starts=i32(c.starts), mask=words, rows=i32(rows), row_starts=i32(row_starts),
                            k_pages=c.kp, v_pages=c.vp, table=i32(c.table), lens=i32(c.lens), refs=refs).items():
        fn.get_buffer(name).torch_view(torch.uint8).copy_(value.contiguous().view(-1).view(torch.uint8))
    want = ref.Cache(1, 16, 2, 16, 64, 2, 6)
    want.k, want.v, want.table, want.lens = c.kp[None].clone(), c.vp[None].clone(), c.table.copy(), np.array(c.lens, np.int32)
    want.refs = refs.numpy().copy()
    for _ in range(3):
        fn()
        c.lens, c.table, c.kp, c.vp = [int(x) for x in want.lens], want.table, want.k[0], want.v[0]
        c.check(gpu, fn.get_buffer("out").to_torch().view(5, 8, 64))
        assert ref.append(want, c.kn[None], c.vn[None], rows, row_starts) == [0, 0]


def test_a_conversation(gpu):
    """The operators together: a prompt in, trees drafted and verified, the accepted rows appended, a fork that goes its own
    way, the parent freed, the pool packed; at every step the attention equals that over the tokens each sequence took."""
    H, Hkv, D, ps, S, MP, P, L, T = 8, 2, 64, 16, 3, 12, 40, 2, 7
    g = torch.Generator().manual_seed(30)
    r = lambda *shape: torch.randn(*shape, generator=g).to(BF16)
    data = dict(num_layers=L, num_kv_heads=Hkv, head_dim=D, num_pages=P, page_size=ps, num_seqs=S, max_pages=MP)
    cache = [torch.full((L, P, Hkv, ps, D), float("nan"), dtype=BF16, device=gpu) for _ in range(2)]
    cache += [torch.full((S, MP), -1, dtype=torch.int32, device=gpu), torch.zeros(S, dtype=torch.int32, device=gpu),
              torch.zeros(P, dtype=torch.int32, device=gpu)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)
    told = torch.zeros(S, dtype=torch.int32, device=gpu)
    history = [[], [], []]  # the (k, v) of every layer that each sequence holds, by position

    def add(kn, vn, rows, starts):
        ops.PagedAppend(num_nodes=kn.shape[1], num_rows=len(rows), **data).get_callable()(kn.to(gpu), vn.to(gpu), i32(rows), i32(starts), *cache, told)
        assert told.tolist() == [0] * S
        for s in range(S):
            history[s] += [(kn[:, i], vn[:, i]) for i in rows[starts[s]:starts[s + 1]]]

    def verify(nodes, seed):
        """The trees' rows and what the attention of each layer made of them."""
        N = sum(nodes) + 1
        starts = [0] + [int(x) for x in np.cumsum(nodes)]
        op = ops.TreeAttention(num_heads=H, num_nodes=N, max_nodes=T, **{k: v for k, v in data.items() if k != "num_layers"})
        parents = [-1] * N
        rng = np.random.default_rng(seed)
        for s in range(S):
            for i in range(1, nodes[s]):
                parents[starts[s] + i] = int(rng.integers(0, i))
        words = op.mask_of_parents(torch.tensor(parents), torch.tensor(starts))
        sees = [[bool(words[i, 0].item() >> j & 1) for j in range(T)] for i in range(N)]
        q, kn, vn = r(L, N, H, D), r(L, N, Hkv, D), r(L, N, Hkv, D)
        for l in range(L):
            prior = torch.full((N, H, D), 7.0, dtype=BF16)
            out = prior.to(gpu)
            op.get_callable()(q[l].to(gpu), kn[l].to(gpu), vn[l].to(gpu), cache[0][l], cache[1][l], cache[2], cache[3], i32(starts), words.to(gpu), out)
            torch.cuda.synchronize()
            lens = [len(h) for h in history]
            assert cache[3].tolist() == lens
            dense = [torch.zeros(S * 20, Hkv, 16, D, dtype=BF16) for _ in range(2)]
            for s, h in enumerate(history):
                for t, kv in enumerate(h):
                    for x in (0, 1):
                        dense[x][s * 20 + t // 16, :, t % 16] = kv[x][l]
            table = [[s * 20 + e for e in range(20)] for s in range(S)]
            want, tol = ref.attention(q[l], kn[l], vn[l], dense[0], dense[1], table, lens, starts, sees, 1 / math.sqrt(D), prior, T)
            assert ((out.cpu().double() - want).abs() <= tol).all(), (l, nodes)
        return kn, vn, starts

    kn, vn = r(L, 90, Hkv, D), r(L, 90, Hkv, D)
    add(kn, vn, list(range(70)) + list(range(75, 90)), [0, 70, 85, 85])
    kn, vn, starts = verify([7, 4, 0], 1)
    add(kn, vn, [0, 2, 5, starts[1], starts[1] + 3], [0, 3, 5, 5])
    two = torch.zeros(1, dtype=torch.int32, device=gpu)
    ops.PageFork(num_forks=1, **data).get_callable()(i32([[0, 2]]), *cache, two)
    assert two.item() == 0
    history[2] = list(history[0])
    kn, vn, starts = verify([3, 1, 5], 2)
    add(kn, vn, [0, 1, starts[1], starts[2], starts[2] + 1, starts[2] + 4], [0, 2, 3, 6])
    verify([2, 2, 2], 3)
    ops.PageFree(num_slots=1, **{k: data[k] for k in ("num_pages", "page_size", "num_seqs", "max_pages")}).get_callable()(i32([0]), *cache[2:], two)
    assert two.item() == 0
    history[0] = []
    verify([1, 1, 6], 4)
    ops.PageCompact(**data).get_callable()(*cache, two)
    torch.cuda.synchronize()
    used = int((cache[4] > 0).sum())
    assert two.item() > 0 and (cache[4][:used] == 1).all() and used == sum(-(-len(h) // ps) for h in history)
    kn, vn, starts = verify([1, 5, 6], 5)
    add(kn, vn, list(range(starts[0], starts[3])), starts)
    verify([7, 7, 7], 6)


def _one_dim(c, q, rows):
    """q and keys with one component: a score is one product, exact in 32 bits. rows: (sequence, position) -> key, the rest 0."""
    c.q[:], c.kp[:], c.kn[:] = 0.0, 0.0, 0.0
    c.q[:, :, 3] = q
    for (s, t), k in rows.items():
        c.kp[c.table[s, t // c.ps], :, t % c.ps, 3] = k


@pytest.mark.parametrize("dtype,D,sizes", [(BF16, 64, (2.0 ** 7, 2.0 ** 12, 2.0 ** 17, 2.0 ** 30)), (BF16, 128, (2.0 ** 13, 2.0 ** 25)),
                                           (FP16, 64, (2.0 ** 7, 2.0 ** 10, 2.0 ** 13, 2.0 ** 15)), (FP16, 128, (2.0 ** 12, 2.0 ** 14))])
@pytest.mark.parametrize("nodes", [3, 30])  # 12 and 120 rows to a KV head
@pytest.mark.parametrize("length", [70, 5000])  # keys of one workgroup or two, and of many
def test_scores_far_from_zero(gpu, dtype, D, sizes, nodes, length):
    """Scores up to 2^62, far enough apart that all weight is the largest one's, or shared by two that are equal: the row is
    that value, or the mean of the two, whatever the size and the sign of the scores."""
    for size in sizes:
        for sign in (1.0, -1.0):
            print(f"scores of {size} squared, sign {sign}, {dtype} D {D} nodes {nodes}", flush=True)
            c = Case(4, 1, D, 16, [length, 33], [nodes, 2], dtype, seed=35, mask="none", scale=1.0)
            row = torch.arange(c.N * 4, dtype=torch.float32).view(c.N, 4)
            _one_dim(c, (size * (1 + row % 61 / 64)).to(dtype), {})
            c.kp[c.table[0, :-(-length // 16)], :, :, 3] = -size * 1.5
            c.kp[c.table[1, :3], :, :, 3] = -size * 1.5
            at = [(0, 21), (0, 66), (1, 32)]
            for s, t in at:
                c.kp[c.table[s, t // 16], :, t % 16, 3] = sign * size
            t = c.tensors(gpu)
            c.op.get_callable()(*t)
            torch.cuda.synchronize()
            got = t[-1].cpu().double()
            v = [c.vp[c.table[s, t // 16], 0, t % 16].double() for s, t in at]
            want = torch.cat([((v[0] + v[1]) / 2).expand(nodes, 4, D), v[2].expand(2, 4, D)])
            size_of = torch.cat([((v[0].abs() + v[1].abs()) / 2).expand(nodes, 4, D), v[2].abs().expand(2, 4, D)])
            tol = want.abs() * torch.finfo(dtype).eps / 2 + size_of * 2.0 ** -15  # equal weights of 16 bits, and their sum's
            assert ((got[:nodes + 2] - want).abs() <= tol).all(), (size, sign)



@pytest.mark.parametrize("infinity", [False, True])
@pytest.mark.parametrize("nodes", [3, 30])
def test_values_behind_far_lower_scores(gpu, nodes, infinity):
    """Keys whose weight is e^-200: values of 1e36 there do not show in rows of small ones, however many workgroups the keys
    went to, and not where an infinity in another dimension has the row done over."""
    c = Case(4, 1, 64, 16, [5000, 20], [nodes, 2], seed=36, mask="none", scale=1.0)
    _one_dim(c, 8.0, {(0, t): -25.0 if t % 5000 != 4321 else 0.0 for t in range(5000)})
    c.vp[:] = 1e36
    c.vp[c.table[0, 4321 // 16], :, 4321 % 16] = torch.randn(64, generator=torch.Generator().manual_seed(37)).to(BF16)
    c.vp[c.table[1, :2]] = 1.0
    if infinity:
        c.vp[c.table[0, 7], :, 9, 40] = float("inf")
    t = c.tensors(gpu)
    c.op.get_callable()(*t)
    torch.cuda.synchronize()
    got = t[-1].cpu().double()
    dims = [d for d in range(64) if not infinity or d != 40]
    want = c.vp[c.table[0, 4321 // 16], 0, 4321 % 16].double()
    assert ((got[:nodes] - want).abs() <= want.abs() * 2.0 ** -8)[:, :, dims].all(), (got[:nodes] - want).abs()[:, :, dims].max()
    if infinity:
        assert (got[:nodes, :, 40] == float("inf")).all()
    assert (got[nodes:nodes + 2] == 1).all()


@pytest.mark.parametrize("nodes,ps,infinity", [(30, 64, False), (30, 16, False), (30, 64, True), (4, 16, True)])  # 60 and 8 rows to a KV head
def test_cache_past_32_bits_wide_and_done_over(gpu, nodes, ps, infinity):
    """The same for the kernel of many rows, for pages that hold half a block of its keys, and for rows that an infinity
    has done over key by key."""
    print(f"{nodes} nodes, pages of {ps}, infinity {infinity}", flush=True)
    P, Hkv, D = 70000 * 64 // ps, 8, 64  # 4.6 GB each of K and V
    c = Case(16, Hkv, D, ps, [300], [nodes], seed=38)
    n = -(-300 // ps)
    if infinity:
        c.vp[c.table[0, n - 2], 3, 5, 9] = float("inf")
    kp, vp = (torch.empty(P, Hkv, ps, D, dtype=BF16, device=gpu) for _ in range(2))
    t = c.tensors(gpu)
    ids = [P - 1 - 3 * e for e in range(n)]
    assert min(ids) * Hkv * ps * D * 2 > 1 << 32
    kp[ids], vp[ids] = t[3][t[5][0, :n].long()], t[4][t[5][0, :n].long()]
    t[3], t[4], t[5][0, :n] = kp, vp, torch.tensor(ids, dtype=torch.int32, device=gpu)
    ops.TreeAttention(num_heads=16, num_kv_heads=Hkv, head_dim=D, num_pages=P, page_size=ps, num_seqs=1, max_pages=c.MP, num_nodes=c.N,
                      max_nodes=c.T).get_callable()(*t)
    torch.cuda.synchronize()
    if not infinity:
        c.check(gpu, t[-1])
        return
    got = t[-1].cpu().double()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[:nodes, 6:8, 9] = True
    assert (got[hit] == float("inf")).all()
    c.vp[c.table[0, n - 2], 3, 5, 9] = 0.0
    want, tol = c.want()
    assert ((got - want).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (128, FP16)])
def test_a_chunk_beside_single_tokens(gpu, D, dtype):
    """A prompt's chunk of hundreds of rows and decode steps of other sequences in one call, some of them behind nothing."""
    lens = [700, 40, 0, 300, 5, 1000, 16, 63, 64, 65, 0, 128]
    Case(8, 2, D, 16, lens, [300] + [1] * 6 + [0] + [1] * 3 + [2], dtype, seed=39, mask="chain").check(gpu)


def test_as_many_sequences_as_there_can_be(gpu):
    rng = np.random.default_rng(42)
    lens, nodes = [int(x) for x in rng.integers(0, 40, 8192)], [0] * 8192
    for s in [0, 8191, *rng.choice(8192, 700, replace=False)]:
        nodes[s] = int(rng.integers(1, 4))
    lens[5000], nodes[5000] = 3000, 1
    Case(2, 1, 64, 16, lens, nodes, seed=42).check(gpu)
    Case(2, 1, 64, 16, lens, nodes[:5000] + [30] + nodes[5001:], seed=43).check(gpu)  # 60 rows: the kernel of many rows
