"""GPU: DraftVerify against a walk in 64 bits, its odd inputs, its distribution, streams and graphs."""

import math

import pytest
import torch

import iron_amd.operators as ops
from iron_amd import _lib
from tests import int4_reference as ref

pytestmark = pytest.mark.gpu


def tree(nodes, most, g):
    """Parents: each node's is one before it with fewer than `most` children."""
    up, count = [-1], [0] * nodes
    for i in range(1, nodes):
        free = [p for p in range(i) if count[p] < most]
        p = i - 1 if most == 1 else free[int(torch.randint(0, len(free), (1,), generator=g))]
        count[p] += 1
        up.append(p)
    return up


def make(V, counts, most, dtype, draft=True, greedy=0.0, seed=0, spare=0, near=0.5):
    """CPU arguments of a call: drafted tokens are drawn from the drafter's rows."""
    g = torch.Generator().manual_seed(seed)
    N = sum(counts) + spare
    d = torch.randn(N, V, generator=g) * 2
    d.scatter_(1, torch.randint(0, V, (N, min(8, V)), generator=g), 4.0 + 3 * torch.rand(N, min(8, V), generator=g))
    t = (d + near * torch.randn(N, V, generator=g)).to(dtype)
    d = d.to(dtype)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    parents = sum((tree(n, most, g) for n in counts if n), []) + [-1] * spare
    temps = torch.rand(len(counts), generator=g) + 0.3
    temps[torch.rand(len(counts), generator=g) < greedy] = 0
    tokens = torch.zeros(N, dtype=torch.int32)
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        for i in range(a, b):
            p = torch.softmax(d[a + max(parents[i], 0)].float() / max(float(temps[s]), 0.3), 0)
            tokens[i] = torch.multinomial(p, 1, generator=g)
    return dict(logits=t, draft=d if draft else None, tokens=tokens, parents=torch.tensor(parents, dtype=torch.int32),
                starts=torch.tensor(starts, dtype=torch.int32), temps=temps, accept=torch.rand(N, generator=g),
                sample=torch.rand(len(counts), generator=g))


def call(gpu, c, max_nodes, most, fn=None):
    N, V = c["logits"].shape
    S = len(c["temps"])
    if fn is None:
        fn = ops.DraftVerify(vocab=V, num_seqs=S, num_nodes=N, max_nodes=max_nodes, max_children=most,
                             draft=c["draft"] is not None, dtype=c["logits"].dtype).get_callable()
    args = [c[k].to(gpu) for k in ("logits", "draft", "tokens", "parents", "starts", "temps", "accept", "sample") if c[k] is not None]
    out = [torch.full((n,), 77, dtype=torch.int32, device=gpu) for n in (N, S + 1, S)]
    fn(*args, *out)
    return [o.tolist() for o in out]


def expect(c, most):
    rows, starts, nexts, margin = ref.verify(c["logits"], c["draft"], c["tokens"], c["parents"].tolist(), c["starts"].tolist(),
                                             c["temps"], c["accept"], c["sample"], most)
    # sums of 2^20 terms in 64 bits: 2^-53 each, exponentials 2^-50 of their argument
    assert margin > 1e-12, "the inputs put a decision on its border"
    return [rows, starts, nexts]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("V,counts,most", [
    (1, [3, 1], 1), (7, [1, 4, 0, 9], 2), (63, [5] * 6, 1), (4095, [4, 9, 2], 1), (4096, [12, 1, 7], 3), (4097, [30, 3], 4),
    (32001, [6, 2, 8], 1), (8193, [70, 0, 66], 5), (16384, [5], 1),
])
def test_walks(gpu, dtype, draft, V, counts, most):
    for seed in range(3):
        c = make(V, counts, most, dtype, draft, greedy=0.3, seed=seed, spare=seed)
        assert call(gpu, c, max(counts), most) == expect(c, most)


def test_large_vocabulary(gpu):
    for seed, draft in ((1, True), (2, False)):
        c = make(128256, [8, 5, 1], 2, torch.bfloat16, draft, seed=seed)
        assert call(gpu, c, 8, 2) == expect(c, 2)
    c = make(1 << 20, [3], 1, torch.float32, True, seed=5)
    assert call(gpu, c, 3, 1) == expect(c, 1)


def test_flat_rows_draw_the_right_token(gpu):
    """2^17 tokens of nearly the same probability, where a cumulative sum of fp32 terms draws neighbours."""
    S = 64
    c = make(131071, [1] * S, 1, torch.float32, False, seed=3)
    c["logits"] = c["logits"] * 1e-3
    assert call(gpu, c, 1, 1) == expect(c, 1)


def test_large_tree(gpu):
    """A chain of 1024 nodes that is accepted to its end, and a star."""
    c = make(50, [1024, 1024], 1, torch.float32, True, seed=1)
    c["logits"] = c["draft"].clone()  # p == q: everything is accepted
    c["parents"][1025:] = 0
    c["tokens"][1024:] = (c["logits"][1024].argmax() + 1) % 50
    assert call(gpu, c, 1024, 64) == expect(c, 64)
    assert call(gpu, c, 1024, 64)[1][1] == 1024


def test_children_past_the_bound_are_left_out(gpu):
    c = make(40, [30, 30], 29, torch.float32, False, seed=2)
    c["parents"][:] = 0
    c["accept"][:] = 0.9999
    for most in (1, 2, 7, 29):
        assert call(gpu, c, 30, most) == expect(c, most)


def test_same_token_twice(gpu):
    """Siblings with one token: with draft logits each is tried for itself, without the second has nothing left."""
    for draft in (True, False):
        c = make(12, [5, 5, 5, 5], 4, torch.float32, draft, seed=4)
        c["parents"] = torch.tensor([-1, 0, 0, 0, 0] * 4, dtype=torch.int32)
        c["tokens"] = torch.tensor([3, 5, 5, 2, 5] * 4, dtype=torch.int32)
        for seed in range(8):
            c["accept"] = torch.rand(20, generator=torch.Generator().manual_seed(seed))
            assert call(gpu, c, 5, 4) == expect(c, 4)


def test_no_probability(gpu):
    """-inf and NaN logits, rows of nothing else, infinite ones, tokens that are none, draws outside [0, 1)."""
    inf, nan = math.inf, math.nan
    for draft in (True, False):
        c = make(6, [3, 3, 3, 3, 3, 3, 3], 1, torch.float32, draft, seed=6)
        rows = torch.tensor([[0., -inf, 1, nan, -inf, 2], [-inf] * 6, [nan] * 6, [inf, 0, inf, 0, 0, 0], [1e38, -1e38, 0, 0, 0, 0]])
        for s in range(5):
            c["logits"][3 * s] = rows[s]
        c["tokens"][1], c["tokens"][4], c["tokens"][16], c["tokens"][19] = 1, 0, -1, 6
        c["sample"] = torch.tensor([0.0, 0.5, 0.5, 0.6, 1.0, nan, -1.0])
        c["accept"][7], c["accept"][10], c["accept"][13] = 1.0, nan, 2.0
        for temps in ([1.0] * 7, [0.0] * 7, [-1.0, nan, 1e-40, 1e-30, 1e30, inf, 0.5]):
            c["temps"] = torch.tensor(temps)
            assert call(gpu, c, 3, 1) == expect(c, 1)


def test_equal_rows_leave_nothing(gpu):
    """p == q and a child that was not drawn from q: nothing is left of p, so the token comes from p itself."""
    c = make(9, [2] * 32, 1, torch.float32, True, seed=7)
    c["logits"][:, 4] = -math.inf
    c["draft"] = c["logits"].clone()
    c["tokens"][:] = 4
    got = call(gpu, c, 2, 1)
    assert got == expect(c, 1) and got[1] == list(range(33)) and 4 not in got[2] and len(set(got[2])) > 3
    c = make(9, [4] * 32, 3, torch.float32, True, seed=7)  # and further children of the same node
    c["logits"][:, 4] = -math.inf
    c["draft"] = c["logits"].clone()
    c["tokens"][:] = 4
    c["tokens"][3::4] = 2
    c["parents"] = torch.tensor([-1, 0, 0, 0] * 32, dtype=torch.int32)
    assert call(gpu, c, 4, 3) == expect(c, 3)


def test_greedy_takes_the_first_of_equals(gpu):
    c = make(9000, [3] * 5, 1, torch.bfloat16, False, seed=8)
    c["temps"][:] = 0
    c["logits"][:] = c["logits"].clamp(max=3.0)
    c["tokens"][1] = int((c["logits"][0] == 3.0).nonzero()[0])
    got = call(gpu, c, 3, 1)
    assert got == expect(c, 1) and got[0][1] == 1


def test_odd_structures(gpu):
    """Parents that are no node before the child, a first node with a parent, trees that are cut, starts that do not fit."""
    c = make(30, [6, 6], 1, torch.float32, True, seed=9, spare=3)
    c["logits"] = c["draft"].clone()
    c["parents"][:6] = torch.tensor([4, 0, 5, 9, -7, 1])
    got = call(gpu, c, 6, 2)
    assert got == expect(c, 2) and got[0][:3] == [0, 1, 5]
    cut = {**c, "parents": c["parents"].clone()}
    cut["parents"][3:6] = cut["parents"][9:12] = 99  # out of reach
    assert call(gpu, c, 3, 1) == expect(cut, 1)
    wild = call(gpu, {**c, "starts": torch.tensor([-4, 400, 2], dtype=torch.int32)}, 6, 2)
    assert all(-1 <= r < 15 for r in wild[0]) and len(wild[2]) == 2


def test_many_sequences(gpu):
    S = 8192
    c = make(5, [2] * S, 1, torch.float32, True, seed=10)
    assert call(gpu, c, 2, 1) == expect(c, 1)


@pytest.mark.parametrize("draft,children", [(True, 1), (True, 3), (False, 2)])
def test_tokens_are_distributed_as_the_target(gpu, draft, children):
    """The first token behind the root, accepted or drawn, has the target's distribution whatever the drafter's: over
    8192 sequences with the same rows each frequency is within 5 standard deviations."""
    S, V = 8192, 6
    g = torch.Generator().manual_seed(11 + children)
    n = 1 + children
    p, q = torch.randn(V, generator=g), torch.randn(V, generator=g)
    c = dict(logits=p.repeat(S * n, 1), draft=q.repeat(S * n, 1) if draft else None, parents=torch.tensor(([-1] + [0] * children) * S, dtype=torch.int32),
             starts=torch.arange(0, S * n + 1, n, dtype=torch.int32), temps=torch.full((S,), 0.8), accept=torch.rand(S * n, generator=g), sample=torch.rand(S, generator=g))
    if draft:
        c["tokens"] = torch.multinomial(torch.softmax(q / 0.8, 0), S * n, True, generator=g).to(torch.int32)
    else:
        c["tokens"] = torch.tensor([0, 4, 1, 5][:n] * S, dtype=torch.int32)
    rows, starts, nexts = call(gpu, c, n, children)
    first = [nexts[s] if starts[s + 1] - starts[s] == 1 else int(c["tokens"][rows[starts[s] + 1]]) for s in range(S)]
    want = torch.softmax(p.double() / float(torch.tensor(0.8)), 0)
    for x in range(V):
        sigma = math.sqrt(float(want[x]) * (1 - float(want[x])) / S)
        assert abs(first.count(x) / S - float(want[x])) < 5 * sigma


def test_streams_and_graphs(gpu):
    """On a side stream, and captured twice: every replay takes the inputs as they are then, with eager calls between."""
    a, b = (make(5000, [6, 9, 4], 3, torch.bfloat16, True, seed=s) for s in (12, 13))
    N = len(a["tokens"])
    fn = ops.DraftVerify(vocab=5000, num_seqs=3, num_nodes=N, max_nodes=9, max_children=3).get_callable()
    names = ("logits", "draft", "tokens", "parents", "starts", "temps", "accept", "sample")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert call(gpu, a, 9, 3, fn) == expect(a, 3)
    graphs = []
    for c in (a, b):
        args = [c[k].to(gpu) for k in names]
        out = [torch.zeros(n, dtype=torch.int32, device=gpu) for n in (N, 4, 3)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn(*args, *out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fn(*args, *out)
        graphs.append((graph, args, out))
    for turn in range(3):
        for (graph, args, out), c in zip(graphs, (a, b)):
            c["accept"] = torch.rand(N, generator=torch.Generator().manual_seed(100 + turn))
            args[6].copy_(c["accept"])
            graph.replay()
            assert call(gpu, b, 9, 3, fn) == expect(b, 3)
            torch.cuda.synchronize()
            assert [o.tolist() for o in out] == expect(c, 3)


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0x7f81), (torch.float16, 0x7c01), (torch.float32, 0x7f800001)])
@pytest.mark.parametrize("draft", [True, False])
def test_signalling_nan(gpu, dtype, bits, draft):
    """NaN whose quiet bit is not set count as -inf too, wherever they stand: beside the largest logit, among many, in a
    row (or a part of one) without anything else."""
    whole = torch.int32 if dtype == torch.float32 else torch.int16
    for seed in range(4):
        c = make(3000, [4, 3, 5, 1, 2], 2, dtype, draft, seed=30 + seed)
        c["temps"] = torch.tensor([1.0, 0.03, 0.0, 0.03, 0.5])
        g = torch.Generator().manual_seed(seed)
        for name, shift in (("logits", 0), ("draft", 5)):
            if c[name] is None:
                continue
            raw = c[name].view(whole)
            for n in range(len(raw)):
                top = (int(c["logits"][n].float().nan_to_num(-1e30).argmax()) + shift) % 3000
                raw[n, torch.randint(0, 3000, (60,), generator=g)] = bits
                raw[n, [i for i in range(top // 8 * 8, min(top // 8 * 8 + 8, 3000)) if i > top]] = bits
                c[name][n, top] = 60.0  # far above the others at the smaller temperatures
        last = len(c["logits"]) - 2
        c["logits"][last - 1, 1:] = -math.inf  # one token, then nothing, in a part of the row
        c["logits"].view(whole)[last - 1, [1, 3, 1024, 2500]] = bits
        c["logits"].view(whole)[last] = bits  # nothing at all
        assert call(gpu, c, 5, 2) == expect(c, 2)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("fill", [0x00, 0xff, 0x3f, 0x80])
def test_what_the_workspace_held_does_not_matter(gpu, draft, fill):
    """The entry point on a workspace full of zeros, NaN, ordinary and negative numbers: nothing is read that the call has
    not written. The last nodes of the walk have no, one and more untried children, within and past max_children."""
    for seed in range(4):
        c = make(700, [9, 1, 12, 0, 70], 4, torch.float32, draft, greedy=0.2, seed=60 + seed, spare=2)
        N, V = c["logits"].shape
        for most in (1, 3, 4):
            args = [c[k].to(gpu) if c[k] is not None else None for k in ("logits", "draft", "tokens", "parents", "starts", "temps", "accept", "sample")]
            out = [torch.full((n,), 77, dtype=torch.int32, device=gpu) for n in (N, 6, 5)]
            need = _lib.query("iron_draft_verify_workspace_bytes", V, 5, N, 70, most, int(draft))
            ws = torch.full((need,), fill, dtype=torch.uint8, device=gpu)
            _lib.call("iron_draft_verify", *[_lib.ptr(t) for t in args + out], 2, V, 5, N, 70, most, ws.data_ptr(), need,
                      torch.cuda.current_stream().cuda_stream)
            assert [o.tolist() for o in out] == expect(c, most)
