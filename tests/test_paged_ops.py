"""CPU: what the paged cache's operators refuse before anything runs, their argument specs and the tree masks."""

import pytest
import torch

import iron_amd.operators as ops
from iron_amd import _lib

POOL = dict(num_pages=8, page_size=16, num_seqs=2, max_pages=4)
DATA = dict(num_layers=2, num_kv_heads=2, head_dim=64, **POOL)
TREE = dict(num_heads=4, num_kv_heads=2, head_dim=64, num_nodes=6, max_nodes=5, **POOL)


@pytest.mark.parametrize("cls,fields,bad,match", [
    ("TreeAttention", TREE, dict(head_dim=96), "head_dim 64 and 128"),
    ("TreeAttention", TREE, dict(num_heads=5), "multiple of num_kv_heads"),
    ("TreeAttention", TREE, dict(dtype=torch.float32), "bfloat16 or torch.float16"),
    ("TreeAttention", TREE, dict(max_nodes=1025), "max_nodes"),
    ("TreeAttention", TREE, dict(max_nodes=0), "max_nodes"),
    ("TreeAttention", TREE, dict(num_nodes=0), "num_nodes"),
    ("TreeAttention", TREE, dict(page_size=48), "power of two"),
    ("TreeAttention", TREE, dict(page_size=8), "power of two"),
    ("TreeAttention", TREE, dict(num_seqs=8193), "num_seqs"),
    ("TreeAttention", TREE, dict(max_pages=1 << 27), "2\\*\\*31"),
    ("TreeAttention", TREE, dict(scale=0.0), "scale"),
    ("TreeAttention", TREE, dict(scale=float("nan")), "scale"), ("TreeAttention", TREE, dict(scale=1e31), "scale"),
    ("TreeAttention", TREE, dict(num_pages=2.0), "must be an int"),
    ("PageCompact", DATA, dict(num_seqs=8192, max_pages=1 << 20), "2\\*\\*33"),
    ("PagedAppend", dict(num_nodes=6, num_rows=4, **DATA), dict(num_rows=0), "num_rows"),
    ("PagedAppend", dict(num_nodes=6, num_rows=4, **DATA), dict(head_dim=7), "multiple of 16"),
    ("PagedAppend", dict(num_nodes=6, num_rows=4, **DATA), dict(dtype="bf16"), "torch dtype"),
    ("PageFork", dict(num_forks=2, **DATA), dict(num_forks=8193), "num_forks"),
    ("PageFork", dict(num_forks=2, **DATA), dict(num_forks=8192, max_pages=1 << 19, page_size=16), "num_forks \\* max_pages"),
    ("PageCompact", DATA, dict(num_layers=0), "num_layers"),
    ("PageFree", dict(num_slots=1, **POOL), dict(num_slots=0), "num_slots"),
])
def test_fields_are_checked(cls, fields, bad, match):
    getattr(ops, cls)(**fields)
    with pytest.raises(ValueError, match=match):
        getattr(ops, cls)(**{**fields, **bad})


def test_arg_specs():
    spec = ops.TreeAttention(**TREE).get_arg_spec()
    assert [s.shape for s in spec] == [(6, 4, 64), (6, 2, 64), (6, 2, 64), (8, 2, 16, 64), (8, 2, 16, 64), (2, 4), (2,),
                                       (3,), (6, 1), (6, 4, 64)]
    assert spec[-1].direction == "out" and all(s.dtype == torch.int32 for s in spec[5:9])
    spec = ops.PagedAppend(num_nodes=6, num_rows=4, **DATA).get_arg_spec()
    assert [s.shape for s in spec] == [(2, 6, 2, 64)] * 2 + [(4,), (3,)] + [(2, 8, 2, 16, 64)] * 2 + [(2, 4), (2,), (8,), (2,)]
    assert [s.direction for s in spec] == ["in"] * 4 + ["inout"] * 5 + ["out"]
    assert len(ops.PageFork(num_forks=3, **DATA).get_arg_spec()) == 7
    assert len(ops.PageCompact(**DATA).get_arg_spec()) == 6
    assert len(ops.PageFree(num_slots=3, **POOL).get_arg_spec()) == 5


def test_masks():
    op = ops.TreeAttention(**{**TREE, "num_nodes": 70, "max_nodes": 40, "num_seqs": 2})
    starts = torch.tensor([0, 40, 69])
    parents = torch.tensor([i - 1 for i in range(40)] + [(i - 1) // 2 if i else -1 for i in range(29)] + [-1])
    words = op.mask_of_parents(parents, starts)
    assert words.shape == (70, 2) and words.dtype == torch.int32
    sees = lambda i, j: bool(words[i, j // 32].item() >> (j % 32) & 1)
    for i in range(40):  # a chain: all before it
        assert [sees(i, j) for j in range(40)] == [j <= i for j in range(40)]
    assert [j for j in range(29) if sees(40 + 22, j)] == [0, 1, 4, 10, 22]  # the way up a binary tree
    assert not words[69].any()  # a row of no tree
    with pytest.raises(ValueError, match="before its child"):
        op.mask_of_parents(torch.full((70,), 5), starts)
    with pytest.raises(ValueError, match="does not fit"):
        op.mask_of_parents(parents, torch.tensor([0, 41, 69]))
    with pytest.raises(ValueError, match="entries"):
        op.mask_of_parents(parents[:5], starts)
    with pytest.raises(ValueError, match="bool"):
        op.pack_mask(torch.zeros(70, 40))


def test_callable_refuses_wrong_tensors():
    op = ops.PageFree(num_slots=1, **POOL)
    with pytest.raises(ValueError, match="takes 5 arguments"):
        op.validate_args([torch.zeros(1)])
    with pytest.raises(ValueError, match="must live on the GPU"):
        op.validate_args([torch.zeros(s.shape, dtype=s.dtype) for s in op.get_arg_spec()])


P = 1 << 20  # a 16-byte-aligned stand-in address: nothing is launched


def _tree(q=P, out=2 * P, dtype=0, H=4, Hkv=2, D=64, pages=8, ps=16, S=2, mp=4, N=6, T=5, scale=0.125, ws=P, size=1 << 30, lens=P, vp=P):
    _lib.call("iron_tree_attention", q, P, P, P, vp, P, lens, P, P, out, dtype, H, Hkv, D, pages, ps, S, mp, N, T, scale, ws,
              size, None)


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "null pointer"), (dict(q=P + 2), "16-byte"), (dict(lens=P + 2), "4-byte"), (dict(out=P), "one of the inputs"),
    (dict(vp=2 * P), "one of the inputs"),
    (dict(dtype=2), "dtype=2"), (dict(H=3), "multiple"), (dict(D=32), "64 or 128"), (dict(pages=0), "num_pages=0"),
    (dict(ps=24), "power of two"), (dict(S=0), "num_seqs"), (dict(mp=0), "max_pages"), (dict(N=0), "num_nodes"),
    (dict(T=2000), "max_nodes"), (dict(scale=-1.0), "scale"), (dict(scale=1e31), "scale"), (dict(ws=None), "workspace"), (dict(size=0), "workspace of 0 bytes"),
])
def test_tree_attention_entry_point_refuses(kw, match):
    with pytest.raises(_lib.IronHipError, match=match):
        _tree(**kw)


def _append(k=P, pages=8, ps=16, S=2, mp=4, L=2, Hkv=2, row=128, N=6, M=4, refs=P, kp=P, vp=2 * P, size=1 << 30):
    _lib.call("iron_paged_append", k, P, P, P, kp, vp, P, P, refs, P, L, Hkv, row, pages, ps, S, mp, N, M, P, size, None)


def _fork(forks=P, n=2, mp=4, size=1 << 30, S=2):
    _lib.call("iron_page_fork", forks, P, 2 * P, P, P, P, P, 2, 2, 128, 8, 16, S, mp, n, 1, P, size, None)


def _compact(size=1 << 30, L=2, moved=P, S=2, mp=4):
    _lib.call("iron_page_compact", P, 2 * P, P, P, P, moved, L, 2, 128, 8, 16, S, mp, P, size, None)


def _free(slots=P, n=1, ps=16):
    _lib.call("iron_page_free", slots, P, P, P, P, 8, ps, 2, 4, n, None)


@pytest.mark.parametrize("fn,kw,match", [
    (_append, dict(k=None), "null pointer"), (_append, dict(k=P + 8), "16-byte"), (_append, dict(refs=P + 4), "page_refs must be 16-byte"),
    (_append, dict(kp=P, vp=P), "same buffer"), (_append, dict(row=100), "rows of 100 bytes"), (_append, dict(N=0), "num_nodes"),
    (_append, dict(M=(1 << 20) + 1), "num_rows"), (_append, dict(size=16), "workspace of 16"), (_append, dict(L=0), "num_layers"),
    (_append, dict(ps=17), "power of two"), (_append, dict(mp=1 << 28), "2\\^31"), (_append, dict(S=9000), "num_seqs"),
    (_fork, dict(forks=None), "forks"), (_fork, dict(n=0), "num_forks"), (_fork, dict(n=8192, mp=1 << 26), "exceeds"),
    (_fork, dict(size=0), "workspace"), (_compact, dict(size=0), "workspace"), (_compact, dict(L=5000), "num_layers"), (_compact, dict(S=8192, mp=1 << 20), "2\\^33"),
    (_compact, dict(moved=None), "null pointer"), (_free, dict(slots=P + 1), "slots"), (_free, dict(n=9000), "num_slots"),
    (_free, dict(ps=0), "power of two"),
])
def test_page_entry_points_refuse(fn, kw, match):
    with pytest.raises(_lib.IronHipError, match=match):
        fn(**kw)


def test_workspace_queries():
    q = _lib.query
    assert q("iron_tree_attention_workspace_bytes", 4, 2, 64, 2, 6, 5, 4, 16) > 0
    assert q("iron_tree_attention_workspace_bytes", 4, 3, 64, 2, 6, 5, 4, 16) == -1
    assert q("iron_paged_append_workspace_bytes", 0, 4, 16) == -1
    assert q("iron_page_fork_workspace_bytes", 2, 2, 4, 8, 1) < q("iron_page_fork_workspace_bytes", 2, 2, 4, 8, 0)
    assert q("iron_page_compact_workspace_bytes", 0) == -1
