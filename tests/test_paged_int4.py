"""CPU: what the operators of a 4-bit cache and the verification of drafted tokens refuse before anything runs, their
argument specs, and the tests' own quantizing."""

import pytest
import torch

import iron_amd.operators as ops
from iron_amd import _lib
from iron_amd.common.paging import int4_row_bytes
from tests import int4_reference as ref

POOL = dict(num_pages=8, page_size=16, num_seqs=2, max_pages=4)
DATA = dict(num_layers=2, num_kv_heads=2, head_dim=64, **POOL)
TREE = dict(num_heads=4, num_kv_heads=2, head_dim=64, num_nodes=6, max_nodes=5, **POOL)
APPEND = dict(num_nodes=6, num_rows=4, **DATA)
VERIFY = dict(vocab=100, num_seqs=2, num_nodes=6, max_nodes=5)


@pytest.mark.parametrize("cls,fields,bad,match", [
    ("TreeAttentionInt4", TREE, dict(head_dim=96), "head_dim 64 and 128"),
    ("TreeAttentionInt4", TREE, dict(dtype=torch.uint8), "bfloat16 or torch.float16"),
    ("TreeAttentionInt4", TREE, dict(num_heads=5), "multiple of num_kv_heads"),
    ("TreeAttentionInt4", TREE, dict(max_nodes=1025), "max_nodes"),
    ("TreeAttentionInt4", TREE, dict(page_size=48), "power of two"),
    ("TreeAttentionInt4", TREE, dict(scale=-1.0), "scale"),
    ("PagedAppendInt4", APPEND, dict(head_dim=32), "head_dim 64 and 128"),
    ("PagedAppendInt4", APPEND, dict(dtype=torch.float32), "bfloat16 or torch.float16"),
    ("PagedAppendInt4", APPEND, dict(num_rows=0), "num_rows"),
    ("PagedAppendInt4", APPEND, dict(num_layers=1025), "num_layers"),
    ("PagedGatherInt4", dict(num_rows=4, **DATA), dict(head_dim=256), "head_dim 64 and 128"),
    ("PagedGatherInt4", dict(num_rows=4, **DATA), dict(num_rows=(1 << 20) + 1), "num_rows"),
    ("PagedGatherInt4", dict(num_rows=4, **DATA), dict(dtype=torch.uint8), "bfloat16 or torch.float16"),
    ("PagedGatherInt4", dict(num_rows=4, **DATA), dict(num_seqs=0), "num_seqs"),
    ("DraftVerify", VERIFY, dict(vocab=0), "vocab"),
    ("DraftVerify", VERIFY, dict(vocab=(1 << 20) + 1), "vocab"),
    ("DraftVerify", VERIFY, dict(num_nodes=1 << 20, vocab=1 << 20), "2\\*\\*23"),
    ("DraftVerify", VERIFY, dict(max_nodes=1025), "max_nodes"),
    ("DraftVerify", VERIFY, dict(max_children=65), "max_children"),
    ("DraftVerify", VERIFY, dict(max_children=0), "max_children"),
    ("DraftVerify", VERIFY, dict(num_seqs=8193), "num_seqs"),
    ("DraftVerify", VERIFY, dict(num_seqs=2.0), "must be an int"),
    ("DraftVerify", VERIFY, dict(dtype=torch.float64), "float32"),
])
def test_fields_are_checked(cls, fields, bad, match):
    getattr(ops, cls)(**fields)
    with pytest.raises(ValueError, match=match):
        getattr(ops, cls)(**{**fields, **bad})


def test_arg_specs():
    assert int4_row_bytes(64) == 48 and int4_row_bytes(128) == 80
    spec = ops.TreeAttentionInt4(**TREE).get_arg_spec()
    assert [s.shape for s in spec] == [(6, 4, 64), (6, 2, 64), (6, 2, 64), (8, 2, 16, 48), (8, 2, 16, 48), (2, 4), (2,), (3,), (6, 1), (6, 4, 64)]
    assert [s.dtype for s in spec[3:5]] == [torch.uint8] * 2 and spec[0].dtype == torch.bfloat16
    spec = ops.PagedAppendInt4(**{**APPEND, "head_dim": 128}).get_arg_spec()
    assert [s.shape for s in spec] == [(2, 6, 2, 128)] * 2 + [(4,), (3,)] + [(2, 8, 2, 16, 80)] * 2 + [(2, 4), (2,), (8,), (2,)]
    assert [s.direction for s in spec] == ["in"] * 4 + ["inout"] * 5 + ["out"]
    spec = ops.PagedGatherInt4(num_rows=4, **DATA).get_arg_spec()
    assert [s.shape for s in spec] == [(2,), (3,)] + [(2, 8, 2, 16, 48)] * 2 + [(2, 4), (2,)] + [(2, 4, 2, 64)] * 2
    assert [s.direction for s in spec] == ["in"] * 6 + ["out"] * 2
    assert len(ops.DraftVerify(**VERIFY).get_arg_spec()) == 11
    spec = ops.DraftVerify(draft=False, dtype=torch.float32, **VERIFY).get_arg_spec()
    assert [s.shape for s in spec] == [(6, 100), (6,), (6,), (3,), (2,), (6,), (2,), (6,), (3,), (2,)]
    # the pages of such a cache are the page operators' with rows of bytes
    assert ops.PageFork(num_forks=1, dtype=torch.uint8, **{**DATA, "head_dim": 48}).get_arg_spec()[1].shape == (2, 8, 2, 16, 48)


def test_cpu_tensors_are_refused():
    op = ops.DraftVerify(**VERIFY)
    args = [torch.zeros(s.shape, dtype=s.dtype) for s in op.get_arg_spec()]
    with pytest.raises(ValueError, match="must live on the GPU"):
        op.validate_args(args)


P = 4096  # an address that is never read: the entry points refuse before a launch


def tree(q=P, kp=P, out=2 * P, lens=P, dtype=0, H=4, Hkv=2, D=64, pages=8, ps=16, S=2, mp=4, N=6, T=5, scale=1.0, ws=P, size=1 << 30):
    _lib.call("iron_tree_attention_int4", q, P, P, kp, P, P, lens, P, P, out, dtype, H, Hkv, D, pages, ps, S, mp, N, T, scale, ws, size, None)


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "null pointer"), (dict(kp=P + 8), "16-byte aligned"), (dict(lens=P + 2), "4-byte aligned"), (dict(out=P), "out is one of the inputs"),
    (dict(D=96), "head_dim must be 64 or 128"), (dict(H=5), "multiple of n_kv_heads"), (dict(dtype=2), "neither 0"), (dict(ps=24), "power of two"),
    (dict(T=0), "max_nodes"), (dict(scale=0.0), "scale"), (dict(ws=None), "workspace must be given"), (dict(size=16), "needed"), (dict(pages=0), "num_pages"),
])
def test_tree_attention_entry_point_refuses(kw, match):
    with pytest.raises(_lib.IronHipError, match=match):
        tree(**kw)


def append(k=P, rows=P, kp=P, vp=2 * P, refs=P, dtype=0, L=2, Hkv=2, D=64, pages=8, ps=16, S=2, mp=4, N=6, M=4, ws=P, size=1 << 30):
    _lib.call("iron_paged_append_int4", k, P, rows, P, kp, vp, P, P, refs, P, dtype, L, Hkv, D, pages, ps, S, mp, N, M, ws, size, None)


@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "null pointer"), (dict(rows=P + 1), "4-byte aligned"), (dict(kp=2 * P), "same buffer"), (dict(vp=P + 4), "16-byte aligned"),
    (dict(refs=P + 4), "16-byte aligned"), (dict(dtype=-1), "neither 0"), (dict(D=80), "head_dim"), (dict(L=0), "num_layers"), (dict(M=0), "num_rows"),
    (dict(N=0), "num_nodes"), (dict(S=9000), "num_seqs"), (dict(ws=P + 8), "workspace must be given"), (dict(size=4), "needed"),
])
def test_append_entry_point_refuses(kw, match):
    with pytest.raises(_lib.IronHipError, match=match):
        append(**kw)


def gather(begins=P, starts=P, kp=P, vp=2 * P, table=P, ko=3 * P, vo=4 * P, dtype=0, L=2, Hkv=2, D=64, pages=8, ps=16, S=2, mp=4, M=4):
    _lib.call("iron_paged_gather_int4", begins, starts, kp, vp, table, P, ko, vo, dtype, L, Hkv, D, pages, ps, S, mp, M, None)


@pytest.mark.parametrize("kw,match", [
    (dict(begins=None), "int32 arrays must be given"), (dict(starts=P + 2), "int32 arrays must be given"), (dict(kp=None), "null pointer"), (dict(table=None), "null pointer"),
    (dict(ko=None), "k_out and v_out must be given"), (dict(vo=P + 8), "k_out and v_out must be given"), (dict(vo=3 * P), "same buffer"), (dict(ko=P), "one of the inputs"),
    (dict(dtype=3), "neither 0"), (dict(D=63), "head_dim"), (dict(ps=8), "power of two"), (dict(M=0), "num_rows"), (dict(pages=0), "num_pages"), (dict(mp=1 << 27), "max_pages"),
])
def test_gather_entry_point_refuses(kw, match):
    with pytest.raises(_lib.IronHipError, match=match):
        gather(**kw)


def verify(logits=P, draft=P, tokens=P, nexts=P, dtype=0, V=100, S=2, N=6, T=5, K=2, ws=P, size=1 << 30):
    _lib.call("iron_draft_verify", logits, draft, tokens, P, P, P, P, P, P, P, nexts, dtype, V, S, N, T, K, ws, size, None)


@pytest.mark.parametrize("kw,match", [
    (dict(logits=None), "logits must be given"), (dict(draft=P + 8), "16-byte aligned"), (dict(tokens=None), "must be given"), (dict(nexts=P + 1), "4-byte aligned"),
    (dict(dtype=3), "dtype"), (dict(V=0), "vocab"), (dict(V=(1 << 20) + 1), "vocab"), (dict(S=0), "num_seqs"), (dict(N=0), "num_nodes"), (dict(T=1025), "max_nodes"),
    (dict(K=65), "max_children"), (dict(N=1 << 20, V=1 << 20), "2\\^23"), (dict(ws=None), "workspace must be given"), (dict(size=64), "needed"),
])
def test_verify_entry_point_refuses(kw, match):
    with pytest.raises(_lib.IronHipError, match=match):
        verify(**kw)


def test_workspace_queries():
    q = _lib.query
    assert q("iron_tree_attention_int4_workspace_bytes", 4, 2, 64, 2, 6, 5, 4, 16) > 0
    assert q("iron_tree_attention_int4_workspace_bytes", 4, 3, 64, 2, 6, 5, 4, 16) == -1
    small, drafted, wide = (q("iron_draft_verify_workspace_bytes", 100, 2, 6, 5, k, d) for k, d in ((1, 0), (1, 1), (3, 1)))
    assert 0 < small < drafted < wide
    assert q("iron_draft_verify_workspace_bytes", 0, 2, 6, 5, 1, 1) == -1


def test_the_reference_rounds_to_the_nearest():
    """Of the tests' own quantizing: every value within half a step (and b's rounding) of its code's, packing loses nothing."""
    g = torch.Generator().manual_seed(0)
    for D in (64, 128):
        x = (torch.randn(200, D, generator=g) * torch.logspace(-3, 3, 200)[:, None]).to(torch.bfloat16)
        x[5] = 1.5
        code, s, b = ref.quantize(x)
        got = ref.values(ref.pack(code, s, b), D)
        each = x.double().reshape(200, 4, -1)
        lo = each.amin(-1)
        # half a step, what the last code may lack of the range (15 s, half a step of fp16 each), b's rounding
        bound = s.double() / 2 + 15 * s.double() * 2.0 ** -11 + (lo - 16 * s.double()).abs() * 2.0 ** -11 + 2.0 ** -24
        assert bool(((got.reshape(each.shape) - each).abs() <= bound[..., None]).all())
        assert bool((got[5] == 1.5).all())


# bytes of each buffer of a call of 6 nodes and 100 bf16 logits
SIZES = dict(logits=1200, draft_logits=1200, tokens=24, parents=24, node_starts=12, temperatures=8, accept_draws=24, sample_draws=8, rows=24, row_starts=12,
             next_tokens=8, workspace=0)
PLACES = {name: (1 + i) << 24 for i, name in enumerate(SIZES)}


@pytest.mark.parametrize("other", list(SIZES))
@pytest.mark.parametrize("out", ["rows", "row_starts", "next_tokens", "workspace"])
def test_verify_refuses_results_over_other_buffers(out, other):
    """The last launch reads trees, numbers, logits and the workspace while other workgroups of it write the results."""
    sizes = {**SIZES, "workspace": _lib.query("iron_draft_verify_workspace_bytes", 100, 2, 6, 5, 2, 1)}
    first, last = PLACES[other], PLACES[other] + (sizes[other] - 4) // 16 * 16
    before = first - (sizes[out] - 4) // 16 * 16  # its last bytes lie there
    for at in {first, last, before}:
        if out != other:
            where = {**PLACES, out: at}
            with pytest.raises(_lib.IronHipError, match="overlap"):
                _lib.call("iron_draft_verify", *[where[k] for k in SIZES if k != "workspace"], 0, 100, 2, 6, 5, 2, where["workspace"], sizes["workspace"], None)


@pytest.mark.parametrize("vocab,nodes", [(100, 6), (128256, 208)])
def test_verify_workspace_holds_sums_behind_the_first_child_only(vocab, nodes):
    """What is left after j children, j = 1 .. max_children - 1: a number to a row and a sum to each 1024 tokens of it."""
    subs = (vocab + 7 + 4095) // 4096 * 4
    sizes = [_lib.query("iron_draft_verify_workspace_bytes", vocab, 2, nodes, 5, k, 1) - 2 * k * (4 + 8) for k in (2, 4, 6)]
    assert sizes[1] - sizes[0] == sizes[2] - sizes[1] == 2 * nodes * (8 + 8 * subs)
    two, one = (_lib.query("iron_draft_verify_workspace_bytes", vocab, 2, nodes, 5, k, 1) for k in (2, 1))
    assert two - one == nodes * (8 + 8 * subs) + 2 * 8  # a sequence's tokens tried, 4 bytes each, fill up to 16
