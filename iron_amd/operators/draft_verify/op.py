"""DraftVerify: which drafted tokens the target accepts, for a batch of sequences
(new operator; the reference samples one token of one sequence on the CPU,
iron/applications/llama_3.2_1b/llama_inference_harness.py:146-169). It stands
between TreeAttention, whose rows end in the logits, and PagedAppend, whose
arguments ``rows`` and ``row_starts`` it makes.

Rows ``node_starts[s]`` .. ``node_starts[s + 1] - 1`` are the nodes of sequence s, as
in TreeAttention: the first is the sequence's last token (always accepted), each
other one a token (``tokens``) drafted behind its parent (``parents``: the index of
a node before it within the tree). With p and q the softmax of a node's row of
logits and draft_logits, divided by the sequence's temperature: at an accepted node,
its children (``max_children`` at most, in row order; further ones are left out) are
tried in turn. A child with token x and accept_draws u is accepted if
u q(x) < p(x); else p becomes max(p - q, 0), scaled to a sum of 1. If none is
accepted, the next token is the first one whose cumulative probability passes
sample_draws: together the tokens are distributed as if drawn from p one by one,
where the children were drawn from q independently. ``draft=False``: no draft_logits;
the children were not drawn (a lookup, the likeliest tokens), q is 1 at x.
A temperature of 0 (or below, or NaN) takes the likeliest token, the lowest of equal ones.

Logits of -inf (a filter's, or padding) and NaN have no probability, +inf counts as the
largest fp32. A row without any gives next token -1; so does an empty tree. A token
outside the vocabulary is not accepted, one without probability neither accepted nor
drawn. Where max(p - q, 0) is zero everywhere, the next token is drawn from p. All of
it is computed in 64 bits, the exponentials to 2^-46 (and 2^-52 of their argument).

Arg spec: logits (num_nodes, vocab), draft_logits (num_nodes, vocab; only with
``draft``; rows of nodes without children are not read), tokens, parents (num_nodes,),
node_starts (num_seqs + 1,) int32, temperatures (num_seqs,), accept_draws
(num_nodes,), sample_draws (num_seqs,) fp32, uniform in [0, 1); out: rows
(num_nodes,) int32, the accepted rows of all sequences from the first on, then -1;
row_starts (num_seqs + 1,), where each sequence's begin; next_tokens (num_seqs,).
bf16, fp16 or fp32 logits (``dtype``). The results are buffers of their own: one that
overlaps another argument is refused. Kernel: iron_draft_verify.
"""

from dataclasses import dataclass, field
from typing import ClassVar

import torch

from ... import _lib
from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@dataclass
class DraftVerify(PagedOperator):
    vocab: int
    num_seqs: int
    num_nodes: int
    max_nodes: int
    max_children: int = 1
    draft: bool = True
    dtype: object = field(default=torch.bfloat16, repr=False)
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("vocab", "num_seqs", "num_nodes", "draft", "dtype")

    def __post_init__(self):
        self._check_counts(vocab=1 << 20, num_seqs=8192, num_nodes=1 << 20, max_nodes=1024, max_children=64)
        if self.num_nodes * -(-(self.vocab + 7) // 4096) >= 1 << 23:
            raise ValueError(f"num_nodes={self.num_nodes}, vocab={self.vocab}: num_nodes * ceil((vocab + 7) / 4096) must be below 2**23")
        if self.dtype not in _DTYPES:
            raise ValueError(f"dtype must be torch.bfloat16, torch.float16 or torch.float32, got {self.dtype!r}")
        PagedOperator.__init__(self, context=self.context)

    def workspace_bytes(self) -> int:
        return _lib.workspace_bytes("iron_draft_verify_workspace_bytes", self.vocab, self.num_seqs, self.num_nodes, self.max_nodes,
                                    self.max_children, int(bool(self.draft)))

    def get_arg_spec(self):
        rows, seqs = (self.num_nodes,), (self.num_seqs,)
        return [
            *[AIERuntimeArgSpec("in", (self.num_nodes, self.vocab), dtype=self.dtype) for _ in range(2 if self.draft else 1)],
            AIERuntimeArgSpec("in", rows, dtype=INT32),
            AIERuntimeArgSpec("in", rows, dtype=INT32),
            AIERuntimeArgSpec("in", (self.num_seqs + 1,), dtype=INT32),
            AIERuntimeArgSpec("in", seqs, dtype=torch.float32),
            AIERuntimeArgSpec("in", rows, dtype=torch.float32),
            AIERuntimeArgSpec("in", seqs, dtype=torch.float32),
            AIERuntimeArgSpec("out", rows, dtype=INT32),
            AIERuntimeArgSpec("out", (self.num_seqs + 1,), dtype=INT32),
            AIERuntimeArgSpec("out", seqs, dtype=INT32),
        ]

    def _launch(self, logits, *tensors, stream):
        draft, rest = (tensors[0], tensors[1:]) if self.draft else (None, tensors)
        self._call("iron_draft_verify", (logits, draft, *rest),
                   (_DTYPES.index(self.dtype), self.vocab, self.num_seqs, self.num_nodes, self.max_nodes, self.max_children), stream)
