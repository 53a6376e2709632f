"""TreeAttention: attention of drafted trees over a paged KV cache, for a batch
of sequences (new operator; the reference decodes one token of one sequence
against a dense cache, iron/applications/llama_3.2_1b/llama_npu.py:486-523).

Rows ``node_starts[s]`` .. ``node_starts[s + 1] - 1`` of q, k_new and v_new are
the nodes of sequence s: tokens that a drafter proposed, every node with its own
context. Node i sees all cached positions of its sequence and the nodes of its
own tree whose bit is set in its row of ``tree_mask`` (``pack_mask`` and
``mask_of_parents`` make it). One node that sees itself is an ordinary decode
step; a chain is a chunk of a prompt. The cache is only read: PagedAppend adds
the rows that were accepted.

Arg spec: q (num_nodes, H, D), k_new and v_new (num_nodes, Hkv, D), one layer's
k_pages and v_pages (num_pages, Hkv, page_size, D), page_table (num_seqs,
max_pages), seq_lens (num_seqs,), node_starts (num_seqs + 1,), tree_mask
(num_nodes, ceil(max_nodes / 32)) int32, out (num_nodes, H, D). q and k_new come
rotated (RoPE with one angle row per node). Head h reads KV head
h // (H / Hkv). bf16 or fp16 (``dtype``), D 64 or 128.

A row that sees nothing gets zeros; rows of out behind the last tree are left
as they were. What a node does not see does not reach its row, whatever it
holds; a key whose score is -inf counts as one that it does not see. Scores,
softmax and sums are fp32; the weights enter the product with V with 16 bits, or rounded
to ``dtype`` (as in MHA) where a KV head has more than 32 rows, max_nodes times
H / Hkv. That rule goes by max_nodes: a sequence of one node in a call with longer
trees is rounded as they are; in a call of its own it keeps the 16 bits. fp16
weights are kept to 2^-30 of a row's largest. Kernel: iron_tree_attention.
"""

import math
from dataclasses import dataclass, field
from typing import ClassVar

import torch

from ... import _lib
from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator


@dataclass
class TreeAttention(PagedOperator):
    num_heads: int
    num_kv_heads: int
    head_dim: int
    num_pages: int
    page_size: int
    num_seqs: int
    max_pages: int
    num_nodes: int
    max_nodes: int
    dtype: object = field(default=torch.bfloat16, repr=False)
    scale: float | None = field(default=None, repr=False)
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("num_heads", "num_kv_heads", "head_dim", "num_pages", "page_size", "num_seqs",
                                     "max_pages", "num_nodes", "max_nodes", "dtype")

    def __post_init__(self):
        self._check_counts(num_heads=1024, num_kv_heads=1024, num_nodes=1 << 20, max_nodes=1024)
        self._check_pool()
        if self.head_dim not in (64, 128):
            raise ValueError(f"Only head_dim 64 and 128 are supported, got {self.head_dim}")
        if self.num_heads % self.num_kv_heads:
            raise ValueError(f"num_heads ({self.num_heads}) must be a multiple of num_kv_heads ({self.num_kv_heads})")
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float16, got {self.dtype!r}")
        if self.scale is None:
            self.scale = 1.0 / math.sqrt(self.head_dim)
        if not 0 < self.scale <= 1e30:
            raise ValueError(f"scale must be positive and at most 1e30, got {self.scale}")
        PagedOperator.__init__(self, context=self.context)

    @property
    def mask_words(self) -> int:
        return (self.max_nodes + 31) // 32

    def workspace_bytes(self) -> int:
        return _lib.workspace_bytes("iron_tree_attention_workspace_bytes", self.num_heads, self.num_kv_heads, self.head_dim,
                                    self.num_seqs, self.num_nodes, self.max_nodes, self.max_pages, self.page_size)

    def get_arg_spec(self):
        new = (self.num_nodes, self.num_kv_heads, self.head_dim)
        pages = (self.num_pages, self.num_kv_heads, self.page_size, self.head_dim)
        rows = (self.num_nodes, self.num_heads, self.head_dim)
        return [
            AIERuntimeArgSpec("in", rows, dtype=self.dtype),
            AIERuntimeArgSpec("in", new, dtype=self.dtype),
            AIERuntimeArgSpec("in", new, dtype=self.dtype),
            AIERuntimeArgSpec("in", pages, dtype=self.dtype),
            AIERuntimeArgSpec("in", pages, dtype=self.dtype),
            AIERuntimeArgSpec("in", (self.num_seqs, self.max_pages), dtype=INT32),
            AIERuntimeArgSpec("in", (self.num_seqs,), dtype=INT32),
            AIERuntimeArgSpec("in", (self.num_seqs + 1,), dtype=INT32),
            AIERuntimeArgSpec("in", (self.num_nodes, self.mask_words), dtype=INT32),
            AIERuntimeArgSpec("out", rows, dtype=self.dtype),
        ]

    def _launch(self, *tensors, stream):
        self._call("iron_tree_attention", tensors,
                   (int(self.dtype == torch.float16), self.num_heads, self.num_kv_heads, self.head_dim,
                    self.num_pages, self.page_size, self.num_seqs, self.max_pages, self.num_nodes, self.max_nodes,
                    float(self.scale)), stream)

    def pack_mask(self, sees: torch.Tensor) -> torch.Tensor:
        """tree_mask from a boolean (num_nodes, max_nodes) tensor on any device:
        ``sees[i, j]`` whether row i sees node j of its own tree."""
        if sees.dtype != torch.bool or sees.shape != (self.num_nodes, self.max_nodes):
            raise ValueError(f"sees must be a bool tensor of shape {(self.num_nodes, self.max_nodes)}, got "
                             f"{sees.dtype} {tuple(sees.shape)}")
        words = self.mask_words
        bits = torch.nn.functional.pad(sees, (0, 32 * words - self.max_nodes)).view(self.num_nodes, words, 32)
        value = (bits.long() << torch.arange(32, device=sees.device)).sum(-1)
        return torch.where(value >= 1 << 31, value - (1 << 32), value).to(INT32)

    def mask_of_parents(self, parents: torch.Tensor, node_starts: torch.Tensor) -> torch.Tensor:
        """tree_mask of trees given by each node's parent: ``parents[i]`` is the
        index of row i's parent within its own tree (a node before it), or -1
        for a root; a node sees itself and all nodes above it. Made on the CPU
        (it is part of a plan) and put on the parents' device."""
        up, starts = parents.reshape(-1).tolist(), node_starts.reshape(-1).tolist()
        if len(up) != self.num_nodes or len(starts) != self.num_seqs + 1:
            raise ValueError(f"parents must have {self.num_nodes} entries and node_starts {self.num_seqs + 1}")
        sees = torch.zeros(self.num_nodes, self.max_nodes, dtype=torch.bool)
        for a, b in zip(starts, starts[1:]):
            if not 0 <= a <= b <= self.num_nodes or b - a > self.max_nodes:
                raise ValueError(f"node_starts: a tree of rows [{a}, {b}) does not fit {self.num_nodes} rows, "
                                 f"{self.max_nodes} to a tree")
            for i in range(a, b):
                if not -1 <= up[i] < i - a:
                    raise ValueError(f"parents[{i}]={up[i]}: a parent is a node of the tree before its child, or -1")
                if up[i] >= 0:
                    sees[i] = sees[a + up[i]]
                sees[i, i - a] = True
        return self.pack_mask(sees).to(parents.device)
