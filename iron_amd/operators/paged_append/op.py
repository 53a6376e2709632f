"""PagedAppend: rows of new keys and values go to the ends of their sequences in
a paged KV cache, in all layers (new operator; the paged form of the cache
append of iron/applications/llama_3.2_1b/llama_npu.py:311-323).

Sequence s takes rows ``rows[row_starts[s]]`` .. ``rows[row_starts[s + 1] - 1]``
of k_new and v_new, in that order: after a verification step the accepted nodes
of its tree, after a prefill the prompt. New pages are taken where the last one
is full, seq_lens grows. A row number outside [0, num_nodes) appends zeros.

Arg spec: k_new and v_new (num_layers, num_nodes, Hkv, D), rows (num_rows,),
row_starts (num_seqs + 1,) int32, the cache (k_pages, v_pages, page_table,
seq_lens, page_refs; iron_amd.common.paging), status (num_seqs,) int32:
0 done, 1 the sequence's length or its range of rows is invalid (the range has
rows and leaves [0, num_rows], ends before its start or starts below an earlier
entry of row_starts), 2 too few free pages or table entries, 3 its partly filled
last page is a hole or shared. A sequence with a status other than 0 is left as
it was. Any dtype whose rows are a multiple of
16 bytes. Kernel: iron_paged_append.
"""

from dataclasses import dataclass, field
from typing import ClassVar

import torch

from ... import _lib
from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator


@dataclass
class PagedAppend(PagedOperator):
    num_layers: int
    num_kv_heads: int
    head_dim: int
    num_pages: int
    page_size: int
    num_seqs: int
    max_pages: int
    num_nodes: int
    num_rows: int
    dtype: object = field(default=torch.bfloat16, repr=False)
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("num_layers", "num_kv_heads", "head_dim", "num_pages", "page_size", "num_seqs",
                                     "max_pages", "num_nodes", "num_rows", "dtype")

    def __post_init__(self):
        self._check_pool()
        self._check_data()
        self._check_counts(num_nodes=(1 << 31) - 1, num_rows=1 << 20)
        PagedOperator.__init__(self, context=self.context)

    def workspace_bytes(self) -> int:
        return _lib.workspace_bytes("iron_paged_append_workspace_bytes", self.num_seqs, self.num_rows, self.page_size)

    def get_arg_spec(self):
        new = (self.num_layers, self.num_nodes, self.num_kv_heads, self.head_dim)
        return [
            AIERuntimeArgSpec("in", new, dtype=self.dtype),
            AIERuntimeArgSpec("in", new, dtype=self.dtype),
            AIERuntimeArgSpec("in", (self.num_rows,), dtype=INT32),
            AIERuntimeArgSpec("in", (self.num_seqs + 1,), dtype=INT32),
            *self._pool_specs(),
            *self._table_specs(),
            AIERuntimeArgSpec("out", (self.num_seqs,), dtype=INT32),
        ]

    def _launch(self, *tensors, stream):
        self._call("iron_paged_append", tensors,
                   (self.num_layers, self.num_kv_heads, self.row_bytes, self.num_pages, self.page_size, self.num_seqs,
                    self.max_pages, self.num_nodes, self.num_rows), stream)
