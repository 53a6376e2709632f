"""PagedGatherInt4: positions of sequences of a 4-bit paged KV cache come back as
16-bit rows, in all layers (new operator, the way back of PagedAppendInt4): for the
dense operators (MHA, GQADecode), to move a sequence to a cache of 16 bits
(PagedAppend), to look at what the cache holds.

Rows ``row_starts[s]`` .. ``row_starts[s + 1] - 1`` of k_out and v_out receive
positions ``begins[s]``, ``begins[s] + 1``, .. of sequence s, each value
b + s (16 + code) rounded to ``dtype``; zeros for a position outside
[0, seq_lens[s]) or in a hole. Rows in no range are left as they were, a row in
several is the first sequence's.

Arg spec: begins (num_seqs,), row_starts (num_seqs + 1,) int32, k_pages and v_pages
(num_layers, num_pages, Hkv, page_size, D / 2 + 16) uint8, page_table (num_seqs,
max_pages), seq_lens (num_seqs,) int32, k_out and v_out (num_layers, num_rows, Hkv,
D). D 64 or 128, bf16 or fp16. Kernel: iron_paged_gather_int4.
"""

from dataclasses import dataclass, field
from typing import ClassVar

import torch

from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator


@dataclass
class PagedGatherInt4(PagedOperator):
    num_layers: int
    num_kv_heads: int
    head_dim: int
    num_pages: int
    page_size: int
    num_seqs: int
    max_pages: int
    num_rows: int
    dtype: object = field(default=torch.bfloat16, repr=False)
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("num_layers", "num_kv_heads", "head_dim", "num_pages", "page_size", "num_seqs",
                                     "max_pages", "num_rows", "dtype")

    def __post_init__(self):
        self._check_int4()
        self._check_pool()
        self._check_data()
        self._check_counts(num_rows=1 << 20)
        PagedOperator.__init__(self, context=self.context)

    def get_arg_spec(self):
        rows = (self.num_layers, self.num_rows, self.num_kv_heads, self.head_dim)
        table, lens, _ = self._table_specs()
        return [
            AIERuntimeArgSpec("in", (self.num_seqs,), dtype=INT32),
            AIERuntimeArgSpec("in", (self.num_seqs + 1,), dtype=INT32),
            *self._int4_specs("in", self.num_layers),
            AIERuntimeArgSpec("in", table.shape, dtype=INT32),
            AIERuntimeArgSpec("in", lens.shape, dtype=INT32),
            AIERuntimeArgSpec("out", rows, dtype=self.dtype),
            AIERuntimeArgSpec("out", rows, dtype=self.dtype),
        ]

    def _launch(self, *tensors, stream):
        self._call("iron_paged_gather_int4", tensors,
                   (int(self.dtype == torch.float16), self.num_layers, self.num_kv_heads, self.head_dim, self.num_pages,
                    self.page_size, self.num_seqs, self.max_pages, self.num_rows), stream)
