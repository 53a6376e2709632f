"""PageCompact: packs the pool of a paged KV cache (new operator, beside the
copies of iron/operators/strided_copy/op.py:15-110).

With L pages in use, those at or above page L move to the free ones below it,
both in ascending order, in every layer; page_table (within seq_lens) and
page_refs follow. Afterwards pages 0 .. L-1 are in use and the rest of the pool
can be cut off or handed to something else.

Arg spec: the cache (k_pages, v_pages, page_table, seq_lens, page_refs;
iron_amd.common.paging), moved (1,) int32: how many pages moved. Any dtype whose
rows are a multiple of 16 bytes. Kernel: iron_page_compact.
"""

from dataclasses import dataclass, field
from typing import ClassVar

import torch

from ... import _lib
from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator


@dataclass
class PageCompact(PagedOperator):
    num_layers: int
    num_kv_heads: int
    head_dim: int
    num_pages: int
    page_size: int
    num_seqs: int
    max_pages: int
    dtype: object = field(default=torch.bfloat16, repr=False)
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("num_layers", "num_kv_heads", "head_dim", "num_pages", "page_size", "num_seqs",
                                     "max_pages", "dtype")

    def __post_init__(self):
        self._check_pool()
        self._check_data()
        if self.num_seqs * -(-self.max_pages // 1024) >= 1 << 23:
            raise ValueError(f"num_seqs={self.num_seqs} with max_pages={self.max_pages}: a table of up to 2**33 entries")
        PagedOperator.__init__(self, context=self.context)

    def workspace_bytes(self) -> int:
        return _lib.workspace_bytes("iron_page_compact_workspace_bytes", self.num_pages)

    def get_arg_spec(self):
        return [*self._pool_specs(), *self._table_specs(), AIERuntimeArgSpec("out", (1,), dtype=INT32)]

    def _launch(self, *tensors, stream):
        self._call("iron_page_compact", tensors,
                   (self.num_layers, self.num_kv_heads, self.row_bytes, self.num_pages, self.page_size, self.num_seqs,
                    self.max_pages), stream)
