"""PageFork: new sequences of a paged KV cache from existing ones (new operator,
beside the copies of iron/operators/strided_copy/op.py:15-110).

For each pair (parent, child) the child, an empty slot of the table, gets the
parent's positions. ``share=True`` forks: the child holds the parent's full
pages too (page_refs count it) and a new page with a copy of the rows of the
last, partly filled one, so that either can grow (several samples, the
branches of a beam). ``share=False`` copies: the child gets new pages with
everything in them. Holes of the parent's table row stay holes.

Arg spec: forks (num_forks, 2) int32, the cache (k_pages, v_pages, page_table,
seq_lens, page_refs; iron_amd.common.paging), status (num_forks,) int32: 0 done,
1 not a pair of slots with an empty child, or a child that an earlier pair
names, 2 too few free pages. Parents are taken as they are before the call; a
pair with a status other than 0 changes nothing, and where the free pages run
out, neither does any later one that needs some. Any dtype whose rows are a
multiple of 16 bytes. Kernel: iron_page_fork.
"""

from dataclasses import dataclass, field
from typing import ClassVar

import torch

from ... import _lib
from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator


@dataclass
class PageFork(PagedOperator):
    num_layers: int
    num_kv_heads: int
    head_dim: int
    num_pages: int
    page_size: int
    num_seqs: int
    max_pages: int
    num_forks: int
    share: bool = True
    dtype: object = field(default=torch.bfloat16, repr=False)
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("num_layers", "num_kv_heads", "head_dim", "num_pages", "page_size", "num_seqs",
                                     "max_pages", "num_forks", "dtype")

    def __post_init__(self):
        self._check_pool()
        self._check_data()
        self._check_counts(num_forks=8192)
        if self.num_forks * self.max_pages >= 1 << 31:
            raise ValueError(f"num_forks * max_pages must be below 2**31, got {self.num_forks * self.max_pages}")
        PagedOperator.__init__(self, context=self.context)

    def workspace_bytes(self) -> int:
        return _lib.workspace_bytes("iron_page_fork_workspace_bytes", self.num_forks, self.num_seqs, self.max_pages,
                                    self.num_pages, int(bool(self.share)))

    def get_arg_spec(self):
        return [
            AIERuntimeArgSpec("in", (self.num_forks, 2), dtype=INT32),
            *self._pool_specs(),
            *self._table_specs(),
            AIERuntimeArgSpec("out", (self.num_forks,), dtype=INT32),
        ]

    def _launch(self, *tensors, stream):
        self._call("iron_page_fork", tensors,
                   (self.num_layers, self.num_kv_heads, self.row_bytes, self.num_pages, self.page_size, self.num_seqs,
                    self.max_pages, self.num_forks, int(bool(self.share))), stream)
