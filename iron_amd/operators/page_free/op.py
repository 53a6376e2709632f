"""PageFree: sequences of a paged KV cache give their pages back (new operator).

Every page of each listed sequence loses one count in page_refs (0 stays 0; at
0 it is free: pages that a fork shares stay until the last holder lets go),
its table entries become -1 and its length 0.

Arg spec: slots (num_slots,) int32, page_table (num_seqs, max_pages), seq_lens
(num_seqs,), page_refs (num_pages,) int32 (iron_amd.common.paging), status
(num_slots,) int32: 0 done, 1 not a slot, one that an earlier entry of the list
names, or one whose length is invalid. Kernel: iron_page_free.
"""

from dataclasses import dataclass, field
from typing import ClassVar

from ...common import AIERuntimeArgSpec
from ...common.paging import INT32, PagedOperator


@dataclass
class PageFree(PagedOperator):
    num_pages: int
    page_size: int
    num_seqs: int
    max_pages: int
    num_slots: int
    context: object = field(default=None, repr=False)

    _spec_fields: ClassVar[tuple] = ("num_pages", "page_size", "num_seqs", "max_pages", "num_slots")

    def __post_init__(self):
        self._check_pool()
        self._check_counts(num_slots=8192)
        PagedOperator.__init__(self, context=self.context)

    def get_arg_spec(self):
        return [
            AIERuntimeArgSpec("in", (self.num_slots,), dtype=INT32),
            *self._table_specs(),
            AIERuntimeArgSpec("out", (self.num_slots,), dtype=INT32),
        ]

    def _launch(self, *tensors, stream):
        self._call("iron_page_free", tensors,
                   (self.num_pages, self.page_size, self.num_seqs, self.max_pages, self.num_slots), stream)
