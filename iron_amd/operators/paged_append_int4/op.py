"""PagedAppendInt4: PagedAppend into a paged KV cache that is held in 4 bits (new
operator; the paged form of the cache append of
iron/applications/llama_3.2_1b/llama_npu.py:311-323, with rows quantized on their way).

Requests, pages, lengths and status are PagedAppend's; k_pages and v_pages are
uint8 (num_layers, num_pages, Hkv, page_size, D / 2 + 16). Each quarter of a row
(D / 4 values from lo to hi) keeps s = fp16((hi - lo) / 15), b = fp16(lo - 16 s)
and for each value the nearest of the 16 codes, of two equally near ones the upper:
a cached value b + s (16 + code) is off by s / 2, what rounding s takes off 15 s, and
the rounding of b at most.
Values are cut to +-20480 first; a NaN makes its quarter NaN. D 64 or 128,
bf16 or fp16 (``dtype``: of k_new and v_new). Kernel: iron_paged_append_int4.
"""

from dataclasses import dataclass
from typing import ClassVar

import torch

from ..paged_append.op import PagedAppend


@dataclass
class PagedAppendInt4(PagedAppend):
    _spec_fields: ClassVar[tuple] = PagedAppend._spec_fields

    def __post_init__(self):
        self._check_int4()
        super().__post_init__()

    def _pool_specs(self):
        return self._int4_specs("inout", self.num_layers)

    def _launch(self, *tensors, stream):
        self._call("iron_paged_append_int4", tensors,
                   (int(self.dtype == torch.float16), self.num_layers, self.num_kv_heads, self.head_dim, self.num_pages,
                    self.page_size, self.num_seqs, self.max_pages, self.num_nodes, self.num_rows), stream)
