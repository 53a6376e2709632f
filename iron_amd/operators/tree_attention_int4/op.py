"""TreeAttentionInt4: TreeAttention over a paged KV cache that is held in 4 bits
(new operator; the reference decodes one token of one sequence against a dense
16-bit cache, iron/applications/llama_3.2_1b/llama_npu.py:486-523).

Everything is TreeAttention's but the pages: one layer's k_pages and v_pages are
uint8 (num_pages, Hkv, page_size, D / 2 + 16), rows as PagedAppendInt4 writes them
(``iron_amd.common.paging.int4_row_bytes`` says how); a value past 65504, which
PagedAppendInt4 does not make, may count as infinite. The tree's own rows k_new and
v_new have 16 bits. With D 64 a position takes 48 bytes instead of 128, with D 128
80 instead of 256.

bf16 calls round cached keys, values and the weights of cached positions once to fp16,
an eighth of the result's own rounding each (weights are kept to 2^-30 of a row's
largest). fp16 calls take cached keys without rounding (but to 2^-24), values rounded
once, and weights in two parts. Weights of the tree's rows are two parts of dtype, or, where a
KV head has more than 32 rows (max_nodes times H / Hkv), one. Kernel:
iron_tree_attention_int4.
"""

from dataclasses import dataclass
from typing import ClassVar

from ..tree_attention.op import TreeAttention


@dataclass
class TreeAttentionInt4(TreeAttention):
    _spec_fields: ClassVar[tuple] = TreeAttention._spec_fields
    _entry: ClassVar[str] = "iron_tree_attention_int4"

    def _page_specs(self):
        return self._int4_specs("in")
