"""TreeAttentionInt4: TreeAttention over a paged KV cache that is held in 4 bits
(new operator; the reference decodes one token of one sequence against a dense
16-bit cache, iron/applications/llama_3.2_1b/llama_npu.py:486-523).

Everything is TreeAttention's but the pages: one layer's k_pages and v_pages are
uint8 (num_pages, Hkv, page_size, D / 2 + 16), rows as PagedAppendInt4 writes them
(``iron_amd.common.paging.int4_row_bytes`` says how). The tree's own rows k_new and
v_new have 16 bits. With D 64 a position takes 48 bytes instead of 128, with D 128
80 instead of 256.

A cached value b + s (16 + code) enters the products rounded once to fp16, in both
types; so do the weights of cached positions (kept to 2^-30 of a row's largest).
Tree rows have bf16 or fp16 weights: two parts of 16 bits, or, where a KV head has
more than 32 rows (max_nodes times H / Hkv), one. Kernel: iron_tree_attention_int4.
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
