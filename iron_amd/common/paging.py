"""What the operators of a paged KV cache share: the checks of the pool's fields,
workspaces and launches.

The pool is ``k_pages`` and ``v_pages`` (num_layers, num_pages, num_kv_heads,
page_size, head_dim); ``page_table`` (num_seqs, max_pages) int32 says which page
holds position t of sequence s (entry ``[s, t // page_size]``, row
``t % page_size``); ``seq_lens`` (num_seqs,) int32 are the lengths and
``page_refs`` (num_pages,) int32 how many table entries hold a page (0: free).
A fresh cache has ``seq_lens`` and ``page_refs`` zero and any table. All of it
lives on the device, so a serving step reads nothing back and can be captured
whole into a graph. The layout and the rules are those of include/iron_hip.h.

A cache may hold its rows in 4 bits (TreeAttentionInt4, PagedAppendInt4,
PagedGatherInt4): pages are then uint8 with ``int4_row_bytes(head_dim)`` in the
place of head_dim, and PageFork, PageCompact and PageFree take them with
``dtype=torch.uint8, head_dim=int4_row_bytes(head_dim)``.

Calls that work on one cache must be stream-ordered. Each call takes its own
workspace from torch's allocator (about 2 us of host time), so one operator may
be called on several streams, for several caches, and captured into several
graphs, with nothing shared between them.
"""

from __future__ import annotations

import torch

from .. import _lib
from .base import AIERuntimeArgSpec, HIPOperator

INT32 = torch.int32


def int4_row_bytes(head_dim: int) -> int:
    """Bytes of a 4-bit row of head_dim values: the codes, eight to a word (even
    values in its low half's nibbles, odd ones in its high half's, both from the
    lowest up), then four fp16 pairs (s, b), one for each quarter of the row. A
    value is ``b + s * (16 + code)``."""
    return head_dim // 2 + 16


class PagedOperator(HIPOperator):
    """Base of the operators that read or change a paged cache."""

    _name_aliases = {
        **HIPOperator._name_aliases,
        "num_layers": "l",
        "num_heads": "h",
        "num_kv_heads": "kv",
        "head_dim": "d",
        "num_pages": "p",
        "page_size": "ps",
        "num_seqs": "s",
        "max_pages": "mp",
    }

    def _check_counts(self, **limits: int) -> None:
        """Each named field is a whole number from 1 to its limit."""
        for name, most in limits.items():
            value = getattr(self, name)
            if isinstance(value, bool) or not isinstance(value, int):
                raise ValueError(f"{name} must be an int, got {value!r}")
            if not 1 <= value <= most:
                raise ValueError(f"{name} must be in [1, {most}], got {value}")

    def _check_pool(self) -> None:
        self._check_counts(num_pages=1 << 27, page_size=1024, num_seqs=8192, max_pages=(1 << 31) - 1)
        if self.page_size < 16 or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {self.page_size}")
        if self.max_pages * self.page_size >= (1 << 31) - (1 << 20):
            raise ValueError(f"max_pages={self.max_pages}: a sequence holds less than 2**31 - 2**20 positions")

    def _check_data(self) -> None:
        self._check_counts(num_layers=1024, num_kv_heads=1024, head_dim=4096)
        if not isinstance(self.dtype, torch.dtype):
            raise ValueError(f"dtype must be a torch dtype, got {self.dtype!r}")
        if self.row_bytes % 16 or not 16 <= self.row_bytes <= 4096:
            raise ValueError(f"head_dim={self.head_dim} of {self.dtype} makes rows of {self.row_bytes} bytes: "
                             "a multiple of 16 up to 4096 is needed")

    @property
    def row_bytes(self) -> int:
        return self.head_dim * self.dtype.itemsize

    def _check_int4(self) -> None:
        """Pages of 4-bit rows, and 16-bit rows beside them."""
        if self.head_dim not in (64, 128):
            raise ValueError(f"Only head_dim 64 and 128 are supported, got {self.head_dim}")
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float16, got {self.dtype!r}")

    def _int4_specs(self, direction: str, *layers: int) -> list[AIERuntimeArgSpec]:
        shape = (*layers, self.num_pages, self.num_kv_heads, self.page_size, int4_row_bytes(self.head_dim))
        return [AIERuntimeArgSpec(direction, shape, dtype=torch.uint8) for _ in range(2)]

    def _pool_specs(self) -> list[AIERuntimeArgSpec]:
        shape = (self.num_layers, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim)
        return [AIERuntimeArgSpec("inout", shape, dtype=self.dtype) for _ in range(2)]

    def _table_specs(self) -> list[AIERuntimeArgSpec]:
        return [AIERuntimeArgSpec("inout", (self.num_seqs, self.max_pages), dtype=INT32),
                AIERuntimeArgSpec("inout", (self.num_seqs,), dtype=INT32),
                AIERuntimeArgSpec("inout", (self.num_pages,), dtype=INT32)]

    def workspace_bytes(self) -> int:
        """Bytes of workspace of one call (a function of the fields; 0: it needs none)."""
        return 0

    def _call(self, entry: str, tensors, numbers, stream: int) -> None:
        """Entry point ``entry`` on the tensors' device: their addresses (None: an
        argument that is not given), the numbers, a workspace (if the operator has
        one) and the stream."""
        device = tensors[0].device
        if device.index != torch.cuda.current_device():
            with torch.cuda.device(device):
                return self._call(entry, tensors, numbers, stream)
        need = self.workspace_bytes()
        space = ()
        if need:
            # below 0: a shape that the entry point refuses, saying why
            ws = torch.empty(max(need, 0), dtype=torch.uint8, device=device)
            space = (ws.data_ptr(), need)
        _lib.call(entry, *[_lib.ptr(t) for t in tensors], *numbers, *space, stream)
