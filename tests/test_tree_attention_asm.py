"""CPU: what the compiler cannot check in the assembly of TreeAttention's kernels. Each M0 write is an LDS-DMA load's
own, one wait state before it, so the compiler keeps nothing in M0 there; no kernel spills. The compiler does wait for
loads of its own (page numbers) among those loads: a count that is too low for it only waits longer."""

import re

import pytest

from tests import test_asm_contracts as contracts

STREAMING, JOIN = ("tree_attention_kernel", "tree_wide_kernel"), "tree_join_kernel"


def test_m0_belongs_to_the_lds_loads():
    loads = {}
    for name, body in contracts.functions(contracts.device_asm("tree_attention.hip")).items():
        for i, ins in enumerate(body):
            if re.search(r"\bm0\b", ins):
                assert ins.startswith("s_mov_b32 m0,") and body[i + 1] == "s_nop 0", (name, body[i:i + 3])
                assert re.match(r"buffer_load_dwordx4 .*\blds$", body[i + 2]), (name, body[i:i + 3])
            if re.match(r"buffer_load_\S+ .*\blds$", ins):
                assert body[i - 1] == "s_nop 0" and body[i - 2].startswith("s_mov_b32 m0,"), (name, body[i - 2:i + 1])
                loads[name] = loads.get(name, 0) + 1
            assert not ins.startswith("global_load_lds"), name
    assert all(any(k in name for k in STREAMING) for name in loads)
    assert sum(STREAMING[0] in name for name in loads) == 8 and sum(STREAMING[1] in name for name in loads) == 4


@pytest.mark.parametrize("kernel", [*STREAMING, JOIN])
def test_no_scratch(kernel):
    asm = contracts.device_asm("tree_attention.hip")
    sizes = re.findall(r"\.amdhsa_kernel (\S+)\n(?:(?!\.end_amdhsa_kernel).*\n)*?\s*\.amdhsa_private_segment_fixed_size (\d+)", asm)
    mine = [int(n) for name, n in sizes if kernel in name]
    assert mine and not any(mine)
