"""CPU: what the compiler cannot check in the assembly of TreeAttentionInt4's kernels. Their v_max3 stand in inline
assembly, which does not wait for a matrix product's result by itself (11 wait states from a 16x16 product, 19 from a 32x32
one): no operand of one may have been written by a product that recently. Nothing uses M0; the kernels of few rows spill nothing."""

import re

from tests import test_asm_contracts as contracts

SOURCE = "tree_attention_int4.hip"


def registers(operand):
    m = re.match(r"v\[(\d+):(\d+)\]$", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.match(r"v(\d+)$", operand)
    return {int(m.group(1))} if m else set()


def early_reads(body):
    """v_max3 that read a register within the wait states of a product that writes it (in the order of the text)."""
    found, products = [], []  # products: (registers, wait states still to pass)
    for ins in body:
        name, _, rest = ins.partition(" ")
        operands = [o.strip() for o in rest.split(",")]
        if name.startswith("v_max3_f32"):
            read = set().union(*(registers(o) for o in operands[1:]))
            found += [ins for regs, left in products if left > 0 and regs & read]
        states = int(operands[0]) + 1 if name == "s_nop" else 1
        products = [(regs, left - states) for regs, left in products if left > states]
        if name.startswith("v_mfma"):
            products.append((registers(operands[0]), 19 if "32x32" in name else 11))
    return found


def test_the_search_finds_one():
    body = ["v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], v[0:3]", "s_nop 3", "v_max3_f32 v9, v2, v20, v21"]
    assert early_reads(body) == [body[2]]
    assert not early_reads([body[0], "s_nop 10", body[2]])
    assert not early_reads([body[0], "v_max3_f32 v9, v4, v20, v21"])


def test_products_have_settled():
    mine = {name: body for name, body in contracts.functions(contracts.device_asm(SOURCE)).items() if "tree4_" in name}
    assert len(mine) == 12
    for name, body in mine.items():
        assert any(ins.startswith("v_max3_f32") for ins in body), name
        assert not early_reads(body), name
        assert not any(re.search(r"\bm0\b", ins) for ins in body), name


def test_few_rows_spill_nothing():
    asm = contracts.device_asm(SOURCE)
    sizes = re.findall(r"\.amdhsa_kernel (\S+)\n(?:(?!\.end_amdhsa_kernel).*\n)*?\s*\.amdhsa_private_segment_fixed_size (\d+)", asm)
    few = [int(n) for name, n in sizes if "tree4_kernel" in name]
    assert len(few) == 8 and not any(few)


def scratch_by_kernel(asm):
    return {name: int(n) for name, n in re.findall(r"\.amdhsa_kernel (\S+)\n(?:(?!\.end_amdhsa_kernel).*\n)*?\s*\.amdhsa_private_segment_fixed_size (\d+)", asm)}


def scratch_depths(asm, kernel):
    """How deep in loops each scratch access of a kernel lies, by what the compiler writes beside its blocks."""
    body = asm[asm.index(f"\n{kernel}:"):]
    depth, fresh, found = 0, False, []
    for line in body[:body.index(".Lfunc_end")].splitlines():
        if re.match(r"\.LBB|; %bb\.", line):
            depth, fresh = 0, True
        elif line.strip() and not line.strip().startswith(";"):
            fresh = False
        if fresh:
            depth = max([depth, *map(int, re.findall(r"Depth=(\d+)", line))])
        if line.strip().startswith("scratch_"):
            found.append(depth)
    return found


def test_scratch_depths_are_found():
    asm = "\nk:\n\tscratch_store_dword off, v3, off\n.LBB0_1: ; =>This Loop Header: Depth=1\n\tscratch_load_dword v3, off, off\n" \
          ".LBB0_2: ;   Parent Loop BB0_1 Depth=1\n                                        ; =>  This Inner Loop Header: Depth=2\n\tscratch_load_dword v3, off, off\n" \
          "; %bb.3: ;   in Loop: Header=BB0_1 Depth=1\n\tscratch_load_dword v3, off, off\n.Lfunc_end0:\n"
    assert scratch_depths(asm, "k") == [0, 1, 2, 1]


def test_many_rows_and_joins_spill_nothing_but_two_addresses():
    """The kernel of many rows with fp16 and head_dim 128 has all 256 registers in use: two addresses are put away at its start
    and fetched once a part (depth 1: the loop over parts), never in the loop over blocks. No other kernel spills."""
    asm = contracts.device_asm(SOURCE)
    sizes = scratch_by_kernel(asm)
    full = [name for name in sizes if "tree4_wide_kernelILi128ELb1" in name]
    assert len(full) == 1 and len(sizes) == 24
    assert not [name for name, n in sizes.items() if n and name not in full]
    depths = scratch_depths(asm, full[0])
    assert sizes[full[0]] <= 12 and len(depths) <= 4 and max(depths, default=0) <= 1
