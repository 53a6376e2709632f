"""CPU: no kernel of this library holds a 64-bit shift whose amount stands in the last vector register that its waves
are allocated (an index that is 7 modulo 8). gfx950 was seen to read a wrong amount there when another wave's registers
follow: v_lshrrev_b64 by v55 of 56 registers, on waves that share a SIMD; the same shift in 32 bits, or by another
register, was right, and no wait or nop before or after it helped. The compiler does not avoid it."""

import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from iron_amd import _build


def _asm(src):
    cmd = [_build._hipcc(), *_build.HIP_FLAGS, *_build.FILE_FLAGS.get(src.name, []), "--cuda-device-only", "-S", str(src), "-o", "-"]
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    return out.stdout


def shifts_by_the_last_register(asm):
    """(kernel, instruction) of every such shift."""
    used = {m.group(1): int(m.group(2)) for m in re.finditer(
        r"\.amdhsa_kernel (\S+)\n(?:(?!\.end_amdhsa_kernel).*\n)*?\s*\.amdhsa_next_free_vgpr (\d+)", asm)}
    name, found = None, []
    for line in asm.splitlines():
        label = re.match(r"^(_Z\S+):", line)
        if label:
            name = label.group(1)
        m = re.match(r"\s*v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)(?:_e64)? v\[\d+:\d+\], v(\d+),", line)
        if m and name in used:
            amount = int(m.group(1))
            if amount % 8 == 7 and amount + 1 >= used[name]:
                found.append((name, line.strip()))
    return found


def test_the_search_finds_one():
    asm = "_Zk:\n\tv_lshrrev_b64 v[0:1], v7, s[0:1]\n.amdhsa_kernel _Zk\n\t.amdhsa_next_free_vgpr 8\n.end_amdhsa_kernel\n"
    assert shifts_by_the_last_register(asm) == [("_Zk", "v_lshrrev_b64 v[0:1], v7, s[0:1]")]
    assert not shifts_by_the_last_register(asm.replace("vgpr 8", "vgpr 12"))


def test_no_64_bit_shift_by_the_last_register():
    try:
        _build._hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    with ThreadPoolExecutor(8) as pool:
        for asm in pool.map(_asm, sorted(_build.CSRC.glob("*.hip"))):
            assert not shifts_by_the_last_register(asm)
