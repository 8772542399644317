"""The product's kernels count their loads: a wait for the copies of a group leaves exactly the
loads behind them in flight (moe_fp8_product.hip).  The built library's own code has to hold what
the counts assume; no GPU needed."""
import re
import subprocess
from pathlib import Path

import pytest

from ainfer_amd._build import HIPCC, LIB
from test_kernel_spills import code_objects

OBJDUMP = Path(HIPCC).resolve().parent.parent / "llvm" / "bin" / "llvm-objdump"


def kernels(tmp_path):
    """{symbol: instructions} of the product's kernels."""
    out = {}
    for i, co in enumerate(code_objects(LIB.read_bytes())):
        if b"k_fp8_tiles" not in co:
            continue
        f = tmp_path / f"{i}.co"
        f.write_bytes(co)
        text = subprocess.run([str(OBJDUMP), "-d", "--no-show-raw-insn", str(f)], capture_output=True,
                              text=True, check=True).stdout
        for m in re.finditer(r"^[0-9a-f]+ <(\S*k_fp8_(?:tiles|split)\S*)>:\n(.*?)(?=^\S|\Z)", text,
                             re.S | re.M):
            out[m.group(1)] = [line.split("//")[0].strip() for line in m.group(2).splitlines()]
    return out


def steps(code):
    """(count waited for, accesses) of every stretch from a wait that leaves loads in flight
    to the next wait or branch, where it holds copies into LDS."""
    found, wait, ops = [], 0, []
    for line in code + ["s_endpgm"]:
        m = re.match(r"s_waitcnt vmcnt\((\d+)\)$", line)
        if m or re.match(r"s_(c?branch|endpgm|setpc)", line):
            if wait and "copy" in ops:
                found.append((wait, ops))
            wait, ops = int(m.group(1)) if m else 0, []
        elif re.match(r"buffer_load_\w+ .*\blds\b", line):
            ops.append("copy")
        elif re.match(r"(global|buffer|flat)_load", line):
            ops.append("load")
        elif re.match(r"(global|buffer|flat)_(store|atomic)", line):
            ops.append("other")
    return found


def test_waits_match_the_loads(tmp_path):
    if not LIB.exists() or not OBJDUMP.exists():
        pytest.skip("library or llvm-objdump missing")
    found = kernels(tmp_path)
    tiles = {k: v for k, v in found.items() if "tiles" in k}
    split = {k: v for k, v in found.items() if "split" in k}
    assert len(tiles) == 4 and len(split) == 8
    for name, code in found.items():
        if name in tiles:
            ahead, per = int(re.search(r"ELi\d+ELi(\d)E", name).group(1)), 9
        else:
            ahead, per = 2, 2 * int(re.search(r"splitILb\dELi(\d)E", name).group(1)) + 1
        n = 0
        for wait, ops in steps(code):
            copies, loads = ops.count("copy"), ops.count("load")
            if loads == 2 * per:
                continue  # the first two groups, ahead of the loop
            # copies first, then the weights' loads, nothing else
            assert ops == ["copy"] * copies + ["load"] * per, (name, wait, ops)
            assert wait == (per if ahead == 1 else per + copies + per), (name, wait, ops)
            n += 1
        assert n >= (8 if name in tiles else 3), (name, n)
