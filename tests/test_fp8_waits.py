"""The product's kernels count their loads: a wait for the copies of a group leaves exactly the
loads and copies behind them in flight (moe_fp8_product.hip).  The built library's own code has to hold what
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


def access(line):
    if re.match(r"buffer_load_\w+ .*\blds\b", line):
        return "copy"
    if re.match(r"(global|buffer|flat)_load", line):
        return "load"
    if re.match(r"(global|buffer|flat)_(store|atomic)", line):
        return "other"
    return None


def tile_steps(code):
    """(count waited for in front of the barrier, accesses behind it up to the next barrier or
    branch) of every step that sends for more, and what is in flight ahead of the loop."""
    found, wait, last, ops, ahead = [], None, None, None, []
    for line in code + ["s_endpgm"]:
        m = re.match(r"s_waitcnt vmcnt\((\d+)\)", line)
        if re.match(r"s_(barrier|c?branch|endpgm|setpc)", line):
            if ops and wait:
                found.append((wait, ops))
            elif ops and ops.count("copy") and ops.count("load") > 9:
                ahead.append(ops)
            ops = [] if line.startswith("s_barrier") else None
            wait = last if line.startswith("s_barrier") else None
            last = None
        elif m:
            last = int(m.group(1)) if last is None else min(last, int(m.group(1)))
        elif access(line):
            last = None
            if ops is not None:
                ops.append(access(line))
    return found, ahead


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
        elif access(line):
            ops.append(access(line))
    return found


def test_waits_match_the_loads(tmp_path):
    if not LIB.exists() or not OBJDUMP.exists():
        pytest.skip("library or llvm-objdump missing")
    found = kernels(tmp_path)
    tiles = {k: v for k, v in found.items() if "tiles" in k}
    split = {k: v for k, v in found.items() if "split" in k}
    assert len(tiles) == 4 and len(split) == 8
    for name, code in tiles.items():
        ahead = int(re.search(r"ELi\d+ELi(\d)E", name).group(1))
        found, first = tile_steps(code)
        for wait, ops in found:
            copies = ops.count("copy")
            # copies of the group two ahead, then its step's weights: behind the copies waited for
            # are the weights of that step, the next step's copies and its weights
            assert copies and ops == ["copy"] * copies + ["load"] * 9, (name, wait, ops)
            assert wait == 9 + copies + 9, (name, wait, ops)
        for ops in first:  # as many behind the first group's copies
            copies = ops.count("copy") // 2
            lead = ["load"] * 9 if ahead == 2 else []
            assert ops == lead + (["copy"] * copies + ["load"] * 9) * 2, (name, ops)
        assert len(found) >= 4 * (ahead + 1) and len(first) >= 4, (name, len(found), len(first))
    for name, code in split.items():
        per, n = 2 * int(re.search(r"splitILb\dELi(\d)E", name).group(1)) + 1, 0
        for wait, ops in steps(code):
            copies, loads = ops.count("copy"), ops.count("load")
            if loads == 2 * per:
                continue  # the first two groups, ahead of the loop
            # copies first, then the weights' loads, nothing else
            assert ops == ["copy"] * copies + ["load"] * per, (name, wait, ops)
            assert wait == per + copies + per, (name, wait, ops)
            n += 1
        assert n >= 3, (name, n)
