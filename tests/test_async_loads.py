"""The loads that go from memory straight into LDS, in the machine code of the library that was built: each reads the LDS address
from M0, and one wait state has to lie between a scalar write of M0 and such a load (five between a vector instruction that writes a
scalar register and a memory instruction that reads it).  The compiler keeps these distances in its own code, not inside inline assembly."""
import os
import re
import shutil
import subprocess

import pytest

import alignedkv_amd
from alignedkv_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def scalar_registers(text):
    found = {int(m) for m in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    return found


def too_close(lines):
    """(number of loads into LDS, those that follow a write of M0 or of their descriptor too closely)."""
    loads, bad, before, where = 0, [], [], ""
    for line in lines:
        head = re.match(r"^[0-9a-f]* ?<(\w+)>:", line)
        if head:
            where, before = head[1], []
            continue
        code = line.split("//")[0].strip()
        if not code or code.endswith(":"):
            continue
        op, _, args = code.partition(" ")
        if op.startswith(("buffer_load", "global_load")) and code.endswith(" lds"):
            loads += 1
            reads, states = scalar_registers(args.partition(",")[2]), 0
            for o, a in reversed(before[-8:]):
                to = a.split(",")[0].strip()
                if (to == "m0" and states < 1) or (o.startswith("v_") and states < 5 and scalar_registers(to) & reads):
                    bad.append(f"{where}: {o} {a} -> {code}")
                states += int(a, 0) + 1 if o == "s_nop" else 1
        before.append((op, args))
    return loads, bad


def test_the_check_tells_them_apart():
    good = ["s_mov_b32 m0, s4", "s_nop 0", "buffer_load_dwordx4 v1, s[0:3], 0 offen lds"]
    assert too_close(good) == (1, [])
    assert too_close(["s_mov_b32 m0, s4", "v_add_u32 v2, v2, v3", good[2]]) == (1, [])
    assert len(too_close([good[0], good[2]])[1]) == 1
    assert len(too_close(["v_readfirstlane_b32 s2, v7", *good])[1]) == 1
    assert too_close(["v_readfirstlane_b32 s2, v7", "s_nop 4", *good]) == (1, [])
    assert too_close(["v_readfirstlane_b32 s9, v7", *good, "buffer_load_dwordx4 v[0:3], v1, s[0:3], 0 offen"]) == (1, [])


def test_loads_into_lds_keep_their_distance(tmp_path):
    if not os.path.exists(_lib.LIB_PATH):
        alignedkv_amd.build()
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    lib = shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], cwd=tmp_path, check=True, capture_output=True)
    loads, bad = 0, []
    for f in sorted(os.listdir(tmp_path)):
        if "gfx950" in f:
            out = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(tmp_path / f)], check=True, capture_output=True, text=True).stdout
            n, b = too_close(out.splitlines())
            loads, bad = loads + n, bad + b
    assert loads > 0
    assert not bad, f"{len(bad)} of {loads} loads into LDS come too close behind what they read: {bad[:3]}"
