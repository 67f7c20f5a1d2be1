"""Wait states in the built library's code.  On gfx950 five wait states have to lie
between a vector instruction that writes a scalar register (v_readfirstlane_b32, the
reload of a spilled one by v_readlane_b32, a compare into a pair) and a vector memory
instruction that reads it: the hardware does not interlock the two, and the load would go
by the old descriptor.  The compiler inserts them before its own loads; inside inline
assembly it does not look, so what the assembly issues is checked here in the code as it
was built, whatever the scheduler and the register allocator put before it."""

import os
import re
import shutil
import subprocess

import pytest

from evo2_flash_amd.build import LIB_PATH

NEED = 5
OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump"))
                if p and os.path.exists(p)), None)
_SGPR = re.compile(r"^s(?:(\d+)|\[(\d+):(\d+)\])$")


def _scalars(operand):
    m = _SGPR.match(operand)
    if not m:
        return ()
    lo, hi = (m.group(1), m.group(1)) if m.group(1) else m.groups()[1:]
    return range(int(lo), int(hi) + 1)


def _short(text):
    """[(kernel, instruction, wait states)] of the vector memory instructions of a listing
    that read a scalar register fewer than NEED wait states after a vector instruction
    wrote it, along the code as it lies and along each branch taken forward or back."""
    found, kernel, now, written = [], "", 0, {}
    code, at = [], {}
    for line in text.splitlines():
        if line.endswith(">:"):
            code.append((None, line.split("<", 1)[1][:-2], ()))
            continue
        m = re.match(r"^\s+([a-z]\w+)\s*(.*?)\s*//\s*([0-9A-F]+):", line)
        if m:
            at[int(m.group(3), 16)] = len(code)
            code.append((m.group(1), m.group(2), int(m.group(3), 16)))

    def step(i, now, written):
        op, args, _ = code[i]
        args = [a.strip() for a in args.replace(" offen", "").split(",")] if args else []
        args = [a.split(" ")[0] for a in args]
        if op.startswith(("buffer_", "global_", "flat_", "scratch_")):
            for a in args:
                for r in _scalars(a):
                    if r in written and now - written[r] < NEED:
                        found.append((kernel, f"{op} {code[i][1]}", now - written[r]))
        now += int(args[0], 0) + 1 if op == "s_nop" else 1
        if op.startswith("v_"):
            for a in args[:2] if "_co_" in op else args[:1]:
                for r in _scalars(a):
                    written[r] = now
        return now

    for i, (op, args, where) in enumerate(code):
        if op is None:
            kernel, now, written = args, 0, {}
            continue
        now = step(i, now, written)
        if op == "s_branch" or op.startswith("s_cbranch"):
            offset = int(args.split()[0], 0)
            to = at.get(where + 4 + 4 * (offset - 65536 if offset >= 32768 else offset))
            there, then = now, dict(written)
            for j in range(to if to is not None else len(code), min(len(code), (to or 0) + NEED)):
                if code[j][0] is None:
                    break
                there = step(j, there, then)
        if op in ("s_branch", "s_endpgm", "s_setpc_b64"):
            written = {}
    return sorted(set(found))


def test_the_check_sees_a_short_distance():
    def listing(*ops):
        return "0000 <kernel>:\n" + "".join(f"\t{o}   // {4 * i:012X}: 00000000\n"
                                            for i, o in enumerate(ops))

    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    near = listing("v_readfirstlane_b32 s6, v0", "s_mov_b32 m0, s9", "s_nop 2", load)
    assert [f[2] for f in _short(near)] == [4]
    assert not _short(near.replace("s_nop 2", "s_nop 3"))
    assert not _short(near.replace("s6, v0", "s8, v0"))
    assert _short(listing("v_cmp_gt_i32_e64 s[4:5], v0, v1", "s_nop 3", load))
    assert _short(listing("v_readlane_b32 s7, v0, 3", "s_branch 1", "s_nop 7", load))
    assert not _short(listing("v_readlane_b32 s7, v0, 3", "s_branch 0", "s_nop 7", load))
    assert _short(listing("s_nop 0", load, "v_readlane_b32 s7, v0, 3", "s_cbranch_scc1 65532"))


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_loads_wait_for_their_scalar_operands(tmp_path):
    lib = tmp_path / "lib.so"  # (the code objects are written beside the file)
    shutil.copy(LIB_PATH, lib)
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    parts = sorted(p for p in os.listdir(tmp_path) if "amdgcn" in p and os.path.getsize(tmp_path / p))
    assert parts
    loads, short = 0, []
    for p in parts:
        text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(tmp_path / p)], check=True,
                              capture_output=True, text=True).stdout
        loads += text.count(" offen lds")
        short += _short(text)
    assert loads > 100
    assert not short, short[:8]
