"""Wait states in front of memory instructions of the built kernels.

A vector memory instruction may read a scalar register five wait states after a vector instruction has written it.  The compiler
counts them in front of its own loads, and not in front of those written as inline assembly (sq_common.h: load_to_lds_*), whose
base address may come out of v_readfirstlane or, where a scalar register was spilled, out of v_readlane.  So the assembly of the
library as built here is looked through.
"""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
NEEDED = 5
SGPR = re.compile(r"(?<![\w])s\[(\d+):(\d+)\]|(?<![\w])s(\d+)(?!\w)")
MEMORY = ("global_", "buffer_", "flat_", "scratch_")


def registers(text):
    out = set()
    for a, b, c in SGPR.findall(text):
        out |= set(range(int(a), int(b) + 1)) if a else {int(c)}
    return out


def parse(text):
    """Instructions of a listing, [(address, mnemonic, operands, address of a branch's target or None)]."""
    out, base = [], {}
    for line in text.splitlines():
        m = re.match(r"([0-9a-f]+) <(.+)>:$", line)
        if m:
            base[m[2]] = int(m[1], 16)
            continue
        m = re.match(r"\s+(\w+)\s*(.*?)\s*// ([0-9A-F]+):[^<]*(?:<(.+?)(?:\+0x([0-9a-f]+))?>)?\s*$", line)
        if m:
            target = (m[4], int(m[5] or "0", 16)) if m[4] and m[1].startswith(("s_branch", "s_cbranch")) else None
            out.append((int(m[3], 16), m[1], m[2], target))
    return [(a, op, args, base[t[0]] + t[1] if t else None) for a, op, args, t in out]


def written_by_vector(op, args):
    """Scalar registers that a vector instruction writes: its first operand, or, beside vector registers, the second (a carry)."""
    if not op.startswith("v_"):
        return set()
    parts = re.findall(r"[^,\[\]]+(?:\[[^\]]*\])?", args)
    if parts and registers(parts[0]):
        return registers(parts[0])
    carry = re.match(r"v_(add_co|addc_co|sub_co|subb_co|subrev_co|subbrev_co|mad_u64_u32|mad_i64_i32|div_scale)", op)
    return registers(parts[1]) if carry and len(parts) > 1 else set()


def too_early(code):
    at = {a: i for i, (a, _, _, _) in enumerate(code)}
    found = []
    for i, (_, op, args, _) in enumerate(code):
        written = written_by_vector(op, args)
        paths = [(i + 1, 0, written)] if written else []
        while paths:
            j, waited, live = paths.pop()
            if j >= len(code) or waited >= NEEDED:
                continue
            _, o, a, target = code[j]
            if o.startswith(MEMORY) and registers(a) & live:
                found.append("%s %s | %d wait states | %s %s" % (op, args, waited, o, a))
                continue
            if o.startswith("s_") and not o.startswith(("s_cmp", "s_cbranch", "s_waitcnt", "s_nop", "s_barrier")):
                live = live - registers(a.split(",")[0])  # (written anew by a scalar instruction, for which nothing has to wait)
            waited += int(a, 0) + 1 if o == "s_nop" else 1
            if target is not None and target in at:
                paths.append((at[target], waited, live))
            if live and o not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                paths.append((j + 1, waited, live))
    return found


def test_the_scan_finds_what_it_looks_for():
    listing = """
0000000000001000 <kernel>:
\tv_readfirstlane_b32 s10, v3                                // 000000001000: 7E140503
\ts_nop 0                                                    // 000000001004: BF800000
\ts_cbranch_scc1 3                                           // 000000001008: BF850003 <kernel+0x18>
\ts_nop 4                                                    // 00000000100C: BF800004
\tglobal_load_lds_dwordx4 v1, s[10:11]                       // 000000001010: DDF48000 000A0001
\tv_readlane_b32 s4, v9, 2                                   // 000000001014: D2890004 00010509
\tglobal_load_lds_dwordx4 v1, s[10:11]                       // 000000001018: DDF48000 000A0001
\ts_mov_b32 s4, s9                                           // 00000000101C: BE840009
\tglobal_load_dword v2, v1, s[4:5]                           // 000000001020: DC508000 02040001
\tv_add_co_u32_e64 v2, s[6:7], v3, v4                        // 000000001024: D1190602 00020903
\tglobal_store_dword v1, v2, s[6:7]                          // 000000001028: DC708000 00060201
\ts_endpgm                                                   // 00000000102C: BF810000
"""
    code = parse(listing)
    assert len(code) == 12 and code[2][3] == 0x1018
    found = too_early(code)
    # through the branch two wait states lie in between, and the carry is read at once; the rewritten register is no case
    assert len(found) == 2 and "| 2 wait states |" in found[0] and "v_add_co" in found[1]


def test_no_memory_instruction_reads_a_scalar_register_too_early(built_lib, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    lib = shutil.copy(built_lib, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, cwd=tmp_path, stdout=subprocess.DEVNULL)
    parts = [p for p in sorted(glob.glob(lib + ".*gfx950")) if os.path.getsize(p)]
    loads, found = 0, []
    for part in parts:
        code = parse(subprocess.run([OBJDUMP, "-d", part], check=True, stdout=subprocess.PIPE, text=True).stdout)
        loads += sum(op.startswith("global_load_lds") for _, op, _, _ in code)
        found += too_early(code)
    assert loads > 100, "the listing holds no direct loads: it was not read as it should be"
    assert not found, "\n".join(found[:20])
