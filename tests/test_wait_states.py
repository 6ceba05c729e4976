"""A matrix instruction's result may be read by other instructions only some cycles later, and the hardware does not wait by itself.  hipcc counts
these wait states along straight code and has missed them where a branch stands between (wrong gradients, the same every run), so the
built kernels are checked: along every path, nothing but another matrix instruction's accumulator reads such a result too early."""
import os
import re
import shutil
import struct
import subprocess

import pytest

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gat_amd", "libgatmi.so")
OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
KERNELS = ("dot_fwd_kernel", "ns_gemm_kernel", "dense_attn")


def device_code(path):
    """The gfx950 code objects in the library's offload bundles."""
    data = open(path, "rb").read()
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        entries, p = struct.unpack_from("<Q", data, at + 24)[0], at + 32
        for _ in range(entries):
            offset, size, n = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + n]:
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 1)


def registers(operand):
    m = re.match(r"^\s*-?\|?([av])(?:\[(\d+):(\d+)\]|(\d+)\b)", operand)
    if not m:
        return frozenset()
    lo, hi = (int(m.group(2)), int(m.group(3))) if m.group(4) is None else (int(m.group(4)),) * 2
    return frozenset((m.group(1), i) for i in range(lo, hi + 1))


def states_needed(op):
    """Upper bounds: passes (4 cycles each) of the instruction + 3, of the fp32 ones + 2; double precision 19."""
    if "f64" in op:
        return 19
    if "_f32_16x16x4_f32" in op:
        return 10
    if "_f32_32x32x2_f32" in op:
        return 18
    return 7 if "16x16x32" in op or "16x16x16" in op else 11


READS_FIRST = ("store", "write", "ds_add", "ds_bpermute", "ds_swizzle", "readlane", "readfirstlane", "cmp")


def too_early(code):
    """[(op, reader, states between, states needed)] of one function: [(op, operands, branch target or None)]."""
    bad = []
    def successors(i):
        op, _, target = code[i]
        if op in ("s_endpgm", "s_setpc_b64"):
            return ()
        if op == "s_branch":
            return (target,)
        return (i + 1, target) if op.startswith("s_cbranch") else (i + 1,)
    for i, (op, operands, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        need, seen = states_needed(op), {}
        todo = [(j, 0, registers(operands[0])) for j in successors(i)]
        while todo:
            j, states, live = todo.pop()
            if j >= len(code) or states >= need or not live or seen.get(j, need) <= states:
                continue
            seen[j] = states
            reader, args, _ = code[j]
            if reader.startswith("v_mfma"):
                if (registers(args[1]) | registers(args[2])) & live:
                    bad.append((op, reader, states, need))
                live = live - registers(args[0])                        # chained through the accumulator: the later one is looked at itself
            elif reader.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                first = 0 if any(s in reader for s in READS_FIRST) or "fmac" in reader else 1
                if any(registers(x) & live for x in args[first:]):
                    bad.append((op, reader, states, need))
                if first == 1 and args:
                    live = live - registers(args[0])
            states += int(args[0], 0) + 1 if reader == "s_nop" else 1
            todo.extend((k, states, live) for k in successors(j))
    return bad


def functions(listing):
    """name -> [(op, operands, branch target)] of a disassembly"""
    name, base, rows = None, 0, []
    for line in listing.splitlines():
        head = re.match(r"^([0-9a-f]+) <(\S+)>:$", line)
        if head:
            if rows:
                yield name, rows
            name, base, rows = head.group(2), int(head.group(1), 16), []
            continue
        m = re.match(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):(.*)$", line)
        if m and name:
            target = re.search(r"<\S+?(?:\+0x([0-9a-f]+))?>\s*$", m.group(4)) if m.group(1).startswith(("s_branch", "s_cbranch")) else None
            rows.append((m.group(1), m.group(2).split(",") if m.group(2) else [], int(m.group(3), 16) - base, int(target.group(1) or "0", 16) if target else None))
    if rows:
        yield name, rows


@pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(OBJDUMP)), reason="no built library or no llvm-objdump")
def test_results_of_matrix_instructions_are_waited_for(tmp_path):
    checked = 0
    for n, code in enumerate(c for c in device_code(LIB) if any(k.encode() in c for k in KERNELS)):
        path = tmp_path / ("%d.elf" % n)
        path.write_bytes(code)
        listing = subprocess.run([OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout
        for name, rows in functions(listing):
            place = {offset: i for i, (_, _, offset, _) in enumerate(rows)}
            body = [(op, args, place.get(target, len(rows)) if target is not None else None) for op, args, _, target in rows]
            if any(op.startswith("v_mfma") for op, _, _ in body):
                checked += 1
                assert not too_early(body), (name, too_early(body)[:3])
    assert checked > 50


def test_the_check_finds_a_missing_wait():
    mfma = ("v_mfma_f32_16x16x32_bf16", ["v[0:3]", " v[4:7]", " v[8:11]", " v[0:3]"], None)
    read, end = ("v_add_f32_e32", ["v12", " v0", " v13"], None), ("s_endpgm", [], None)
    assert too_early([mfma, read, end])
    assert too_early([mfma, ("s_nop", ["5"], None), read, end])
    assert not too_early([mfma, ("s_nop", ["6"], None), read, end])
    assert too_early([mfma, ("s_cbranch_vccz", ["2"], 3), ("s_nop", ["9"], None), read, end])          # the path that skips the wait
    assert not too_early([mfma, mfma, ("s_nop", ["9"], None), read, end])
