"""A 64-bit shift whose amount lies in the last vector register that its wave has been given reads the amount wrong: the hardware fetches the register
behind it too.  hipcc avoids that on older targets only.  One kernel of the library had it (the flag of a bias in masks with few entries, fp32 heads wider than
64): right in the first wave of a SIMD, wrong and different every time in the next ones.  No kernel of the built library may have it."""
import os
import re
import subprocess

import pytest

from tests import test_wait_states as waits

FUNCTION = re.compile(r"^[0-9a-f]+ <(\S+)>:\n", re.M)
SHIFT = re.compile(r"^\s+v_(?:lshlrev|lshrrev|ashrrev)_[bi]64\S*\s+v\[\d+:\d+\], v(\d+),", re.M)
REGISTER = re.compile(r"\bv(?:\[\d+:(\d+)\]|(\d+)\b)")


def shifts_by_the_last_register(code):
    """(64-bit shifts by a vector register, those whose amount is the highest register in use) of the text of one function"""
    amounts = [int(m) for m in SHIFT.findall(code)]
    last = max(int(a or b) for a, b in REGISTER.findall(code)) if amounts else -1
    return amounts, [a for a in amounts if a == last]


@pytest.mark.skipif(not (os.path.exists(waits.LIB) and os.path.exists(waits.OBJDUMP)), reason="no built library or no llvm-objdump")
def test_no_shift_takes_its_amount_from_the_last_register(tmp_path):
    shifts = 0
    for n, code in enumerate(waits.device_code(waits.LIB)):
        path = tmp_path / ("%d.elf" % n)
        path.write_bytes(code)
        listing = subprocess.run([waits.OBJDUMP, "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True, check=True).stdout
        parts = FUNCTION.split(listing)
        for name, body in zip(parts[1::2], parts[2::2]):
            amounts, bad = shifts_by_the_last_register(re.sub(r"//.*", "", body))
            shifts += len(amounts)
            assert not bad, (name, bad)
    assert shifts > 100


def test_the_check_finds_one():
    shift = "\tv_lshrrev_b64 v[62:63], v79, v[22:23]\n"
    assert shifts_by_the_last_register(shift) == ([79], [79])
    assert shifts_by_the_last_register(shift + "\tv_mov_b32_e32 v80, v0\n") == ([79], [])
    assert shifts_by_the_last_register(shift + "\tglobal_load_dwordx4 v[80:83], v[8:9], off\n") == ([79], [])
    assert shifts_by_the_last_register("\tv_lshrrev_b64 v[62:63], s79, v[22:23]\n") == ([], [])
    assert shifts_by_the_last_register("\tv_lshlrev_b64 v[78:79], v3, v[78:79]\n") == ([3], [])
