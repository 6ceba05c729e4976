"""The check of tests/test_wait_states.py over every code object of the built library, with the states that hipcc itself puts before the first
reader on gfx950: 8 for the 16-bit products of 16 x 16 (s_nop 7), 12 for the larger ones, 10 for fp32's, 19 in double precision."""
import os
import subprocess

import pytest

from tests import test_wait_states as waits

STATES = {7: 8, 11: 12}


def _functions(path, code):
    path.write_bytes(code)
    listing = subprocess.run([waits.OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout
    for name, rows in waits.functions(listing):
        place = {offset: i for i, (_, _, offset, _) in enumerate(rows)}
        body = [(op, args, place.get(target, len(rows)) if target is not None else None) for op, args, _, target in rows]
        if any(op.startswith("v_mfma") for op, _, _ in body):
            yield name, body


@pytest.mark.skipif(not (os.path.exists(waits.LIB) and os.path.exists(waits.OBJDUMP)), reason="no built library or no llvm-objdump")
def test_every_kernel_with_matrix_instructions_waits(tmp_path, monkeypatch):
    before = waits.states_needed
    monkeypatch.setattr(waits, "states_needed", lambda op: STATES.get(before(op), before(op)))
    checked = []
    for n, code in enumerate(waits.device_code(waits.LIB)):
        for name, body in _functions(tmp_path / ("%d.elf" % n), code):
            early = waits.too_early(body)
            assert not early, (name, early[:3])
            checked.append(name)
    assert len(checked) > 500
    for family in ("dot_fwd_kernel", "dot_bwd_q_kernel", "dot_bwd_kv_kernel", "ns_gemm_kernel", "ns_piece_kernel", "ns_gram_kernel", "dense_attn", "bnf", "ipd", "proj"):
        assert any(family in name for name in checked), family


def test_seven_states_are_too_few(monkeypatch):
    before = waits.states_needed
    monkeypatch.setattr(waits, "states_needed", lambda op: STATES.get(before(op), before(op)))
    mfma = ("v_mfma_f32_16x16x32_bf16", ["v[0:3]", " v[4:7]", " v[8:11]", " v[0:3]"], None)
    read, end = ("v_add_f32_e32", ["v12", " v0", " v13"], None), ("s_endpgm", [], None)
    assert waits.too_early([mfma, ("s_nop", ["6"], None), read, end])
    assert not waits.too_early([mfma, ("s_nop", ["7"], None), read, end])
