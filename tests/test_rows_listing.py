"""What the compiler made of the products on plain rows, whose MFMAs are assembly statements: read from the listing of the built library, no GPU needed."""
import os
import re
import subprocess

import pytest

from tests.test_kernel_resources import OBJDUMP, VALU_RESULT, _code_objects, _hazards, _registers


def _code(listing):
    return [m.groups() for m in (re.match(r"\s+(\S+)\s*(.*?)\s*// [0-9A-F]+:", line) for line in listing.splitlines()) if m]


def _reads(name, operands):
    """The registers that an instruction takes, its own sums among them; of an MFMA onto zeros not those that it only writes."""
    parts = re.split(r",\s*(?![^\[]*\])", operands)
    if name.startswith("v_mfma") and parts[3].strip() == "0":
        return _registers(",".join(parts[1:]))
    return _registers(operands)


def _young(listing):
    """As ``_hazards``, but for vector instructions in front of an MFMA onto zeros that writes the same register and does not read it: it does so many cycles later."""
    code = _code(listing)
    found = []
    for i, name, ops in _hazards(listing):
        if not name.startswith("v_mfma"):
            result, waited, j = _registers(ops.split(",")[0]), 0, i + 1
            while waited < VALU_RESULT and j < len(code) and not code[j][0].startswith(("s_branch", "s_cbranch")):
                if code[j][0].startswith("v_mfma") and result & _reads(*code[j]):
                    break
                waited += 1 + (int(code[j][1]) if code[j][0] == "s_nop" else 0)
                j += 1
            else:
                if waited >= VALU_RESULT or j == len(code):
                    continue
        found.append((i, name, ops))
    return found


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="llvm-objdump is not installed")
def test_nothing_touches_a_product_before_it_is_there(tmp_path):
    import __graft_entry__
    import pika_h3_flex_amd as pk

    __graft_entry__.ensure_built()
    forms = {}
    for i, image in enumerate(_code_objects(pk._lib.LIB_PATH)):
        f = tmp_path / f"{i}.elf"
        f.write_bytes(image)
        text = subprocess.run([OBJDUMP, "-d", str(f)], check=True, capture_output=True, text=True).stdout
        for name, listing in re.findall(r"^[0-9a-f]+ <(\S*4pkh3\d+product_kernel\S*)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", text, re.M | re.S):
            forms[name] = _young(listing)
            assert listing.count("v_mfma") >= 48, name
    assert len(forms) == 29, sorted(forms)      # five sizes of tiles, six kinds of product, of which one is not there with tiles of 96 rows
    assert not {n: h[:3] for n, h in forms.items() if h}


def test_the_look_finds_what_it_looks_for():
    first = "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[4:7], 0// 000000000100: 00\n"
    onto = "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[4:7], v[0:3]// 000000000100: 00\n"
    write = "\tv_mov_b32_e32 v{}, v20           // 0000000000FC: 00\n"
    assert not _young(write.format(1) + first) and len(_young(write.format(9) + first)) == 1 and len(_young(write.format(1) + onto)) == 1
    assert len(_young(first + "\tv_mov_b32_e32 v30, v2           // 000000000108: 00\n")) == 1
