"""Waits that the hardware leaves to the program, at the copies into LDS that the kernels write in inline assembly, where the
compiler adds none: read from the assembly that hipcc writes for them; nothing is launched."""

import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from forgeserve_amd.build import CSRC, FLAGS, HIPCC, SOURCES

COPY = re.compile(r"(global_load_lds_|buffer_load_\w+ .*\blds\b)")
INSTRUCTION = re.compile(r"(s|v|ds|global|buffer|flat|scratch)_\w")


def instructions(lines):
    """A listing's instructions in text order, without comments; what begins a block is kept as None."""
    out = []
    for line in lines:
        line = line.split(";")[0].split("//")[0].strip()
        if INSTRUCTION.match(line):
            out.append(line)
        elif re.match(r"[.\w$]+:", line):
            out.append(None)
    return out


def target(ins):
    return ins.split(None, 1)[1].split(",")[0].strip() if ins and " " in ins else ""


def copies_right_behind_m0(lines):
    """(copies into LDS, those with no instruction between them and the one before that writes m0). A block's first copy
    counts as right behind it."""
    code = instructions(lines)
    at = [i for i, ins in enumerate(code) if ins and COPY.match(ins)]
    return len(at), [code[i] for i in at if i == 0 or code[i - 1] is None or target(code[i - 1]) == "m0"]


def test_the_reading_itself():
    text = """
      s_mov_b32 m0, s4
      global_load_lds_dwordx4 v1, s[2:3]     ; one
      s_add_i32 m0, s4, 64
      s_nop 0
      global_load_lds_dword v1, s[2:3]
    .LBB0_1:
      buffer_load_dwordx4 v5, s[4:7], 0 offen lds
      global_load_dwordx4 v[0:3], v9, s[2:3]
    """
    assert copies_right_behind_m0(text.splitlines()) == (3, ["global_load_lds_dwordx4 v1, s[2:3]", "buffer_load_dwordx4 v5, s[4:7], 0 offen lds"])


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    """Of every source that has such copies, its own or an included file's."""
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    to = tmp_path_factory.mktemp("asm")

    def text(name):
        with open(os.path.join(CSRC, name)) as f:
            body = f.read()
        return body + "".join(text(i) for i in re.findall(r'#include "(\w+\.h)"', body))

    def listing(name):
        path = str(to / (name + ".s"))
        subprocess.run([HIPCC, *FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, name), "-o", path], check=True,
                       stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
        with open(path) as f:
            return name, f.readlines()

    with ThreadPoolExecutor(4) as pool:
        return dict(pool.map(listing, [s for s in SOURCES if "global_load_lds" in text(s)]))


def test_a_copy_waits_for_m0(listings):
    """A copy into LDS reads m0, and needs one wait state behind the scalar instruction that wrote it."""
    assert {"gemm.hip", "gemm_e4m3.hip", "linear_e4m3.hip", "attention.hip"} <= set(listings)
    for name, lines in listings.items():
        copies, early = copies_right_behind_m0(lines)
        assert copies > 100 and not early, (name, copies, len(early), early[:3])
