"""The order of LDS reads and copies in the compiled projections with their epilogues, read from the assembly that hipcc
writes for them; nothing is launched. The kernels with tiles order copies against reads by barriers, as gemm_e4m3's; the
streaming kernels' waves each copy into places that they alone read, so no read of a wave's may be out at any of its copies."""

import os
import re
import subprocess

import pytest

from forgeserve_amd.build import CSRC, FLAGS, HIPCC
from test_e4m3_schedule import reads_at_barriers

COPY = re.compile(r"(global_load_lds_|buffer_load_\w+ .*\blds\b)")


def reads_at_copies(lines):
    """The most LDS reads that may be out at each copy into LDS."""
    return reads_at_barriers(["s_barrier" if COPY.match(line.strip()) else line for line in lines
                              if not line.strip().startswith("s_barrier")])


def test_the_walk_itself():
    text = """
      global_load_lds_dwordx4 v1, s[2:3]
      ds_read_b128 v[0:3], v4
      s_barrier
      buffer_load_dwordx4 v5, s[4:7], 0 offen lds
      s_waitcnt lgkmcnt(0)
      buffer_load_dwordx4 v[5:8], v9, s[4:7], 0 offen
      global_load_lds_dwordx4 v1, s[2:3]
      s_endpgm
    """
    assert reads_at_copies([line.strip() for line in text.splitlines()]) == [0, 1, 0]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    to = str(tmp_path_factory.mktemp("asm") / "linear_e4m3.s")
    subprocess.run([HIPCC, *FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, "linear_e4m3.hip"), "-o", to], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    out, name = {}, None
    for line in open(to):
        start = re.match(r"(_Z\w*kernel\w*):", line)
        if start:
            name = start.group(1)
            out[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            out[name].append(line)
    return out


@pytest.mark.parametrize("kernel", ["gemm_e4m3_long_kernel", "gemm_e4m3_tile_kernel"])
def test_no_read_is_out_at_a_barrier(kernels, kernel):
    mine = {name: lines for name, lines in kernels.items() if kernel in name}
    assert len(mine) >= 4, sorted(kernels)
    for name, lines in mine.items():
        at = reads_at_barriers(lines)
        assert len(at) >= 2 and not any(at), (name, at)


def test_no_read_is_out_at_a_streaming_waves_copy(kernels):
    mine = {name: lines for name, lines in kernels.items() if "linear_e4m3_stream_kernel" in name}
    assert len(mine) >= 4, sorted(kernels)
    for name, lines in mine.items():
        at = reads_at_copies(lines)
        assert len(at) >= 8 and not any(at), (name, at)
