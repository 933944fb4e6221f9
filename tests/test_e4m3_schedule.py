"""The order of LDS reads and copies in the compiled 8-bit projections, read from the assembly that hipcc writes for them;
nothing is launched.

The tile kernels' copies land straight in LDS, over operands of an earlier stage, and are ordered against the waves that
read those by barriers alone. A barrier orders what a wave has issued only if it has also come back: so each wave waits for
its LDS reads before every barrier."""

import os
import re
import subprocess

import pytest

from forgeserve_amd.build import CSRC, FLAGS, HIPCC

BRANCH = re.compile(r"s_(c?branch\w*)\s+(\.L\w+)")


def blocks_of(lines):
    """A kernel's basic blocks: [(instructions, labels it may go on to)] in text order, and the label of each."""
    blocks, names = [([], [])], {}
    for line in lines:
        label = re.match(r"(\.L\w+):", line)
        if label:
            if blocks[-1][0] or blocks[-1][1]:
                blocks.append(([], []))
            names[label.group(1)] = len(blocks) - 1
            continue
        line = line.strip()
        if not line or line[0] in ".;":
            continue
        blocks[-1][0].append(line)
        to = BRANCH.match(line)
        if to or line.startswith("s_endpgm"):
            blocks[-1][1].append((to.group(1), to.group(2)) if to else ("endpgm", None))
            blocks.append(([], []))
    return blocks, names


def reads_at_barriers(lines):
    """The most LDS reads that may be out at each s_barrier, over every path to it."""
    blocks, names = blocks_of(lines)
    entry = [-1] * len(blocks)   # (not reached)
    entry[0], todo, found = 0, [0], {}
    while todo:
        i = todo.pop()
        out = entry[i]
        for j, ins in enumerate(blocks[i][0]):
            op = ins.split()[0]
            if op.startswith("ds_read"):
                out = min(out + 1, 64)
            elif op == "s_waitcnt":
                left = re.search(r"lgkmcnt\((\d+)\)", ins)
                out = min(out, int(left.group(1))) if left else out
            elif op == "s_barrier":
                found[i, j] = max(found.get((i, j), 0), out)
        end = blocks[i][1]
        then = [names[label] for _, label in end if label]
        if not (end and end[0][0] in ("branch", "endpgm")) and i + 1 < len(blocks):
            then.append(i + 1)
        for t in then:
            if out > entry[t]:
                entry[t] = out
                todo.append(t)
    return list(found.values())


def test_the_walk_itself():
    text = """
      ds_read_b128 v[0:3], v4
      ds_read_b128 v[8:11], v4
      s_cbranch_scc1 .LBB0_2
      s_waitcnt lgkmcnt(0)
    .LBB0_2:
      s_barrier
      s_waitcnt vmcnt(2) lgkmcnt(1)
      s_barrier
      s_waitcnt lgkmcnt(0)
      s_barrier
      s_branch .LBB0_4
      ds_read_b32 v1, v4
    .LBB0_4:
      s_barrier
      s_endpgm
    """
    assert reads_at_barriers([line.strip() for line in text.splitlines()]) == [2, 1, 0, 0]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    to = str(tmp_path_factory.mktemp("asm") / "gemm_e4m3.s")
    subprocess.run([HIPCC, *FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, "gemm_e4m3.hip"), "-o", to], check=True,
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


@pytest.mark.parametrize("kernel,copies", [("gemm_e4m3_long_kernel", 4), ("gemm_e4m3_tile_kernel", 6), ("gemm_e4m3_short_kernel", 12)])
def test_no_read_is_out_at_a_barrier(kernels, kernel, copies):
    mine = {name: lines for name, lines in kernels.items() if kernel in name}
    assert len(mine) == copies, sorted(kernels)
    for name, lines in mine.items():
        at = reads_at_barriers(lines)
        assert len(at) >= 2 and not any(at), (name, at)
