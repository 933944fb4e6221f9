"""A plan that no kernel of the projections over codes takes is refused: the host's half of the library's source, compiled by
itself and called with plans, also with such as its rule does not make. Launches are counted by stand-ins for the runtime's
functions; no GPU is asked for anything."""

import ctypes
import os
import subprocess

import pytest

from forgeserve_amd.build import CSRC, FLAGS, HIPCC
from test_gpu_linear_e4m3 import SIZES

CALL = """
#include "%s/linear_e4m3.hip"

extern "C" int try_plan(int m, int n, int bm, int bn, int splits, int join, int stream, int gated, int codes) {
  fs_linear c{};
  c.x = c.x_scales = c.w = c.w_scales = c.out = reinterpret_cast<void*>(256);
  c.out_scales = codes ? c.out : nullptr;
  c.ldx = c.ldw = c.K = 4096;
  c.ldo = c.N = n;
  c.M = m;
  c.dtype = FS_BF16;
  c.gated = gated;
  return linear(c, Plan{bm, bn, splits, join != 0, stream != 0}, reinterpret_cast<char*>(256), nullptr);
}
"""
STAND_INS = """
#include <stddef.h>
char __hip_fatbin[8];
int launches;
void **__hipRegisterFatBinary(const void *p) { return NULL; }
void __hipUnregisterFatBinary(void **p) {}
void __hipRegisterFunction(void) {}
int __hipPushCallConfiguration(void) { return 0; }
int __hipPopCallConfiguration(void) { return 0; }
int hipLaunchKernel(void) { return ++launches, 0; }
int _ZN2fs13launch_statusEPKc(const char *what) { return 0; }
int _ZN2fs9arg_errorEPKcz(const char *fmt, ...) { return -1; }
void _ZN2fs18quantize_rows_e4m3EPKvllliPhlPjP12ihipStream_t(void) {}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    to = str(tmp_path_factory.mktemp("plans"))
    for name, text in (("call.hip", CALL % CSRC), ("stand_ins.c", STAND_INS)):
        with open(os.path.join(to, name), "w") as f:
            f.write(text)
    flags = [f for f in FLAGS if f != "-O3"] + ["--cuda-host-only", "-fuse-cuid=none"]
    subprocess.run([HIPCC, *flags, "-c", "call.hip", "-o", "call.o"], cwd=to, check=True, stderr=subprocess.DEVNULL)
    subprocess.run(["gcc", "-w", "-shared", "-fPIC", "stand_ins.c", "call.o", "-lstdc++", "-o", "plans.so"], cwd=to, check=True)
    return ctypes.CDLL(os.path.join(to, "plans.so"))


def tried(host, bm, bn, splits, join, stream, gated, codes, m=None, n=256):
    """(status, launches)"""
    count = ctypes.c_int.in_dll(host, "launches")
    count.value = 0
    m = m or (min(bm, 100) if stream else 100)
    return host.try_plan(m, n, bm, bn, splits, join, stream, gated, codes), count.value


def plans_of_the_rule():
    """(rows, columns, splits, through memory, streamed, gated, codes out), each as the rule gives it for some size."""
    return sorted({(bm, bn, splits, join, int(bn < 64 or bn == 112 or (bm < 64 and bn == 64)), int(gated), int(codes))
                   for (_, _, _, gated, codes), (bm, bn, splits, join) in SIZES.items()})


def test_the_rules_plans_are_launched(host):
    for plan in plans_of_the_rule():
        assert tried(host, *plan) == (0, 2 if plan[3] else 1), plan


def test_other_plans_are_refused(host):
    good, refused = set(plans_of_the_rule()), 0
    for bm in (16, 32, 48, 64, 128, 192, 256, 512):
        for bn in (16, 32, 48, 64, 112, 128, 256, 512):
            for splits in (1, 2, 3, 4, 8, 16):
                for join in (0, 1):
                    for stream in (0, 1):
                        for gated in (0, 1):
                            for codes in (0, 1):
                                plan = bm, bn, splits, join, stream, gated, codes
                                status, launches = tried(host, *plan)
                                # launched in full, or refused with nothing launched
                                assert (status, launches) in ((0, 1 + join), (-1, 0)), (plan, status, launches)
                                assert status == 0 or plan not in good
                                refused += status != 0
    assert refused > 1000


def test_rows_and_columns_beyond_a_streaming_plan_are_refused(host):
    assert tried(host, 16, 16, 1, 0, 1, 0, 0) == (0, 1)
    for m, n, bn, launched in ((17, 256, 16, False), (16, 256 * 16, 16, True), (16, 256 * 16 + 1, 16, False),
                               (16, 256 * 16 + 1, 32, True), (16, 256 * 112, 112, True), (16, 256 * 48, 32, False)):
        assert tried(host, 16, bn, 1, 0, 1, 0, 0, m=m, n=n) == ((0, 1) if launched else (-1, 0)), (m, n, bn)
