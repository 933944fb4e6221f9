"""The kernels' sources as the compiler reads them; nothing is launched."""

import os
import subprocess

import pytest

from forgeserve_amd.build import CSRC, FLAGS, HIPCC, SOURCES

# the host pass does not know the GPU's feature flag, and nothing is linked
EXPECTED = ("is not a recognized feature for this target", "'--hip-link'")


@pytest.mark.parametrize("source", SOURCES)
def test_no_warnings(source):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    done = subprocess.run([HIPCC, *FLAGS, "-fsyntax-only", os.path.join(CSRC, source)], stdout=subprocess.PIPE,
                          stderr=subprocess.STDOUT, text=True)
    said = [line for line in done.stdout.splitlines() if "warning:" in line and not any(e in line for e in EXPECTED)]
    assert done.returncode == 0 and not said, said[:5]
