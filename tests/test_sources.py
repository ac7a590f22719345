"""What the compiler's analyzer says about the kernels' sources: nothing is read before it is set, no null pointer is followed.  Needs hipcc, no GPU."""
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from chadslab_amd import build

ANALYZE = ["--cuda-device-only", "--analyze", "--analyzer-output", "text", "-Xclang", "-analyzer-checker=core", "-Xclang", "-analyzer-config", "-Xclang", "max-nodes=2000"]


@pytest.mark.skipif(shutil.which(build.HIPCC) is None, reason="no hipcc")
def test_nothing_is_read_before_it_is_set():
    def found(source):
        p = subprocess.run([build.HIPCC, "--offload-arch=gfx950", "-std=c++17", "-w", *ANALYZE, str(source)], capture_output=True, text=True)
        return p.returncode, [line for line in p.stderr.splitlines() if "warning:" in line or "error:" in line]

    sources = sorted(build.CSRC.glob("*.hip"), key=os.path.getsize, reverse=True)
    with ThreadPoolExecutor(max_workers=8) as pool:
        said = {s.name: f for s, f in zip(sources, pool.map(found, sources)) if f != (0, [])}
    assert not said
