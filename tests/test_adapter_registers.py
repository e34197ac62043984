"""The adapters' kernels hold what they work on in registers: none of them, at any rank and type, keeps some of it in scratch memory, which
made those of rank 128 two to three times slower and slower than dense products over all adapters."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_no_scratch():
    flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    run = subprocess.run([HIPCC, *flags, "--cuda-device-only", f"-I{ROOT}/include", "-Rpass-analysis=kernel-resource-usage", "-c",
                          f"{ROOT}/dsh-moss-tts_amd/csrc/adapters.hip", "-o", os.devnull], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", run.stderr)
    scratch = [int(n) for n in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", run.stderr)]
    assert len(names) == len(scratch) >= 17  # four pairs of types, four ranks, and the packing
    assert not any(scratch), [n for n, s in zip(names, scratch) if s]
