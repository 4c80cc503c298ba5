"""The host side of the paged cache's operators where a GPU test cannot go: launches that fail, and
rows that take several launches. tests/cached_host.cpp on the CPU, with a HIP runtime and launchers of
its own that record what they are given."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tenferro-decision-rs_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def test_host_side_of_the_cache(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    sources = [os.path.join(ROOT, "tests", "cached_host.cpp"), os.path.join(CSRC, "tfd_host.cpp")]
    objects = [str(tmp_path / f"{i}.o") for i in range(2)]
    for source, out in zip(sources, objects):
        subprocess.run([HIPCC, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-w", "-fno-pie",
                        "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-c", source, "-o", out],
                       check=True, timeout=300)
    program = tmp_path / "cached_host"
    # What the other entries call is not there, and not called.
    subprocess.run(["g++", "-no-pie", *objects, "-Wl,--unresolved-symbols=ignore-all", "-o",
                    str(program)], check=True, timeout=300)
    got = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0, got.stdout + got.stderr
