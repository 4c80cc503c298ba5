"""Which of its two kernels the attention over a cache takes, by the library's own rule (CPU only), for
the sizes of the GPU tests: a changed rule would otherwise leave one kernel's tests on the other."""
import os
import shutil
import subprocess

import pytest

import test_cached_attention as single
import test_cached_decision as decision
import test_cached_scales as scales

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "tenferro-decision-rs_amd")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

SOURCE = """
#include <cstdio>
#include <cstdlib>
#include "tfd_internal.hpp"
int main(int n, char **v) {
  for (int i = 1; i + 3 < n; i += 4) {
    tfd::CachedArgs a{};
    a.rows = atoi(v[i]);
    a.group = atoi(v[i + 1]) / atoi(v[i + 2]);
    a.cache.kv_heads = atoi(v[i + 2]);
    a.cache.L = atoi(v[i + 3]);
    a.cache.wide = 64;
    a.cus = 256;
    tfd::cached_plan(a);
    printf("%d", (int)a.prompt);
  }
}
"""


def rows_and_prompts():
    """(rows, heads, kv_heads, length), for the rows kernel and for the prompt kernel."""
    case = lambda i: (len(single.CASES[i][7]), *single.CASES[i][:2], single.CASES[i][6])
    shape = lambda i: (*list(decision.shapes())[i][:3], list(decision.shapes())[i][4])
    call = lambda i: (*decision.CALLS[i][:3], decision.CALLS[i][4])
    few = [case(i) for i in (0, 1, 2, 3, 4, 5, 7, 8)] + [shape(i) for i in (4, 5, 9, 10)]
    few += [call(i) for i in (0, 2, 3, 5)] + [(2, 8, 1, 1), (33, 8, 1, 2), scales.SINGLE, (256, 1, 1, 1)]
    many = [case(i) for i in (6, 9)] + [shape(i) for i in (0, 1, 2, 3, 6, 7, 8, 11, 12, 13)]
    many += [call(i) for i in (1, 4)] + [(33, 8, 1, L) for L in (9, 17, 20, 33, 131)] + [scales.PROMPT]
    return few, many


def test_the_kernel_of_each_case(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    source, program = tmp_path / "choice.hip", tmp_path / "choice"
    source.write_text(SOURCE)
    build = os.path.join(PKG, "_build")
    subprocess.run([HIPCC, "--cuda-host-only", "-std=c++17", "-w", "-I" + os.path.join(PKG, "csrc"),
                    "-I" + os.path.join(ROOT, "include"), str(source), "-L" + build, "-ltfd_attention",
                    "-Wl,-rpath," + build, "-o", str(program)], check=True, timeout=300)
    few, many = rows_and_prompts()
    args = [str(x) for s in few + many for x in s]
    got = subprocess.run([str(program), *args], capture_output=True, text=True, check=True, timeout=60)
    wrong = [s for s, kernel, want in zip(few + many, got.stdout, "0" * len(few) + "1" * len(many))
             if kernel != want]
    assert len(got.stdout) == len(few) + len(many) and not wrong
