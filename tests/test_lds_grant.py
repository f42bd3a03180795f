"""The grant of dynamic LDS (csrc/lds_grant.h), compiled for the host: one for every kernel and device."""
import os
import subprocess

from helpers import ROOT

CSRC = os.path.join(ROOT, "itak-torch-rebuild_amd", "csrc")

PROGRAM = r"""
#include "lds_grant.h"
#include <cstdio>
template <int N> void kernel(int) {}
int calls[2];
template <int N> int ask(int device, int answer = 0) {
    return itak::granted_once<&kernel<N>>(device, [&] { ++calls[N]; return answer; });
}
int main() {
    // Two kernels of one type, two devices, a grant that fails first, a device beyond the marks.
    if (ask<0>(0, 7) != 7 || ask<0>(0) != 0 || ask<0>(0) != 0 || ask<1>(0) != 0 || ask<1>(0) != 0) return 1;
    if (calls[0] != 2 || calls[1] != 1) return 2;
    if (ask<0>(3) || ask<0>(3) || ask<0>(0) || calls[0] != 3) return 3;
    if (ask<1>(64) || ask<1>(64) || calls[1] != 3) return 4;
    puts("fine");
}
"""


def test_every_kernel_and_device_has_a_grant_of_its_own(tmp_path):
    src, exe = tmp_path / "grant.cpp", tmp_path / "grant"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert (out.returncode, out.stdout) == (0, "fine\n")


def test_many_rows_over_pages_ask_by_kernel():
    text = open(os.path.join(CSRC, "paged_chunk_kernel.h")).read()
    assert "granted_once<Kernel>" in text and "static const hipError_t granted" not in text
