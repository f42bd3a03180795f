"""Where the kernels look up the records of a batch's rows, without a GPU."""
import os
import subprocess

from helpers import ROOT

PROGRAM = r"""
#include "paged_tree.h"
#include <cstdio>
using namespace itak;
int main() {
    // Of a handle whose trees have up to `most` rows: every word of a record that a kernel may read of row `row`, with records and without.
    const uint64_t most = 2, rows[] = {0, 1, 2, 63, 8191, (1ull << 24) - 1};
    for (uint64_t row : rows) {
        const uint64_t last = tree_record_at(false, row) + kTreeStride - 1;
        printf("%d", int(last < most * kTreeStride));
    }
    printf(" %d%d\n", int(tree_record_at(true, 1) == kTreeStride), int(tree_record_at(true, (1ull << 24) - 1) == ((1ull << 24) - 1) * kTreeStride));
}
"""


def test_rows_without_records_are_looked_up_where_there_is_one(tmp_path):
    src, exe = tmp_path / "at.cpp", tmp_path / "at"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "itak-torch-rebuild_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "111111 11\n"
