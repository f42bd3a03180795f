"""The calls of trees and of batches that the device makes, without a GPU: what the compiled front module takes, and the words that trees become."""
import os
import subprocess

import numpy as np
import pytest

from helpers import ROOT, pkg
from test_paged_front import REFUSED, front

PROGRAM = r"""
#include "paged_table.h"
#include "paged_tree.h"
#include <cstdlib>
using namespace itak;
int main(int argc, char **argv) {
    std::vector<int32_t> parents;
    for (int i = 1; i < argc; ++i) parents.push_back(atoi(argv[i]));
    printf("%d %llu\n", int(tree_is_chain(parents.data(), parents.size())), (unsigned long long)tree_first_wrong(parents.data(), parents.size()));
    // Sequences without rows keep their number where a handle takes trees.
    const itak_paged_item items[3] = {{3, 2, 1}, {9, 0, 1}, {0, 1, 1}};
    const uint32_t ids[3] = {4, 0, 2};
    std::vector<uint32_t> marks(8, 0);
    uint32_t stamp = 0;
    for (bool keep : {false, true}) {
        PagedBatch b;
        const PagedRefusal r = make_paged_batch(PagedLimits{8, 16, 3, 8}, items, 3, ids, 3, marks, stamp, b, keep);
        printf("%d %u:", r.code, b.items);
        for (uint32_t w : b.head) printf(" %u", w);
        printf("\n");
    }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("tree")
    src, exe = folder / "tree.cpp", folder / "tree"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=address,undefined", "-D_GLIBCXX_DEBUG", "-I",
                    os.path.join(ROOT, "itak-torch-rebuild_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    return lambda *args: subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True).stdout.splitlines()


def test_parents(program):
    for parents, chain, wrong in (([-1], 1, 1), ([-1, 0, 1, 2], 1, 4), ([-1, 0, 0], 0, 3), ([-1, -1], 0, 2), ([0], 0, 0), ([-1, 1], 0, 1),
                                  ([-1, 0, -2], 0, 2), ([-1, 0, 1, 7], 0, 3), ([], 1, 0)):
        assert program(*parents)[0] == f"{chain} {wrong}", parents
    without, with_ = program(-1)[1:]
    assert without == "0 2: 2 3 0 0 3 2 0 16 0 1 2 18"
    assert with_ == "0 3: 3 3 0 0 3 2 0 16 9 0 2 17 0 1 2 18"


def test_only_plain_arguments_are_taken():
    f = front()
    ids, parents = np.array([3, 1], np.uint32), np.array([-1, 0], np.int32)
    assert f.set_batch_tree(0, [(0, 2)], [ids], parents) == REFUSED
    for odd in ([-1, 0], parents.astype(np.int64), parents.astype(np.uint32), parents[:1], parents[:0], np.array([[-1, 0]], np.int32), None):
        assert f.set_batch_tree(0, [(0, 2)], [ids], odd) == -1
    assert f.fit_tables(0, 0, 2, 0, None, 0) == f.fit_tables(0, 0, 2, 0, [1, 2], 0) == f.fit_tables(0, 0, 2, 0, (0, 5), 0) == REFUSED
    done = f.set_batch_device(0, 0, 2, 0, [1, 2], 5, 0, 0)
    assert done >> 32 == REFUSED and done & 0xFFFFFFFF == 3
    for rows in ([1], [1, 2, 3], [1, -1], [1, 1 << 32], [1, 2.0], np.array([1, 2]), [1, np.int64(2)], 5):
        assert f.fit_tables(0, 0, 2, 0, rows, 0) == f.set_batch_device(0, 0, 2, 0, rows, 5, 0, 0) == -1
    assert f.set_batch_device(0, 0, 2, 0, [(1 << 32) - 1, 1], 5, 0, 0) == -1
    assert f.set_batch_device(0, 0, 1025, 0, [1] * 1025, 5, 0, 0) == f.set_batch_device(0, 0, 1, 0, [1], -5, 0, 0) == -1
    assert f.batch_rows(0, 0, 0) == f.accept(0, 0, 0, 0, 0) == f.keep(0, 0, 0) == REFUSED
    assert f.batch_rows(0, None, 0) == f.accept(0, 0, 0, 0, np.int64(0)) == f.keep(0, 1.0, 0) == -1
    for call in (f.batch_rows, f.accept, f.keep, f.fit_tables, f.set_batch_device, f.set_batch_tree, f.bind_trees):
        with pytest.raises(TypeError):
            call(0)


def test_tables_are_of_integers_of_32_bits():
    P = pkg()
    with pytest.raises(ValueError):
        P.PageTables(0, 1 << 64, 0, 1)
    with pytest.raises(ValueError):
        P.PageTables(0, 1, 0, 1 << 32)
    import torch

    table, pages = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        P.PageTables.of(table, pages)  # (not on a GPU)
