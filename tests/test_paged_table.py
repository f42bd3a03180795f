"""The paged cache without a GPU: what a batch's tables become and are refused for (csrc/paged_table.h), the frequencies of a
rotation (csrc/rotation_table.h), and the refusals of the constructors."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import paged_cases as PC
from helpers import ROOT, pkg

PROGRAM = r"""
#include "paged_table.h"
#include "rotation_table.h"
#include <cstdlib>
#include <cstring>
using namespace itak;
int main(int argc, char **argv) {
    if (!strcmp(argv[1], "frequencies")) {
        itak_rotation_config c{};
        c.rotary_dim = atoi(argv[2]), c.base = atof(argv[3]), c.scaling = atoi(argv[4]), c.factor = atof(argv[5]);
        c.original_positions = atof(argv[6]);
        if (const char *wrong = rotation_refusal(c)) return printf("%s\n", wrong), 0;
        for (double f : rotation_frequencies(c)) printf("%.17g ", f);
        printf("%.17g\n", rotation_amplitude(c));
        return 0;
    }
    // page_count page_rows max_sequences max_table_pages, then batches: n, n x (position rows pages), ids, the ids
    int at = 1;
    auto next = [&] { return strtoull(argv[at++], nullptr, 0); };
    PagedLimits lim;
    lim.page_count = next(), lim.page_rows = next(), lim.max_sequences = next(), lim.max_table_pages = next();
    std::vector<uint32_t> marks(lim.page_count, 0);
    uint32_t stamp = 0xfffffffd;  // (about to wrap)
    PagedBatch b;
    while (at < argc) {
        std::vector<itak_paged_item> items(next());
        for (auto &it : items) it.position = next(), it.rows = next(), it.pages = next();
        std::vector<uint32_t> ids(next());
        for (auto &id : ids) id = next();
        const PagedRefusal r = make_paged_batch(lim, items.data(), items.size(), ids.data(), ids.size(), marks, stamp, b);
        if (r.code) { printf("%d %s\n", r.code, r.text.c_str()); continue; }
        printf("0 rows=%u most=%u", b.rows, b.most_rows);
        for (uint32_t w : b.head) printf(" %u", w);
        printf(" |");
        for (uint32_t w : b.ids) printf(" %u", w);
        printf("\n");
    }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("paged")
    src, exe = folder / "table.cpp", folder / "table"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=address,undefined", "-D_GLIBCXX_DEBUG", "-I",
                    os.path.join(ROOT, "itak-torch-rebuild_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    return lambda *args: subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True).stdout.splitlines()


def batch(items, tables):
    flat = [x for it, t in zip(items, tables) for x in (*it, len(t))]
    ids = [p for t in tables for p in t]
    return [len(items), *flat, len(ids), *ids]


def test_a_batch_becomes_words(program):
    limits = (10, 16, 4, 8)
    out, = program(*limits, *batch([(0, 1), (17, 0), (31, 2)], [[5], [1, 2], [7, 0, 9]]))
    # Two active items of three rows; ids begin at word 4 + 4 * 4, the idle sequence's among them.
    assert out == "0 rows=3 most=2 2 3 0 0 0 1 0 20 31 2 1 23 | 5 1 2 7 0 9"
    assert program(*limits, *batch([], [])) == ["0 rows=0 most=0 0 0 0 0 |"]


def test_what_a_batch_is_refused_for(program):
    limits = (10, 16, 2, 4)
    one = lambda items, tables: program(*limits, *batch(items, tables))[0]  # noqa: E731
    assert one([(0, 1)] * 3, [[0], [1], [2]]).startswith("19 a batch of 3 sequences")
    assert one([(60, 20)], [[0, 1, 2, 3, 4]]).startswith("19 a batch of 5 page ids")
    assert one([(0, 1)], [[10]]).startswith("17 page 10 out of range")
    assert one([(16, 1)], [[3]]).startswith("4 item 0: 17 positions need 2 pages, got 1")
    assert one([(2 ** 31 - 1, 1)], [[3]]).startswith("3 item 0: positions reach 2^31")
    assert one([(2 ** 64 - 1, 1)], [[3]]).startswith("3 ")
    assert program(*limits, 1, 0, 1, 2, 1, 0)[0].startswith("4 page_ids: got 1, the items name 2")
    # A page that takes new rows: twice in one table, in two tables as written, as read, of an idle sequence, as spare.
    for items, tables in ([(16, 1)], [[3, 3]]), ([(0, 1), (0, 1)], [[3], [3]]), ([(0, 1), (16, 1)], [[3], [3, 4]]), \
                         ([(0, 1), (5, 0)], [[3], [3]]), ([(0, 1), (0, 1)], [[3], [4, 3]]), ([(15, 2)], [[3, 4, 3]]):
        assert one(items, tables).startswith("17 page 3 takes new rows and is named"), (items, tables)
    # Shared pages that are only read are fine, also between calls (the marks of a refused one do not stay).
    good = batch([(16, 1), (20, 2)], [[3, 4], [3, 5]])
    bad = batch([(16, 1), (0, 1)], [[3, 4], [3]])
    outs = program(*limits, *good, *bad, *good, *bad, *good)
    assert [o.split()[0] for o in outs] == ["0", "17", "0", "17", "0"] and outs[0] == outs[2] == outs[4]


@pytest.mark.parametrize("scaling,factor", [("plain", 1.0), ("linear", 4.0), ("yarn", 8.0)])
@pytest.mark.parametrize("rotary,base", [(128, 1e6), (64, 1e4), (2, 10.0)])
def test_frequencies(program, scaling, factor, rotary, base):
    got = [float(x) for x in program("frequencies", rotary, base, ["plain", "linear", "yarn"].index(scaling), factor, 4096)[0].split()]
    want, amplitude = PC.frequencies(rotary, base, scaling, factor, 4096)
    assert np.allclose(got[:-1], want.numpy(), rtol=1e-14, atol=0) and abs(got[-1] - amplitude) < 1e-15
    if scaling == "yarn" and rotary == 128:
        plain, _ = PC.frequencies(rotary, base)
        assert got[0] == plain[0] and math.isclose(got[-2], plain[-1] / factor, rel_tol=1e-14)


def test_rotations_are_refused_by_name(program):
    for args, text in (((3, 1e4, 0, 1, 0), "rotary_dim"), ((0, 1e4, 0, 1, 0), "rotary_dim"), ((258, 1e4, 0, 1, 0), "rotary_dim"),
                       ((64, 1, 0, 1, 0), "base"), ((64, "inf", 0, 1, 0), "base"), ((64, 1e4, 3, 1, 0), "scaling"),
                       ((64, 1e4, 1, 0.5, 0), "factor"), ((64, 1e4, 2, "nan", 9), "factor"), ((64, 1e4, 2, 2, 0), "original_positions")):
        assert text in program("frequencies", *args)[0]
    for kw in (dict(rotary_dim=3), dict(rotary_dim=64, base=1.0), dict(rotary_dim=64, amplitude=-1.0),
               dict(rotary_dim=64, scaling="yarn", factor=2.0, original_positions=64.0, beta_fast=1.0, beta_slow=2.0)):
        with pytest.raises(pkg().AttentionError) as e:
            pkg().Rotation(**kw)
        assert e.value.variant == "InvalidArgument"


def test_paged_caches_are_refused_by_name():
    def refused(variant, **kw):
        with pytest.raises(pkg().AttentionError) as e:
            pkg().PagedKv(**{**dict(layers=1, num_kv_heads=2, head_dim=64, page_count=4), **kw})
        assert e.value.variant == variant, (kw, e.value)

    refused("ZeroDimension", layers=0)
    refused("ZeroDimension", num_kv_heads=0)
    refused("ZeroDimension", head_dim=0)
    refused("ZeroDimension", page_count=0)
    refused("ZeroDimension", max_sequences=0)
    refused("InvalidArgument", elem="f32")
    refused("Unsupported", head_dim=12)
    refused("Unsupported", head_dim=264)
    refused("Unsupported", page_rows=8)
    refused("Unsupported", page_rows=48)
    refused("Unsupported", page_rows=2048)
    refused("SizeOverflow", page_count=2 ** 31)
    refused("SizeOverflow", max_sequences=1025)
    refused("SizeOverflow", num_kv_heads=4096, head_dim=256, page_rows=1024, page_count=2 ** 31 - 1, layers=2 ** 32 - 1)
    refused("ShapeMismatch", storage_ptr=1 << 20, storage_bytes=4 * 2 * 2 * 64 * 64 * 2 - 1)
    refused("InvalidArgument", storage_ptr=(1 << 20) + 2, storage_bytes=1 << 30)
    assert pkg().PagedKv.bytes_for(3, 2, 64, page_count=4, page_rows=32) == 3 * 4 * 2 * 2 * 32 * 64 * 2
    assert pkg().PagedKv.bytes_for(3, 2, 65, page_count=4) == 0


def test_calls_without_a_handle_are_refused():
    N = pkg()._native
    lib = N.load()
    rows = N.Rows()
    assert lib.itak_paged_set_batch(None, None, 0, None, 0) == 17
    assert lib.itak_paged_append_device(None, 0, C.byref(rows), C.byref(rows), None) == 17
    assert lib.itak_paged_attention_device(None, 0, C.byref(rows), C.byref(rows), 1.0, 0.0, 0, None) == 17
    assert lib.itak_paged_synchronize(None) == 17 and lib.itak_paged_set_stream(None, None) == 17
    assert lib.itak_rotate_device(None, None, 64, 1, None, None, None, 1, 0) == 17
    assert lib.itak_rotation_frequencies(None, None, None) == 17
    assert not lib.itak_paged_storage(None)
    lib.itak_paged_destroy(None)
    lib.itak_rotation_destroy(None)


def test_views_of_tensors():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="not on a GPU"):
        pkg().Rows.of(torch.zeros(2, 3, 8))
