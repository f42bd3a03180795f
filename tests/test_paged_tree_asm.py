"""The wait states before loads from assembly (test_paged_asm.py) in the kernel of trees and in the kernel of many rows over batches of trees."""
import os
import subprocess
import sys

import pytest

from helpers import ROOT
from test_paged_asm import CSRC, HIPCC, early


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is not installed")
@pytest.mark.parametrize("src", [f"paged_{kernel}_{form}.hip" for kernel in ("trees", "chunk_tree") for form in ("f16", "f16_f32", "bf16", "bf16_f32")])
def test_addresses_are_old_enough_for_the_loads_that_read_them(tmp_path, src):
    sys.path.insert(0, ROOT)
    from __graft_entry__ import _load_builder

    build = _load_builder()
    out = str(tmp_path / "kernel.s")
    flags = [f for f in build.FLAGS if not f.startswith("-Rpass")]
    subprocess.run([HIPCC, *flags, *build.source_flags(src), "--cuda-device-only", "-S", os.path.join(CSRC, src), "-o", out],
                   check=True, capture_output=True)
    bad, loads = early(open(out).read().split("\n"))
    # (Of the kernel of trees at least two places that send loads, with 1, 2 and 8 of them for 64, 128 and 256 channels.)
    assert loads >= 2 * 2 * (1 + 2 + 8) and not bad, bad[:5]
