"""The wait states before loads from assembly (test_paged_asm.py) in the other forms of the kernel of many rows: f32 tensors, bf16 pages.
Their loops are other schedules of the same source."""
import os
import subprocess
import sys

import pytest

from helpers import ROOT
from test_paged_asm import CSRC, HIPCC, early


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is not installed")
@pytest.mark.parametrize("form", ["f16_f32", "bf16", "bf16_f32"])
def test_addresses_are_old_enough_for_the_loads_that_read_them(tmp_path, form):
    sys.path.insert(0, ROOT)
    from __graft_entry__ import _load_builder

    build = _load_builder()
    src, out = f"paged_chunk_{form}.hip", str(tmp_path / "kernel.s")
    flags = [f for f in build.FLAGS if not f.startswith("-Rpass")]
    subprocess.run([HIPCC, *flags, *build.source_flags(src), "--cuda-device-only", "-S", os.path.join(CSRC, src), "-o", out],
                   check=True, capture_output=True)
    bad, loads = early(open(out).read().split("\n"))
    assert loads > 100 and not bad, bad[:5]
