"""The largest batches and rotations: what a launch does not hold is refused before one is made."""
import pytest
import torch

from helpers import pkg
from test_paged_table import batch, program  # noqa: F401

LAUNCH = (1 << 32) // 256  # rows, a workgroup of 256 threads each, whose threads 32 bits do not count any more


def test_rows_of_a_batch_are_what_a_launch_holds(program):  # noqa: F811
    pages = LAUNCH // 1024
    limits = (pages, 1024, 2, pages)
    most = batch([(0, LAUNCH - 1)], [range(pages)])
    more = batch([(0, LAUNCH)], [range(pages)])
    both = batch([(0, LAUNCH // 2), (0, LAUNCH // 2)], [range(pages // 2), range(pages // 2, pages)])
    fits, *refused = program(*limits, *most, *more, *both)
    assert fits.startswith(f"0 rows={LAUNCH - 1} ")
    for line in refused:
        assert line.startswith("3 more than 2^24 - 1 rows"), line


@pytest.mark.gpu
def test_rows_of_a_rotation_are_what_a_launch_holds():
    P = pkg()
    rotation, x = P.Rotation(8), torch.ones(8, device="cuda")
    positions = torch.zeros(1, dtype=torch.int64, device="cuda")
    for rows in (LAUNCH, LAUNCH + 1, 1 << 40):
        with pytest.raises(P.AttentionError) as e:  # (refused by the count alone: nothing lies behind the pointers)
            rotation.rotate_device([P.Rows(x.data_ptr(), "f32", 1)], [P.Rows(x.data_ptr(), "f32", 1)], positions.data_ptr(), rows, 8)
        assert e.value.variant == "SizeOverflow"
    torch.cuda.synchronize()
    assert bool((x == 1.0).all())
