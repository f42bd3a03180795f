"""The largest batches and rotations: what a launch does not hold is refused before one is made."""
import numpy as np
import pytest
import torch

from helpers import pkg, refusal
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


# One token of 32 KV heads at 2^30 positions are 32 units of 2^25 blocks. Of such a batch a captured call, which finds its work on the device,
# would lose count; with a window it goes through three blocks. (All pages but the one the token stands in are one.)
@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 64])
def test_positions_that_a_replay_cannot_count_are_refused(window):
    P, heads, d, far = pkg(), 32, 8, 1 << 30
    storage = torch.randn(1, 2, 2, heads, 1024, d, device="cuda").half()
    paged = P.PagedKv(1, heads, d, page_rows=1024, page_count=2, max_sequences=1, max_table_pages=far // 1024 + 1,
                      storage_ptr=storage.data_ptr(), storage_bytes=storage.numel() * 2)
    stream, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    paged.set_stream(stream.cuda_stream)
    q = torch.randn(1, heads, d, device="cuda").half()
    out = torch.zeros_like(q)
    attend = lambda: paged.attention_device(0, P.Rows.of(q), P.Rows.of(out), window=window)  # noqa: E731
    near = ([(900, 1)], [np.array([1], np.uint32)])
    table = np.zeros(far // 1024 + 1, np.uint32)
    table[-1] = 1
    paged.set_batch([(far, 1)], [table])  # (nothing has been captured)
    paged.set_batch(*near)
    attend()
    torch.cuda.synchronize()
    want = out.clone()
    paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        attend()
    paged.set_stream(stream.cuda_stream)
    if window:
        paged.set_batch([(far, 1)], [table])
        attend()
        torch.cuda.synchronize()
        want = out.clone()
    else:
        assert refusal(lambda: paged.set_batch([(far, 1)], [table])) == "SizeOverflow"
    for _ in range(3):  # (over the far batch, or the one before the refused)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # (An eager call cuts the keys otherwise: two outputs of up to 4 rounded to f16, and weights too.)
        assert bool(((out - want).abs() <= 2.0 ** -7).all()) and bool(out.any())
