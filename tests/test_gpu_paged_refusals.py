"""Calls over pages that are refused late, for their size or for memory they cannot have: nothing of them has been enqueued."""
import pytest
import torch

import paged_cases as PC
from helpers import pkg, refusal
from test_gpu_paged import view
from test_gpu_paged_serving import filled

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


class Call:
    """A batch and its tensors."""

    def __init__(self, cache, items, q_heads, rotation=None):
        self.cache, self.items, self.rotation = cache, items, rotation
        rows = sum(r for _, r in items)
        self.q, self.k, self.v = (cache.normal(rows, h, cache.d).half().cuda() for h in (q_heads, cache.kv_heads, cache.kv_heads))
        self.out = torch.full_like(self.q, 7.0)

    def set(self):
        self.cache.paged.set_batch(self.items, self.cache.tables[:len(self.items)])

    def step(self):
        self.cache.paged.attention_step_device(0, view(self.q), view(self.k), view(self.v), view(self.out), rotation=self.rotation)

    def attend(self):
        self.cache.paged.attention_device(0, view(self.q), view(self.out), rotation=self.rotation)


# A capture that needs more memory holds nothing of the refused call: not the append before the attention, not the few rows' part of
# a batch before the many rows'. `earlier`: calls that made a part of the memory.
@pytest.mark.parametrize("items,earlier,rotated,attend", [
    ([(3999, 1)], [], False, False),
    ([(3999, 1)], [], True, True),
    ([(3999, 1)], [[(0, 64)]], True, False),        # the rotated queries' memory is there, that of the parts is not
    ([(3999, 1)], [[(0, 64)]], True, True),
    ([(1999, 1), (2000, 60)], [[(1999, 1)]], False, False),
    ([(1999, 1), (2000, 60)], [[(1999, 1)]], False, True),
])
def test_a_refused_capture_is_empty(items, earlier, rotated, attend):
    P = pkg()
    cache = filled([4096, 4096], kv_heads=8, d=256, page_rows=64, seed=len(items))
    rotation = P.Rotation(256) if rotated else None
    for batch in earlier:
        call = Call(cache, batch, 64 if rotated else 8, rotation)
        call.set()
        call.attend()
    call = Call(cache, items, 8, rotation)
    call.set()
    torch.cuda.synchronize()
    side, graph, mark = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    before = cache.storage.clone()
    torch.cuda.synchronize()
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        refused = refusal(call.attend if attend else call.step)
        mark.add_(1.0)
    assert refused == "CapacityExceeded"
    for n in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert float(mark) == n + 1.0
        assert same(before, cache.storage) and bool((call.out == 7.0).all())
    (call.attend if attend else call.step)()  # (uncaptured it gets what it needs)
    cache.paged.synchronize()
    assert not bool((call.out == 7.0).any())


def test_a_step_of_too_many_query_vectors_has_not_appended():
    # 2^20 rows of 64 heads over one, 8 channels: 2^26 query vectors a KV head.
    P, rows = pkg(), 1 << 20
    storage = torch.zeros(1, 1024, 2, 1, 1024, 8, dtype=torch.float16, device="cuda")
    paged = P.PagedKv(1, 1, 8, page_rows=1024, page_count=1024, max_sequences=1, storage_ptr=storage.data_ptr(),
                      storage_bytes=storage.numel() * 2)
    paged.set_stream(torch.cuda.current_stream().cuda_stream)
    q = torch.ones(1, 64, 8, dtype=torch.float16, device="cuda").expand(rows, 64, 8)
    k = torch.ones(rows, 1, 8, dtype=torch.float16, device="cuda")
    out = torch.full((rows, 64, 8), 7.0, dtype=torch.float16, device="cuda")
    paged.set_batch([(0, rows)], [list(range(1024))])
    for rotation in (None, P.Rotation(8)):
        assert refusal(lambda: paged.attention_step_device(0, view(q), view(k), view(k), view(out), rotation=rotation)) == "SizeOverflow"
        torch.cuda.synchronize()
        assert not bool(storage.any()) and bool((out == 7.0).all())
