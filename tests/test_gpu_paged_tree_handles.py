"""Handles that take trees beside what else a program does with them: plain prompts in graphs that hold more rows than trees may have, sequences
without rows in graphs from before, what memory calls take and when, and windows that graphs hold trees to."""
import pytest
import torch

import paged_cases as PC
from helpers import pkg
from test_gpu_paged import check_attention
from test_gpu_paged_trees import view

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def captured(paged, call):
    """A graph of a call of `paged`, whose stream is the current one before and after."""
    stream, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        call()
    paged.set_stream(stream.cuda_stream)
    return graph


# A captured call over a prompt of more rows than trees may have looks no record up: there are none behind the last. (8,192 rows of 4 vectors a KV head are
# the kernel of many rows', smaller batches the kernel of trees', and the tokens beside them that of few rows.)
@pytest.mark.parametrize("prompt,kv_heads,heads,d,pages,tensors", [
    (8192, 1, 4, 128, "f16", "f16"), (8192, 1, 4, 64, "bf16", "f32"), (700, 2, 4, 64, "bf16", "bf16"), (300, 1, 2, 256, "f16", "f32")])
def test_captured_prompts_of_more_rows_than_trees_may_have(prompt, kv_heads, heads, d, pages, tensors):
    items = [(40, 1), (100, prompt), (7, 2)]
    cache = PC.Cache(pkg(), [p + r for p, r in items], kv_heads=kv_heads, d=d, pages=pages, page_rows=64, seed=prompt)
    cache.paged.enable_trees(2)
    q = cache.normal(prompt + 3, heads, d).to(PC.DTYPES[tensors])
    qd = q.cuda()
    out = torch.zeros_like(qd)
    attend = lambda: cache.paged.attention_device(0, view(qd), view(out))  # noqa: E731
    cache.paged.set_batch(items, cache.tables)
    attend()
    graph = captured(cache.paged, attend)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert bool(out.isfinite().all())
        check_attention(cache, 0, [(40, 1)], q[:1], out[:1], tensors)
        check_attention(cache, 0, [(40, 0), (100, 0), (7, 2)], q[-2:], out[-2:], tensors)
        for row in (0, 60, prompt // 2, prompt - 5):  # (some rows of the prompt: all of them in 64 bits take minutes)
            mine = slice(1 + row, 1 + row + 5)
            check_attention(cache, 0, [(40, 0), (100 + row, 5)], q[mine], out[mine], tensors)
