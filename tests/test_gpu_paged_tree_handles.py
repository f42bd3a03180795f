"""Handles that take trees beside what else a program does with them: plain prompts in graphs that hold more rows than trees may have, sequences
without rows in graphs from before, what memory calls take and when, and calls that are refused."""
import pytest
import torch

import paged_cases as PC
import tree_cases as TC
from helpers import pkg, refusal
from test_gpu_paged import check_attention
from test_gpu_paged_trees import cache_of, view

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


# A graph looks at all sequences of the batch that is there when it runs, also where it was captured over one without those that have no rows: once trees
# are taken, and of a batch that the device makes, these count too.
@pytest.mark.parametrize("later", ["trees are taken", "from the device"])
@pytest.mark.parametrize("rows,heads", [(1, 4), (20, 8), (300, 4)])
def test_graphs_captured_over_a_batch_that_left_sequences_out(rows, heads, later):
    new = [rows, 0, rows, 0, rows]
    items = list(zip([20, 9, 33, 0, 70], new))
    cache = PC.Cache(pkg(), [p + r for p, r in items], kv_heads=2, d=64, page_rows=16, seed=rows)
    q = cache.normal(3 * rows, heads, 64).half()
    qd = q.cuda()
    out = torch.zeros_like(qd)
    positions, slots = (torch.zeros(3 * rows, dtype=torch.int64, device="cuda") for _ in range(2))

    def forward():
        cache.paged.attention_device(0, view(qd), view(out))
        cache.paged.batch_rows_device(positions.data_ptr(), slots.data_ptr())

    cache.paged.set_batch(items, cache.tables)
    forward()
    graph = captured(cache.paged, forward)
    if later == "trees are taken":
        cache.paged.enable_trees(3 * rows)
        cache.paged.set_batch(items, cache.tables)
    else:
        width = max(len(t) for t in cache.tables)
        tables = pkg().PageTables.of(i32([t + [0] * (width - len(t)) for t in cache.tables]), i32([len(t) for t in cache.tables]))
        held = i32([p for p, _ in items])
        cache.paged.set_batch_device(tables, held.data_ptr(), new, 100)
    for _ in range(3):
        out.fill_(7.0), positions.fill_(-7), slots.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(cache, 0, items, q, out, "f16")
        assert positions.tolist() == [p + r for p, n in items for r in range(n)]
        assert slots.tolist() == [cache.tables[s][x // 16] * 16 + x % 16 for s, (p, n) in enumerate(items) for x in range(p, p + n)]


def test_a_plain_call_takes_the_memory_that_it_needs_and_a_graph_finds_its_own():
    # What graphs of trees may need lies there from enable_trees on. (A handle that takes none makes the same call first, so that its kernels are loaded; its
    # own partials are below 32 MiB.)
    P, items = pkg(), [(100, 600)]
    q = torch.randn(600, 8, 128, generator=torch.Generator().manual_seed(1)).half()
    qd = q.cuda()
    out = torch.zeros_like(qd)
    free = lambda: (torch.cuda.synchronize(), torch.cuda.mem_get_info()[0])[1]  # noqa: E731
    for trees in (False, True):
        cache = PC.Cache(P, [700], kv_heads=2, d=128, page_rows=64)
        if trees:
            cache.paged.enable_trees(8)
        cache.paged.set_batch(items, cache.tables)
        before = free()
        cache.paged.attention_device(0, view(qd), view(out))
        took = before - free()
    assert took < 32 << 20, took
    graph = captured(cache.paged, lambda: cache.paged.attention_device(0, view(qd), view(out)))
    assert before - free() < (32 << 20) + (64 << 20)  # (the graph's kernels)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(cache, 0, [(100, 5)], q[:5], out[:5], "f16")
        check_attention(cache, 0, [(695, 5)], q[-5:], out[-5:], "f16")


# What a call was refused for it says itself: the next one, of the handle or of the program's own, does not.
def test_a_call_refused_for_memory_leaves_the_next_alone():
    P, heads, kv_heads, d, rows = pkg(), 64000, 1000, 8, 1 << 19
    cache = PC.Cache(P, [40], kv_heads=kv_heads, d=d, page_rows=16, seed=2)
    rotation = P.Rotation(d)
    tables = P.PageTables.of(i32([cache.tables[0]]), i32([len(cache.tables[0])]))
    nowhere, held = i32([-1]), i32([30])
    x = torch.zeros(8, dtype=torch.float32, device="cuda")
    cache.paged.set_batch_device(tables, nowhere.data_ptr(), [rows], 30)
    # (1 TB of turned queries; nothing is launched, so nothing lies behind the pointers.)
    q, out = P.Rows(x.data_ptr(), "f32", heads), P.Rows(x.data_ptr() + 16, "f32", heads)
    assert refusal(lambda: cache.paged.attention_device(0, q, out, rotation=rotation)) == "HipError"
    q = cache.normal(3, kv_heads, d).half()
    qd = q.cuda()
    out = torch.zeros_like(qd)
    cache.paged.set_batch_device(tables, held.data_ptr(), [3], 30)
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    check_attention(cache, 0, [(30, 3)], q, out, "f16")


def test_trees_that_a_graph_has_too_short_a_window_for_are_refused_by_name():
    items = [(100, 9)]
    cache = cache_of(items, kv_heads=1, d=64, page_rows=16)
    q = cache.normal(9, 2, 64).half()
    qd = q.cuda()
    out = torch.zeros_like(qd)
    attend = lambda: cache.paged.attention_device(0, view(qd), view(out), window=8)  # noqa: E731
    cache.paged.set_batch(items, cache.tables)
    attend()
    graph = captured(cache.paged, attend)
    wide, parents = [-1] + [0] * 8, i32([-1] + [0] * 8)
    tables, held = pkg().PageTables.of(i32([cache.tables[0]]), i32([len(cache.tables[0])])), i32([100])
    for call in (lambda: cache.paged.set_batch(items, cache.tables, TC.flat([wide])),
                 lambda: cache.paged.set_batch_device(tables, held.data_ptr(), [9], 100, parents.data_ptr())):
        try:
            call()
            said = None
        except pkg().AttentionError as e:
            said = e.variant, e.message
        assert said and said[0] == "Unsupported" and "a window of 8" in said[1] and "a tree of 9 rows" in said[1] and "captured" in said[1]
        out.zero_()
        graph.replay()  # (over the batch before)
        torch.cuda.synchronize()
        check_attention(cache, 0, items, q, out, "f16", window=8)
    cache.paged.set_batch(items, cache.tables, TC.flat([TC.chain(9)]))
    cache.paged.set_batch([(100, 8)], cache.tables, TC.flat([wide[:8]]))


# A graph may set a batch that the host does not see: attention that is captured afterwards is refused what it could not do over it.
def test_attention_captured_behind_a_graph_that_sets_larger_trees():
    items, star = [(100, 9)], [-1] + [0] * 8
    cache = cache_of(items, kv_heads=1, d=64, page_rows=16)
    q = cache.normal(9, 2, 64).half()
    qd = q.cuda()
    out = torch.zeros_like(qd)
    tables, held, parents = pkg().PageTables.of(i32([cache.tables[0]]), i32([len(cache.tables[0])])), i32([100]), i32(star)
    sets = captured(cache.paged, lambda: cache.paged.set_batch_device(tables, held.data_ptr(), [9], 100, parents.data_ptr()))
    cache.paged.set_batch(items, cache.tables)
    said, graphs = [], []
    for window in (8, 9):
        attend = lambda: cache.paged.attention_device(0, view(qd), view(out), window=window)  # noqa: E731
        attend()
        graphs.append(captured(cache.paged, lambda: said.append(refusal(attend))))
    assert said == ["Unsupported", None]
    for _ in range(3):
        out.zero_()
        sets.replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        TC.check(cache, 0, items, [star], q, out, "f16", window=9)


def test_attention_captured_behind_a_graph_that_sets_more_blocks_than_it_can_count():
    # 32 heads' 2^25 blocks each at 2^30 positions.
    P, heads, d, far = pkg(), 32, 8, 1 << 30
    storage = torch.randn(1, 2, 2, heads, 1024, d, device="cuda").half()
    paged = P.PagedKv(1, heads, d, page_rows=1024, page_count=2, max_sequences=1, max_table_pages=far // 1024 + 1,
                      storage_ptr=storage.data_ptr(), storage_bytes=storage.numel() * 2)
    paged.set_stream(torch.cuda.current_stream().cuda_stream)
    q = torch.randn(1, heads, d, device="cuda").half()
    out = torch.zeros_like(q)
    tables, held = P.PageTables.of(i32([[1]]), i32([1])), i32([900])
    sets = captured(paged, lambda: paged.set_batch_device(tables, held.data_ptr(), [1], far))
    paged.set_batch([(900, 1)], [[1]])
    said, graphs = [], []
    for window in (0, 64):
        attend = lambda: paged.attention_device(0, view(q), view(out), window=window)  # noqa: E731
        attend()
        graphs.append(captured(paged, lambda: said.append(refusal(attend))))
    assert said == ["SizeOverflow", None]
    torch.cuda.synchronize()
    want = out.clone()
    for _ in range(3):
        out.zero_()
        sets.replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        # (Captured the keys are cut otherwise: two outputs of up to 4 rounded to f16, and weights too.)
        assert bool(((out - want).abs() <= 2.0 ** -7).all()) and bool(out.any())


def test_joins_of_more_vectors_than_a_launch_has_in_one_dimension():
    # Of 2^20 rows by 64 heads, all rows but the last are of a sequence that the device leaves out.
    rows, heads, d = 1 << 20, 64, 8
    cache = PC.Cache(pkg(), [16, 31], kv_heads=heads, d=d, page_rows=16, seed=4)
    cache.paged.enable_trees(rows)
    qd, out = torch.zeros(rows, heads, d, dtype=torch.float16, device="cuda"), torch.full((rows, heads, d), 7.0, dtype=torch.float16, device="cuda")
    q = cache.normal(1, heads, d).half()
    qd[-1:] = q.cuda()
    parents = torch.arange(-1, rows - 1, dtype=torch.int32, device="cuda")
    parents[-1] = -1
    tables, held, status = pkg().PageTables.of(i32([[0, 0], cache.tables[1]]), i32([1, 2])), i32([-1, 30]), i32([9, 9])
    cache.paged.set_batch_device(tables, held.data_ptr(), [rows - 1, 1], 30, parents.data_ptr(), status.data_ptr())
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    assert status.tolist() == [1, 0] and bool((out[:-1] == 7.0).all())
    check_attention(cache, 0, [(0, 0), (30, 1)], q, out[-1:], "f16")


def test_a_graph_that_sets_its_own_batch_goes_by_it_alone():
    # Trees of nine rows in a graph without windows, and of eight in another with one of eight.
    star = [-1] + [0] * 8
    cache = cache_of([(100, 9)], kv_heads=1, d=64, page_rows=16)
    q = cache.normal(9, 2, 64).half()
    qd = q.cuda()
    outs = [torch.zeros_like(qd) for _ in range(2)]
    tables, held, parents = pkg().PageTables.of(i32([cache.tables[0]]), i32([len(cache.tables[0])])), i32([100]), i32(star)

    def forward(rows, window):
        cache.paged.set_batch_device(tables, held.data_ptr(), [rows], 100, parents.data_ptr())
        cache.paged.attention_device(0, view(qd[:rows]), view(outs[rows - 8][:rows]), window=window)

    forms = (9, 0), (8, 8)
    for form in forms:
        forward(*form)
    graphs = [captured(cache.paged, lambda: forward(*form)) for form in forms]
    for _ in range(3):
        for graph, (rows, window) in zip(graphs, forms):
            outs[rows - 8].zero_()
            graph.replay()
            torch.cuda.synchronize()
            TC.check(cache, 0, [(100, rows)], [star[:rows]], q[:rows], outs[rows - 8][:rows], "f16", window=window)
