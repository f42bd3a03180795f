"""Trees over pages and batches from the device at their edges: sequences left out of batches of long splits, replays over long chains beside
trees, layers that differ over one batch, pages far into the storage, handles at work at once, and what is refused."""
import numpy as np
import pytest
import torch

import paged_cases as PC
import tree_cases as TC
from helpers import pkg, refusal
from test_gpu_paged_trees import attend, cache_of, view

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tables_of(cache):
    width = max(len(t) for t in cache.tables)
    return pkg().PageTables.of(i32([t + [0] * (width - len(t)) for t in cache.tables]), i32([len(t) for t in cache.tables]))


def check_one(cache, items, trees, seq, q, out, tensors, window=0):
    """What sequence `seq`'s rows came to."""
    first = sum(r for _, r in items[:seq])
    mine = slice(first, first + items[seq][1])
    alone = [(p, r if s == seq else 0) for s, (p, r) in enumerate(items)]
    TC.check(cache, 0, alone, trees, q[mine], out[mine], tensors, window)


# The host plans for all sequences, the device leaves some out: nothing of theirs is written, also where their parts are joined.
@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("tensors", ["f16", "f32"])
@pytest.mark.parametrize("out_of", [(0,), (1, 2), (0, 1, 2, 3)])
def test_long_sequences_that_the_device_leaves_out(trees, tensors, out_of):
    items = [(6000, 40), (5000, 2), (90, 33), (3000, 1)]
    cache = cache_of(items, kv_heads=1, d=64, page_rows=64, seed=3) if trees else PC.Cache(pkg(), [p + r for p, r in items], kv_heads=1, d=64,
                                                                                           page_rows=64, fill="nan", seed=3)
    if not trees:
        for seq, (p, r) in enumerate(items):
            x = cache.normal(2, p + r, 1, 64).half()
            cache.place(0, seq, 0, x[0], x[1])
    parents = [TC.tree(r, 4) if trees else TC.chain(r) for _, r in items]
    q = cache.normal(76, 4, 64).to(PC.DTYPES[tensors])
    qd, out, status = q.cuda(), torch.full_like(q, 7.0, device="cuda"), i32([9] * 4)
    held = i32([-1 if s in out_of else p for s, (p, _) in enumerate(items)])
    up, tables = torch.from_numpy(TC.flat(parents)).cuda(), tables_of(cache)
    cache.paged.set_batch_device(tables, held.data_ptr(), [r for _, r in items], 6000, up.data_ptr() if trees else 0, status.data_ptr())
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    assert status.tolist() == [int(s in out_of) for s in range(4)]
    first = 0
    for s, (_, r) in enumerate(items):
        if s in out_of:
            assert bool((out[first:first + r] == 7.0).all())
        else:
            check_one(cache, items, parents, s, q, out, tensors)
        first += r


@pytest.mark.parametrize("tensors", ["f16", "f32"])
@pytest.mark.parametrize("window", [0, 64])
def test_replays_over_long_chains_beside_trees(tensors, window):
    now, later = [(0, 400), (40, 1), (500, 30)], [(1700, 400), (0, 1), (64, 30)]
    cache = cache_of([(1700, 400), (500, 1), (500, 30)], kv_heads=1, d=128, pages="bf16", page_rows=32, seed=window)
    q = cache.normal(431, 2, 128).to(PC.DTYPES["bf16" if tensors == "f16" else "f32"])
    kind = "bf16" if tensors == "f16" else "f32"
    qd, out = q.cuda(), torch.empty_like(q, device="cuda")
    stream, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    chains = [TC.chain(400), [-1], TC.chain(30)]
    cache.paged.set_batch(now, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), window=window)
    torch.cuda.synchronize()
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        cache.paged.attention_device(0, view(qd), view(out), window=window)
    cache.paged.set_stream(stream.cuda_stream)
    for n, items in enumerate((later, now, later)):
        trees = chains if n == 1 else [TC.chain(400), [-1], TC.tree(30, n)]
        cache.paged.set_batch(items, cache.tables, None if n == 1 else TC.flat(trees))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s in (0, 1, 2) if n == 0 else (1, 2):
            check_one(cache, items, trees, s, q, out, kind, window)
        again = torch.empty_like(out)
        cache.paged.attention_device(0, view(qd), view(again), window=window)
        torch.cuda.synchronize()
        check_one(cache, items, trees, 2, q, again, kind, window)


# More sequences than a wavefront has lanes, in a graph of the batch, its attention and the lengths' own: cut by the device, split and whole, other sequences
# left out at every replay.
@pytest.mark.parametrize("kv_heads", [1, 4])
def test_replays_over_many_sequences(kv_heads):
    n, nodes, d = 70, 20, 64
    most = [(37 * s) % 701 for s in range(n)]
    cache = cache_of([(p, nodes) for p in most], kv_heads=kv_heads, d=d, page_rows=32, max_sequences=n, seed=kv_heads)
    trees = [TC.tree(nodes, s) for s in range(n)]
    tables, parents = tables_of(cache), torch.from_numpy(TC.flat(trees)).cuda()
    q = cache.normal(n * nodes, 4 * kv_heads, d).half()
    qd, out, held, status = q.cuda(), torch.empty_like(q, device="cuda"), i32(most), i32([9] * n)
    stream, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def forward():
        cache.paged.set_batch_device(tables, held.data_ptr(), [nodes] * n, 700, parents.data_ptr(), status.data_ptr())
        cache.paged.attention_device(0, view(qd), view(out))

    forward()
    torch.cuda.synchronize()
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        forward()
    cache.paged.set_stream(stream.cuda_stream)
    for turn, shrink in enumerate((1, 2, 50)):
        now = [-1 if (s + turn) % 9 == 4 else p // shrink for s, p in enumerate(most)]
        held.copy_(i32(now))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [int(p < 0) for p in now]
        items = [(max(p, 0), nodes) for p in now]
        for s in range(turn, n, 9):
            if now[s] < 0:
                assert bool((out[s * nodes:(s + 1) * nodes] == 7.0).all())
            else:
                check_one(cache, items, trees, s, q, out, "f16")


# Query heads of a KV head that are no power of two or the most there may be, and more KV heads than parts leave room for.
@pytest.mark.parametrize("heads,kv_heads,d,tensors", [(64, 1, 64, "f16"), (33, 1, 128, "f32"), (96, 2, 96, "f16"), (390, 130, 8, "f16"), (64, 1, 256, "f32")])
def test_many_heads(heads, kv_heads, d, tensors):
    items = [(1500 if kv_heads < 100 else 90, 1), (31, 13), (0, 2), (130, 5)]
    trees = [[-1], TC.tree(13, 1), [-1, -1], TC.tree(5, 2)]
    cache = cache_of(items, kv_heads=kv_heads, d=d, page_rows=32, seed=heads)
    q, out = attend(cache, items, trees, heads, tensors)
    stream, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    qd, again = q.cuda(), torch.empty_like(q, device="cuda")
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        cache.paged.attention_device(0, view(qd), view(again))
    cache.paged.set_stream(stream.cuda_stream)
    for _ in range(2):
        again.zero_()
        graph.replay()
        torch.cuda.synchronize()
        TC.check(cache, 0, items, trees, q, again, tensors)


def test_layers_that_differ_over_one_batch():
    # Heads, types and windows in turn, over one batch and each over a batch of its own: the same cut, so the same bits.
    items, trees = [(900, 40), (2500, 21), (64, 5)], [TC.tree(40, 1), TC.tree(21, 2), TC.tree(5, 3)]
    cache = cache_of(items, kv_heads=2, d=64, page_rows=32, seed=8)
    calls = [(4, "f16", 0), (16, "f16", 0), (4, "f16", 700), (4, "f32", 0), (4, "f16", 900), (4, "f16", 0)]
    queries = {(h, t): cache.normal(66, h, 64).to(PC.DTYPES[t]).cuda() for h, t, _ in calls}

    def run(fresh):
        outs = []
        for n, (h, t, window) in enumerate(calls):
            if fresh or n == 0:
                cache.paged.set_batch(items, cache.tables, TC.flat(trees))
            q = queries[h, t]
            outs.append(torch.empty_like(q))
            cache.paged.attention_device(0, view(q), view(outs[-1]), window=window)
        torch.cuda.synchronize()
        return outs

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


# Pages that begin beyond 2^32 elements of the storage: the results of the same rows in its first pages.
@pytest.mark.parametrize("rows,heads", [(4, 4), (30, 4), (200, 4)])
def test_pages_far_into_the_storage(rows, heads):
    P, d, page_rows, held = pkg(), 128, 64, 1000
    need = -(-(held + rows) // page_rows)
    page_count = (9 << 30) // (2 * page_rows * d * 2)
    storage = torch.zeros(page_count * 2 * page_rows * d, dtype=torch.float16, device="cuda")
    paged = P.PagedKv(1, 1, d, page_rows=page_rows, page_count=page_count, max_sequences=1, max_table_pages=64,
                      storage_ptr=storage.data_ptr(), storage_bytes=2 * storage.numel())
    paged.set_stream(torch.cuda.current_stream().cuda_stream)
    paged.enable_trees(rows)
    g = torch.Generator().manual_seed(rows)
    content = torch.randn(need, 2 * page_rows * d, generator=g).half().cuda()
    parents, pages = TC.flat([TC.tree(rows, 6)]), storage.view(page_count, -1)
    q, k, v = (torch.randn(rows, h, d, generator=g).half().cuda() for h in (heads, 1, 1))
    path = i32([r for r in range(rows) if r % 3 == 0] + [-1] * (rows - (rows + 2) // 3))
    got = []
    for first in (0, page_count - need):
        pages[first:first + need] = content
        out, lengths = torch.empty_like(q), i32([0])
        paged.set_batch([(held, rows)], [list(range(first, first + need))], parents)
        paged.attention_step_device(0, view(q), view(k), view(v), view(out))
        paged.keep_device(path.data_ptr(), lengths.data_ptr())
        torch.cuda.synchronize()
        got.append((out, pages[first:first + need].clone(), lengths.tolist()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and got[0][2] == got[1][2] == [held + (rows + 2) // 3]
    assert bool(got[0][0].isfinite().all()) and not torch.equal(got[0][1], content)
    assert not bool(pages[need:page_count - need].any())


def test_handles_at_work_at_once():
    P = pkg()
    items, trees = [(4000, 40), (700, 3)], [TC.tree(40, 1), TC.tree(3, 2)]
    cache = cache_of(items, kv_heads=2, d=128, page_rows=64, seed=4)
    other = P.PagedKv(1, 2, 128, page_rows=64, page_count=cache.page_count, storage_ptr=cache.storage.data_ptr(),
                      storage_bytes=cache.storage.numel() * 2)
    other.enable_trees(43)
    q = cache.normal(43, 8, 128).half().cuda()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.empty_like(q) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    for s, paged in zip(streams, (cache.paged, other)):
        paged.set_stream(s.cuda_stream)
        paged.set_batch(items, cache.tables, TC.flat(trees))
    for a, b in zip(*outs):
        cache.paged.attention_device(0, view(q), view(a))
        other.attention_device(0, view(q), view(b))
    torch.cuda.synchronize()
    TC.check(cache, 0, items, trees, q, outs[0][0], "f16")
    assert all(torch.equal(x, outs[0][0]) for out in outs for x in out)


def test_refusals():
    P = pkg()
    cache = PC.Cache(P, [40, 30], kv_heads=1, d=64, page_rows=16)
    x = i32([0] * 4)
    cache.paged.set_batch([(20, 0), (3, 2)], cache.tables)
    cache.paged.enable_trees(10)
    # Items and sequences were not the same then.
    assert refusal(lambda: cache.paged.keep_device(x.data_ptr())) == "InvalidArgument"
    assert refusal(lambda: cache.paged.accept_device(*[x.data_ptr()] * 4)) == "InvalidArgument"
    cache.paged.set_batch([(20, 0), (3, 2)], cache.tables)
    tokens, chosen, path, following = i32([5, 6]), i32([6, 7]), i32([9, 9]), i32([9, 9])
    cache.paged.accept_device(tokens.data_ptr(), chosen.data_ptr(), path.data_ptr(), following.data_ptr())
    torch.cuda.synchronize()
    assert path.tolist() == [0, 1] and following.tolist() == [9, 7]
    # Free lists shorter than the pages may be many, and counts that are no single word.
    table, pages, count = i32([[0] * 4] * 2), i32([0, 0]), i32([0])
    short = P.PageTables.of(table, pages, i32([0] * (cache.page_count - 1)), count)
    for call in (lambda: cache.paged.fit_tables_device(short, x.data_ptr()), lambda: P.PageTables.of(table, pages, i32([0] * 9), i32([]))):
        with pytest.raises(ValueError):
            call()
    assert refusal(lambda: cache.paged.fit_tables_device(P.PageTables.of(table, pages), x.data_ptr())) == "InvalidArgument"
    np.testing.assert_array_equal(count.cpu(), [0])
