"""Trees of drafted tokens over a paged cache on the GPU, against plain attention in 64 bits over what each row sees: types, head sizes and
groups on both kernels, trees from one row to the largest, positions around block and page borders, masked rows that hold NaN, windows, the
rotation by depth, and captured calls replayed over batches with trees and without."""
import numpy as np
import pytest
import torch

import paged_cases as PC
import tree_cases as TC
from helpers import pkg, refusal
from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu


def view(t):
    return pkg().Rows.of(t)


def cache_of(items, spare_rows=0, **kw):
    """A cache whose sequences hold the items' positions and new rows; everything else in its pages is NaN."""
    cache = PC.Cache(pkg(), [p + r + spare_rows for p, r in items], fill="nan", **kw)
    cache.paged.enable_trees(max(1, sum(r for _, r in items)))
    for layer in range(cache.host.shape[0]):
        for seq, (p, r) in enumerate(items):
            x = cache.normal(2, p + r, cache.kv_heads, cache.d).to(PC.DTYPES[cache.pages])
            cache.place(layer, seq, 0, x[0], x[1])
    return cache


def attend(cache, items, trees, heads, tensors, layout="dense", window=0, softcap=0.0, layer=0):
    rows = sum(r for _, r in items)
    q = cache.normal(rows, heads, cache.d).to(PC.DTYPES[tensors])
    qd, out = PC.laid_out(q, layout), PC.laid_out(torch.full_like(q, 7.0), layout)
    cache.paged.set_batch(items, cache.tables, TC.flat(trees))
    cache.paged.attention_device(layer, view(qd), view(out), window=window, softcap=softcap)
    torch.cuda.synchronize()
    TC.check(cache, layer, items, trees, q, out, tensors, window, softcap)
    return q, out


TYPES = [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")]


@pytest.mark.parametrize("pages,tensors", TYPES)
@pytest.mark.parametrize("d,kv_heads,heads,page_rows,layout", [
    (128, 2, 8, 16, "dense"), (64, 1, 8, 32, "slice"), (80, 3, 3, 16, "heads"), (96, 2, 2, 64, "odd"), (256, 1, 5, 128, "dense"), (8, 2, 4, 16, "slice"),
])
def test_trees(pages, tensors, d, kv_heads, heads, page_rows, layout):
    # A row alone on nothing, one on a block's border, small and middle trees around borders, a chain among them, a sequence without rows.
    items = [(0, 1), (32, 1), (31, 3), (97, 17), (5, 0), (64, 9), (300, 40)]
    trees = [[-1], [-1], [-1, 0, 0], TC.tree(17, d), [], TC.chain(9), TC.tree(40, 1)]
    cache = cache_of(items, kv_heads=kv_heads, d=d, pages=pages, page_rows=page_rows, seed=d)
    attend(cache, items, trees, heads, tensors, layout)


@pytest.mark.parametrize("pages,tensors", TYPES)
@pytest.mark.parametrize("position", [0, 1, 31, 1000])
def test_the_largest_trees(pages, tensors, position):
    items = [(position, 256), (position + 16, 255)]
    trees = [TC.tree(256, 3, 20), TC.tree(255, 4, 200)]
    cache = cache_of(items, kv_heads=1, d=64, pages=pages, page_rows=16, seed=position)
    attend(cache, items, trees, 2, tensors)


@pytest.mark.parametrize("heads,d,tensors", [(1, 128, "f16"), (2, 64, "f32"), (16, 128, "f16"), (4, 256, "f32")])
def test_long_sequences_are_split(heads, d, tensors):
    items = [(5000, 13), (70, 2), (9000, 30)]
    trees = [TC.tree(13, 1), [-1, -1], TC.tree(30, 2)]
    cache = cache_of(items, kv_heads=1, d=d, page_rows=64, seed=heads)
    attend(cache, items, trees, heads, tensors)


@pytest.mark.parametrize("tensors", ["f16", "f32"])
@pytest.mark.parametrize("window,softcap", [(40, 0.0), (64, 30.0), (0, 5.0), (1 << 33, 0.0)])
def test_windows_and_caps(tensors, window, softcap):
    # A chain longer than the window, trees at and far behind its length.
    items = [(200, 40), (10, 33), (0, 100), (41, 1), (2000, 7)]
    trees = [TC.tree(40, 5), TC.tree(33, 6), TC.chain(100), [-1], TC.tree(7, 7)]
    cache = cache_of(items, kv_heads=2, d=64, page_rows=16, seed=9)
    attend(cache, items, trees, 4, tensors, window=window, softcap=softcap)
    small = [(p, min(r, 5)) for p, r in items]
    attend(cache, small, [t[:5] for t in trees], 4, tensors, window=window, softcap=softcap)


@pytest.mark.parametrize("pages,tensors", TYPES)
@pytest.mark.parametrize("rows,heads", [(6, 2), (60, 4)])
@pytest.mark.parametrize("d", [64, 128])
def test_a_drafted_row_that_is_not_finite_reaches_those_below_it(pages, tensors, rows, heads, d):
    items = [(50, rows), (7, rows)]
    trees = [TC.tree(rows, 11), TC.tree(rows, 12)]
    cache = cache_of(items, kv_heads=2, d=d, pages=pages, page_rows=16, seed=rows)
    hit = max(set(trees[0][1:]) - {-1})  # (a row with rows below it, and rows beside it)
    keys, values = cache.rows(0, 0, 50 + rows)
    keys, values = keys.clone(), values.clone()
    values[50 + hit, 1, 3] = float("nan")
    values[50 + rows - 1, 0, 5] = float("inf")
    keys[50 + hit, 0, 1] = float("-inf")
    cache.place(0, 0, 0, keys, values)
    q, out = attend(cache, items, trees, heads, tensors)
    beside = [r for r in range(rows) if hit not in [s - 50 for s in TC.seen(50, trees[0], r, 0)] and r != rows - 1]
    assert beside and bool(out[beside].isfinite().all()) and bool(out[hit].isnan().any())


@pytest.mark.parametrize("pages,tensors,interleaved", [("f16", "f16", True), ("bf16", "f32", False), ("f16", "f32", True)])
@pytest.mark.parametrize("scale", [1, 8])
def test_a_step_turns_by_depth_and_lies_by_number(pages, tensors, interleaved, scale):
    d, kv_heads, heads = 64, 2, 4
    items = [(33, 5 * scale), (0, 1), (47, 0), (100, 3 * scale), (15, 2)]
    trees = [TC.tree(5 * scale, 2), [-1], [], TC.tree(3 * scale, 3), [-1, -1]]
    rotation = pkg().Rotation(d, base=1e4, interleaved=interleaved)
    cache = cache_of(items, layers=2, kv_heads=kv_heads, d=d, pages=pages, page_rows=16, seed=scale)
    rows = sum(r for _, r in items)
    at = torch.tensor([p + x for (p, _), t in zip(items, trees) for x in TC.depths(t)])
    q, k, v = (cache.normal(rows, h, d).to(PC.DTYPES[tensors]) for h in (heads, kv_heads, kv_heads))
    out = torch.empty(rows, heads, d, dtype=q.dtype, device="cuda")
    before = cache.storage.clone()
    cache.paged.set_batch(items, cache.tables, TC.flat(trees))
    cache.paged.attention_step_device(1, view(q.cuda()), view(k.cuda()), view(v.cuda()), view(out), rotation=rotation)
    torch.cuda.synchronize()
    assert torch.equal(cache.storage[0].view(torch.int16), before[0].view(torch.int16))
    freq = PC.frequencies(d)
    (kt, kerr), (qt, qerr) = PC.rotated(k, at, *freq, interleaved), PC.rotated(q, at, *freq, interleaved)
    stored, first, touched = cache.storage[1].cpu(), 0, torch.zeros(cache.page_count, 16, dtype=torch.bool)
    for seq, (p, r) in enumerate(items):
        for i in range(r):
            page, row = cache.tables[seq][(p + i) // 16], (p + i) % 16
            touched[page, row] = True
            tol = kerr[first + i] + (kt[first + i].abs() + kerr[first + i]) * PC.HALF_STEP[pages] + 2.0 ** -25
            assert bool(((stored[page, 0, :, row].double() - kt[first + i]).abs() <= tol).all()), (seq, i)
            assert torch.equal(stored[page, 1, :, row], v[first + i].to(stored.dtype))
        first += r
    same = stored.view(torch.int16) == before[1].cpu().view(torch.int16)
    assert bool(same.permute(0, 3, 1, 2, 4)[~touched].all())
    # Attention over the rows as they were stored, of the queries as they turn (a type of 16 bits rounds them once more, which moves a score
    # by at most half a step of q times |k|): by the same calls one after the other, which the step is.
    cache.host[1] = stored
    turned = torch.empty_like(out)
    positions = at.cuda()
    rotation.rotate_device([view(q.cuda())], [view(turned)], positions.data_ptr(), rows, d, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool(((turned.cpu().double() - qt).abs() <= qerr + (qt.abs() + qerr) * PC.HALF_STEP[tensors] + 2.0 ** -25).all())
    TC.check(cache, 1, items, trees, turned, out, tensors)
    again = torch.empty_like(out)
    cache.paged.attention_device(1, view(q.cuda()), view(again), rotation=rotation)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


def test_a_chain_is_an_ordinary_batch_and_batches_follow_one_another():
    items = [(20, 40), (3, 2), (64, 1)]
    cache = cache_of(items, kv_heads=2, d=64, page_rows=16, seed=2)
    rows = sum(r for _, r in items)
    q = cache.normal(rows, 8, 64).half().cuda()
    outs = [torch.empty_like(q) for _ in range(4)]
    chains, trees = [TC.chain(r) for _, r in items], [TC.tree(r, 8) for _, r in items]
    for out, parents in zip(outs, (None, chains, trees, None)):
        cache.paged.set_batch(items, cache.tables, None if parents is None else TC.flat(parents))
        cache.paged.attention_device(0, view(q), view(out))
    torch.cuda.synchronize()
    check_attention(cache, 0, items, q, outs[0], "f16")
    check_attention(cache, 0, items, q, outs[1], "f16")
    TC.check(cache, 0, items, trees, q, outs[2], "f16")
    assert torch.equal(outs[0], outs[3])
    # A list in place of an array, and results that are the same from call to call.
    cache.paged.set_batch(items, cache.tables, TC.flat(trees).tolist())
    cache.paged.attention_device(0, view(q), view(outs[3]))
    torch.cuda.synchronize()
    assert torch.equal(outs[2], outs[3])


@pytest.mark.parametrize("rows,heads", [(3, 2), (24, 8)])
def test_replays_are_right_over_batches_with_trees_and_without(rows, heads):
    items, far = [(40, rows), (7, rows)], [(131, rows), (64, rows)]
    cache = cache_of([(131, rows), (131, rows)], kv_heads=2, d=64, page_rows=16, seed=rows)
    q = cache.normal(2 * rows, heads, 64).half().cuda()
    out = torch.empty_like(q)
    stream, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    cache.paged.set_batch(far, cache.tables)
    cache.paged.attention_device(0, view(q), view(out))  # (what a capture needs of memory)
    torch.cuda.synchronize()
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        cache.paged.attention_device(0, view(q), view(out))
    cache.paged.set_stream(stream.cuda_stream)
    for n, batch in enumerate((items, far, items, far, far)):
        trees = [TC.tree(rows, n), TC.tree(rows, n + 20)] if n != 2 else None
        cache.paged.set_batch(batch, cache.tables, None if trees is None else TC.flat(trees))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        if trees:
            TC.check(cache, 0, batch, trees, q, out, "f16")
        else:
            check_attention(cache, 0, batch, q, out, "f16")
        assert float(q.sum().isfinite())  # (the program's own work between the replays)


def test_refusals():
    P = pkg()
    items = [(20, 6), (3, 2)]
    cache = PC.Cache(P, [400, 30], kv_heads=2, d=64, page_rows=16)
    paged = cache.paged
    good = TC.flat([TC.tree(6), [-1, 0]])
    assert refusal(lambda: paged.set_batch(items, cache.tables, good)) == "Unsupported"  # takes no trees
    x = torch.zeros(8, dtype=torch.int32, device="cuda").data_ptr()
    assert refusal(lambda: paged.accept_device(x, x, x, x)) == refusal(lambda: paged.keep_device(x)) == "Unsupported"
    assert refusal(lambda: paged.enable_trees(0)) == "ZeroDimension"
    assert refusal(lambda: paged.enable_trees(1 << 24)) == "SizeOverflow"
    paged.enable_trees(300)
    assert refusal(lambda: paged.enable_trees(300)) == "InvalidArgument"
    paged.set_batch(items, cache.tables, good)
    for at, parent in ((0, 0), (0, 5), (3, 3), (3, -2), (6, 0), (7, 1), (2, 1 << 20), (5, -(1 << 31))):
        bad = good.copy()
        bad[at] = parent
        assert refusal(lambda: paged.set_batch(items, cache.tables, bad)) == "InvalidArgument", (at, parent)
    assert refusal(lambda: paged.set_batch([(20, 301)], cache.tables[:1], TC.flat([TC.chain(301)]))) == "CapacityExceeded"
    assert refusal(lambda: paged.set_batch([(20, 257)], cache.tables[:1], TC.flat([TC.chain(256) + [0]]))) == "Unsupported"
    paged.set_batch([(20, 257)], cache.tables[:1], TC.flat([TC.chain(257)]))
    for wrong in (good[:-1], np.append(good, 0), good.astype(np.float32), good[None]):
        with pytest.raises(ValueError):
            paged.set_batch(items, cache.tables, wrong)
    with pytest.raises(ValueError):
        paged.set_batch(items, cache.tables, np.full(8, 1 << 40))
    # A window within a tree's reach.
    paged.set_batch(items, cache.tables, good)
    q = torch.zeros(8, 4, 64, dtype=torch.float16, device="cuda")
    out = torch.zeros_like(q)
    assert refusal(lambda: paged.attention_device(0, view(q), view(out), window=5)) == "Unsupported"
    paged.attention_device(0, view(q), view(out), window=6)
    paged.set_batch(items, cache.tables)  # (chains have no reach)
    paged.attention_device(0, view(q), view(out), window=1)
    paged.set_batch([(20, 0)], cache.tables[:1], [])
    paged.set_batch([], [], [])
    torch.cuda.synchronize()
