"""The paged cache as a serving program uses it: many sequences, captured forwards that are replayed over other batches, several
handles and streams, and the calls that are refused."""
import math

import numpy as np
import pytest
import torch

import paged_cases as PC
from helpers import pkg
from test_gpu_paged import check_attention, view

pytestmark = pytest.mark.gpu


def filled(lengths, layer=0, **kw):
    cache = PC.Cache(pkg(), lengths, fill="nan", **kw)
    for seq, n in enumerate(lengths):
        if n:
            at = cache.host[layer][cache.tables[seq]]  # [pages][2][kv_heads][page_rows][d]
            rows = torch.randn(at.shape, generator=cache.g).to(at.dtype)
            past = torch.arange(len(at) * cache.page_rows).view(len(at), 1, 1, cache.page_rows, 1) >= n
            cache.host[layer][cache.tables[seq]] = rows.masked_fill(past, float("nan"))
    cache.storage.copy_(cache.host)
    return cache


# Batches of more sequences than travel with a launch, more than a wavefront looks at in one go, and more heads of them than workgroups.
@pytest.mark.parametrize("count,kv_heads,q_heads,d,rows", [
    (9, 2, 8, 64, [1]), (64, 1, 8, 128, [1]), (65, 2, 4, 64, [1, 1, 3]), (130, 8, 8, 64, [1, 0, 2]), (200, 2, 32, 128, [1, 1, 1, 1, 30])])
@pytest.mark.parametrize("pages,tensors", [("f16", "f16"), ("bf16", "f32")])
def test_many_sequences(count, kv_heads, q_heads, d, rows, pages, tensors):
    items = [((37 * i * i) % 301, rows[i % len(rows)]) for i in range(count)]
    cache = filled([p + r for p, r in items], kv_heads=kv_heads, d=d, pages=pages, page_rows=16, max_sequences=count, seed=count)
    total = sum(r for _, r in items)
    q = cache.normal(total, q_heads, d).to(PC.DTYPES[tensors])
    qd = q.cuda()
    out = torch.full((total + 1, q_heads, d), 5.0, dtype=q.dtype, device="cuda")
    cache.paged.set_batch(items, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out[:total]), window=77)
    torch.cuda.synchronize()
    check_attention(cache, 0, items, q, out[:total], tensors, window=77)
    assert bool((out[total] == 5.0).all())


# One KV head, so that a unit's keys are all the work there is: more parts of it than a wavefront of the merge has lanes.
@pytest.mark.parametrize("q_heads,tensors", [(64, "f16"), (64, "f32"), (8, "f16")])
def test_one_unit_in_many_parts(q_heads, tensors):
    cache = filled([90001], kv_heads=1, d=64, page_rows=256, seed=q_heads)
    q = cache.normal(1, q_heads, 64).to(PC.DTYPES[tensors])
    qd = q.cuda()
    out = torch.empty_like(qd)
    cache.paged.set_batch([(90000, 1)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    check_attention(cache, 0, [(90000, 1)], q, out, tensors)


def test_appends_of_many_sequences():
    items = [((53 * i) % 90, (i * 7) % 4) for i in range(150)]
    cache = PC.Cache(pkg(), [p + r for p, r in items], kv_heads=2, d=64, page_rows=16, max_sequences=150)
    total = sum(r for _, r in items)
    k, v = (cache.normal(total, 2, 64).half() for _ in range(2))
    kd, vd = k.cuda(), v.cuda()
    want, at = cache.host.clone(), 0
    for seq, (p, r) in enumerate(items):
        for i in range(r):
            page, row = cache.tables[seq][(p + i) // 16], (p + i) % 16
            want[0, page, 0, :, row], want[0, page, 1, :, row] = k[at], v[at]
            at += 1
    cache.paged.set_batch(items, cache.tables)
    cache.paged.append_device(0, view(kd), view(vd))
    torch.cuda.synchronize()
    assert torch.equal(cache.storage.cpu(), want)


# A captured forward is right for every batch of the same rows, whatever the positions: single tokens, blocks, a chunk among tokens.
@pytest.mark.parametrize("rows", [[1, 1, 1], [1, 60, 1], [7, 7], [300], [1] * 12])
@pytest.mark.parametrize("pages,tensors", [("f16", "f16"), ("bf16", "f32")])
def test_replays_over_other_positions(rows, pages, tensors):
    kv_heads, q_heads, d, room = 2, 8, 64, 2000
    cache = filled([room + r for r in rows], kv_heads=kv_heads, d=d, pages=pages, page_rows=32, max_sequences=16, seed=len(rows))
    total = sum(rows)
    q, k, v = (cache.normal(total, h, d).to(PC.DTYPES[tensors]).cuda() for h in (q_heads, kv_heads, kv_heads))
    out, again = torch.empty_like(q), torch.empty_like(q)
    rotation = pkg().Rotation(d, base=1e4)
    first = [(0, r) for r in rows]
    cache.paged.set_batch(first, cache.tables)
    stream, side = torch.cuda.current_stream(), torch.cuda.Stream()

    def forward(out):
        cache.paged.attention_step_device(0, view(q), view(k), view(v), view(out), rotation=rotation)

    forward(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        forward(out)
    cache.paged.set_stream(stream.cuda_stream)
    torch.cuda.synchronize()
    for n in range(4):
        held = [((n * 997 + 131 * i * i) % room if n else room, r) for i, r in enumerate(rows)]
        cache.paged.set_batch(held, cache.tables)
        out.fill_(3.0)
        graph.replay()
        forward(again)
        torch.cuda.synchronize()
        cache.host = cache.storage.cpu()
        turned = torch.empty_like(q)
        positions = torch.cat([torch.arange(p, p + r) for p, r in held]).cuda()
        rotation.rotate_device([view(q)], [view(turned)], positions.data_ptr(), total, d, stream.cuda_stream)
        check_attention(cache, 0, held, turned.cpu(), out, tensors)
        check_attention(cache, 0, held, turned.cpu(), again, tensors)
        if n == 3:
            before = out.clone()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(before, out)


def test_a_capture_that_needs_more_memory_is_refused_and_one_after_it_is_not():
    cache = filled([4000], kv_heads=2, d=64, page_rows=64)
    q = cache.normal(1, 8, 64).half().cuda()
    out = torch.empty_like(q)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    cache.paged.set_batch([(3999, 1)], cache.tables)
    torch.cuda.synchronize()
    cache.paged.set_stream(side.cuda_stream)
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(pkg().AttentionError) as e:
            cache.paged.attention_device(0, view(q), view(out))
    assert e.value.variant == "CapacityExceeded"
    cache.paged.attention_device(0, view(q), view(out))
    cache.paged.synchronize()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.paged.attention_device(0, view(q), view(out))
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) or bool(((out - want).abs() <= 2.0 ** -9).all())


def test_two_handles_over_one_storage_on_two_streams():
    # Another handle's batch, workspace and stream are its own: two halves of a batch at a time.
    one = filled([900, 500], kv_heads=2, d=128, page_rows=32, seed=8)
    two = pkg().PagedKv(1, 2, 128, page_rows=32, page_count=one.page_count, max_sequences=8,
                        storage_ptr=one.storage.data_ptr(), storage_bytes=one.storage.numel() * 2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    q = one.normal(2, 8, 128).half()
    qd = q.cuda()
    outs = torch.zeros(20, 2, 8, 128, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    for handle, s in zip((one.paged, two), streams):
        handle.set_stream(s.cuda_stream)
    one.paged.set_batch([(899, 1)], one.tables[:1])
    two.set_batch([(499, 1)], one.tables[1:])
    for i in range(20):
        one.paged.attention_device(0, view(qd[:1]), view(outs[i, :1]))
        two.attention_device(0, view(qd[1:]), view(outs[i, 1:]))
    one.paged.synchronize()
    two.synchronize()
    for i in range(20):
        check_attention(one, 0, [(899, 1), (499, 1)], q, outs[i], "f16")
        assert torch.equal(outs[i], outs[0])


def test_empty_batches_do_nothing():
    cache = filled([50], kv_heads=1, d=64, page_rows=16)
    q = torch.ones(0, 2, 64, dtype=torch.float16, device="cuda")
    k = torch.ones(0, 1, 64, dtype=torch.float16, device="cuda")
    before = cache.storage.clone()
    for items, tables in (([], []), ([(20, 0)], cache.tables), ([(0, 0)], [[]])):
        cache.paged.set_batch(items, tables)
        cache.paged.append_device(0, view(k), view(k))
        cache.paged.attention_device(0, view(q), view(q))
        cache.paged.attention_step_device(0, view(q), view(k), view(k), view(q))
    torch.cuda.synchronize()
    assert torch.equal(before.view(torch.int16), cache.storage.view(torch.int16))


@pytest.mark.parametrize("window", [1, 50, 51, 1 << 20, 1 << 40])
def test_windows_from_one_position_to_more_than_there_are(window):
    items = [(50, 1), (0, 1), (49, 3)]
    cache = filled([p + r for p, r in items], kv_heads=2, d=64, page_rows=16)
    q = cache.normal(5, 4, 64).half()
    qd, out = q.cuda(), torch.empty(5, 4, 64, dtype=torch.float16, device="cuda")
    cache.paged.set_batch(items, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), window=window)
    torch.cuda.synchronize()
    check_attention(cache, 0, items, q, out, "f16", window=min(window, 1 << 20))


def test_positions_near_the_largest():
    # 2^31 - 64 positions of which a window sees 40: pages of a short storage, named again and again.
    page_rows, d = 1024, 64
    position = (1 << 31) - 64
    pages = (position + 2 + page_rows - 1) // page_rows
    storage = torch.randn(1, 4, 2, 1, page_rows, d, device="cuda").half()
    paged = pkg().PagedKv(1, 1, d, page_rows=page_rows, page_count=4, max_sequences=1, max_table_pages=pages,
                          storage_ptr=storage.data_ptr(), storage_bytes=storage.numel() * 2)
    paged.set_stream(torch.cuda.current_stream().cuda_stream)
    table = np.arange(pages, dtype=np.uint32) % 3
    table[-1] = 3  # (the page that takes the new rows is nobody else's)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, h, d, generator=g).half() for h in (4, 1, 1))
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    out = torch.empty_like(qd)
    paged.set_batch([(position, 2)], [table])
    paged.attention_step_device(0, view(qd), view(kd), view(vd), view(out), window=40)
    torch.cuda.synchronize()
    host = storage.cpu()
    seen = [(int(table[p // page_rows]), p % page_rows) for p in range(position - 39, position + 2)]
    keys, values = (torch.stack([host[0, page, side, :, row] for page, row in seen]) for side in (0, 1))
    assert torch.equal(keys[-2:], k) and torch.equal(values[-2:], v)
    want, spread, most = PC.attention(q, keys, values, 39, 40, 0.0, d ** -0.5)
    assert bool(((out.cpu().double() - want).abs() <= PC.tolerance(want, spread, most, "f16", "f16", d, 41)).all())


def test_f32_queries_beyond_the_range_of_f16():
    cache = filled([90], kv_heads=1, d=64, page_rows=16, seed=1)
    q = cache.normal(3, 2, 64)
    q[1] *= 1e5
    qd, out = q.cuda(), torch.empty(3, 2, 64, device="cuda")
    cache.paged.set_batch([(87, 3)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    check_attention(cache, 0, [(87, 3)], q, out, "f32")


def test_refusals_leave_everything_as_it_was():
    P = pkg()
    cache = filled([40, 40], kv_heads=2, d=64, page_rows=16, layers=2)
    paged, (a, b) = cache.paged, cache.tables
    paged.set_batch([(30, 2), (39, 1)], cache.tables)
    t = lambda rows, heads, dtype=torch.float16, d=64: torch.full((rows, heads, d), 2.0, dtype=dtype, device="cuda")  # noqa: E731
    q, k, out = t(3, 4), t(3, 2), t(3, 4)
    before = cache.storage.clone()
    R, wide = P.Rows, P.Rotation(128)
    attend = lambda **kw: paged.attention_device(kw.pop("layer", 0), kw.pop("q", view(q)), kw.pop("out", view(out)), **kw)  # noqa: E731
    wrong = [
        ("InvalidLayer", lambda: attend(layer=2)),
        ("InvalidLayer", lambda: paged.append_device(2, view(k), view(k))),
        ("ShapeMismatch", lambda: attend(out=view(t(3, 2)))),
        ("ShapeMismatch", lambda: paged.append_device(0, view(t(3, 4)), view(k))),
        ("ShapeMismatch", lambda: attend(rotation=wide)),
        ("NonDivisibleHeads", lambda: attend(q=view(t(3, 3)), out=view(t(3, 3)))),
        ("Unsupported", lambda: attend(q=view(t(3, 130)), out=view(t(3, 130)))),
        ("Unsupported", lambda: attend(q=view(t(3, 4, torch.bfloat16)), out=view(t(3, 4, torch.bfloat16)))),
        ("Unsupported", lambda: attend(softcap=1e-38, scale=3e5)),
        ("InvalidArgument", lambda: attend(out=view(t(3, 4, torch.float32)))),
        ("InvalidArgument", lambda: attend(out=view(q))),
        ("InvalidArgument", lambda: paged.append_device(0, view(k), view(t(3, 2, torch.float32)))),
        ("InvalidArgument", lambda: attend(scale=math.inf)),
        ("InvalidArgument", lambda: attend(softcap=-1.0)),
        ("InvalidArgument", lambda: attend(softcap=math.nan)),
        ("InvalidArgument", lambda: attend(softcap=math.inf)),
        ("InvalidArgument", lambda: attend(out=R(out.data_ptr(), "f16", 4, 64, 64))),      # rows over one another
        ("InvalidArgument", lambda: attend(out=R(out.data_ptr(), "f16", 4, 256, 32))),     # heads over one another
        ("InvalidArgument", lambda: attend(q=R(0, "f16", 4))),
        ("InvalidArgument", lambda: attend(q=R(q.data_ptr() + 1, "f16", 4))),
        ("ZeroDimension", lambda: attend(q=R(q.data_ptr(), "f16", 0))),
        ("ShapeMismatch", lambda: paged.set_batch([(47, 2)], [a])),                        # too few pages
        ("InvalidArgument", lambda: paged.set_batch([(30, 2)], [[a[0], cache.page_count, a[2]]])),
        ("InvalidArgument", lambda: paged.set_batch([(30, 2), (30, 2)], [a, a])),          # both write the same page
        ("InvalidArgument", lambda: paged.set_batch([(30, 2), (20, 1)], [a, [a[1], b[1]]])),
        ("SizeOverflow", lambda: paged.set_batch([((1 << 31) - 1, 1)], [a])),
    ]
    for name, call in wrong:
        with pytest.raises(P.AttentionError) as e:
            call()
        assert e.value.variant == name, (name, str(e.value))
    torch.cuda.synchronize()
    assert torch.equal(before.view(torch.int16), cache.storage.view(torch.int16)) and bool((out == 2.0).all())
    attend()  # (the batch before the refused ones is in force)
    torch.cuda.synchronize()
    check_attention(cache, 0, [(30, 2), (39, 1)], q, out, "f16")
