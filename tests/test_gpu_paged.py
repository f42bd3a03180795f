"""The paged cache on the GPU against a plain implementation in 64 bits (paged_cases.py): rotation, append, attention and their
step, over types, head layouts, page sizes and lengths where they can go wrong."""
import math

import pytest
import torch

import paged_cases as PC
from helpers import pkg

pytestmark = pytest.mark.gpu


def view(t):
    return pkg().Rows.of(t)


def check_attention(cache, layer, items, q, got, tensors, window=0, softcap=0.0, scale=None):
    scale = 1 / math.sqrt(cache.d) if scale is None else scale
    at = 0
    for seq, (position, rows) in enumerate(items):
        if rows == 0:
            continue
        n = position + rows
        keys, values = cache.rows(layer, seq, n)
        want, spread, most = PC.attention(q[at:at + rows].cpu(), keys, values, position, window, softcap, scale)
        tol = PC.tolerance(want, spread, most, cache.pages, tensors, cache.d, n)
        mine = got[at:at + rows].cpu().double()
        assert torch.equal(mine.isnan(), want.isnan()), "NaN reaches other outputs than it should"
        off = ((mine - want).abs() / tol).nan_to_num(0.0)
        assert off.max() <= 1.0, (seq, float(off.max()), float((mine - want).abs().nan_to_num().max()))
        at += rows


# ------------------------------------------------------------------------------------- rotation

@pytest.mark.parametrize("tensors", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,rotary,interleaved,scaling,layout", [
    (128, 128, False, "plain", "dense"), (128, 64, True, "yarn", "slice"), (64, 64, True, "linear", "heads"),
    (80, 40, False, "yarn", "dense"), (80, 80, True, "plain", "slice"), (6, 2, False, "plain", "dense"),
    (7, 6, True, "plain", "odd"), (256, 256, False, "yarn", "odd"), (96, 20, True, "linear", "dense"), (300, 128, False, "plain", "heads"),
])
def test_rotation(tensors, d, rotary, interleaved, scaling, layout):
    g = torch.Generator().manual_seed(d * 7 + rotary)
    kw = dict(scaling=scaling, factor=4.0 if scaling != "plain" else 1.0)
    rotation = pkg().Rotation(rotary, base=5e5, interleaved=interleaved, original_positions=8192, **kw)
    freq, amplitude = PC.frequencies(rotary, 5e5, original=8192, **kw)
    got_freq, got_amplitude = rotation.frequencies()
    assert torch.allclose(torch.from_numpy(got_freq), freq, rtol=1e-14, atol=0) and abs(got_amplitude - amplitude) < 1e-15
    for rows in (1, 5, 130):
        positions = torch.randint(0, 200000, (rows,), generator=g)
        positions[0] = 0
        if rows > 1:
            positions[1] = -77
        x = [torch.randn(rows, h, d, generator=g).to(PC.DTYPES[tensors]) for h in (6, 1)]
        src = [PC.laid_out(t, layout) for t in x]
        dst = [torch.full((rows, t.shape[1] + 1, d), 7.0, dtype=t.dtype, device="cuda") for t in x]
        out = [t[:, :-1] for t in dst]
        for inverse in (False, True):
            rotation.rotate_device([view(t) for t in src], [view(t) for t in out], positions.cuda().data_ptr(), rows, d,
                                   torch.cuda.current_stream().cuda_stream, inverse)
            torch.cuda.synchronize()
            for t, o, whole in zip(x, out, dst):
                want, err = PC.rotated(t, positions, freq, amplitude, interleaved, inverse)
                tol = err + (want.abs() + err) * PC.HALF_STEP[tensors] + (2.0 ** -25 if tensors == "f16" else 0.0)
                assert bool(((o.cpu().double() - want).abs() <= tol).all())
                assert torch.equal(o.cpu()[..., rotary:], t[..., rotary:])  # channels past the rotary part pass through
                assert bool((whole[:, -1] == 7.0).all())
        # In place.
        rotation.rotate_device([view(t) for t in src], [view(t) for t in src], positions.cuda().data_ptr(), rows, d,
                               torch.cuda.current_stream().cuda_stream, True)
        torch.cuda.synchronize()
        for t, o in zip(src, out):
            assert torch.equal(t, o)


def test_inverse_rotation_is_the_gradient():
    # L = sum(w * rotate(x)): dL/dx is the inverse rotation of w, against differences of the operator in f32.
    rows, heads, d = 3, 2, 16
    g = torch.Generator().manual_seed(3)
    rotation = pkg().Rotation(12, base=100.0, interleaved=True, scaling="yarn", factor=8.0, original_positions=64)
    positions = torch.tensor([0, 5, 90], device="cuda")
    x, w = (torch.randn(rows, heads, d, generator=g).cuda() for _ in range(2))
    out, grad = torch.empty_like(x), torch.empty_like(x)
    run = lambda a, b, inverse: rotation.rotate_device([view(a)], [view(b)], positions.data_ptr(), rows, d,  # noqa: E731
                                                       torch.cuda.current_stream().cuda_stream, inverse)
    run(w, grad, True)
    loss = []
    for e in (1.0, -1.0):  # (the operator is linear: a step of one loses nothing)
        stepped = x.clone()
        stepped[1, 1, 3] += e
        run(stepped, out, False)
        loss.append(float((w.double() * out.double()).sum()))
    # The loss sums 96 terms of at most a few units, each within 2^-21 of its row's magnitude.
    assert abs((loss[0] - loss[1]) / 2 - float(grad[1, 1, 3])) < 96 * 8 * 2.0 ** -21


# --------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("pages,tensors", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("d,page_rows,layout,rotary,interleaved", [
    (64, 16, "dense", 64, False), (128, 32, "slice", 64, True), (80, 64, "heads", 80, False), (8, 16, "odd", 6, True),
    (256, 128, "slice", 256, True), (128, 16, "dense", 0, False),
])
def test_append(pages, tensors, d, page_rows, layout, rotary, interleaved):
    items = [(0, 1), (page_rows - 1, 2), (37, 0), (5, 3 * page_rows), (1000, 1)]
    cache = PC.Cache(pkg(), [p + r for p, r in items], layers=2, kv_heads=3, d=d, pages=pages, page_rows=page_rows, seed=d)
    rows = sum(r for _, r in items)
    positions = torch.cat([torch.arange(p, p + r) for p, r in items])
    k, v = (cache.normal(rows, 3, d).to(PC.DTYPES[tensors]) for _ in range(2))
    rotation = pkg().Rotation(rotary, base=1e4, interleaved=interleaved) if rotary else None
    before = cache.host.clone()
    cache.paged.set_batch(items, cache.tables)
    kd, vd = PC.laid_out(k, layout), PC.laid_out(v, layout)
    cache.paged.append_device(1, view(kd), view(vd), rotation)
    torch.cuda.synchronize()
    got = cache.storage.cpu()
    assert torch.equal(got[0], before[0])  # the other layer
    want, err = PC.rotated(k, positions, *PC.frequencies(rotary), interleaved) if rotary else (k.double(), torch.zeros_like(k.double()))
    touched = torch.zeros(cache.page_count, page_rows, dtype=torch.bool)
    at = 0
    for seq, (position, n) in enumerate(items):
        for r in range(n):
            page, row = cache.tables[seq][(position + r) // page_rows], (position + r) % page_rows
            touched[page, row] = True
            tol = err[at] + (want[at].abs() + err[at]) * PC.HALF_STEP[pages] + (2.0 ** -25 if pages == "f16" else 0.0)
            assert bool(((got[1, page, 0, :, row].double() - want[at]).abs() <= tol).all())
            assert torch.equal(got[1, page, 1, :, row], v[at].to(PC.DTYPES[pages]))
            at += 1
    untouched = ~touched
    assert torch.equal(got[1].permute(0, 3, 1, 2, 4)[untouched], before[1].permute(0, 3, 1, 2, 4)[untouched])


# ------------------------------------------------------------------------------------ attention

ATTENTION = [
    # q heads, kv heads, d, page rows, [(position, rows)], window, softcap, layout
    (8, 2, 64, 16, [(0, 1)], 0, 0.0, "dense"),
    (8, 1, 128, 32, [(31, 1), (32, 1), (0, 1), (700, 1)], 0, 0.0, "dense"),
    (32, 4, 128, 64, [(1000, 1)], 0, 0.0, "slice"),
    (6, 6, 80, 16, [(99, 1), (0, 5), (300, 2), (50, 0), (17, 33)], 0, 0.0, "heads"),
    (10, 2, 96, 16, [(211, 7), (5, 7)], 0, 30.0, "odd"),
    (16, 2, 128, 128, [(500, 9), (127, 1), (129, 40)], 100, 0.0, "dense"),
    (3, 3, 256, 16, [(150, 3), (0, 20)], 33, 5.0, "slice"),
    (64, 1, 64, 32, [(260, 2)], 1, 0.0, "dense"),
    (5, 1, 8, 16, [(77, 70)], 0, 0.0, "dense"),
    (2, 1, 112, 16, [(0, 300)], 64, 0.0, "heads"),
    (4, 4, 192, 64, [(400, 2)], 0, 0.0, "odd"),
    (12, 4, 128, 16, [(0, 130), (1, 129), (640, 64)], 0, 0.0, "slice"),
    # Tiles of many rows beside single tokens, parts of their keys, every head size's form of them.
    (16, 2, 128, 16, [(0, 1), (1500, 70), (33, 9), (900, 1)], 0, 0.0, "dense"),
    (8, 2, 64, 32, [(777, 100), (3, 1)], 0, 20.0, "heads"),
    (4, 2, 256, 64, [(100, 90)], 40, 0.0, "odd"),
    (6, 2, 144, 16, [(70, 61)], 0, 0.0, "dense"),
    (8, 8, 40, 16, [(19, 200), (0, 65)], 0, 0.0, "slice"),
    (8, 1, 128, 1024, [(2000, 33)], 1000, 0.0, "dense"),
]


@pytest.mark.parametrize("pages,tensors", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("case", ATTENTION, ids=[str(i) for i in range(len(ATTENTION))])
def test_attention(pages, tensors, case):
    q_heads, kv_heads, d, page_rows, items, window, softcap, layout = case
    # (Rows that nobody wrote hold NaN: a right kernel never lets one through.)
    cache = PC.Cache(pkg(), [p + r for p, r in items], layers=2, kv_heads=kv_heads, d=d, pages=pages, page_rows=page_rows,
                     seed=q_heads * d, fill="nan")
    for seq, (p, r) in enumerate(items):
        cache.place(1, seq, 0, *(cache.normal(p + r, kv_heads, d).to(PC.DTYPES[pages]) for _ in range(2)))
    rows = sum(r for _, r in items)
    q = cache.normal(rows, q_heads, d).to(PC.DTYPES[tensors])
    out = PC.laid_out(torch.full((rows + 1, q_heads, d), 9.0, dtype=q.dtype), layout)
    cache.paged.set_batch(items, cache.tables)
    qd = PC.laid_out(q, layout)
    cache.paged.attention_device(1, view(qd), view(out[:rows]), softcap=softcap, window=window)
    torch.cuda.synchronize()
    check_attention(cache, 1, items, q, out[:rows], tensors, window, softcap)
    assert bool((out[rows] == 9.0).all())
    assert torch.equal(cache.storage.cpu().view(torch.int16), cache.host.view(torch.int16))


@pytest.mark.parametrize("pages", ["f16", "bf16"])
@pytest.mark.parametrize("rows,position", [(1, 4096), (3, 5000), (1, 9000), (200, 3000)])
def test_attention_over_many_splits(pages, rows, position):
    cache = PC.Cache(pkg(), [position + rows, 40], kv_heads=2, d=128, pages=pages, page_rows=64, fill="nan", seed=rows)
    items = [(position, rows), (39, 1)]
    for seq, (p, r) in enumerate(items):
        cache.place(0, seq, 0, *(cache.normal(p + r, 2, 128).to(PC.DTYPES[pages]) for _ in range(2)))
    q = cache.normal(rows + 1, 8, 128).to(PC.DTYPES[pages])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch(items, cache.tables)
    first = None
    for _ in range(2):  # the same bits from call to call
        out.fill_(0)
        cache.paged.attention_device(0, view(qd), view(out), scale=0.2)
        torch.cuda.synchronize()
        assert first is None or torch.equal(first, out)
        first = out.clone()
    check_attention(cache, 0, items, q, out, pages, scale=0.2)


@pytest.mark.parametrize("pages,tensors", [("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows", [1, 6, 14, 40])
@pytest.mark.parametrize("window", [0, 50])
def test_rows_that_are_not_finite_reach_the_queries_that_see_them(pages, tensors, rows, window):
    position = 120
    cache = PC.Cache(pkg(), [position + rows], kv_heads=2, d=128, pages=pages, page_rows=16, fill="nan", seed=5)
    items = [(position, rows)]
    keys, values = (cache.normal(position + rows, 2, 128).to(PC.DTYPES[pages]) for _ in range(2))
    values[position + rows - 1, 0, 3] = float("inf")     # the newest row only
    values[position + rows // 2, 0, 40] = float("nan")   # from the middle on
    values[position + rows - 50, 0, 77] = float("-inf")  # with a window of 50: not the newest row
    keys[position + rows // 3, 1, 9] = float("nan")
    cache.place(0, 0, 0, keys, values)
    q = cache.normal(rows, 8, 128).to(PC.DTYPES[tensors])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch(items, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), window=window)
    torch.cuda.synchronize()
    got = out.cpu().double()
    want, spread, most = PC.attention(q, keys, values, position, window, 0.0, 1 / math.sqrt(128))
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    tol = PC.tolerance(want, spread, most.nan_to_num(0.0), pages, tensors, 128, position + rows)
    fine = want.isfinite()
    assert bool(((got - want).abs()[fine] <= tol[fine]).all())


# One key has most of the weight and thousands share the rest evenly, 2^-16 of it each: what a rounding takes of one it takes of all.
@pytest.mark.parametrize("pages,tensors,off", [("f16", "f16", 2.0 ** -11), ("f16", "f32", 2.0 ** -19), ("bf16", "f32", 2.0 ** -19)])
@pytest.mark.parametrize("rows", [1, 40])
def test_many_small_weights_beside_a_large_one(pages, tensors, off, rows):
    n, d = 20000, 64
    cache = PC.Cache(pkg(), [n], kv_heads=1, d=d, pages=pages, page_rows=256, fill="nan", seed=2)
    keys, values = torch.zeros(n, 1, d), torch.full((n, 1, d), 0.75)
    keys[7, 0, 0] = 11.2  # a score of 11.2 above the others' 0: their weights are e^-11.2 of its
    keys[7] = keys[7].to(PC.DTYPES[pages]).float()
    values[7] = -0.5
    cache.place(0, 0, 0, keys.to(PC.DTYPES[pages]), values.to(PC.DTYPES[pages]))
    q = torch.zeros(rows, 2, d)
    q[:, :, 0] = 1.0
    q = q.to(PC.DTYPES[tensors])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch([(n - rows, rows)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), scale=1.0)
    torch.cuda.synchronize()
    # f16: weights are within 2^-11 of themselves in the numerator, where the large one brings at most 0.5 and the others together
    # at most 0.75 * 0.22, and the output, at most 0.5, is rounded within 2^-11 of itself: below 2^-11 in all. f32: second and
    # third pieces leave 2^-21 of a weight, and a workgroup adds at most 20 blocks, 2^-24 each in numerator and denominator.
    w = math.exp(-float(keys[7, 0, 0]))
    at = torch.arange(n - rows + 1, n + 1).double() - 1
    want = (-0.5 + 0.75 * w * at) / (1 + w * at)
    assert bool(((out.cpu().double() - want[:, None, None]).abs() <= off).all())


# Small queries before large keys: the scores are what they are of ordinary ones.
@pytest.mark.parametrize("rows", [1, 40])
def test_small_f32_queries_keep_their_bits(rows):
    cache = PC.Cache(pkg(), [200 + rows], kv_heads=2, d=64, page_rows=16, fill="nan", seed=3)
    items = [(200, rows)]
    keys, values = (cache.normal(200 + rows, 2, 64) for _ in range(2))
    cache.place(0, 0, 0, (keys * 64).half(), values.half())
    q = cache.normal(rows, 4, 64) * 2.0 ** -6
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch(items, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    at, scale = 0, 1 / math.sqrt(64)
    k16, v16 = cache.rows(0, 0, 200 + rows)
    want, spread, most = PC.attention(q, k16, v16, 200, 0, 0.0, scale)
    # A query channel is off by 2^-22 of itself or by 2^-29: over 64 channels of keys up to 4 * 64, beside the tolerance of any other.
    extra = 2 * 64 * 4 * 64 * 2.0 ** -29 * scale
    tol = PC.tolerance(want, spread, most, "f16", "f32", 64, 200 + rows) + spread * extra
    assert bool(((out.cpu().double() - want).abs() <= tol).all())


# A cap far above the scores changes them little, and one below them much: both leave f32 tensors their precision. (Of 8 channels,
# where the bound on a product's sum is no wider than that.)
@pytest.mark.parametrize("pages", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("softcap", [1000.0, 30.0, 2.0])
def test_a_cap_keeps_the_precision_of_f32(pages, rows, softcap):
    cache = PC.Cache(pkg(), [300 + rows], kv_heads=2, d=8, pages=pages, page_rows=32, fill="nan", seed=11)
    items = [(300, rows)]
    cache.place(0, 0, 0, *(cache.normal(300 + rows, 2, 8).to(PC.DTYPES[pages]) for _ in range(2)))
    q = cache.normal(rows, 8, 8)
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch(items, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), softcap=softcap, scale=0.3)
    torch.cuda.synchronize()
    check_attention(cache, 0, items, q, out, "f32", softcap=softcap, scale=0.3)


# ------------------------------------------------------------------------------------ the step

@pytest.mark.parametrize("pages,tensors", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
def test_steps_from_prompts_to_tokens(pages, tensors):
    # Prompts, then a block, then single tokens, on a windowed rotated layer and a global plain one.
    kv_heads, q_heads, d, page_rows = 2, 8, 64, 16
    plan = [[33, 1, 70], [2, 5, 0], [1, 1, 1], [1, 1, 1]]
    totals = [sum(f[s] for f in plan) for s in range(3)]
    cache = PC.Cache(pkg(), totals, layers=2, kv_heads=kv_heads, d=d, pages=pages, page_rows=page_rows, fill="nan")
    rotation = pkg().Rotation(32, base=1e4)
    freq, amplitude = PC.frequencies(32)
    held = [0, 0, 0]
    for new in plan:
        items = list(zip(held, new))
        rows = sum(new)
        cache.paged.set_batch(items, cache.tables)
        positions = torch.cat([torch.arange(p, p + r) for p, r in items])
        for layer, (window, turn) in enumerate([(20, rotation), (0, None)]):
            q, k, v = (cache.normal(rows, h, d).to(PC.DTYPES[tensors]) for h in (q_heads, kv_heads, kv_heads))
            qd, kd, vd = (PC.laid_out(t, "slice") for t in (q, k, v))
            out = torch.empty(rows, q_heads, d, dtype=q.dtype, device="cuda")
            cache.paged.attention_step_device(layer, view(qd), view(kd), view(vd), view(out), window=window, rotation=turn)
            torch.cuda.synchronize()
            cache.host = cache.storage.cpu()
            turned = q
            if turn:
                q64, q_err = PC.rotated(q, positions, freq, amplitude, False)
                k64, k_err = PC.rotated(k, positions, freq, amplitude, False)
                at = 0
                for seq, (p, r) in enumerate(items):
                    stored = cache.rows(layer, seq, p + r)[0][p:]
                    tol = k_err[at:at + r] + (k64[at:at + r].abs() + k_err[at:at + r]) * PC.HALF_STEP[pages]
                    assert bool(((stored.double() - k64[at:at + r]).abs() <= tol + 2.0 ** -25).all())
                    at += r
                # (The rotated queries as the operator itself rounds them: what attends.)
                turned_dev = torch.empty_like(q, device="cuda")
                turn.rotate_device([view(qd)], [view(turned_dev)], positions.cuda().data_ptr(), rows, d,
                                   torch.cuda.current_stream().cuda_stream)
                turned = turned_dev.cpu()
            check_attention(cache, layer, items, turned, out, tensors, window)
            again = torch.empty_like(out)
            cache.paged.attention_device(layer, view(qd), view(again), window=window, rotation=turn)
            torch.cuda.synchronize()
            assert torch.equal(again, out)
        held = [p + r for p, r in items]


@pytest.mark.parametrize("pages", ["f16", "bf16"])
def test_shared_prefix_pages_are_read_by_both(pages):
    cache = PC.Cache(pkg(), [64, 16, 16], kv_heads=2, d=64, pages=pages, page_rows=16, fill="nan")
    shared = cache.tables[0][:3]
    tables = [cache.tables[0], shared + cache.tables[1], shared + cache.tables[2]]
    cache.tables = tables
    cache.place(0, 0, 0, *(cache.normal(50, 2, 64).to(PC.DTYPES[pages]) for _ in range(2)))
    for seq in (1, 2):
        cache.place(0, seq, 48, *(cache.normal(4, 2, 64).to(PC.DTYPES[pages]) for _ in range(2)))
    items = [(49, 1), (50, 2), (51, 1)]
    q = cache.normal(4, 4, 64).to(PC.DTYPES[pages])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch(items, tables)
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    check_attention(cache, 0, items, q, out, pages)


def test_pages_beyond_32_bits():
    # 9 GB of one layer's pages: the last ones lie past 2^32 elements and 2^33 bytes.
    pages, kv_heads, d, page_rows = 70000, 4, 128, 64
    storage = torch.empty(1, pages, 2, kv_heads, page_rows, d, dtype=torch.float16, device="cuda")
    paged = pkg().PagedKv(1, kv_heads, d, page_count=pages, page_rows=page_rows, max_sequences=2, max_table_pages=64,
                          storage_ptr=storage.data_ptr(), storage_bytes=storage.numel() * 2)
    paged.set_stream(torch.cuda.current_stream().cuda_stream)
    table, n = [pages - 1, 2, pages - 2], 150
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, d, generator=g).half() for h in (8, kv_heads, kv_heads))
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    out = torch.empty_like(qd)
    paged.set_batch([(0, n)], [table])
    paged.attention_step_device(0, view(qd), view(kd), view(vd), view(out))
    torch.cuda.synchronize()
    assert torch.equal(storage[0, pages - 1, 0, :, 5].cpu(), k[5]) and torch.equal(storage[0, pages - 2, 1, :, 3].cpu(), v[131])
    want, spread, most = PC.attention(q[-20:], k, v, n - 20, 0, 0.0, d ** -0.5)
    assert bool(((out[-20:].cpu().double() - want).abs() <= PC.tolerance(want, spread, most, "f16", "f16", d, n)).all())


# ------------------------------------------------------------------------- streams and graphs

def test_replays_see_the_batch_that_is_set():
    kv_heads, q_heads, d = 2, 8, 64
    cache = PC.Cache(pkg(), [400, 90], layers=2, kv_heads=kv_heads, d=d, page_rows=16, fill="nan")
    for layer in range(2):
        for seq, n in enumerate((400, 90)):
            cache.place(layer, seq, 0, *(cache.normal(n, kv_heads, d).half() for _ in range(2)))
    rotation = pkg().Rotation(64, base=1e4, interleaved=True)
    q, k, v = (cache.normal(2, h, d).half().cuda() for h in (q_heads, kv_heads, kv_heads))
    outs = [torch.empty_like(q) for _ in range(2)]

    def forward():
        for layer in range(2):
            cache.paged.attention_step_device(layer, view(q), view(k), view(v), view(outs[layer]), rotation=rotation)

    stream = torch.cuda.current_stream()
    cache.paged.set_batch([(300, 1), (20, 1)], cache.tables)
    forward()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(stream)
    with torch.cuda.stream(side):
        cache.paged.set_stream(side.cuda_stream)
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(pkg().AttentionError) as e:
                cache.paged.set_batch([(1, 1)], [cache.tables[0]])
            assert e.value.variant == "InvalidArgument"
            forward()
    torch.cuda.synchronize()
    cache.paged.set_stream(stream.cuda_stream)
    for held in ([(300, 1), (20, 1)], [(301, 1), (21, 1)], [(5, 1), (88, 1)], [(398, 1), (0, 1)]):
        before = cache.storage.clone()
        q.copy_(torch.randn(q.shape, generator=cache.g))
        cache.paged.set_batch(held, cache.tables)
        forward()
        torch.cuda.synchronize()
        eager, stored = [o.clone() for o in outs], cache.storage.clone()
        cache.storage.copy_(before)
        for o in outs:
            o.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, outs):
            assert torch.equal(a, b)
        assert torch.equal(cache.storage.view(torch.int16), stored.view(torch.int16))


def test_work_on_a_stream_of_its_own():
    side = torch.cuda.Stream()
    cache = PC.Cache(pkg(), [200], kv_heads=2, d=128, page_rows=32)
    cache.paged.set_stream(side.cuda_stream)
    q, k, v = (cache.normal(3, h, 128).half().cuda() for h in (4, 2, 2))
    out = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.paged.set_batch([(197, 3)], cache.tables)
        cache.paged.attention_step_device(0, view(q), view(k), view(v), view(out))
    cache.paged.synchronize()
    cache.host = cache.storage.cpu()
    check_attention(cache, 0, [(197, 3)], q, out, "f16")
