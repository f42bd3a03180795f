"""Attention over bf16 pages whose values reach the ends of the type's range: a weighted mean of finite values is finite."""
import pytest
import torch

import paged_cases as PC
from helpers import pkg
from test_gpu_paged import check_attention, view

pytestmark = pytest.mark.gpu

CASES = [
    # q heads, kv heads, d, page rows, [(position, rows)], window
    (4, 2, 64, 16, [(0, 1)], 0),
    (8, 2, 128, 16, [(700, 1), (5, 1)], 0),        # few rows, whole
    (4, 1, 128, 64, [(6000, 1)], 0),               # few rows in parts that the merge joins
    (4, 1, 80, 64, [(5000, 3)], 4000),
    (8, 2, 128, 16, [(120, 40), (33, 1)], 0),      # many rows, whole
    (4, 1, 64, 64, [(3000, 20)], 0),               # many rows in parts
    (4, 2, 256, 16, [(90, 30)], 50),
    (8, 1, 96, 32, [(2000, 9)], 0),
]


# Beside ordinary values: a channel of large ones, one of the largest throughout, one of the largest with both signs, and one of small
# ones. The tolerance is relative to the weighted sum of magnitudes in the channel; f32 sums and a rounding to bf16 of numbers that are
# 2^-7 below the type's end do not reach it.
@pytest.mark.parametrize("tensors", ["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_finite_values_come_out_finite(tensors, case):
    q_heads, kv_heads, d, page_rows, items, window = case
    cache = PC.Cache(pkg(), [p + r for p, r in items], kv_heads=kv_heads, d=d, pages="bf16", page_rows=page_rows, fill="nan", seed=d)
    for seq, (p, r) in enumerate(items):
        n = p + r
        keys, values = (cache.normal(n, kv_heads, d) for _ in range(2))
        if seq == 0:
            values[..., 3] *= 1e37
            values[..., 5] = 3.3e38
            values[..., 6] = torch.where(torch.arange(n) % 3 == 0, -3.2e38, 3.0e38)[:, None]
            values[..., 7] *= 1e-20
        cache.place(0, seq, 0, keys.bfloat16(), values.bfloat16())
    rows = sum(r for _, r in items)
    q = cache.normal(rows, q_heads, d).to(PC.DTYPES[tensors])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch(items, cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), window=window)
    torch.cuda.synchronize()
    assert bool(out.isfinite().all())
    check_attention(cache, 0, items, q, out, tensors, window)


# Beside them a row that is not finite, which reaches the queries that see it and no others.
@pytest.mark.parametrize("tensors", ["bf16", "f32"])
@pytest.mark.parametrize("position,rows", [(100, 2), (100, 40), (5000, 3), (3000, 20)])
def test_infinities_beside_the_largest_values(tensors, position, rows):
    n = position + rows
    cache = PC.Cache(pkg(), [n], kv_heads=1, d=64, pages="bf16", page_rows=64, fill="nan", seed=rows)
    keys, values = (cache.normal(n, 1, 64) for _ in range(2))
    values[..., 5] = 3.3e38
    values[n - 1, 0, 5] = float("inf")   # the newest row's
    values[n - 1, 0, 9] = float("-inf")
    values[n // 2, 0, 11] = float("nan")
    cache.place(0, 0, 0, keys.bfloat16(), values.bfloat16())
    q = cache.normal(rows, 4, 64).to(PC.DTYPES[tensors])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch([(position, rows)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out))
    torch.cuda.synchronize()
    got = out.cpu().double()
    want, spread, most = PC.attention(q, *cache.rows(0, 0, n), position, 0, 0.0, 64 ** -0.5)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    tol, fine = PC.tolerance(want, spread, most, "bf16", tensors, 64, n), want.isfinite()
    assert bool(((got - want).abs()[fine] <= tol[fine]).all())


# Every key scores the same 10^10 and more, beyond which 32 is lost in f32: parts with values that a sum cannot hold and parts without them
# weigh alike all the same. Of powers of two the score is the scale, 24 bits, times one of them, which f32 holds: weights are 1 to the bit and the
# output is the mean, whose sums of up to 6,001 values in pieces of 32 and a merge of up to 256 stay within 2^-14, beside the rounding
# of the output. Of 10^5 squared the product with the scale is rounded, by up to 2^9 where a weight's exponent is the difference of two of
# them, so that any mean of the values is right.
@pytest.mark.parametrize("tensors", ["bf16", "f32"])
@pytest.mark.parametrize("position,rows", [(6000, 1), (3000, 20)])
@pytest.mark.parametrize("channel", [2.0 ** 17, 1e5])
def test_parts_weigh_alike_at_large_scores(tensors, position, rows, channel):
    n = position + rows
    cache = PC.Cache(pkg(), [n], kv_heads=1, d=64, pages="bf16", page_rows=64, fill="nan")
    keys, values = torch.zeros(n, 1, 64), torch.ones(n, 1, 64)
    keys[..., 0] = channel
    values[n // 2:, 0, 4] = 3e38
    cache.place(0, 0, 0, keys.bfloat16(), values.bfloat16())
    q = torch.zeros(rows, 4, 64)
    q[..., 0] = channel
    q = q.to(PC.DTYPES[tensors])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch([(position, rows)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), scale=1.0)
    torch.cuda.synchronize()
    got, values = out.cpu().double(), cache.rows(0, 0, n)[1].double()
    tol = 2.0 ** -14 + PC.HALF_STEP[tensors]
    if channel == 1e5:
        assert bool((got >= values.amin(0) * (1 - tol)).all()) and bool((got <= values.amax(0) * (1 + tol)).all())
        return
    mean = values.cumsum(0)[position:] / torch.arange(position + 1, n + 1).double()[:, None, None]
    off = float((got / mean - 1).abs().max())
    assert off <= tol, off
