"""Caps far above the scores: cap * tanh(s / cap) is then nearly s, and the softmax is that of the scores."""
import math

import pytest
import torch

import paged_cases as PC
from helpers import pkg
from test_gpu_paged import check_attention, view

pytestmark = pytest.mark.gpu

TYPES = [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")]


# A capped score is within a few roundings of itself, which the tolerance of a score without a cap has room for, whatever the cap: the
# scale's and the maximum's 2^-22 of it are two roundings of 2^-24 each, and the series of tanh takes five more. `nan`: a value of
# the newest row is none, and the unit is done over.
@pytest.mark.parametrize("pages,tensors", TYPES)
@pytest.mark.parametrize("position,rows", [(300, 1), (300, 40), (4000, 2)])
@pytest.mark.parametrize("softcap", [300.0, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("nan", [False, True])
def test_large_caps(pages, tensors, position, rows, softcap, nan):
    d, n = 64, position + rows
    cache = PC.Cache(pkg(), [n], kv_heads=2, d=d, pages=pages, page_rows=64, fill="nan", seed=rows)
    keys, values = (cache.normal(n, 2, d) for _ in range(2))
    if nan:
        values[n - 1, 1, 8] = float("nan")
    cache.place(0, 0, 0, keys.to(PC.DTYPES[pages]), values.to(PC.DTYPES[pages]))
    q = cache.normal(rows, 8, d).to(PC.DTYPES[tensors])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch([(position, rows)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), softcap=softcap, scale=0.3)
    torch.cuda.synchronize()
    check_attention(cache, 0, [(position, rows)], q, out, tensors, softcap=softcap, scale=0.3)


# Caps where the short form of the 16-bit types ends: its error is 2^-22 of the cap, in a weight's numerator and denominator.
@pytest.mark.parametrize("pages", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("softcap", [1.0, 30.0, 255.0, 256.0, 257.0])
def test_caps_of_both_forms(pages, rows, softcap):
    cache = PC.Cache(pkg(), [200 + rows], kv_heads=2, d=128, pages=pages, page_rows=64, fill="nan", seed=rows)
    keys, values = (cache.normal(200 + rows, 2, 128).to(PC.DTYPES[pages]) for _ in range(2))
    cache.place(0, 0, 0, keys, values)
    q = cache.normal(rows, 4, 128).to(PC.DTYPES[pages])
    out, qd = torch.empty_like(q, device="cuda"), q.cuda()
    cache.paged.set_batch([(200, rows)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), softcap=softcap)
    torch.cuda.synchronize()
    want, spread, most = PC.attention(q, keys, values, 200, 0, softcap, 128 ** -0.5)
    tol = PC.tolerance(want, spread, most, pages, pages, 128, 200 + rows) + spread * 2 * softcap * 2.0 ** -22
    assert bool(((out.cpu().double() - want).abs() <= tol).all())


def test_caps_beyond_what_f32_holds_are_refused():
    P = pkg()
    cache = PC.Cache(P, [40], kv_heads=1, d=64, page_rows=16)
    for dtype in (torch.float16, torch.float32):
        q, out = (torch.full((1, 2, 64), x, dtype=dtype, device="cuda") for x in (1.0, 7.0))
        cache.paged.set_batch([(39, 1)], cache.tables)
        for softcap, scale in ((3e38, 1.0), (1e38, None), (1e30, 1e-10)):
            with pytest.raises(P.AttentionError) as e:
                cache.paged.attention_device(0, view(q), view(out), softcap=softcap, scale=scale)
            assert e.value.variant == "Unsupported"
        torch.cuda.synchronize()
        assert bool((out == 7.0).all())
        cache.paged.attention_device(0, view(q), view(out), softcap=30.0, scale=0.0)  # (scores of zero: the mean of the values)
        torch.cuda.synchronize()
        check_attention(cache, 0, [(39, 1)], q.cpu(), out, "f32" if dtype == torch.float32 else "f16", softcap=30.0, scale=0.0)
        assert not math.isnan(float(out.float().sum()))
