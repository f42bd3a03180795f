"""f32 tensors over bf16 pages: queries and softmax weights enter the products as three bf16 pieces each, 24 bits of them; of two pieces
16 to 18 bits would be left, and these outputs show it."""
import pytest
import torch

import paged_cases as PC
from helpers import pkg
from test_gpu_paged import view

pytestmark = pytest.mark.gpu


def left(x):
    """What two bf16 pieces leave of each number, relative to it."""
    first = x.float().bfloat16().double()
    second = (x - first).float().bfloat16().double()
    return (x - first - second).abs() / x.abs()


def outputs(position, rows, keys, values, q, scale):
    n, d = position + rows, keys.shape[-1]
    cache = PC.Cache(pkg(), [n], kv_heads=1, d=d, pages="bf16", page_rows=16, fill="nan")
    cache.place(0, 0, 0, keys.bfloat16(), values.bfloat16())
    out, qd = torch.empty(q.shape, device="cuda"), q.float().cuda()
    cache.paged.set_batch([(position, rows)], cache.tables)
    cache.paged.attention_device(0, view(qd), view(out), scale=scale)
    torch.cuda.synchronize()
    return out.cpu().double()


# Eight keys of one weight w beside one of the weight 1, values 1 and 0: the output is 8 w / (1 + 8 w), and what the pieces leave out of w
# is missing from the numerator alone. Errors, relative to the output: at most 9 additions, the division, the product and the output's
# rounding 2^-24 each in numerator and denominator, 2^-19.7 of 20 in all; w's own error (its exponential and its score, 2^-21) counts for
# 1 / (1 + 8 w), below a fifth: 2^-23.3. Together below 2^-19.5.
@pytest.mark.parametrize("rows", [1, 40])  # the kernels of few and of many rows
def test_weights_keep_24_bits(rows):
    scores = torch.arange(0.25, 0.7, 2.0 ** -9, dtype=torch.float64)  # of eight bits or fewer: what bf16 holds
    scores = scores[scores.bfloat16().double() == scores]
    lost = left(torch.exp(-scores))
    score = float(scores[lost.argmax()])
    position, n, tol = 8, 8 + rows, 2.0 ** -19.5
    keys, values = torch.zeros(n, 1, 64), torch.zeros(n, 1, 64)
    keys[1:9, 0, 0], values[1:9] = -score, 1.0
    keys[9:, 0, 0] = -200.0  # (weights of e^-200: zero)
    q = torch.zeros(rows, 4, 64)
    q[..., 0] = 1.0
    w = torch.exp(torch.tensor(-score, dtype=torch.float64))
    want = float(8 * w / (1 + 8 * w))
    off = (outputs(position, rows, keys, values, q, 1.0) / want - 1).abs().max()
    assert float(lost.max()) > 1.5 * tol  # (two pieces would be seen)
    assert float(off) <= tol, float(off)


# Two keys, values 0 and 1: the output is w / (1 + w), w = e^(-16 q) of a query channel q near 0.25 with 24 bits, and an error of the score counts
# for 1 / (1 + w) = 0.98 of the output. A score of 4 (5.8 in the log2 domain) is rounded three times, as a sum, by the scale and by the scale's
# own rounding: 12 * 2^-24 = 2^-20.4. The exponential takes 2^-22, the sum, the division, the product and the output 5 * 2^-24. Together
# below 2^-19.5, where two pieces of q leave up to 4 * 2^-17 of the score out.
@pytest.mark.parametrize("rows", [1, 40])
def test_queries_keep_24_bits(rows):
    g = torch.Generator().manual_seed(1)
    some = (0.25 + 0.05 * torch.rand(4096, generator=g)).double()
    lost = left(some)
    channel = float(some[lost.argmax()])
    position, n, tol = 1, 1 + rows, 2.0 ** -19.5
    keys, values = torch.zeros(n, 1, 64), torch.zeros(n, 1, 64)
    keys[1, 0, 3], values[1] = -16.0, 1.0
    keys[2:, 0, 3] = -800.0  # (weights of e^-200: zero)
    q = torch.zeros(rows, 4, 64, dtype=torch.float64)
    q[..., 3] = channel
    w = torch.exp(torch.tensor(-16.0 * channel, dtype=torch.float64))
    want = float(w / (1 + w))
    off = (outputs(position, rows, keys, values, q, 1.0) / want - 1).abs().max()
    assert 0.98 * 4 * float(lost.max()) > 2 * tol  # (two pieces would be seen)
    assert float(off) <= tol, float(off)
