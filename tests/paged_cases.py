"""A paged cache of the tests: inputs, a plain implementation in 64 bits, and how far a right kernel may be from it."""
import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Half a step of each type, relative to the value.
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def frequencies(rotary_dim, base=1e4, scaling="plain", factor=1.0, original=0.0, fast=32.0, slow=1.0):
    """Radians a position of every pair, and the amplitude."""
    out, amplitude = [], 1.0
    if scaling == "yarn":
        edge = [rotary_dim * math.log(original / (2 * math.pi * n)) / (2 * math.log(base)) for n in (fast, slow)]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rotary_dim - 1)
        amplitude = 0.1 * math.log(factor) + 1
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            m = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = f * (1 - m) + f / factor * m
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), amplitude


def rotated(x, positions, freq, amplitude, interleaved, inverse=False):
    """x [rows][heads][channels] turned in 64 bits, and the bound of a kernel's error before it rounds to its type: sine and cosine
    are within 2^-22 (the angle, at most half a turn, is rounded to 24 bits: 2^-25 turns, 2 pi 2^-25 = 1.9e-7 radians, and the
    functions to two units: 2^-23), and two products and a sum are rounded: 2^-21 of |a| + |b| covers the two."""
    x = x.double()
    half = len(freq)
    t = positions.double()[:, None, None] * freq * (-1 if inverse else 1)
    c, s = t.cos() * amplitude, t.sin() * amplitude
    y, err = x.clone(), torch.zeros_like(x)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    err[..., first] = err[..., second] = (a.abs() + b.abs()) * amplitude * 2.0 ** -21
    return y, err


def attention(q, keys, values, position, window, softcap, scale):
    """One sequence in 64 bits: q [rows][heads][d] at positions position .., keys and values [n][kv_heads][d]. The outputs, and for
    the bound of each the sum of its weights times |v| and the largest sum over channels of |q k| * scale it saw."""
    rows, heads, d = q.shape
    n, kv_heads, _ = keys.shape
    group = heads // kv_heads
    q, keys, values = q.double(), keys.double(), values.double()
    out, spread, most = torch.empty_like(q), torch.empty_like(q), torch.empty(rows, heads, dtype=torch.float64)
    at, key = position + torch.arange(rows)[:, None], torch.arange(n)[None]
    seen = key <= at
    if window:
        seen &= key > at - window
    for h in range(heads):
        k, v = keys[:, h // group], values[:, h // group]
        for r in range(rows):  # (a row reads the keys and values it sees and no others)
            mine = seen[r]
            kk, vv = k[mine], v[mine]
            s = kk @ q[r, h] * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            w = torch.softmax(s, 0)
            out[r, h] = (w[:, None] * vv).sum(0)
            spread[r, h] = (w[:, None] * vv.abs()).sum(0)
            most[r, h] = ((kk * q[r, h]).abs().sum(1) * abs(scale)).max()
    return out, spread, most


def tolerance(out, spread, most, pages, tensors, d, n):
    """How far a right kernel's output may be from the one in 64 bits, element by element.

    Weights: rounded to the pages' type (two pieces of it for f32 tensors), relative to each, in the numerator: `weight`. A score's error
    e makes a weight's relative error e: the products' f32 sum of d terms is within d 2^-24 of the sum of |q k|, and f32 queries enter
    as 22 (f16) or 24 (bf16) bits; the scale and the maximum's subtraction round twice more. Numerator and denominator carry it: twice.
    The exponential is within 2^-22, sums over n keys in pieces of 32 within (n / 32 + 40) 2^-24, twice. The output is rounded once."""
    if tensors == "f32":
        weight = 2.0 ** -22 if pages == "f16" else 2.0 ** -16
        query = 2.0 ** -22 if pages == "f16" else 2.0 ** -24
    else:
        weight, query = HALF_STEP[pages], 0.0
    score = (most * (d * 2.0 ** -24 + query) + (most + 16) * 2.0 ** -22)[..., None]
    rel = weight + 2 * score + 2.0 ** -21 + 2 * (n / 32 + 40) * 2.0 ** -24
    return spread * rel * 1.01 + out.abs() * HALF_STEP[tensors] + 1e-30 + (2.0 ** -25 if tensors == "f16" else 0.0)


class Cache:
    """Pages on the GPU with sequences scattered over them, and the same rows on the CPU."""

    def __init__(self, pkg, lengths, *, layers=1, kv_heads=2, d=64, pages="f16", page_rows=16, spare=3, max_sequences=8, seed=0,
                 fill="normal", device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.g, self.pages, self.page_rows, self.d, self.kv_heads = g, pages, page_rows, d, kv_heads
        counts = [-(-n // page_rows) for n in lengths]
        self.page_count = sum(counts) + spare
        order = torch.randperm(self.page_count, generator=g).tolist()
        self.tables, at = [], 0
        for n in counts:
            self.tables.append(order[at:at + n])
            at += n
        self.host = torch.randn(layers, self.page_count, 2, kv_heads, page_rows, d, generator=g).to(DTYPES[pages])
        if fill == "nan":  # rows nobody may look at
            self.host[:] = float("nan")
        self.storage = self.host.to(device)
        self.paged = pkg.PagedKv(layers, kv_heads, d, elem=pages, page_rows=page_rows, page_count=self.page_count,
                                 max_sequences=max_sequences, max_table_pages=sum(counts) + 8,
                                 storage_ptr=self.storage.data_ptr(), storage_bytes=self.storage.numel() * 2)
        self.paged.set_stream(torch.cuda.current_stream().cuda_stream)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g)

    def place(self, layer, seq, first, keys, values):
        """Rows [n][kv_heads][d] of a sequence from position `first` on, on the host and the device."""
        for r in range(len(keys)):
            p = first + r
            page, row = self.tables[seq][p // self.page_rows], p % self.page_rows
            self.host[layer, page, 0, :, row], self.host[layer, page, 1, :, row] = keys[r], values[r]
        self.storage.copy_(self.host)

    def rows(self, layer, seq, n):
        """The first n positions' keys and values [n][kv_heads][d] as the host's pages hold them."""
        at = self.host[layer][self.tables[seq]]  # [pages][2][kv_heads][page_rows][d]
        flat = at.permute(1, 0, 3, 2, 4).reshape(2, -1, self.kv_heads, self.d)
        return flat[0, :n], flat[1, :n]


def laid_out(x, layout, device="cuda"):
    """x [rows][heads][d] on the device as `layout` says: dense, heads first, a slice of wider rows, or one element off 16 bytes."""
    rows, heads, d = x.shape
    if layout == "heads":
        return x.transpose(0, 1).contiguous().to(device).transpose(0, 1)
    if layout == "slice":
        wide = torch.zeros(rows, heads + 3, d, dtype=x.dtype, device=device)
        wide[:, 1:1 + heads] = x.to(device)
        return wide[:, 1:1 + heads]
    if layout == "odd":
        flat = torch.zeros(rows * (heads * d + 1) + 1, dtype=x.dtype, device=device)
        view = flat[1:1 + rows * (heads * d + 1)].view(rows, heads * d + 1)[:, :heads * d].view(rows, heads, d)
        view.copy_(x.to(device))
        return view
    return x.to(device).contiguous()
