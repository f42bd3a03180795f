"""What is timed of the paged cache: the rotation of queries and keys, the append of new rows to pages with that
rotation on the way, attention over the pages, and the step that joins them.

  listed()             the named cases
  draw(rng)            one more case of the ranges behind them
  prepare(case, seed)  what a serving program has in hand before the call: pages, tables, new rows, the handles it keeps
  run(state)           one pass through an operator, and its outputs
  exact(case, seed)    the same outputs in 64 bits
  work(case)           the bytes and operations a pass cannot do without

Kinds of case:
  rotate     the queries and keys of `rows` tokens turned by their positions, out of place.
  append     every sequence's new keys (rotated) and values written into its pages.
  attention  every sequence's new queries over its pages, which hold their keys already.
  step       one forward's attention, layer by layer: the batch is set, then on each layer the new queries and keys are
             rotated, keys and values appended, and the queries attend. With `window`, three layers in four are
             windowed and rotated, and the fourth is global and not, which is the pattern of the hybrid models served here.

The pages are one tensor [layer][page][side][kv_head][row of the page][channel], side 0 keys and 1 values; a sequence's
table names its pages in order, scattered over the storage.
`own` = False computes with elementary torch operations in f32, True with this repository's kernels.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BASE = 1e6
ORIGINAL = 32768  # positions a scaled rotation's model was trained on


def _case(kind, name, **kw):
    case = {"kind": kind, "name": name, "layers": 1, "seqs": 1, "rows": 1, "ctx": 4096, "ragged": False, "pages": "f16",
            "tensors": "f16", "page_rows": 64, "head_dim": 128, "q_heads": 32, "kv_heads": 4, "window": 0, "softcap": 0.0,
            "layout": "dense", "rotary_dim": 128, "interleaved": False, "scaling": "plain", "factor": 1.0}
    case.update(kw)
    return case


def listed():
    return [
        # One token's queries and keys between their projections and the cache: the smallest call, all of it latency.
        _case("rotate", "rotate_1row", interleaved=True),
        # A prompt's chunk far behind the trained length, f32 activations as slices of one projection, half of the head turned.
        _case("rotate", "rotate_2048rows_yarn_f32", rows=2048, ctx=90112, tensors="f32", layout="fused", rotary_dim=64,
              scaling="yarn", factor=4.0),
        # Continuous batching: 16 sequences' next tokens into their pages.
        _case("append", "append_16seqs", seqs=16, ctx=16384, ragged=True, pages="bf16", tensors="bf16", layout="fused"),
        # A long prompt's chunk into its pages.
        _case("append", "append_2048_on_30720", rows=2048, ctx=30720, interleaved=True, layout="fused"),
        # One token of one sequence at the context of the headline workload.
        _case("attention", "decode_ctx4096"),
        # Continuous batching: 16 sequences of very different lengths, one token each.
        _case("attention", "decode_ragged16_to_16384", seqs=16, ctx=16384, ragged=True, pages="bf16", tensors="bf16"),
        # A small batch of a model with an unusual head size, small pages, f32 activations.
        _case("attention", "decode_8x1500_d80_f32", seqs=8, ctx=1500, ragged=True, tensors="f32", page_rows=16, head_dim=80,
              kv_heads=8, rotary_dim=80),
        # Speculative verify: four sequences, seven drafted rows each.
        _case("attention", "verify_4x7_ctx8192", seqs=4, rows=7, ctx=8192),
        # A prompt going through a windowed layer in a short block: odd sizes, capped logits.
        _case("attention", "block61_window2048_ctx4099", rows=61, ctx=4099, window=2048, softcap=30.0, layout="heads"),
        # The largest: a long prompt's last chunk.
        _case("attention", "chunk_2048_on_30720", rows=2048, ctx=30720),
        # A long conversation's next token through the hybrid pattern.
        _case("step", "step_hybrid_ctx32768", layers=4, ctx=32768, window=2048, pages="bf16", tensors="bf16", layout="fused",
              interleaved=True),
        # Four short prompts start together, head size 64.
        _case("step", "step_4prompts_509rows_d64", layers=2, seqs=4, rows=509, ctx=0, ragged=True, head_dim=64, kv_heads=8,
              rotary_dim=64, layout="fused"),
    ]


# ------------------------------------------------------------------------------------- drawing

HEADS = [(32, 4), (32, 8), (16, 4), (20, 4), (8, 8), (8, 1)]  # query heads, KV heads
LARGEST = 2048 * (30720 + 1024) * 32 * 128  # query rows x positions x heads x channels of the largest listed case


def _log(rng, low, high):
    return int(round(float(low) * (float(high) / low) ** rng.random())) if high > low else int(low)


def draw(rng):
    kind = rng.choice(["rotate", "append", "attention", "attention", "attention", "step"])
    q_heads, kv_heads = HEADS[0] if rng.random() < 0.3 else rng.choice(HEADS)
    head_dim = rng.choice([128, 128, 64, 80, 96, 112, 192, 256])
    pages = rng.choice(["f16", "bf16"])
    case = _case(kind, "", pages=pages, tensors=rng.choice([pages, pages, "f32"]), page_rows=rng.choice([16, 32, 64, 128]),
                 head_dim=head_dim, q_heads=q_heads, kv_heads=kv_heads, layout=rng.choice(["dense", "fused", "heads"]),
                 rotary_dim=rng.choice([head_dim, head_dim // 2]), interleaved=rng.random() < 0.5,
                 scaling=rng.choice(["plain", "linear", "yarn"]))
    case["factor"] = 1.0 if case["scaling"] == "plain" else rng.choice([2.0, 4.0, 8.0])
    case.pop("name")
    if kind == "rotate":
        case.update(rows=_log(rng, 1, 4096), ctx=_log(rng, 1, 120000), seqs=_log(rng, 1, 8))
    elif kind == "append":
        seqs = _log(rng, 1, 32)
        case.update(seqs=seqs, rows=rng.choice([1, _log(rng, 2, 2048 // seqs + 1)]), ctx=_log(rng, 1, 65536 // seqs),
                    ragged=seqs > 1)
    elif kind == "attention":
        form = rng.choice(["token", "token", "block", "chunk"])
        seqs = {"token": _log(rng, 1, 32), "block": _log(rng, 1, 8), "chunk": rng.choice([1, 1, 2, 3])}[form]
        rows = {"token": 1, "block": rng.randint(2, 9), "chunk": _log(rng, 10, 2048 // seqs)}[form]
        case.update(seqs=seqs, rows=rows, ctx=_log(rng, 30, min(65536, 200000 // seqs)), ragged=seqs > 1 and rng.random() < 0.7,
                    window=rng.choice([0, 0, 512, 2048]), softcap=rng.choice([0.0, 0.0, 30.0]))
    else:
        seqs = _log(rng, 1, 8)
        case.update(layers=rng.choice([2, 4]), seqs=seqs, rows=rng.choice([1, 1, rng.randint(2, 300)]),
                    ctx=rng.choice([0, _log(rng, 30, 32768 // seqs)]), ragged=seqs > 1, window=rng.choice([0, 2048]))
    if kind in ("attention", "step"):
        # (A padded batch costs what its longest sequence costs.)
        most = LARGEST // (case["layers"] * case["seqs"] * case["rows"] * q_heads * head_dim)
        case["ctx"] = max(0 if kind == "step" else 1, min(case["ctx"], most - case["rows"]))
    return case


# ------------------------------------------------------------------------------ what a pass takes

def _spread(case):
    """Every sequence's positions before the pass and its new rows: `ctx` and `rows`, or spread from a 64th of them up to them."""
    n, ctx, rows = case["seqs"], case["ctx"], case["rows"]
    if not case["ragged"] or n == 1:
        return [ctx] * n, [rows] * n
    at = np.random.RandomState(n * 7919 + ctx + rows)
    return ([ctx] + [int(x) for x in at.randint(ctx // 64, ctx + 1, n - 1)],
            [rows] + [int(x) for x in at.randint(max(1, rows // 64), rows + 1, n - 1)])


def _windows(case):
    return [case["window"] if case["kind"] == "attention" or (i + 1) % 4 else 0 for i in range(case["layers"])]


def _rotated(case):
    """Which layers' queries and keys are rotated: all of them, or of the hybrid pattern the windowed ones."""
    return [case["window"] == 0 or w > 0 for w in _windows(case)]


def _bytes(elem):
    return 4 if elem == "f32" else 2


def work(case):
    d, qh, kh, size = case["head_dim"], case["q_heads"], case["kv_heads"], _bytes(case["tensors"])
    held, new = _spread(case)
    rows = sum(new)
    pair = case["rotary_dim"] // 2 * 6
    if case["kind"] == "rotate":
        return {"bytes": rows * ((qh + kh) * d * size * 2 + 8), "flops": rows * (qh + kh) * pair}
    append = {"bytes": 2 * rows * kh * d * (size + 2), "flops": rows * kh * pair}
    if case["kind"] == "append":
        return append
    total = {"bytes": 0, "flops": 0}
    for w, turned in zip(_windows(case), _rotated(case)):
        total["bytes"] += 2 * rows * qh * d * size
        for n, r in zip(held, new):
            seen = min(n + r, w + r - 1) if w else n + r
            fresh = r if case["kind"] == "step" else 0  # a step's new rows are read where the caller left them
            total["bytes"] += 2 * (seen - fresh) * kh * d * 2
            at = np.arange(n + 1, n + r + 1)
            total["flops"] += 4 * d * qh * int((np.minimum(at, w) if w else at).sum())
        if case["kind"] == "step":
            total["bytes"] += append["bytes"]
            total["flops"] += rows * (qh + kh) * pair if turned else 0
    return total


# ------------------------------------------------------------------------------------ inputs

class State:
    pass


def _rows(layout, parts, rows, d, dtype, normal):
    """Tensors of `rows` x heads x d: dense, slices of one projection's output, or heads first."""
    if layout == "fused":
        whole = normal(rows, sum(parts), d).to(dtype)
        return list(whole.split(parts, dim=1))
    if layout == "heads":
        return [normal(h, rows, d).to(dtype).transpose(0, 1) for h in parts]
    return [normal(rows, h, d).to(dtype) for h in parts]


def _inputs(case, seed):
    s = State()
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    d, qh, kh, layers = case["head_dim"], case["q_heads"], case["kv_heads"], case["layers"]
    s.held, s.new = _spread(case)
    rows, dtype = sum(s.new), DTYPES[case["tensors"]]
    s.positions = torch.from_numpy(np.concatenate([np.arange(n, n + r) for n, r in zip(s.held, s.new)])).cuda()
    parts = [_rows(case["layout"], [qh, kh, kh], rows, d, dtype, normal) for _ in range(layers)]
    s.q, s.k, s.v = zip(*parts)
    if case["kind"] == "rotate":
        return s
    # Pages: every sequence's table, scattered; some pages between them are nobody's.
    size = case["page_rows"]
    counts = [-(-(n + r) // size) for n, r in zip(s.held, s.new)]
    s.page_count = sum(counts) + sum(counts) // 8 + 1
    order = np.random.RandomState(seed % (1 << 31)).permutation(s.page_count)
    s.tables = np.split(order[:sum(counts)].astype(np.uint32), np.cumsum(counts)[:-1])
    s.storage = torch.empty(layers, s.page_count, 2, kh, size, d, device="cuda", dtype=DTYPES[case["pages"]])
    s.storage.normal_(generator=g)
    # The batch as tensors: a row's sequence and its place there, tables padded to the longest.
    s.row_seq = torch.from_numpy(np.repeat(np.arange(len(s.new)), s.new)).cuda()
    s.row_in = torch.from_numpy(np.concatenate([np.arange(r) for r in s.new])).cuda()
    table = np.zeros((len(counts), max(counts)), np.int64)
    for at, pages in zip(table, s.tables):
        at[:len(pages)] = pages
    s.table = torch.from_numpy(table).cuda()
    s.first = torch.tensor(s.held, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s.out = [torch.empty_like(q) for q in s.q]
    s.k_out = [torch.empty_like(k) for k in s.k]
    s.freq, s.amplitude = _frequencies(case)
    if own:
        from __graft_entry__ import load_package

        pkg = load_package()
        view = pkg.Rows.of
        s.rotation = pkg.Rotation(case["rotary_dim"], base=BASE, interleaved=case["interleaved"], scaling=case["scaling"],
                                  factor=case["factor"], original_positions=ORIGINAL)
        s.views = [[view(t) for t in layer] for layer in zip(s.q, s.k, s.v, s.out, s.k_out)]
        s.stream = torch.cuda.current_stream().cuda_stream
        if case["kind"] != "rotate":
            s.batch = list(zip(s.held, s.new))
            s.paged = pkg.PagedKv(case["layers"], case["kv_heads"], case["head_dim"], elem=case["pages"],
                                  page_rows=case["page_rows"], page_count=s.page_count, max_sequences=case["seqs"],
                                  storage_ptr=s.storage.data_ptr(), storage_bytes=s.storage.numel() * 2)
            s.paged.set_stream(s.stream)
            s.paged.set_batch(s.batch, s.tables)
    return s


# ------------------------------------------------------------------------------------- passes

def _frequencies(case):
    """Radians a position of every pair, in 64 bits, and what cosine and sine are multiplied by."""
    r, factor = case["rotary_dim"], case["factor"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    plain = BASE ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return plain / factor, 1.0
    if case["scaling"] == "yarn":
        # Pairs that turn more than 32 times over the trained length stay, those below one turn are stretched.
        low, high = (r * math.log(ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(BASE)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return plain * (1 - ramp) + plain / factor * ramp, 0.1 * math.log(factor) + 1
    return plain, 1.0


def _turn(s, x):
    """x [rows][heads][d] rotated by the rows' positions, in f32."""
    x = x.float()
    half, interleaved = s.case["rotary_dim"] // 2, s.case["interleaved"]
    angle = s.positions.double()[:, None, None] * s.freq
    cos, sin = (angle.cos() * s.amplitude).float(), (angle.sin() * s.amplitude).float()
    a = x[..., 0:2 * half:2] if interleaved else x[..., :half]
    b = x[..., 1:2 * half:2] if interleaved else x[..., half:2 * half]
    pair = [a * cos - b * sin, a * sin + b * cos]
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _store(s, layer, k, v):
    at = s.positions // s.case["page_rows"]
    page, row = s.table[s.row_seq, at], s.positions % s.case["page_rows"]
    s.storage[layer, page, 0, :, row] = k.to(s.storage.dtype)
    s.storage[layer, page, 1, :, row] = v.to(s.storage.dtype)


def _attend(s, layer, q, window):
    case = s.case
    n, (qh, kh, d) = case["seqs"], (case["q_heads"], case["kv_heads"], case["head_dim"])
    most = max(s.new)
    held = s.storage[layer][s.table].float()  # [seqs][pages][side][kv_heads][rows][d]
    keys, values = (held[:, :, i].transpose(1, 2).flatten(2, 3) for i in (0, 1))
    padded = torch.zeros(n, most, qh, d, device="cuda")
    padded[s.row_seq, s.row_in] = q.float()
    queries = padded.view(n, most, kh, qh // kh, d).permute(0, 2, 1, 3, 4).reshape(n, kh, -1, d)
    scores = queries @ keys.transpose(2, 3) / math.sqrt(d)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    at = (s.first[:, None] + torch.arange(most, device="cuda")).repeat_interleave(qh // kh, 1)[:, None, :, None]
    key = torch.arange(keys.shape[2], device="cuda")
    hidden = key > at
    if window:
        hidden |= key + window <= at
    scores.masked_fill_(hidden, float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = weights @ values / weights.sum(-1, keepdim=True)
    out = out.view(n, kh, most, qh // kh, d).permute(0, 2, 1, 3, 4).reshape(n, most, qh, d)
    return out[s.row_seq, s.row_in].to(q.dtype)


def _run_plain(s):
    kind = s.case["kind"]
    if kind == "rotate":
        return [_turn(s, s.q[0]).to(s.q[0].dtype), _turn(s, s.k[0]).to(s.k[0].dtype)]
    if kind == "append":
        _store(s, 0, _turn(s, s.k[0]), s.v[0])
        return s.storage
    if kind == "attention":
        return _attend(s, 0, s.q[0], s.case["window"])
    outs = []
    for layer, (w, turned) in enumerate(zip(_windows(s.case), _rotated(s.case))):
        q, k = s.q[layer], s.k[layer]
        _store(s, layer, _turn(s, k) if turned else k, s.v[layer])
        outs.append(_attend(s, layer, _turn(s, q).to(q.dtype) if turned else q, w))
    return [outs, s.storage]


def _run_own(s):
    case = s.case
    q, k, v, out, k_out = s.views[0]
    if case["kind"] == "rotate":
        s.rotation.rotate_device([q, k], [out, k_out], s.positions.data_ptr(), len(s.positions), case["head_dim"], s.stream)
        return [s.out[0], s.k_out[0]]
    if case["kind"] == "append":
        s.paged.append_device(0, k, v, rotation=s.rotation)
        return s.storage
    if case["kind"] == "attention":
        s.paged.attention_device(0, q, out, softcap=case["softcap"], window=case["window"])
        return s.out[0]
    s.paged.set_batch(s.batch, s.tables)
    for layer, (w, turned) in enumerate(zip(_windows(case), _rotated(case))):
        q, k, v, out, _ = s.views[layer]
        s.paged.attention_step_device(layer, q, k, v, out, window=w, rotation=s.rotation if turned else None)
    return [s.out, s.storage]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------- in 64 bits

def _exact_turn(s, x):
    """The rotation as a product of complex numbers."""
    case, r = s.case, s.case["rotary_dim"]
    freq, amplitude = _frequencies(case)
    turn = torch.polar(torch.full((len(s.positions), 1, r // 2), amplitude, dtype=torch.float64, device="cuda"),
                       (s.positions.double()[:, None] * freq)[:, None, :].contiguous())
    y = x.double().clone()
    if case["interleaved"]:
        first, second = slice(0, r, 2), slice(1, r, 2)
    else:
        first, second = slice(0, r // 2), slice(r // 2, r)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attend(s, q, pages, layer_window):
    """Sequence by sequence and KV head by KV head, over the rows as they lie in `pages` [page][side][kv_head][row][d]."""
    case, out, at = s.case, torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    group = case["q_heads"] // case["kv_heads"]
    for n, r, table in zip(s.held, s.new, s.tables):
        ids = torch.from_numpy(table.astype(np.int64)).cuda()
        position = torch.arange(n, n + r, device="cuda")[:, None, None]
        key = torch.arange(n + r, device="cuda")
        seen = key <= position
        if layer_window:
            seen = seen & (key > position - layer_window)
        for h in range(case["kv_heads"]):
            k, v = (pages[ids, side, h].double().flatten(0, 1)[:n + r] for side in (0, 1))
            mine = slice(h * group, (h + 1) * group)
            x = torch.tensordot(q[at:at + r, mine].double(), k, ([2], [1])) * case["head_dim"] ** -0.5
            if case["softcap"]:
                x = (x / case["softcap"]).tanh() * case["softcap"]
            out[at:at + r, mine] = torch.tensordot(torch.softmax(x.where(seen, -math.inf), -1), v, ([2], [0]))
        at += r
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotate":
        return [_exact_turn(s, s.q[0]), _exact_turn(s, s.k[0])]
    if case["kind"] == "attention":
        return _exact_attend(s, s.q[0], s.storage[0], case["window"])
    page = torch.cat([torch.from_numpy(t.astype(np.int64)).cuda()[torch.arange(n, n + r, device="cuda") // case["page_rows"]]
                      for n, r, t in zip(s.held, s.new, s.tables)])
    row = s.positions % case["page_rows"]
    stored, outs = s.storage.double(), []
    for layer, (w, turned) in enumerate(zip(_windows(case), _rotated(case))):
        k = _exact_turn(s, s.k[layer]) if turned else s.k[layer].double()
        stored[layer, page, 0, :, row], stored[layer, page, 1, :, row] = k, s.v[layer].double()
        if case["kind"] == "step":  # what the cache holds are rows of its own type
            s.storage[layer, page, 0, :, row] = k.to(s.storage.dtype)
            s.storage[layer, page, 1, :, row] = s.v[layer].to(s.storage.dtype)
            q = _exact_turn(s, s.q[layer]) if turned else s.q[layer]
            outs.append(_exact_attend(s, q, s.storage[layer], w))
    return stored if case["kind"] == "append" else [outs, stored]
