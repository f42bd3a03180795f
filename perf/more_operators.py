"""What is timed of a paged cache that serves trees of drafted tokens: attention over the cache and the tree, the step that
appends first, the walk that accepts a path of the tree and keeps its rows, and the page tables that the device keeps itself.

  listed()             the named cases
  draw(rng)            one more case of the ranges behind them
  prepare(case, seed)  what a serving program has in hand before the call: pages, tables, drafted trees, the handle it keeps
  run(state)           one pass through an operator, and its outputs
  exact(case, seed)    the same outputs in 64 bits
  work(case)           the bytes and operations a pass cannot do without

A drafted tree is `nodes` new rows of a sequence behind its held positions, each with the number of an earlier row it continues,
or -1 of one that continues the sequence itself. Row r of the tree lies in the pages at position held + r, stands in the text
at position held + its depth, and sees the held positions, its ancestors and itself.

Kinds of case:
  attention  every tree's queries over the held positions and the tree, whose keys and values the pages hold already.
  step       one forward: the batch and its trees are set, then on each layer queries and keys are rotated by the depths, keys and
             values appended, and the queries attend. With `window`, three layers in four are windowed and rotated, and the
             fourth is global and not.
  keep       after a forward: from row 0 on the walk goes to the lowest-numbered child whose token is the one that the model chose at
             its parent; the rows it went through move to the front of the tree in every layer, and the lengths grow by them.
  tables     between forwards: pages are taken from the free list for the new rows of every sequence, the batch and its trees are set from
             lengths and tables on the device, every row's position in the text and place in the storage are written out, and the
             pages behind the lengths go back.

The pages are one tensor [layer][page][side][kv_head][row of the page][channel], side 0 keys and 1 values; a sequence's
table names its pages in order, scattered over the storage.
`own` = False computes with elementary torch operations in f32, True with this repository's kernels.
"""
import math
import zlib

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BASE = 1e6
VOCAB = 32000


def _case(kind, name, **kw):
    case = {"kind": kind, "name": name, "layers": 1, "seqs": 1, "nodes": 16, "depth": 6, "ctx": 4096, "ragged": False,
            "pages": "f16", "tensors": "f16", "page_rows": 64, "head_dim": 128, "q_heads": 32, "kv_heads": 4, "window": 0,
            "softcap": 0.0, "layout": "dense", "interleaved": False}
    case.update(kw)
    return case


def listed():
    return [
        # A small tree of one conversation at the context of the headline workload: latency.
        _case("attention", "tree16_ctx4096"),
        # A tree as deep models draft them, one conversation, f16.
        _case("attention", "tree64_ctx8192", nodes=64, depth=8, ctx=8192),
        # Continuous batching: 16 conversations of very different lengths, their trees of very different sizes.
        _case("attention", "trees26_ragged16_to_16384", seqs=16, nodes=26, ctx=16384, ragged=True, pages="bf16", tensors="bf16"),
        # Very small trees of a model with an unusual head size, small pages, f32 activations.
        _case("attention", "trees5_8x1500_d80_f32", seqs=8, nodes=5, depth=3, ctx=1500, ragged=True, tensors="f32", page_rows=16,
              head_dim=80, kv_heads=8),
        # A windowed layer with capped logits; odd sizes, heads first.
        _case("attention", "trees61_window2048_4x4099", seqs=4, nodes=61, depth=8, ctx=4099, window=2048, softcap=30.0, layout="heads"),
        # The largest: wide trees of eight long conversations.
        _case("attention", "trees256_8x16384", seqs=8, nodes=256, depth=12, ctx=16384, pages="bf16", tensors="bf16"),
        # A long conversation's tree through the hybrid pattern of windowed and global layers.
        _case("step", "step_tree32_hybrid_ctx32768", layers=4, nodes=32, ctx=32768, window=2048, pages="bf16", tensors="bf16",
              layout="fused", interleaved=True),
        # Small trees of many conversations, head size 64.
        _case("step", "step_trees8_16x2000_d64", layers=2, seqs=16, nodes=8, depth=4, ctx=2000, ragged=True, head_dim=64, kv_heads=8,
              layout="fused"),
        # One conversation's walk and its rows: the smallest call.
        _case("keep", "keep_tree16", layers=4, ctx=700),
        # Many conversations', over the layers of a deep model.
        _case("keep", "keep_trees64_16x300_24layers", layers=24, seqs=16, nodes=64, depth=8, ctx=300, ragged=True, pages="bf16"),
        # Tables of a few conversations.
        _case("tables", "tables_4x2000", seqs=4, ctx=2000, ragged=True, page_rows=16),
        # Tables of a full batch of long ones.
        _case("tables", "tables_256x32768", seqs=256, nodes=64, depth=8, ctx=32768, ragged=True),
    ]


# ------------------------------------------------------------------------------------- drawing

HEADS = [(32, 4), (32, 8), (16, 4), (20, 4), (8, 8), (8, 1)]  # query heads, KV heads
LARGEST = 8 * 256 * (16384 + 256) * 32 * 128  # query rows x positions x heads x channels of the largest listed case


def _log(rng, low, high):
    return int(round(float(low) * (float(high) / low) ** rng.random())) if high > low else int(low)


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "step", "keep", "tables"])
    q_heads, kv_heads = HEADS[0] if rng.random() < 0.3 else rng.choice(HEADS)
    pages = rng.choice(["f16", "bf16"])
    case = _case(kind, "", pages=pages, tensors=rng.choice([pages, pages, "f32"]), page_rows=rng.choice([16, 32, 64, 128]),
                 head_dim=rng.choice([128, 128, 64, 80, 96, 112, 192, 256]), q_heads=q_heads, kv_heads=kv_heads,
                 layout=rng.choice(["dense", "fused", "heads"]), interleaved=rng.random() < 0.5)
    case.pop("name")
    seqs = _log(rng, 1, {"attention": 32, "step": 16, "keep": 16, "tables": 256}[kind])
    case.update(seqs=seqs, nodes=_log(rng, 1, 256 if kind in ("attention", "tables") else 64), depth=rng.randint(2, 12),
                ragged=seqs > 1 and rng.random() < 0.7)
    if kind == "attention":
        case.update(ctx=_log(rng, 30, min(65536, 200000 // seqs)), window=rng.choice([0, 0, 512, 2048]),
                    softcap=rng.choice([0.0, 0.0, 30.0]))
    elif kind == "step":
        case.update(layers=rng.choice([2, 4]), ctx=rng.choice([0, _log(rng, 30, 32768 // seqs)]), window=rng.choice([0, 2048]))
    elif kind == "keep":
        case.update(layers=_log(rng, 1, 24), ctx=_log(rng, 1, 500))
    else:
        case.update(ctx=_log(rng, 30, 32768))
    if kind in ("attention", "step"):
        # (A padded batch costs what its longest sequence and its largest tree cost.)
        each = case["layers"] * seqs * q_heads * case["head_dim"]
        case["nodes"] = max(1, min(case["nodes"], LARGEST // (each * 1024)))
        most = LARGEST // (each * case["nodes"])
        case["ctx"] = max(0 if kind == "step" else 1, min(case["ctx"], most - case["nodes"]))
    return case


# ------------------------------------------------------------------------------ what a pass takes

def _spread(case):
    """Every sequence's held positions and its nodes: `ctx` and `nodes`, or spread from a 64th and a quarter of them up to them."""
    n, ctx, nodes = case["seqs"], case["ctx"], case["nodes"]
    if not case["ragged"] or n == 1:
        return [ctx] * n, [nodes] * n
    at = np.random.RandomState(n * 7919 + ctx + nodes)
    return ([ctx] + [int(x) for x in at.randint(ctx // 64, ctx + 1, n - 1)],
            [nodes] + [int(x) for x in at.randint(max(1, nodes // 4), nodes + 1, n - 1)])


def _trees(case):
    """Every sequence's tree (the parent of each row, row 0 the only one without) and an accepted path of it, from row 0 down. The
    trees are as a program orders them, level by level. A path's rows are moved only from behind its end, so that a pass may
    be made again on what it left."""
    at = np.random.RandomState(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()) % (1 << 31))
    trees, paths = [], []
    for nodes in _spread(case)[1]:
        depth = [0]
        for _ in range(nodes - 1):
            deepest = depth[-1]
            deeper = deepest == 0 or (deepest + 1 < case["depth"] and at.rand() < 0.5)
            depth.insert(-1, int(at.randint(1, deepest + 1))) if not deeper else depth.append(deepest + 1)
        depth.sort()
        parents = [-1]
        for r in range(1, nodes):
            above = [i for i in range(r) if depth[i] == depth[r] - 1]
            parents.append(above[min(int(at.geometric(0.4)) - 1, len(above) - 1)])
        level = int(at.randint(0, depth[-1] + 1))
        path = [int(at.choice([i for i in range(nodes) if depth[i] == level]))]
        while path[0]:
            path.insert(0, parents[path[0]])
        while any(p != i and p < len(path) for i, p in enumerate(path)):
            path.pop()
        trees.append(parents), paths.append(path)
    return trees, paths


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


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
    trees, paths = _trees(case)
    if case["kind"] == "keep":
        moved = sum(p != i for path in paths for i, p in enumerate(path))
        return {"bytes": moved * case["layers"] * 2 * kh * d * 2 * 2 + rows * 16 + case["seqs"] * 12, "flops": rows}
    if case["kind"] == "tables":
        taken = sum(-(-(n + r) // case["page_rows"]) + -n // case["page_rows"] for n, r in zip(held, new))
        return {"bytes": case["seqs"] * 16 + rows * 20 + taken * 16, "flops": rows}
    pair = d // 2 * 6
    total = {"bytes": 0, "flops": 0}
    for w, turned in zip(_windows(case), _rotated(case)):
        total["bytes"] += 2 * rows * qh * d * size + 4 * rows
        for n, r, parents in zip(held, new, trees):
            depth = np.array(_depths(parents))
            seen = np.minimum(n, w - 1 - depth) if w else np.full(r, n)  # of the held positions, by each row
            fresh = 0 if case["kind"] == "step" else r  # a step's new rows are read where the caller left them
            total["bytes"] += 2 * (int(seen.max()) + fresh) * kh * d * 2
            total["flops"] += 4 * d * qh * int((seen + depth + 1).sum())
        if case["kind"] == "step":
            total["bytes"] += 2 * rows * kh * d * (size + 2)
            total["flops"] += rows * (qh + kh) * pair if turned else 0
    return total


# ------------------------------------------------------------------------------------ inputs

class State:
    pass


def _rows(layout, parts, rows, d, dtype, normal):
    """Tensors of `rows` x heads x d: dense, slices of one projection's output, or heads first."""
    if layout == "fused":
        return list(normal(rows, sum(parts), d).to(dtype).split(parts, dim=1))
    if layout == "heads":
        return [normal(h, rows, d).to(dtype).transpose(0, 1) for h in parts]
    return [normal(rows, h, d).to(dtype) for h in parts]


def _inputs(case, seed):
    s = State()
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    host = np.random.RandomState(seed % (1 << 31))
    d, qh, kh, layers, n = case["head_dim"], case["q_heads"], case["kv_heads"], case["layers"], case["seqs"]
    s.held, s.new = _spread(case)
    s.trees, s.paths = _trees(case)
    rows, size = sum(s.new), case["page_rows"]
    s.parents = torch.tensor([p for tree in s.trees for p in tree], dtype=torch.int32, device="cuda")
    # The batch as tensors: a row's sequence and its place there.
    s.row_seq = torch.from_numpy(np.repeat(np.arange(n), s.new)).cuda()
    s.row_in = torch.from_numpy(np.concatenate([np.arange(r) for r in s.new])).cuda()
    s.first = torch.tensor(s.held, device="cuda")
    s.rows_each = torch.tensor(s.new, device="cuda")
    s.row0 = torch.from_numpy(np.concatenate([[0], np.cumsum(s.new)[:-1]])).cuda()
    # Pages: every sequence's table, scattered; some pages between them are nobody's. (Of "tables" the free list has those of the new rows.)
    counts = [-(-(a + r) // size) for a, r in zip(s.held, s.new)]
    s.page_count = sum(counts) + sum(counts) // 8 + 1
    order = host.permutation(s.page_count)
    if case["kind"] == "tables":
        s.width = max(counts)
        s.held_pages = [-(-a // size) for a in s.held]
        s.taken = sum(s.held_pages)
        table = np.full((n, s.width), -1, np.int32)
        for at, start, count in zip(table, np.cumsum([0] + s.held_pages), s.held_pages):
            at[:count] = order[start:start + count]
        s.table = torch.from_numpy(table).cuda()
        s.pages = torch.tensor(s.held_pages, dtype=torch.int32, device="cuda")
        s.free = torch.from_numpy(np.append(order[s.taken:], np.full(s.taken, -1)).astype(np.int32)).cuda()
        s.free_count = torch.tensor([s.page_count - s.taken], dtype=torch.int32, device="cuda")
        s.lengths = torch.tensor(s.held, dtype=torch.int32, device="cuda")
        return s
    s.tables = np.split(order[:sum(counts)].astype(np.uint32), np.cumsum(counts)[:-1])
    table = np.zeros((n, max(counts)), np.int64)
    for at, pages in zip(table, s.tables):
        at[:len(pages)] = pages
    s.table = torch.from_numpy(table).cuda()
    s.storage = torch.empty(layers, s.page_count, 2, kh, size, d, device="cuda", dtype=DTYPES[case["pages"]])
    s.storage.normal_(generator=g)
    if case["kind"] == "keep":
        tokens, chosen = host.randint(0, VOCAB, rows), host.randint(0, VOCAB, rows)
        at = 0
        for tree, path in zip(s.trees, s.paths):  # (siblings' tokens differ, and the model chooses none of them at the path's end)
            for r in range(len(tree)):
                tokens[at + r] = (tokens[at + max(tree[r], 0)] * 7 + 13 * r + 1) % VOCAB
            for a, b in zip(path, path[1:]):
                chosen[at + a] = tokens[at + b]
            chosen[at + path[-1]] = VOCAB + host.randint(0, 100)
            at += len(tree)
        s.tokens, s.chosen = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (tokens, chosen))
        return s
    parts = [_rows(case["layout"], [qh, kh, kh], rows, d, DTYPES[case["tensors"]], normal) for _ in range(layers)]
    s.q, s.k, s.v = zip(*parts)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    i32 = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = sum(s.new)
    if kind in ("attention", "step"):
        s.out = [torch.empty_like(q) for q in s.q]
        s.freq = _frequencies(case)
    elif kind == "keep":
        s.path, s.next, s.lengths = i32(rows), i32(case["seqs"]), i32(case["seqs"])
    else:
        s.positions, s.slots = (torch.empty(rows, dtype=torch.int64, device="cuda") for _ in range(2))
    if own:
        from __graft_entry__ import load_package

        pkg = load_package()
        s.stream = torch.cuda.current_stream().cuda_stream
        storage = torch.empty(s.page_count * case["page_rows"] * 16, device="cuda", dtype=torch.float16) if kind == "tables" else s.storage
        s.keep_alive = storage
        s.paged = pkg.PagedKv(case["layers"], 1 if kind == "tables" else case["kv_heads"], 8 if kind == "tables" else case["head_dim"],
                              elem=case["pages"], page_rows=case["page_rows"], page_count=s.page_count, max_sequences=case["seqs"],
                              storage_ptr=storage.data_ptr(), storage_bytes=storage.numel() * 2)
        s.paged.set_stream(s.stream)
        s.paged.enable_trees(rows)
        if kind == "tables":
            s.page_tables = pkg.PageTables.of(s.table, s.pages, s.free, s.free_count)
        else:
            s.batch = list(zip(s.held, s.new))
            s.flat = np.concatenate([np.array(t, np.int32) for t in s.trees])
            s.paged.set_batch(s.batch, s.tables, s.flat)
        if kind in ("attention", "step"):
            s.rotation = pkg.Rotation(case["head_dim"], base=BASE, interleaved=case["interleaved"])
            s.views = [[pkg.Rows.of(t) for t in layer] for layer in zip(s.q, s.k, s.v, s.out)]
    elif kind == "attention":
        s.depth, s.above = _plan(s)
    return s


# ------------------------------------------------------------------------------------- passes

def _frequencies(case):
    """Radians a position of every pair, in 64 bits."""
    i = torch.arange(case["head_dim"] // 2, dtype=torch.float64, device="cuda")
    return BASE ** (-2.0 * i / case["head_dim"])


def _plan(s):
    """Every row's depth, and [row][row of its sequence] whether that is the row itself or above it: as many rounds as the trees are deep."""
    here = s.row0[s.row_seq]
    up = torch.where(s.parents < 0, -1, s.parents + here)  # rows of the batch
    depth = torch.zeros_like(up)
    above = torch.zeros(len(up), max(s.new), dtype=torch.bool, device="cuda")
    row = torch.arange(len(up), device="cuda")
    at = row
    for _ in range(s.case["depth"]):
        on = at >= 0
        above[row, torch.where(on, at - here, s.row_in)] = True
        at = torch.where(on, up[at.clamp(min=0)], -1)
        depth += at >= 0
    return depth, above


def _turn(s, x, positions):
    """x [rows][heads][d] rotated by the rows' positions, in f32."""
    x = x.float()
    angle = positions.double()[:, None, None] * s.freq
    cos, sin = angle.cos().float(), angle.sin().float()
    half, interleaved = x.shape[-1] // 2, s.case["interleaved"]
    a = x[..., 0::2] if interleaved else x[..., :half]
    b = x[..., 1::2] if interleaved else x[..., half:]
    pair = [a * cos - b * sin, a * sin + b * cos]
    return torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)


def _store(s, layer, k, v):
    place = s.first[s.row_seq] + s.row_in
    page, row = s.table[s.row_seq, place // s.case["page_rows"]], place % s.case["page_rows"]
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
    key = torch.arange(keys.shape[2], device="cuda")
    seen = torch.zeros(n, most, keys.shape[2], dtype=torch.bool, device="cuda")
    mine = key < s.first[s.row_seq][:, None]
    if window:
        mine &= key + window > (s.first[s.row_seq] + s.depth)[:, None]
    in_tree = key - s.first[s.row_seq][:, None]
    mine |= (in_tree >= 0) & (in_tree < most) & s.above.gather(1, in_tree.clamp(0, most - 1))
    seen[s.row_seq, s.row_in] = mine
    scores.masked_fill_(~seen.repeat_interleave(qh // kh, 1)[:, None], float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    out = weights @ values / weights.sum(-1, keepdim=True)
    out = out.view(n, kh, most, qh // kh, d).permute(0, 2, 1, 3, 4).reshape(n, most, qh, d)
    return out[s.row_seq, s.row_in].to(q.dtype)


def _walk(s):
    """The accepted paths: from row 0 on the lowest-numbered child whose token was chosen at its parent. Every path as rows of its
    sequence (-1 behind its end), how many, and the model's choice at its last."""
    n, most = s.case["seqs"], max(s.new)
    pad = lambda x, fill: torch.full((n, most), fill, dtype=torch.int64, device="cuda").index_put_((s.row_seq, s.row_in), x.long())  # noqa: E731
    parents, tokens, chosen = pad(s.parents, -2), pad(s.tokens, -1), pad(s.chosen, -1)
    seq = torch.arange(n, device="cuda")
    at, on = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.ones(n, dtype=torch.bool, device="cuda")
    path, last = [], at
    for _ in range(min(s.case["depth"], most)):
        path.append(torch.where(on, at, -1))
        last = torch.where(on, at, last)
        fits = (parents == at[:, None]) & (tokens == chosen[seq, at][:, None])
        on = on & fits.any(1)
        at = torch.where(on, fits.byte().argmax(1), 0)
    path = torch.nn.functional.pad(torch.stack(path, 1), (0, most - len(path)), value=-1)
    return path, chosen[seq, last]


def _run_keep(s):
    path, choice = _walk(s)
    kept = (path >= 0).sum(1)
    seq, to = (path >= 0).nonzero(as_tuple=True)
    a, b = s.first[seq] + path[seq, to], s.first[seq] + to
    size = s.case["page_rows"]
    s.storage[:, s.table[seq, b // size], :, :, b % size] = s.storage[:, s.table[seq, a // size], :, :, a % size]
    return [path[s.row_seq, s.row_in].int(), choice.int(), (s.first + kept).int(), s.storage]


def _run_tables(s):
    size, width = s.case["page_rows"], s.width
    column = torch.arange(width, device="cuda")
    # Pages for the new rows from the end of the free list, sequence by sequence.
    need = -(-(s.lengths + s.rows_each) // size)
    new = (column >= s.pages[:, None]) & (column < need[:, None])
    number = new.flatten().cumsum(0).view_as(new) - 1
    s.table = torch.where(new, s.free[(s.free_count - 1 - number).clamp(min=0)], s.table)
    s.free_count, s.pages = s.free_count - new.sum().int(), need.int()
    # The rows.
    depth, _ = _plan(s)
    place = s.lengths.long()[s.row_seq] + s.row_in
    positions = s.lengths.long()[s.row_seq] + depth
    slots = s.table[s.row_seq, place // size].long() * size + place % size
    # The pages behind the lengths, back to where they were taken.
    fewer = -(-s.lengths // size)
    old = (column >= fewer[:, None]) & (column < s.pages[:, None])
    number = old.flatten().cumsum(0).view_as(old) - 1
    back = old.sum().int()
    s.free[(s.free_count + back - 1 - number)[old]] = s.table[old]
    s.free_count, s.pages = s.free_count + back, fewer.int()
    return [positions, slots, s.table, s.pages, s.free, s.free_count]


def _run_plain(s):
    kind = s.case["kind"]
    if kind == "keep":
        return _run_keep(s)
    if kind == "tables":
        return _run_tables(s)
    if kind == "attention":
        return _attend(s, 0, s.q[0], s.case["window"])
    s.depth, s.above = _plan(s)
    positions = s.first[s.row_seq] + s.depth
    outs = []
    for layer, (w, turned) in enumerate(zip(_windows(s.case), _rotated(s.case))):
        q, k = s.q[layer], s.k[layer]
        _store(s, layer, _turn(s, k, positions) if turned else k, s.v[layer])
        outs.append(_attend(s, layer, _turn(s, q, positions).to(q.dtype) if turned else q, w))
    return [outs, s.storage]


def _run_own(s):
    case, paged = s.case, s.paged
    if case["kind"] == "keep":
        paged.accept_device(s.tokens.data_ptr(), s.chosen.data_ptr(), s.path.data_ptr(), s.next.data_ptr())
        paged.keep_device(s.path.data_ptr(), s.lengths.data_ptr())
        return [s.path, s.next, s.lengths, s.storage]
    if case["kind"] == "tables":
        paged.fit_tables_device(s.page_tables, s.lengths.data_ptr(), s.new)
        paged.set_batch_device(s.page_tables, s.lengths.data_ptr(), s.new, case["ctx"], s.parents.data_ptr())
        paged.batch_rows_device(s.positions.data_ptr(), s.slots.data_ptr())
        paged.fit_tables_device(s.page_tables, s.lengths.data_ptr())
        return [s.positions, s.slots, s.table, s.pages, s.free, s.free_count]
    if case["kind"] == "attention":
        q, k, v, out = s.views[0]
        paged.attention_device(0, q, out, softcap=case["softcap"], window=case["window"])
        return s.out[0]
    paged.set_batch(s.batch, s.tables, s.flat)
    for layer, (w, turned) in enumerate(zip(_windows(case), _rotated(case))):
        q, k, v, out = s.views[layer]
        paged.attention_step_device(layer, q, k, v, out, window=w, rotation=s.rotation if turned else None)
    return [s.out, s.storage]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------- in 64 bits

def _exact_turn(s, x, positions):
    """The rotation as a product of complex numbers."""
    half = x.shape[-1] // 2
    freq = _frequencies(s.case)
    turn = torch.polar(torch.ones(len(positions), 1, half, dtype=torch.float64, device="cuda"),
                       (positions[:, None] * freq)[:, None, :].contiguous())
    y = x.double().clone()
    first, second = (slice(0, None, 2), slice(1, None, 2)) if s.case["interleaved"] else (slice(0, half), slice(half, None))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attend(s, q, pages, window):
    """Sequence by sequence and KV head by KV head, over the rows as they lie in `pages` [page][side][kv_head][row][d]; what a row
    sees is written down by going from it up to its root."""
    case, out, at = s.case, torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    group = case["q_heads"] // case["kv_heads"]
    for n, r, table, parents in zip(s.held, s.new, s.tables, s.trees):
        ids = torch.from_numpy(table.astype(np.int64)).cuda()
        seen = np.zeros((r, n + r), bool)
        for i in range(r):
            up, steps = i, 0
            while up >= 0:
                seen[i, n + up] = True
                up, steps = parents[up], steps + 1
            seen[i, (max(0, n + steps - window) if window else 0):n] = True
        seen = torch.from_numpy(seen).cuda()[:, None]
        for h in range(case["kv_heads"]):
            k, v = (pages[ids, side, h].double().flatten(0, 1)[:n + r] for side in (0, 1))
            mine = slice(h * group, (h + 1) * group)
            x = torch.tensordot(q[at:at + r, mine].double(), k, ([2], [1])) * case["head_dim"] ** -0.5
            if case["softcap"]:
                x = (x / case["softcap"]).tanh() * case["softcap"]
            out[at:at + r, mine] = torch.tensordot(torch.softmax(x.where(seen, -math.inf), -1), v, ([2], [0]))
        at += r
    return out


def _exact_keep(s):
    path, choice, length = [], [], []
    stored, size, at = s.storage.double(), s.case["page_rows"], 0
    chosen = s.chosen.tolist()
    for n, r, table, mine in zip(s.held, s.new, s.tables, s.paths):
        path += mine + [-1] * (r - len(mine))
        choice.append(chosen[at + mine[-1]])
        length.append(n + len(mine))
        place = lambda p: (int(table[p // size]), p % size)  # noqa: E731
        for to, one in enumerate(mine):
            (page, row), (old_page, old_row) = place(n + to), place(n + one)
            stored[:, page, :, :, row] = s.storage[:, old_page, :, :, old_row].double()
        at += r
    return [*(torch.tensor(x, dtype=torch.int32) for x in (path, choice, length)), stored]


def _exact_tables(s):
    size = s.case["page_rows"]
    table, free = s.table.cpu().numpy(), s.free.cpu().numpy()
    count, positions, slots = int(s.free_count), [], []
    for at, n, r, held, parents in zip(table, s.held, s.new, s.held_pages, s.trees):
        for page in range(held, -(-(n + r) // size)):
            count -= 1
            at[page] = free[count]
        positions += [n + d for d in _depths(parents)]
        slots += [int(at[p // size]) * size + p % size for p in range(n, n + r)]
    # (What was taken went back to where it had been.)
    return [torch.tensor(positions), torch.tensor(slots), torch.from_numpy(table), s.pages, s.free, s.free_count]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "keep":
        return _exact_keep(s)
    if case["kind"] == "tables":
        return _exact_tables(s)
    if case["kind"] == "attention":
        return _exact_attend(s, s.q[0], s.storage[0], case["window"])
    place = np.concatenate([np.arange(n, n + r) for n, r in zip(s.held, s.new)])
    page = torch.from_numpy(np.concatenate([t[np.arange(n, n + r) // case["page_rows"]].astype(np.int64)
                                            for n, r, t in zip(s.held, s.new, s.tables)])).cuda()
    row = torch.from_numpy(place % case["page_rows"]).cuda()
    positions = torch.tensor([n + x for n, parents in zip(s.held, s.trees) for x in _depths(parents)], dtype=torch.float64, device="cuda")
    stored, outs = s.storage.double(), []
    for layer, (w, turned) in enumerate(zip(_windows(case), _rotated(case))):
        k = _exact_turn(s, s.k[layer], positions) if turned else s.k[layer].double()
        stored[layer, page, 0, :, row], stored[layer, page, 1, :, row] = k, s.v[layer].double()
        # (What the cache holds are rows of its own type.)
        s.storage[layer, page, 0, :, row] = k.to(s.storage.dtype)
        s.storage[layer, page, 1, :, row] = s.v[layer].to(s.storage.dtype)
        q = _exact_turn(s, s.q[layer], positions) if turned else s.q[layer]
        outs.append(_exact_attend(s, q, s.storage[layer], w))
    return [outs, stored]
