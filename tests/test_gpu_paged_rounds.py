"""Rounds of trees that the device keeps the books of: page tables that grow and shrink, batches from lengths and tables there, the walk
down a tree, the rows that are kept, and all of it in turn as a serving program runs it, eagerly and as one captured graph."""
import numpy as np
import pytest
import torch

import paged_cases as PC
import tree_cases as TC
from helpers import pkg, refusal

pytestmark = pytest.mark.gpu


def view(t):
    return pkg().Rows.of(t)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


KEPT = []


def at(values):
    """Where these words lie on the device; they stay there."""
    KEPT.append(i32(values))
    return KEPT[-1].data_ptr()


@pytest.fixture(autouse=True)
def kept():
    yield
    torch.cuda.synchronize()
    KEPT.clear()


class Tables:
    """Page tables on the device and, as lists, by hand."""

    def __init__(self, sequences, width, page_count, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.table = [[-1] * width for _ in range(sequences)]
        self.pages, self.count = [0] * sequences, page_count
        self.free = torch.randperm(page_count, generator=g).tolist()
        self.dev = [i32(self.table), i32(self.pages), i32(self.free), i32([page_count])]
        self.raw = pkg().PageTables.of(*self.dev)

    def fit(self, wanted):
        self.count, refused = TC.fit(self.table, self.pages, self.free, self.count, wanted)
        return refused

    def same(self):
        table, pages, free, count = (t.cpu().tolist() for t in self.dev)
        assert pages == self.pages and count == [self.count] and free[:self.count] == self.free[:self.count]
        for a, b, n in zip(table, self.table, pages):
            assert a[:n] == b[:n]
        live = free[:count[0]] + [p for a, n in zip(table, pages) for p in a[:n]]
        assert sorted(live) == sorted(set(live)) and len(live) == len(self.free)  # every page is somewhere, once


def small(**kw):
    kw = {"layers": 1, "kv_heads": 1, "d": 8, "page_rows": 16, "page_count": 64, "max_sequences": 1024, **kw}
    paged = pkg().PagedKv(kw["layers"], kw["kv_heads"], kw["d"], page_rows=kw["page_rows"], page_count=kw["page_count"],
                          max_sequences=kw["max_sequences"], max_table_pages=kw.get("max_table_pages", 0))
    paged.set_stream(torch.cuda.current_stream().cuda_stream)
    return paged


@pytest.mark.parametrize("sequences,page_count,width", [(1, 3, 3), (5, 40, 12), (70, 300, 9), (1000, 2000, 5)])
def test_tables_grow_and_shrink(sequences, page_count, width):
    paged, tables = small(page_count=page_count), Tables(sequences, width, page_count, sequences)
    rng = np.random.RandomState(sequences)
    for turn in range(6):
        lengths = rng.randint(0, 16 * width + 1 - 20, sequences)
        rows = rng.randint(0, 21, sequences) if turn % 2 else None
        status = i32([-1] * sequences)
        paged.fit_tables_device(tables.raw, at(lengths), rows, status.data_ptr())
        refused = tables.fit([-(-int(x) // 16) for x in (lengths if rows is None else lengths + rows)])
        torch.cuda.synchronize()
        assert [bool(x) for x in status.tolist()] == refused and set(status.tolist()) <= {0, 6}
        tables.same()


def test_pages_that_go_back_are_the_ones_taken_next():
    paged, tables = small(), Tables(3, 20, 64, 7)
    held, more = i32([17, 0, 160]), [30, 100, 1]
    paged.fit_tables_device(tables.raw, held.data_ptr())
    before = [t.clone() for t in tables.dev]
    paged.fit_tables_device(tables.raw, held.data_ptr(), more)
    grown = [t.clone() for t in tables.dev]
    paged.fit_tables_device(tables.raw, held.data_ptr())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(tables.dev[1:], before[1:]))
    paged.fit_tables_device(tables.raw, held.data_ptr(), more)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(tables.dev, grown))


def test_tables_that_are_none_are_left_as_they_are():
    paged = small(page_count=8)
    for pages, count, lengths, status in (([1, -1, 9, 1], 4, [20, 20, 20, 16], [0, 2, 2, 0]), ([0, 1, 1, 0], 4, [-1, 16, 16 * 4 + 1, 0], [1, 0, 1, 0]),
                                          ([1, 1, 0, 0], 9, [0, 16, 16, 0], [6, 0, 6, 0]), ([1, 1, 0, 0], -1, [0, 16, 16, 0], [6, 0, 6, 0]),
                                          ([4, 4, 0, 0], 7, [0, 64, 0, 0], [6, 0, 0, 0])):
        table, got, free = i32([[0, 1, 2, 3], [4, 5, 6, 7], [0] * 4, [0] * 4]), i32([9] * 4), i32(range(8))
        have, left = i32(pages), i32([count])
        paged.fit_tables_device(pkg().PageTables.of(table, have, free, left), at(lengths), None, got.data_ptr())
        torch.cuda.synchronize()
        assert got.tolist() == status, (got.tolist(), status)
        want = [-(-n // 16) if s == 0 and n >= 0 else p for n, s, p in zip(lengths, status, pages)]
        assert have.tolist() == want and left.tolist() == [count - sum(max(0, w - max(p, 0)) for w, p in zip(want, pages)) if 0 <= count <= 8 else count]


@pytest.mark.parametrize("trees", [True, False])
@pytest.mark.parametrize("sequences", [1, 6, 300])
def test_a_batch_from_the_device_is_the_one_from_the_host(sequences, trees):
    rng = np.random.RandomState(sequences)
    held = rng.randint(0, 90, sequences).tolist()
    new = rng.randint(0, 8, sequences).tolist()
    new[0] = 40
    items = list(zip(held, new))
    cache = PC.Cache(pkg(), [p + r + 1 for p, r in items], kv_heads=1, d=8, page_rows=16, max_sequences=sequences, seed=sequences)
    parents = [TC.tree(r, i) if i % 3 else TC.chain(r) for i, r in enumerate(new)]
    parents[0] = TC.tree(40, 9)
    if trees:
        cache.paged.enable_trees(sum(new))
    width = max(len(t) for t in cache.tables)
    table = i32([t + [0] * (width - len(t)) for t in cache.tables])
    tables = pkg().PageTables.of(table, i32([len(t) for t in cache.tables]))
    flat = torch.from_numpy(TC.flat(parents)).cuda()
    rows = sum(new)
    q = cache.normal(rows, 2, 8).half().cuda()
    got = []
    for host in (True, False):
        status, out = i32([-1] * sequences), torch.zeros_like(q)
        positions, slots = (torch.full((rows,), -7, device="cuda") for _ in range(2))
        if host:
            cache.paged.set_batch(items, cache.tables, TC.flat(parents) if trees else None)
        else:
            cache.paged.set_batch_device(tables, at(held), new, 100, flat.data_ptr() if trees else 0, status.data_ptr())
        cache.paged.batch_rows_device(positions.data_ptr(), slots.data_ptr())
        cache.paged.attention_device(0, view(q), view(out))
        torch.cuda.synchronize()
        got.append((positions, slots, out))
    assert status.tolist() == [0] * sequences
    stand = [p + x for (p, r), t in zip(items, parents) for x in (TC.depths(t) if trees else range(r))]
    place = [cache.tables[s][x // 16] * 16 + x % 16 for s, (p, r) in enumerate(items) for x in range(p, p + r)]
    for positions, slots, out in got:
        assert positions.tolist() == stand and slots.tolist() == place
        TC.check(cache, 0, items, parents if trees else [TC.chain(r) for r in new], q, out, "f16")
    # Either output alone.
    positions.fill_(-7)
    cache.paged.batch_rows_device(positions.data_ptr())
    torch.cuda.synchronize()
    assert positions.tolist() == stand
    # Back to one that the host sets.
    cache.paged.set_batch(items[:1], cache.tables[:1], TC.flat(parents[:1]) if trees else None)
    out.zero_()
    cache.paged.attention_device(0, view(q[:40]), view(out[:40]))
    torch.cuda.synchronize()
    TC.check(cache, 0, items[:1], parents[:1] if trees else [TC.chain(40)], q, out[:40], "f16")


def test_sequences_that_the_device_leaves_out():
    new = [3, 2, 4, 3, 2, 5, 0, 2]
    held = [17, -1, 40, 101, 20, 0, -5, 60]
    cache = PC.Cache(pkg(), [40, 40, 44, 120, 40, 40, 5, 62], kv_heads=1, d=8, page_rows=16, max_sequences=8, seed=1)
    cache.paged.enable_trees(64)
    table = i32([t + [0] * (8 - len(t)) for t in cache.tables])
    pages = [len(t) for t in cache.tables]
    pages[4] = 1                                  # too few for 22 positions
    table[5, 0] = cache.page_count                # no page
    parents = [[-1, 0, 0], [-1, 0], [-1, 0, 2, 1], [-1, 0, 0], [-1, 0], [-1, 0, 0, 0, 0], [], [-1, -1]]  # (the third's second goes nowhere)
    status, rows = i32([9] * 8), sum(new)
    q, k, v = (cache.normal(rows, h, 8).half().cuda() for h in (2, 1, 1))
    out, before = torch.full_like(q, 7.0), cache.storage.clone()
    positions, slots = (torch.zeros(rows, dtype=torch.int64, device="cuda") for _ in range(2))
    path, following, lengths = i32([9] * rows), i32([9] * 8), i32([9] * 8)
    tokens = i32([1] * rows)
    tables = pkg().PageTables.of(table, i32(pages))
    cache.paged.set_batch_device(tables, at(held), new, 100, at([p for t in parents for p in t]), status.data_ptr())
    cache.paged.attention_step_device(0, view(q), view(k), view(v), view(out))
    cache.paged.batch_rows_device(positions.data_ptr(), slots.data_ptr())
    cache.paged.accept_device(tokens.data_ptr(), tokens.data_ptr(), path.data_ptr(), following.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [0, 1, 4, 1, 2, 3, 0, 0]
    in_ = [s in (0, 7) for s, r in enumerate(new) for _ in range(r)]
    assert [x >= 0 for x in positions.tolist()] == in_ and [x >= 0 for x in slots.tolist()] == in_
    for r, taken in enumerate(in_):
        assert taken != bool((out[r] == 7.0).all())
    assert path.tolist() == [x if t else -1 for x, t in zip([0, 1, -1] + [0] * 16 + [0, -1], in_)]
    assert following.tolist() == [1, 9, 9, 9, 9, 9, 9, 1]
    written = torch.zeros(cache.page_count * 16, dtype=torch.bool)
    written[[x for x in slots.tolist() if x >= 0]] = True
    same = (cache.storage.view(torch.int16) == before.view(torch.int16)).cpu()[0].permute(0, 3, 1, 2, 4).reshape(cache.page_count * 16, -1)
    assert bool(same[~written].all()) and not bool(same[written].any(1).logical_not().any() and same[written].all())
    cache.paged.keep_device(path.data_ptr(), lengths.data_ptr())
    torch.cuda.synchronize()
    assert lengths.tolist() == [19, 9, 9, 9, 9, 9, 9, 61]


def test_more_page_ids_than_a_batch_takes():
    paged = small(page_count=16, max_table_pages=5)
    table = i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    status, rows = i32([9] * 3), [1, 1, 1]
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    tables = pkg().PageTables.of(table, i32([3, 3, 3]))
    paged.set_batch_device(tables, at([40, 40, 15]), rows, 40, 0, status.data_ptr())
    paged.batch_rows_device(0, slots.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [0, 5, 5] and slots.tolist() == [2 * 16 + 8, -1, -1]


@pytest.mark.parametrize("largest", [1, 2, 16, 64, 65, 256])
def test_walks(largest):
    rng = np.random.RandomState(largest)
    new = [largest, 1, 0, max(1, largest // 2), largest, 300 if largest == 256 else 3]
    parents = [TC.tree(r, i, 20) for i, r in enumerate(new[:-1])] + [TC.chain(new[-1])]
    parents[2] = []
    items = [(5, r) for r in new]
    cache = PC.Cache(pkg(), [5 + r for r in new], kv_heads=1, d=8, page_rows=16, seed=3)
    cache.paged.enable_trees(sum(new))
    for vocabulary in (1, 2, 3):  # (of one token every walk goes as deep as its lowest-numbered rows do)
        tokens, chosen = (rng.randint(-1, vocabulary, sum(new)).astype(np.int32) for _ in range(2))
        if vocabulary == 1:
            tokens[:], chosen[:] = -5, -5
        path, following = i32([9] * sum(new)), i32([9] * 6)
        for flat in ((TC.flat(parents), None) if vocabulary == 2 else (TC.flat(parents),)):
            cache.paged.set_batch(items, cache.tables, flat)
            t, c = torch.from_numpy(tokens).cuda(), torch.from_numpy(chosen).cuda()
            cache.paged.accept_device(t.data_ptr(), c.data_ptr(), path.data_ptr(), following.data_ptr())
            torch.cuda.synchronize()
            first, want, ends = 0, [], []
            for p, r in zip(parents, new):
                if r:
                    mine, end = TC.walk(p if flat is not None else TC.chain(r), tokens[first:first + r], chosen[first:first + r])
                    want += mine + [-1] * (r - len(mine))
                ends.append(int(end) if r else 9)
                first += r
            assert path.tolist() == want and following.tolist() == ends


@pytest.mark.parametrize("pages,d,kv_heads,page_rows", [("f16", 64, 2, 16), ("bf16", 8, 1, 32), ("f16", 256, 3, 16)])
def test_kept_rows(pages, d, kv_heads, page_rows):
    new = [40, 12, 1, 0, 256, 300, 6, 5]
    items = [(p, r) for p, r in zip([30, 16, 0, 5, 7, 3, 9, 11], new)]
    paths = [[2, 3, 5, 6, 7, 20, 39], [0, 4, 11], [0], [], list(range(0, 256, 3)), list(range(290)), [], [0, 3, 3]]
    cache = PC.Cache(pkg(), [p + r for p, r in items], layers=3, kv_heads=kv_heads, d=d, pages=pages, page_rows=page_rows, seed=d)
    cache.paged.enable_trees(sum(new))
    cache.paged.set_batch(items, cache.tables)
    path, lengths = i32([x for p, r in zip(paths, new) for x in p + [-1] * (r - len(p))]), i32([-9] * 8)
    want = cache.host.clone()
    for seq, ((p, r), mine) in enumerate(zip(items, paths)):
        if seq == 7:
            continue  # (it does not ascend)
        for to, one in enumerate(mine):
            (a, b), (c, e) = (divmod(p + to, page_rows), divmod(p + one, page_rows))
            want[:, cache.tables[seq][a], :, :, b] = cache.host[:, cache.tables[seq][c], :, :, e]
    cache.paged.keep_device(path.data_ptr(), lengths.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(cache.storage.cpu(), want)
    assert lengths.tolist() == [37, 19, 1, -9, 93, 293, 9, -1]
    beyond = path.clone()
    beyond[0] = 40
    cache.paged.keep_device(beyond.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(cache.storage[:, cache.tables[0]].cpu(), want[:, cache.tables[0]])


@pytest.mark.parametrize("sequences", [64, 65, 200])
def test_walks_and_rows_of_many_sequences(sequences):
    rng = np.random.RandomState(sequences)
    new, held = rng.randint(0, 9, sequences).tolist(), rng.randint(0, 40, sequences).tolist()
    new[0], new[-1] = 8, 8
    items, parents = list(zip(held, new)), [TC.tree(r, i, 6) if r else [] for i, r in enumerate(new)]
    cache = PC.Cache(pkg(), [p + r + 1 for p, r in items], layers=2, kv_heads=1, d=8, page_rows=16, max_sequences=sequences, seed=1)
    cache.paged.enable_trees(sum(new))
    cache.paged.set_batch(items, cache.tables, TC.flat(parents))
    tokens, chosen = (rng.randint(0, 2, sum(new)).astype(np.int32) for _ in range(2))
    path, following, lengths = i32([9] * sum(new)), i32([9] * sequences), i32([9] * sequences)
    t, c = torch.from_numpy(tokens).cuda(), torch.from_numpy(chosen).cuda()
    want_path, want_next, want_length, want, first = [], [], [], cache.host.clone(), 0
    for (p, r), mine, table in zip(items, parents, cache.tables):
        if r:
            walk, end = TC.walk(mine, tokens[first:first + r], chosen[first:first + r])
            for to, one in enumerate(walk):
                want[:, table[(p + to) // 16], :, :, (p + to) % 16] = cache.host[:, table[(p + one) // 16], :, :, (p + one) % 16]
            want_path += walk + [-1] * (r - len(walk))
        want_next.append(int(end) if r else 9)
        want_length.append(p + len(walk) if r else 9)
        first += r
    cache.paged.accept_device(t.data_ptr(), c.data_ptr(), path.data_ptr(), following.data_ptr())
    cache.paged.keep_device(path.data_ptr(), lengths.data_ptr())
    torch.cuda.synchronize()
    assert path.tolist() == want_path and following.tolist() == want_next and lengths.tolist() == want_length
    assert torch.equal(cache.storage.cpu(), want)


def test_both_ways_make_the_same_call(monkeypatch):
    # Plain arguments go through the compiled front module, every other kind through ctypes.
    P, got = pkg(), []
    for way in ("front", "ctypes", "arrays"):
        with monkeypatch.context() as m:
            if way == "ctypes":
                m.setattr(P.hip_compute, "_front", P._native.NoFront)
            cast = (lambda x: np.asarray(x, np.uint32)) if way == "arrays" else list
            paged, tables = small(max_sequences=3), Tables(3, 8, 64, 2)
            paged.enable_trees(20)
            held, status = i32([5, 30, 0]), i32([7] * 3)
            parents, chosen = i32([-1, 0, 0, 1, -1, 0, -1]), i32([4, 9, 4, 9, 2, 2, 1])
            tokens, path, following = i32([1, 3, 4, 9, 5, 2, 0]), i32([7] * 7), i32([7] * 3)
            places = torch.zeros(2, 7, dtype=torch.int64, device="cuda")
            paged.fit_tables_device(tables.raw, held.data_ptr(), cast([4, 2, 1]), status.data_ptr())
            paged.set_batch_device(tables.raw, held.data_ptr(), cast([4, 2, 1]), 30, parents.data_ptr(), status.data_ptr())
            assert paged._rows == 7
            paged.batch_rows_device(places[0].data_ptr(), places[1].data_ptr())
            paged.accept_device(tokens.data_ptr(), chosen.data_ptr(), path.data_ptr(), following.data_ptr())
            paged.keep_device(path.data_ptr(), held.data_ptr())
            paged.fit_tables_device(tables.raw, held.data_ptr())
            torch.cuda.synchronize()
            got.append([t.tolist() for t in (places, path, following, held, status, *tables.dev)])
    assert got[0] == got[1] == got[2]
    assert got[0][0][0] == [5, 6, 6, 7, 30, 31, 0] and got[0][1] == [0, 2, -1, -1, 0, 1, 0] and got[0][2] == [4, 2, 1] and got[0][3] == [7, 32, 1]


class Model:
    """What stands around the cache in a round: fixed projections of a token, and what it would choose behind a row of attention outputs."""

    def __init__(self, layers, heads, kv_heads, d, vocabulary=50):
        g = torch.Generator().manual_seed(5)
        self.q, self.k, self.v = (torch.randn(layers, vocabulary, h, d, generator=g).half().cuda() for h in (heads, kv_heads, kv_heads))
        self.vocabulary = vocabulary


def rounds(cache_kw, sequences, nodes, turns, device, graph=False):
    """`turns` rounds of `sequences` trees over one cache, the books kept by the device or by hand on the host. What was accepted each
    round, and the cache's rows at the end."""
    P, layers, heads, kv_heads, d = pkg(), 2, 4, 2, 64
    model = Model(layers, heads, kv_heads, d)
    page_count, width = 80, 12
    paged = P.PagedKv(layers, kv_heads, d, page_rows=16, page_count=page_count, max_sequences=sequences)
    stream = torch.cuda.current_stream()
    paged.set_stream(stream.cuda_stream)
    paged.enable_trees(sequences * nodes)
    rotation = P.Rotation(d)
    tables = Tables(sequences, width, page_count, 1)
    rows, new = sequences * nodes, [nodes] * sequences
    lengths = i32([0] * sequences)
    parents, tokens, path, chosen = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(4))
    following = i32([0] * sequences)
    q = torch.zeros(rows, heads, d, dtype=torch.float16, device="cuda")
    k, v = (torch.zeros(rows, kv_heads, d, dtype=torch.float16, device="cuda") for _ in range(2))
    out = [torch.zeros_like(q) for _ in range(layers)]
    answers = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def forward(on):
        paged.set_stream(on.cuda_stream)
        if device:
            paged.fit_tables_device(tables.raw, lengths.data_ptr(), new)
            paged.set_batch_device(tables.raw, lengths.data_ptr(), new, 16 * width - nodes, parents.data_ptr())
        for layer in range(layers):
            token = tokens.long()
            q.copy_(model.q[layer][token]), k.copy_(model.k[layer][token]), v.copy_(model.v[layer][token])
            paged.attention_step_device(layer, view(q), view(k), view(v), view(out[layer]), rotation=rotation)
        chosen.copy_(answers)
        paged.accept_device(tokens.data_ptr(), chosen.data_ptr(), path.data_ptr(), following.data_ptr())
        paged.keep_device(path.data_ptr(), lengths.data_ptr())
        if device:
            paged.fit_tables_device(tables.raw, lengths.data_ptr())

    seen, captured, host_lengths = [], None, [0] * sequences
    for turn in range(turns):
        trees = [TC.tree(nodes, 10 * turn + s, 5) for s in range(sequences)]
        rng = np.random.RandomState(turn)
        parents.copy_(torch.from_numpy(TC.flat(trees)))
        tokens.copy_(torch.from_numpy(rng.randint(0, model.vocabulary, rows).astype(np.int32)))
        picks = rng.randint(0, model.vocabulary, rows).astype(np.int32)
        known = tokens.cpu().numpy()
        for s, t in enumerate(trees):  # (the model chooses a child's token more often than not)
            for r in range(1, nodes):
                if t[r] >= 0 and rng.rand() < 0.6:
                    picks[s * nodes + t[r]] = known[s * nodes + r]
        answers.copy_(torch.from_numpy(picks))
        if not device:
            tables.fit([-(-(n + nodes) // 16) for n in host_lengths])
            paged.set_batch([(n, nodes) for n in host_lengths], [np.array(t[:c], np.uint32) for t, c in zip(tables.table, tables.pages)],
                            TC.flat(trees))
        if graph and turn == 1:
            torch.cuda.synchronize()
            side, captured = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=side):
                forward(side)
            paged.set_stream(stream.cuda_stream)
        if captured:
            captured.replay()
        else:
            forward(stream)
        torch.cuda.synchronize()
        if not device:
            host_lengths = lengths.tolist()
            tables.fit([-(-n // 16) for n in host_lengths])
        seen.append((path.tolist(), following.tolist(), lengths.tolist(), [o.clone() for o in out]))
    storage = torch.empty(0)
    if device:
        table, held = tables.dev[0].cpu(), tables.dev[1].tolist()
    else:
        table, held = torch.tensor(tables.table), tables.pages
    return seen, (table, held, storage)


def test_whole_rounds():
    kw = dict(sequences=3, nodes=9, turns=5)
    by_host, host_tables = rounds({}, device=False, **kw)
    by_device, device_tables = rounds({}, device=True, **kw)
    by_graph, graph_tables = rounds({}, device=True, graph=True, **kw)
    assert max(by_host[-1][2]) > 10
    for a, b, c in zip(by_host, by_device, by_graph):
        assert a[:3] == b[:3] == c[:3]
        for x, y, z in zip(a[3], b[3], c[3]):
            # The same rows in other pieces: an output, a mean of values up to 5 in magnitude, is two roundings of weights (2^-11 of it
            # each) and its own from another.
            assert float((x.double() - y.double()).abs().max()) <= 5 * 3 * 2.0 ** -11 and torch.equal(y, z)
    for (t, n, _) in (device_tables, graph_tables):
        assert n == host_tables[1] and all(torch.equal(a[:m], b[:m].int()) for a, b, m in zip(t, host_tables[0], n))


def test_refusals():
    P = pkg()
    paged, tables = small(max_sequences=4, page_count=8), Tables(4, 4, 8)
    x = at([0] * 16)
    rows = [1] * 4
    fit, batch = paged.fit_tables_device, paged.set_batch_device
    bad = lambda **kw: P.PageTables(**{**dict(table_ptr=x, stride=4, pages_ptr=x, sequences=4, free_ptr=x, free_count_ptr=x), **kw})  # noqa: E731
    for kw, variant in ((dict(table_ptr=0), "InvalidArgument"), (dict(pages_ptr=0), "InvalidArgument"), (dict(stride=0), "ZeroDimension"),
                        (dict(stride=1 << 29), "SizeOverflow"), (dict(sequences=0), "ZeroDimension"), (dict(sequences=5), "CapacityExceeded")):
        t = bad(**kw)
        assert refusal(lambda: fit(t, x)) == refusal(lambda: batch(t, x, [1] * t.sequences, 10)) == variant, kw
    assert refusal(lambda: fit(bad(free_ptr=0), x)) == refusal(lambda: fit(bad(free_count_ptr=0), x)) == refusal(lambda: fit(tables.raw, 0)) == "InvalidArgument"
    assert refusal(lambda: batch(tables.raw, 0, rows, 10)) == "InvalidArgument"
    for most in (1 << 31, (1 << 31) - 1, 1 << 63):
        assert refusal(lambda: batch(tables.raw, x, rows, most)) == "SizeOverflow"
    assert refusal(lambda: batch(tables.raw, x, [1 << 23, 1 << 23, 0, 0], 10)) == "SizeOverflow"
    assert refusal(lambda: batch(tables.raw, x, rows, 10, x)) == "Unsupported"
    paged.enable_trees(3)
    assert refusal(lambda: batch(tables.raw, x, rows, 10, x)) == "CapacityExceeded"
    for call in (lambda: fit(tables.raw, x, rows[:3]), lambda: batch(tables.raw, x, rows + [1], 10), lambda: batch(tables.raw, x, [1, 1, 1, -1], 10),
                 lambda: fit(tables.raw, x, np.ones(4)), lambda: batch(tables.raw, x, rows, -1)):
        with pytest.raises(ValueError):
            call()
    for wrong in (dict(table=tables.dev[0].long()), dict(pages=tables.dev[1].cpu()), dict(table=tables.dev[1]), dict(pages=tables.dev[1][:2]),
                  dict(free=tables.dev[2][::2])):
        with pytest.raises(ValueError):
            P.PageTables.of(**{**dict(table=tables.dev[0], pages=tables.dev[1], free=tables.dev[2], free_count=tables.dev[3]), **wrong})
    # Nothing to do is no error, and nothing is read.
    paged.accept_device(0, 0, 0, 0)
    paged.keep_device(0)
    batch(tables.raw, x, [0] * 4, 10)
    paged.batch_rows_device(x)
    paged.accept_device(0, 0, 0, 0)
    fit(tables.raw, at([16] * 4))
    batch(tables.raw, x, [1, 1, 0, 0], 15)
    assert refusal(lambda: paged.accept_device(x, x, x, 0)) == refusal(lambda: paged.keep_device(0)) == "InvalidArgument"
    assert refusal(lambda: paged.batch_rows_device()) == "InvalidArgument"
    torch.cuda.synchronize()
