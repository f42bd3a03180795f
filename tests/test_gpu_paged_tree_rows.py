"""What a cache holds after rounds of trees: the rows of every accepted token at its place, the same where the books were kept by the host, by the
device and in a graph."""
import numpy as np
import pytest
import torch

import paged_cases as PC
import test_gpu_paged_rounds as R
from helpers import pkg

pytestmark = pytest.mark.gpu

LAYERS, HEADS, KV_HEADS, D, PAGE_ROWS = 2, 4, 2, 64, 16  # as the rounds have them


def rows_after(monkeypatch, **kw):
    """What was accepted in each of the rounds, and every sequence's rows at their end: [layer][side][kv_head][position][channel]."""
    P, made = pkg(), []

    class Owned(P.PagedKv):
        def __init__(self, layers, kv_heads, d, *, page_rows, page_count, max_sequences):
            made.append(torch.full((layers, page_count, 2, kv_heads, page_rows, d), float("nan"), dtype=torch.float16, device="cuda"))
            super().__init__(layers, kv_heads, d, page_rows=page_rows, page_count=page_count, max_sequences=max_sequences,
                             storage_ptr=made[0].data_ptr(), storage_bytes=made[0].numel() * 2)

    class Package:
        def __getattr__(self, name):
            return Owned if name == "PagedKv" else getattr(P, name)

    with monkeypatch.context() as m:
        m.setattr(R, "pkg", lambda: Package())
        seen, (table, held, _) = R.rounds({}, **kw)
    (storage,), rows = made, []
    for pages, count, length in zip(table.tolist(), held, seen[-1][2]):
        assert count == -(-length // PAGE_ROWS)
        mine = storage[:, pages[:count]].cpu().permute(0, 2, 3, 1, 4, 5)
        rows.append(mine.reshape(LAYERS, 2, KV_HEADS, -1, D)[:, :, :, :length])
    return seen, rows


# (Five rounds end within the sequences' first page, twelve behind it.)
@pytest.mark.parametrize("turns", [5, 12])
def test_rows_at_the_end_of_whole_rounds(monkeypatch, turns):
    sequences, nodes = 3, 9
    kw = dict(sequences=sequences, nodes=nodes, turns=turns)
    ways = [rows_after(monkeypatch, device=device, graph=graph, **kw) for device, graph in ((False, False), (True, False), (True, True))]
    seen, by_host = ways[0]
    for other, rows in ways[1:]:
        assert [x[:3] for x in other] == [x[:3] for x in seen]
        assert all(torch.equal(a, b) for a, b in zip(rows, by_host))
    # And by the formula: the tokens along the paths, round by round, their keys turned by where they stand.
    model = R.Model(LAYERS, HEADS, KV_HEADS, D)
    kept = [[] for _ in range(sequences)]
    for turn, (path, _, lengths, _) in enumerate(seen):
        tokens = np.random.RandomState(turn).randint(0, model.vocabulary, sequences * nodes)  # as the rounds draw them
        for s in range(sequences):
            kept[s] += [int(tokens[s * nodes + r]) for r in path[s * nodes:(s + 1) * nodes] if r >= 0]
        assert [len(x) for x in kept] == lengths
    assert (max(lengths) > PAGE_ROWS) == (turns > 5)
    freq = PC.frequencies(D, 1e4)
    for tokens, rows in zip(kept, by_host):
        for layer in range(LAYERS):
            k, v = (x[layer].cpu()[tokens] for x in (model.k, model.v))
            assert torch.equal(rows[layer, 1].transpose(0, 1), v)
            turned, err = PC.rotated(k, torch.arange(len(tokens)), *freq, False)
            tol = err + (turned.abs() + err) * PC.HALF_STEP["f16"] + 2.0 ** -25
            assert bool(((rows[layer, 0].transpose(0, 1).double() - turned).abs() <= tol).all())
