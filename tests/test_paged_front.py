"""The paged calls of the Python front end: plain arguments go through its compiled module, every other kind through ctypes, and
what neither can mean is refused before the library is asked."""
import numpy as np
import pytest
import torch

import paged_cases as PC
from helpers import pkg

REFUSED = 17  # InvalidArgument: no handle


def front():
    hip = pkg().hip_compute
    hip._load()
    return hip._front


def test_only_plain_arguments_are_taken():
    f, P = front(), pkg()
    x = P.Rows(1 << 20, "f16", 2)
    ids = np.array([3, 1], np.uint32)
    assert f.append(0, 1, 64, 0, x, x, 0) == REFUSED
    assert f.paged_attention(0, 1, 64, 0, x, x, None, 0.0, 0, 0) == f.paged_attention(0, 1, 64, 0, x, x, 0.5, 0, 7, 0) == REFUSED
    assert f.paged_step(0, 1, 64, 0, x, x, x, x, None, 0.0, 0, 0) == REFUSED
    assert f.set_batch(0, [(0, 1), (4, 2)], [ids, ids[:1]]) == f.set_batch(0, ((0, 1),), (ids.astype(np.int32),)) == f.set_batch(0, [], []) == REFUSED
    assert f.rotate(0, 0, 64, 1, 0, [x], (x,), False) == REFUSED
    for odd in (x.raw, None, 5):
        assert f.append(0, 1, 64, 0, odd, x, 0) == f.paged_attention(0, 1, 64, 0, x, odd, None, 0.0, 0, 0) == -1
        assert f.paged_step(0, 1, 64, 0, x, x, odd, x, None, 0.0, 0, 0) == f.rotate(0, 0, 64, 1, 0, [odd], [x], False) == -1
    assert f.append(0, 1, 64, 0, x, x, None) == f.append(0, 1, 64, np.int64(0), x, x, 0) == -1  # (None: a rotation that is closed)
    assert f.rotate(0, 0, 64, 1, 0, [x] * 5, [x] * 5, False) == f.rotate(0, 0, 64, 1, 0, [x], [], False) == f.rotate(0, 0, 64, 1, 0, [x], [x], 1) == -1
    for tables in ([[3, 1]], [ids.astype(np.int64)], [np.array([[3, 1]], np.uint32)], [np.arange(4, dtype=np.uint32)[::2]],
                   [ids.astype(">u4")], ids, [ids, ids], []):
        assert f.set_batch(0, [(0, 1)], tables) == -1
    for items in ([[0, 1]], [(0, -1)], [(0, 1 << 32)], [(-1, 1)], [(np.int64(0), 1)], [(0, 1, 2)]):
        assert f.set_batch(0, items, [ids]) == -1
    assert f.set_batch(0, [(0, 1)] * 65, [ids] * 65) == -1
    known = P.Rows(1 << 20, "f16", 2, 128, 64, rows=3, channels=64)  # of a tensor: how much there is of it is known
    assert f.append(0, 3, 64, 0, known, x, 0) == f.append(0, 1, 64, 0, known, known, 0) == REFUSED
    for rows, channels in ((4, 64), (3, 128), (3, 32)):
        assert f.append(0, rows, channels, 0, x, known, 0) == f.paged_attention(0, rows, channels, 0, known, x, None, 0.0, 0, 0) == -1
        assert f.paged_step(0, rows, channels, 0, x, x, x, known, None, 0.0, 0, 0) == f.rotate(0, 0, channels, rows, 0, [known], [x], False) == -1
    with pytest.raises(TypeError):
        f.append(0, 1, 64, 0, x, x)


@pytest.mark.gpu
def test_both_ways_make_the_same_call(monkeypatch):
    P = pkg()
    items, got = [(21, 2), (0, 1)], []
    rotation = P.Rotation(64)
    tables = None
    for way in (lambda t: t, lambda t: [list(map(int, x)) for x in t], lambda t: [np.asarray(x, np.int64) for x in t]):
        for plain in (True, False):
            cache = PC.Cache(P, [23, 1], kv_heads=2, d=64, page_rows=16, seed=4)
            tables = [np.asarray(t, np.uint32) for t in cache.tables]
            q, k, v = (cache.normal(3, h, 64).half().cuda() for h in (4, 2, 2))
            out, turned = torch.empty_like(q), torch.empty_like(q)
            with monkeypatch.context() as m:
                if not plain:
                    m.setattr(P.hip_compute, "_front", P._native.NoFront)
                cache.paged.set_batch(items, way(tables))
                cache.paged.append_device(0, P.Rows.of(k), P.Rows.of(v), rotation)
                cache.paged.attention_device(0, P.Rows.of(q), P.Rows.of(out), scale=0.25, softcap=8.0, window=9, rotation=rotation)
                one = out.clone()
                cache.paged.attention_step_device(0, P.Rows.of(q), P.Rows.of(k), P.Rows.of(v), P.Rows.of(out), scale=0.25, softcap=8.0,
                                                  window=9, rotation=rotation)
                positions = torch.tensor([21, 22, 0], device="cuda")
                rotation.rotate_device([P.Rows.of(q)], [P.Rows.of(turned)], positions.data_ptr(), 3, 64,
                                       torch.cuda.current_stream().cuda_stream, inverse=True)
                torch.cuda.synchronize()
            got.append([t.cpu() for t in (one, out, turned, cache.storage.view(torch.int16))])
            assert torch.equal(one, out)
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("plain", [True, False])
def test_what_neither_way_can_mean_is_refused(monkeypatch, plain):
    P = pkg()
    if not plain:
        P.hip_compute._load()
        monkeypatch.setattr(P.hip_compute, "_front", P._native.NoFront)
    cache = PC.Cache(P, [40], kv_heads=1, d=64, page_rows=16)
    q, k = cache.normal(1, 1, 64).half().cuda(), cache.normal(1, 1, 64).half().cuda()
    out = torch.empty_like(q)
    rotation = P.Rotation(64)
    rotation.close()
    cache.paged.set_batch([(5, 1)], cache.tables)
    before = cache.storage.clone()
    x, y, z = P.Rows.of(q), P.Rows.of(k), P.Rows.of(out)
    two, wide = torch.zeros(2, 1, 64, device="cuda").half(), torch.zeros(1, 1, 128, device="cuda").half()
    cache.paged.set_batch([(5, 2)], cache.tables)  # (of which the tensors above have one row)
    for call in (lambda: cache.paged.append_device(0, y, P.Rows.of(two)),
                 lambda: cache.paged.attention_device(0, x, P.Rows.of(two)),
                 lambda: cache.paged.attention_step_device(0, P.Rows.of(two), P.Rows.of(two), y, P.Rows.of(two)),
                 lambda: cache.paged.attention_device(0, P.Rows.of(two), P.Rows.of(wide)),
                 lambda: P.Rotation(64).rotate_device([x], [z], 0, 2, 64),
                 lambda: P.Rotation(64).rotate_device([x], [z], 0, 1, 128),
                 lambda: P.Rows.of(torch.zeros(1, 1, 64, device="cuda").expand(3, 2, 64))):
        with pytest.raises(ValueError):
            call()
    cache.paged.set_batch([(5, 1)], cache.tables)
    for call in (lambda: cache.paged.append_device(0, y, y, rotation),
                 lambda: cache.paged.attention_device(0, x, z, rotation=rotation),
                 lambda: cache.paged.attention_step_device(0, x, y, y, z, rotation=rotation),
                 lambda: rotation.rotate_device([x], [z], 0, 1, 64),
                 lambda: cache.paged.set_batch([(0, (1 << 32) + 1)], cache.tables),
                 lambda: cache.paged.set_batch([(-1, 1)], cache.tables),
                 lambda: cache.paged.set_batch([(5, 1)], [np.array([1 << 32, 1, 2])]),
                 lambda: cache.paged.set_batch([(5, 1)], [np.array([0.0, 1.0, 2.0])])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(P.AttentionError):
        cache.paged.attention_device(0, x, x)
    torch.cuda.synchronize()
    assert torch.equal(before, cache.storage)
