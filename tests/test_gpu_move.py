"""pa_cache_move: rows of caches copied, forked and moved together, word for word against indexing."""
import random

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError

pytestmark = pytest.mark.gpu


def engine(nKV, hd, rows, n_seqs, kv="f16", layers=1, **kw):
    return AttnEngine(AttnConfig(n_heads=nKV * 2, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e6, max_seq=rows, n_seqs=n_seqs, n_layers=layers, kv_format=kv,
                                 act_dtype=torch.float16, **kw))


def arrays(eng):
    """All that a row has, by layer: views of [n_seqs, max_seq, words]."""
    out = []
    for li in range(eng.cfg.n_layers):
        a = [eng.cache(li, w) for w in "kv"]
        a = [x.view(torch.int32) if x.dtype == torch.float32 else x for x in a]
        if eng.cfg.kv_format == "q8":
            a += [eng.cache_scales(li, w).view(torch.int32) for w in "kv"]
        try:
            a.append(eng.weights(li).view(torch.int32).transpose(1, 2))
        except PaError:
            pass
        out.append(a)
    return out


def fill(eng, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for layer in arrays(eng):
        for x in layer:
            x.copy_(torch.randint(-128, 128, x.shape, generator=g, device="cuda").to(x.dtype) if x.dtype == torch.int8 else
                    torch.randint(-30000, 30000, x.shape, generator=g, device="cuda").to(x.dtype))


def expected(eng, items, lists=None, layers=None):
    want = [[x.clone() for x in layer] for layer in arrays(eng)]
    for li in range(eng.cfg.n_layers) if layers is None else layers:
        for x, y in zip(arrays(eng)[li], want[li]):
            for i, (ss, sr, ds, dr, n) in enumerate(items):
                if lists is None:
                    y[ds, dr:dr + n] = x[ss, sr:sr + n]
                else:
                    count = min(lists[i][0] & 0xffffffff, n, len(lists[i]) - 1)
                    offs = [(j, o & 0xffffffff) for j, o in enumerate(lists[i][1:1 + count]) if (o & 0xffffffff) < n]
                    if offs:
                        j, o = (torch.tensor(t, device="cuda") for t in zip(*offs))
                        y[ds, dr + j] = x[ss, sr + o]
    return want


def same(eng, want):
    eng.sync()
    return all(torch.equal(x, y) for a, b in zip(arrays(eng), want) for x, y in zip(a, b))


FORMATS = [("f16", 2, 256, False), ("f16", 8, 128, True), ("q8", 2, 256, False), ("q8", 1, 64, False), ("f32", 8, 128, False), ("f16", 3, 64, True)]


@pytest.mark.parametrize("kv,nKV,hd,track", FORMATS)
@pytest.mark.parametrize("items", [
    [(0, 0, 1, 0, 1)], [(0, 7, 2, 300, 65)], [(1, 0, 0, 0, 2000)], [(0, 0, s, 0, 777) for s in (1, 2, 3)], [(0, 5, 1, 9, 333), (0, 5, 2, 11, 333), (3, 0, 0, 1000, 1000), (0, 0, 3, 1500, 0)],
    [(0, 10, 0, 3, 40)], [(0, 3, 0, 10, 40)], [(2, 600, 2, 5, 500)], [(1, 64, 1, 63, 1900)], [(1, 63, 1, 64, 1900)], [(0, 700, 0, 0, 1300), (1, 0, 1, 700, 1300), (2, 50, 2, 40, 20), (3, 40, 3, 50, 512)],
    [(1, 513, 1, 0, 513)], [(0, 8, 0, 0, 1992), (2, 0, 2, 1, 1999), (1, 0, 3, 0, 2000)], [(2, 11, 2, 11, 99), (1, 2, 0, 4, 31)]])
def test_ranges(kv, nKV, hd, track, items):
    eng = engine(nKV, hd, 2000, 4, kv, layers=2)
    if track:
        eng.track_weights(1)                                               # one of the two layers
    fill(eng, 1)
    for _ in range(2):                                                     # the order's words are zero again
        want = expected(eng, items)
        eng.move(items)
        assert same(eng, want)


@pytest.mark.parametrize("kv,nKV,hd,track", FORMATS)
@pytest.mark.parametrize("span,stride,over", [(60, 61, True), (60, 20, True), (512, 513, True), (513, 514, True), (1800, 1200, True), (1800, 1801, True), (1, 2, True), (300, 301, False), (1900, 700, False)])
def test_lists(kv, nKV, hd, track, span, stride, over):
    r = random.Random(span + stride)
    eng = engine(nKV, hd, 2000, 6, kv, layers=2)
    if track:
        eng.track_weights(0)
        eng.track_weights(1)
    fill(eng, 2)
    items, lists = [], []
    for s in range(3):
        most = min(span, stride - 1)
        count = [most, r.randint(0, most), 0][s]
        # over one another: ascending; else any order, some twice
        offs = sorted(r.sample(range(span), count)) if over else [r.randrange(span) for _ in range(count)]
        lists.append([count, *offs, *[r.randrange(span) for _ in range(stride - 1 - count)]])
        items.append((s, 90, s, 90 if s else 40, span) if over else (s, 90, 3 + s, 100 - s, span))
    t = torch.tensor(lists, dtype=torch.int32, device="cuda")
    for _ in range(2):
        want = expected(eng, items, lists)
        eng.move(items, lists=t)
        assert same(eng, want)


def test_list_entries_past_their_item_move_nothing():
    eng = engine(2, 256, 500, 2)
    fill(eng, 3)
    lists = [[7, 0, 100, 5, -1, 50, 99, 2 ** 31 - 1, 3], [-1, 1, 2, 3, 4, 5, 6, 7, 120]]         # of 100 rows; a count past the stride
    items = [(0, 0, 1, 0, 100), (0, 200, 1, 200, 100)]
    want = expected(eng, items, lists)
    eng.move(items, lists=torch.tensor(lists, dtype=torch.int32, device="cuda"))
    assert same(eng, want)


def test_random_moves():
    r = random.Random(11)
    for trial in range(25):
        kv, nKV, hd, _ = r.choice(FORMATS)
        rows, seqs = r.choice([64, 700, 3001]), r.randint(2, 6)
        eng = engine(nKV, hd, rows, seqs, kv, layers=r.choice([1, 3]))
        fill(eng, trial)
        items, spans = [], []
        for _ in range(40):
            n = r.choice([0, 1, r.randint(1, rows), r.randint(1, 70) % rows])
            it = (r.randrange(seqs), r.randint(0, rows - n), r.randrange(seqs), r.randint(0, rows - n), n)
            a, b = (it[0], it[1], it[1] + n), (it[2], it[3], it[3] + n)
            meet = lambda x, y: x[0] == y[0] and x[1] < y[2] and y[1] < x[2]
            if all(not meet(b, x) and not meet(b, y) and not meet(a, y) for x, y in spans):
                items.append(it)
                spans.append((a, b))
        want = expected(eng, items)
        eng.move(items)
        assert same(eng, want), items


@pytest.mark.parametrize("gap", [1, 15, 16, 17, 100, 4000, 9000])
@pytest.mark.parametrize("up", [False, True])
def test_long_rows_over_one_another_keep_their_order(gap, up):
    eng = engine(4, 256, 20000, 1)
    fill(eng, 4)
    n = 20000 - gap
    items = [(0, 0, 0, gap, n) if up else (0, gap, 0, 0, n)]
    for _ in range(3):
        want = expected(eng, items)
        eng.move(items)
        assert same(eng, want)
    # lists: every row but some
    kept = [i for i in range(n) if i % gap or not i] if gap > 1 else list(range(0, n, 3))
    lists = [[len(kept), *kept]]
    want = expected(eng, [(0, 0, 0, 0, n)], lists)
    eng.move([(0, 0, 0, 0, n)], lists=torch.tensor(lists, dtype=torch.int32, device="cuda"))
    assert same(eng, want)


def test_rows_past_four_gigabytes():
    # the last of eight sequences of 300000 rows of 2 KB: a fork, a list, rows over one another
    eng = engine(8, 128, 300000, 8)
    caches = [eng.cache(0, w) for w in "kv"]
    for i, x in enumerate(caches):
        x[7, 290000:] = torch.randint(-30000, 30000, (10000, 1024), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").to(torch.int16)
    was = [x[7, 290000:].clone() for x in caches]
    eng.move([(7, 290000, 7, 280000, 9000), (7, 290000, 6, 291000, 9000)])
    eng.move([(7, 290000, 7, 290007, 9000)])
    eng.move([(7, 290007, 0, 5, 100)], lists=torch.tensor([[3, 99, 0, 50]], dtype=torch.int32, device="cuda"))
    eng.sync()
    for x, y in zip(caches, was):
        assert torch.equal(x[7, 280000:289000], y[:9000]) and torch.equal(x[6, 291000:], y[:9000])
        assert torch.equal(x[7, 290000:290007], y[:7]) and torch.equal(x[7, 290007:299007], y[:9000]) and torch.equal(x[7, 299007:], y[9007:])
        assert torch.equal(x[0, 5:8], y[[99, 0, 50]])


def test_some_layers_and_many():
    eng = engine(2, 64, 100, 2, layers=70)                                 # more than one launch takes
    fill(eng, 5)
    items = [(0, 0, 1, 5, 60), (0, 70, 0, 60, 25)]
    want = expected(eng, items)
    eng.move(items)
    assert same(eng, want)
    want = expected(eng, [(1, 0, 1, 1, 99)], layers=[3, 69, 7])
    eng.move([(1, 0, 1, 1, 99)], layers=[3, 69, 7])
    assert same(eng, want)


def test_graphs_and_streams():
    eng = engine(4, 256, 6000, 3, layers=2)
    fill(eng, 6)
    items = [(0, 1000, 0, 0, 5000), (1, 0, 2, 0, 6000)]
    lists = torch.tensor([[3, 1, 5, 9], [2, 0, 4, 0]], dtype=torch.int32, device="cuda")
    path = [(0, 100, 0, 100, 20), (1, 50, 1, 40, 20)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        eng.move(items)
        eng.move(path, lists=lists)
    for new in ([[3, 1, 5, 9], [2, 0, 4, 0]], [[1, 19, 0, 0], [3, 2, 3, 4]]):
        lists.copy_(torch.tensor(new, dtype=torch.int32))
        before = [[x.clone() for x in layer] for layer in arrays(eng)]
        mid = expected(eng, items)
        for layer, m in zip(arrays(eng), mid):
            for x, y in zip(layer, m):
                x.copy_(y)
        want = expected(eng, path, new)
        for layer, b in zip(arrays(eng), before):
            for x, y in zip(layer, b):
                x.copy_(y)
        g.replay()
        assert same(eng, want)
    side = torch.cuda.Stream()
    want = expected(eng, items)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eng.move(items)
        eng.sync()
    assert same(eng, want)


@pytest.mark.parametrize("kv,act", [("f16", torch.float16), ("f16", torch.float32), ("q8", torch.float32), ("f32", torch.float32)])
def test_calls_right_behind_a_move_see_its_rows(kv, act):
    # layers' calls fetch rows ahead of their wait: none that a move may still be storing
    nL, rows = 3, 6000
    cfg = dict(n_heads=16, n_kv_heads=8, head_dim=128, n_rot=128, rope_theta=1e6, max_seq=rows, n_seqs=2, n_layers=nL, kv_format=kv, act_dtype=act, max_cols=64)
    eng, ref = AttnEngine(AttnConfig(**cfg)), AttnEngine(AttnConfig(**cfg))
    g = torch.Generator(device="cuda").manual_seed(7)
    for cols in (1, 4, 64, 1):
        q = torch.empty((cols, 2048), device="cuda").normal_(generator=g).to(act)
        k, v = [torch.empty((cols, 1024), device="cuda").normal_(generator=g).to(act) for _ in "kv"]
        for trial in range(4):
            for li in range(nL):
                for w in "kv":
                    x = torch.empty((2, rows, 1024), device="cuda").normal_(generator=g)
                    if kv == "q8":
                        x, sc = (x * 20).round().clamp(-127, 127).to(torch.int8), torch.rand((2, rows, 32), generator=g, device="cuda") * 0.1
                        for e in (eng, ref):
                            e.cache_scales(li, w).copy_(sc)
                    elif kv == "f16":
                        x = x.half().view(torch.int16)
                    for e in (eng, ref):
                        e.cache(li, w).copy_(x)
            for e in (ref, eng):
                for li in range(nL):
                    for a in arrays(e)[li]:
                        if e is ref:
                            a[0, 10:5000] = a[0, 910:5900].clone()
            torch.cuda.synchronize()
            want = [ref.encode_layer(li, 5000, q, k, v, mode="decode" if cols < 64 else "auto") for li in range(nL)]
            torch.cuda.synchronize()
            eng.move([(0, 910, 0, 10, 4990)])
            got = [eng.encode_layer(li, 5000, q, k, v, mode="decode" if cols < 64 else "auto") for li in range(nL)]
            eng.sync()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (cols, trial)


def test_refusals_write_nothing():
    eng = engine(2, 256, 100, 3, layers=2)
    fill(eng, 8)
    before = [[x.clone() for x in layer] for layer in arrays(eng)]
    t = lambda *rows: torch.tensor(rows, dtype=torch.int32, device="cuda")
    bad = [([], None), ([(3, 0, 0, 0, 1)], None), ([(0, 0, 3, 0, 1)], None), ([(0, 60, 1, 0, 41)], None), ([(0, 0, 1, 60, 41)], None), ([(0, 2 ** 32 - 1, 1, 0, 2)], None),
           ([(0, 0, 1, 0, 2 ** 32 - 1)], None), ([(0, 0, 1, 0, 10), (0, 50, 1, 9, 10)], None), ([(0, 0, 1, 0, 10), (1, 5, 2, 0, 10)], None), ([(0, 0, 0, 5, 10), (0, 4, 1, 0, 10)], None),
           ([(0, i, 1, i, 1) for i in range(65)], None), ([(0, 0, 0, 5, 10)], t([2, 0, 1, 0])), ([(0, 0, 1, 98, 10)], t([2, 0, 1, 0])), ([(0, 0, 1, 0, 10), (0, 0, 1, 2, 10)], t([2, 0, 1, 0], [2, 0, 1, 0])),
           ([(0, 0, 1, 0, 10)], t([2, 0, 1, 0], [2, 0, 1, 0])), ([(0, 0, 1, 0, 10)], t([2, 0, 1, 0]).long()), ([(0, 0, 1, 0, 10)], t([2, 0, 1, 0]).cpu())]
    for items, lists in bad:
        with pytest.raises(PaError):
            eng.move(items, lists=lists)
    with pytest.raises(PaError):
        eng.move([(0, 0, 1, 0, 10)], layers=[0, 0])
    import ctypes as C
    other = engine(2, 256, 101, 3)
    arr = (C.c_void_p * 2)(eng.layers[0].value, other.layers[0].value)
    from pooled_b200 import lib as L
    it = L.PaMoveItem(0, 0, 1, 0, 5, 0)
    assert eng.L.pa_cache_move(arr, 2, C.byref(it), 1, None, 0, None) == -1
    assert eng.L.pa_cache_move(None, 1, C.byref(it), 1, None, 0, None) == -1
    assert eng.L.pa_cache_move(arr, 0, C.byref(it), 1, None, 0, None) == -1
    assert same(eng, before)
    eng.move([(0, 0, 1, 0, 0)])                                            # nothing to move is no error
    eng.move([(0, 3, 0, 3, 50)])
    assert same(eng, before)
