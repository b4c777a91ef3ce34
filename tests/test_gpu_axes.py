"""Rotations of several axes and at positions of the device: pa_rotary_create_axes, pa_rotary_apply, pa_rotary_append_at; and a drafted tree's way
through all of its operators."""
import math
import random

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def engine(hd=128, nH=4, nKV=2, act=F16, rows=64, seqs=1, cols=5000, **kw):
    return AttnEngine(AttnConfig(n_heads=nH, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e4, max_seq=rows, n_seqs=seqs, act_dtype=act, max_cols=cols, **kw))


def angle_of(pairs, order, n_rot, theta, positions):
    """Angles in float64 [cols, n_rot / 2], pair after pair, positions [axes, cols]."""
    half, n = n_rot // 2, len(pairs)
    cols = []
    ends = [sum(pairs[:a + 1]) for a in range(n)]
    for i in range(half):
        if order == "cycled":
            a = i % n
            if a and i >= n * pairs[a]:
                a = 0
            if a == 0 or i >= n * pairs[a]:
                a = 0
            f = theta ** (-2.0 * i / n_rot)
        else:
            a = next(a for a in range(n) if i < ends[a])
            j = i - (ends[a] - pairs[a])
            f = theta ** (-2.0 * j / (2 * pairs[a])) if order == "own" else theta ** (-2.0 * i / n_rot)
        cols.append(positions[a].double() * f)
    return torch.stack(cols, 1)


def turned(x, n_rot, angle, layout):
    """x [cols, heads, hd] in float64, rotated."""
    y = x.double().clone()
    a, b = (slice(0, n_rot // 2), slice(n_rot // 2, n_rot)) if layout == "half" else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    y[..., a], y[..., b] = x.double()[..., a] * c - x.double()[..., b] * s, x.double()[..., b] * c + x.double()[..., a] * s
    return y


def near(got, want, x, pos, n_rot):
    # a pair: 2^-21 of its length, the angle's own 2^-52 (turns) and 2^-53 (frequency) of it; then the type's rounding
    length = x.double().abs().amax(-1, keepdim=True) * math.sqrt(2)
    tol = length * (2.0 ** -21 + pos.double().abs().amax() * 2.0 ** -50) + (2.0 ** -11 * want.abs() + 2.0 ** -25 if got.dtype == F16 else 0)
    assert torch.all((got.double() - want).abs() <= tol)


AXES = [((24, 20, 20), "blocks", 128), ((24, 20, 20), "cycled", 128), ((32, 32), "own", 128), ((11, 21), "blocks", 64), ((16, 16, 16, 16), "cycled", 128), ((8, 4, 4), "cycled", 32),
        ((0, 7, 9), "blocks", 32), ((1, 2, 3, 4), "own", 20), ((64,), "own", 128), ((64,), "cycled", 128), ((62, 1, 1), "cycled", 128)]


@pytest.mark.parametrize("pairs,order,n_rot", AXES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("act,cols", [(F16, 1), (F32, 7), (F16, 999), (F32, 300)])
def test_apply(pairs, order, n_rot, layout, act, cols):
    eng = engine(act=act)
    rot = eng.rotary(n_rot=n_rot, theta=1e4, layout=layout, axes=pairs, axes_order=order)
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.empty((cols, 4 * 136), device="cuda").normal_(generator=g).to(act)
    pos = torch.randint(-3000, 200000, (len(pairs), cols), generator=g, device="cuda", dtype=torch.int32)
    angle = angle_of(pairs, order, n_rot, 1e4, pos)
    xs = x.view(cols, 4, 136)[..., :128]
    want = turned(xs, n_rot, angle, layout)
    got = rot.apply(x, 4, positions=pos, head_stride=136)
    near(got.view(cols, 4, 128), want, xs, pos, n_rot)
    # in place, and by single values (an odd head stride)
    odd = torch.zeros((cols, 4 * 131), dtype=act, device="cuda")
    odd.view(cols, 4, 131)[..., :128] = xs
    rot.apply(odd, 4, positions=pos, head_stride=131, out=odd)
    near(odd.view(cols, 4, 131)[..., :128], want, xs, pos, n_rot)


@pytest.mark.parametrize("order", ["blocks", "cycled"])
def test_equal_positions_are_one_axis(order):
    eng = engine()
    many, one = eng.rotary(axes=(24, 20, 20), axes_order=order, scaling="yarn", factor=4.0, original=4096), eng.rotary(scaling="yarn", factor=4.0, original=4096)
    assert many.freqs() == one.freqs()
    x = torch.randn((77, 512), device="cuda").half()
    p = torch.randint(0, 9000, (77,), device="cuda", dtype=torch.int32)
    assert torch.equal(many.apply(x, 4, positions=p.repeat(3, 1)), one.apply(x, 4, positions=p))
    assert torch.equal(many.apply(x, 4, pos=501), one.apply(x, 4, pos=501))
    own = eng.rotary(axes=(16, 48), axes_order="own", scaling="linear", factor=2.0)
    f, m = own.freqs()
    assert m == 1.0 and all(math.isclose(a, b, rel_tol=1e-14) for a, b in zip(f, [1e4 ** (-j / 16) / 2 for j in range(16)] + [1e4 ** (-j / 48) / 2 for j in range(48)]))


@pytest.mark.parametrize("act,q_dtype", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("pairs", [None, (24, 20, 20)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("sizes", [[1], [5, 1, 64], [700]])
def test_append_at(act, q_dtype, pairs, layout, sizes):
    eng = engine(act=act, rows=800, seqs=3)
    rot = eng.rotary(layout=layout, **(dict(axes=pairs, axes_order="cycled") if pairs else {}))
    cols, n_axes = sum(sizes), len(pairs or [0])
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.empty((cols, 4 * 256), device="cuda").normal_(generator=g).to(act)
    k, v = [torch.empty((cols, 256 + 8), device="cuda").normal_(generator=g).to(act)[:, :256] for _ in "kv"]
    pos = torch.randint(0, 100000, (n_axes, cols), generator=g, device="cuda", dtype=torch.int32)
    items = [(2 - i, 17 * i + 3, n) for i, n in enumerate(sizes)]
    for w in "kv":
        eng.cache(0, w).fill_(77)
    for rows in (None, [40 + i for i in range(len(sizes))]):
        out = eng.rotary_append(0, rot, items, q, k, v, rows=rows, q_head_stride=256, q_dtype=q_dtype, positions=pos if pairs else pos[0])
        eng.sync()
        angle = angle_of(pairs or (64,), "cycled", 128, 1e4, pos)
        near(out.view(cols, 4, 128), turned(q.view(cols, 4, 256)[..., :128], 128, angle, layout), q.view(cols, 4, 256)[..., :128], pos, 128)
        col = 0
        for i, (s, p, n) in enumerate(items):
            r0 = p if rows is None else rows[i]
            kc, vc = (eng.cache(0, w)[s, r0:r0 + n].view(F16) for w in "kv")
            kk = k[col:col + n].reshape(n, 2, 128)
            near(kc.reshape(n, 2, 128), turned(kk, 128, angle[col:col + n], layout), kk, pos, 128)
            assert torch.equal(vc, v[col:col + n].half())
            col += n
    touched = sum(n for n in sizes) * 2
    assert int((eng.cache(0, "k") != 77).any(-1).sum()) <= touched and bool((eng.cache(0, "v")[:, 790:] == 77).all())


def test_the_item_positions_and_the_same_of_the_device_give_the_same_bits():
    eng, two = engine(rows=300, seqs=2), engine(rows=300, seqs=2)
    rot, rot2 = eng.rotary(), two.rotary()
    q, k, v = [torch.randn((60, n), device="cuda").half() for n in (512, 256, 256)]
    items = [(0, 100, 50), (1, 7, 10)]
    pos = torch.tensor([100 + c for c in range(50)] + [7 + c for c in range(10)], dtype=torch.int32, device="cuda")
    a, b = eng.rotary_append(0, rot, items, q, k, v), two.rotary_append(0, rot2, items, q, k, v, positions=pos)
    assert torch.equal(a, b) and torch.equal(eng.cache(0, "k")[0, 100:150], two.cache(0, "k")[0, 100:150]) and torch.equal(eng.cache(0, "k")[1, 7:17], two.cache(0, "k")[1, 7:17])
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(a)
    with torch.cuda.graph(g):
        eng.rotary_append(0, rot, items, q, k, v, positions=pos, q_out=out)
    pos += 11                                                              # read when the graph runs
    g.replay()
    assert torch.equal(out[:50], rot.apply(q[:50].float(), 4, pos=111))


def test_refusals():
    eng = engine()
    for kw in (dict(axes=()), dict(axes=(16, 16, 16, 8, 8)), dict(axes=(24, 20, 19)), dict(axes=(20, 20, 24), axes_order="cycled"), dict(axes=(64, 64)), dict(axes=(2 ** 32 - 1, 65)),
               dict(axes=(63, 1), axes_order="own", scaling="ntk", factor=2.0)):
        with pytest.raises(PaError):
            eng.rotary(**kw)
    with pytest.raises(KeyError):
        eng.rotary(axes=(32, 32), axes_order="none")
    rot, plain = eng.rotary(axes=(24, 20, 20)), eng.rotary()
    x = torch.zeros((5, 512), device="cuda", dtype=F16)
    k = torch.zeros((5, 256), device="cuda", dtype=F16)
    p = torch.zeros((3, 5), device="cuda", dtype=torch.int32)
    for bad in (p[0], p[:2], p[:, :4], p.long(), p.cpu(), p.t(), torch.zeros((3, 10), device="cuda", dtype=torch.int32)[:, ::2]):
        with pytest.raises(PaError):
            rot.apply(x, 4, positions=bad)
        with pytest.raises(PaError):
            eng.rotary_append(0, rot, [(0, 0, 5)], x, k, k, positions=bad)
    for bad in (p, p[0, :4], p[0].float()):
        with pytest.raises(PaError):
            plain.apply(x, 4, positions=bad)
    assert eng.L.pa_rotary_append_at(plain.handle, eng.layers[0], None, 0, None, None, None, 0, 0, None, None, 0, None, 0, 0, None) == -1


@pytest.mark.parametrize("nH,nKV,hd,act", [(16, 8, 128, F16), (16, 2, 256, F32), (8, 2, 64, F32)])
def test_a_drafted_tree_from_its_rows_to_the_next_token(nH, nKV, hd, act):
    # append at the depths, attend, keep the accepted path, go on: what a cache that only ever held the path gives
    r = random.Random(8)
    cfg = dict(n_heads=nH, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e6, max_seq=700, n_seqs=3, act_dtype=act, max_cols=600, n_layers=2)
    eng, ref = AttnEngine(AttnConfig(**cfg)), AttnEngine(AttnConfig(**cfg))
    rot, rrot = eng.rotary(), ref.rotary()
    new = lambda n, d: torch.randn((n, d), device="cuda").to(act)
    lens = [501, 64, 130]
    for s, n in enumerate(lens):
        for li in range(2):
            k, v = new(n, nKV * hd), new(n, nKV * hd)
            for e, ro in ((eng, rot), (ref, rrot)):
                e.rotary_append(li, ro, [(s, 0, n)], None, k, v)
    for step in range(3):
        sizes = [r.randint(3, 40) for _ in lens]
        trees = [[-1 if c == 0 else r.randint(max(0, c - 5), c - 1) for c in range(n)] for n in sizes]
        depth = []
        for s, t in enumerate(trees):
            d = []
            for p in t:
                d.append(lens[s] if p < 0 else d[p] + 1)
            depth += d
        paths = []
        for t in trees:
            a = r.randrange(len(t))
            path = []
            while a >= 0:
                path.append(a)
                a = t[a]
            paths.append(path[::-1])
        parents = torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda")
        pos = torch.tensor(depth, dtype=torch.int32, device="cuda")
        items = [(s, lens[s], n) for s, n in enumerate(sizes)]
        total = sum(sizes)
        for li in range(2):
            q, k, v = new(total, nH * hd), new(total, nKV * hd), new(total, nKV * hd)
            qr = eng.rotary_append(li, rot, items, q, k, v, q_dtype=act, positions=pos)
            got = eng.decode_tree(li, items, qr, parents=parents)
            col = 0
            for s, path in enumerate(paths):                              # the path alone, token after token
                at = torch.tensor([col + c for c in path], device="cuda")
                qq = ref.rotary_append(li, rrot, [(s, lens[s], len(path))], q[at], k[at], v[at], q_dtype=act)
                want = torch.cat([ref.decode(li, [(s, lens[s] + i, 1)], qq[i:i + 1]) for i in range(len(path))])
                tol = (2.0 ** -10 if act == F16 else 2e-5) * want.abs().max()
                assert (got[at].float() - want.float()).abs().max() <= tol
                col += sizes[s]
        stride = 1 + max(sizes)
        lists = torch.tensor([[len(p), *p, *[0] * (stride - 1 - len(p))] for p in paths], dtype=torch.int32, device="cuda")
        eng.move([(s, lens[s], s, lens[s], n) for s, n in enumerate(sizes)], lists=lists)
        lens = [n + len(p) for n, p in zip(lens, paths)]
        for li in range(2):
            for w in "kv":
                for s, n in enumerate(lens):
                    assert torch.equal(eng.cache(li, w)[s, :n], ref.cache(li, w)[s, :n])
        q, k, v = new(3, nH * hd), new(3, nKV * hd), new(3, nKV * hd)
        for li in range(2):
            outs = [e.encode_items(li, [(s, lens[s]) for s in range(3)], q, k, v) for e in (eng, ref)]
            assert torch.equal(*outs)
        lens = [n + 1 for n in lens]
    # the first conversation given to the others
    eng.move([(0, 0, 1, 0, lens[0]), (0, 0, 2, 0, lens[0])])
    q = new(3, nH * hd)
    o = eng.decode_tree(0, [(s, lens[0] - 1, 1) for s in range(3)], q[:1].repeat(3, 1))
    assert torch.equal(o[0], o[1]) and torch.equal(o[0], o[2])
