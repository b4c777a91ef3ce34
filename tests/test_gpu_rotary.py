"""pa_rotary: layouts, scalings, free positions and rows, against the formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def engine(nH=4, nKV=2, hd=128, act=F16, max_seq=64, n_seqs=1, max_cols=256, **kw):
    return AttnEngine(AttnConfig(n_heads=nH, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e6, max_seq=max_seq, n_seqs=n_seqs, act_dtype=act, max_cols=max_cols, **kw))


def frequencies(n, theta, scaling="none", factor=1.0, original=0, fast=0.0, slow=0.0):
    """Radians per position and the factor on cos and sin, one pair after another."""
    out, m = [], 1.0
    if scaling == "ntk":
        theta *= factor ** (n / (n - 2))
    for i in range(n // 2):
        f = theta ** (-2 * i / n)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            at = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(at(fast or 32)), 0), min(math.ceil(at(slow or 1)), n - 1)
            t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f, m = (1 - t) * f + t * f / factor, 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        elif scaling == "bands":
            turns = original * f / (2 * math.pi)
            t = min(1.0, max(0.0, (turns - (slow or 1)) / ((fast or 4) - (slow or 1))))
            f = t * f + (1 - t) * f / factor
        out.append(f)
    return np.array(out), m


def rotated(x, positions, f, m, layout):
    """x [cols, heads, hd] in float64, and the lengths of its pairs (0 for dims that are copied)."""
    x = x.double().cpu().numpy()
    n = 2 * len(f)
    ang = np.asarray(positions, dtype=np.float64)[:, None, None] * f
    c, s = m * np.cos(ang), m * np.sin(ang)
    a, b = (slice(0, n // 2), slice(n // 2, n)) if layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    y, r = x.copy(), np.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    r[..., a] = r[..., b] = m * np.hypot(x[..., a], x[..., b])
    return y, r


def check(got, want, length, extra=0.0):
    # cos and sin of the f32 pair: sincospif's unit in the last place, the correction's and mscale's roundings, 2.5 * 2^-24 together; times
    # a and b at most 3.6 * 2^-24 of the pair's length, two more roundings of the rotation: below 2^-21.  f16: half a step more.
    tol = 2.0 ** -21 * length + extra * length + 1e-37
    if got.dtype == F16:
        tol = tol + 2.0 ** -11 * (np.abs(want) + tol) + 2.0 ** -25
    err = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    assert np.all(err <= tol), f"{np.max(err - tol)} over the tolerance at {np.unravel_index(np.argmax(err - tol), err.shape)}"


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,n_rot", [(64, 64), (128, 2), (128, 6), (128, 24), (256, 64), (256, 256)])
@pytest.mark.parametrize("tin,tout", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
def test_apply(layout, hd, n_rot, tin, tout):
    eng = engine(hd=hd)
    rot = eng.rotary(n_rot=n_rot, theta=1e4, layout=layout)
    f, m = frequencies(n_rot, 1e4)
    g = torch.Generator(device="cuda").manual_seed(n_rot)
    for cols, heads, hs, pos in [(1, 1, hd, 0), (1, 16, 2 * hd, 77), (3, 5, hd, 131071), (700, 2, hd, 5), (37, 24, 2 * hd, 9000)]:
        wide = torch.empty((cols, heads * hs + 8), device="cuda").normal_(generator=g).to(tin)
        x = wide[:, :heads * hs]
        out = torch.full((cols, heads * hd + 16), 7.0, dtype=tout, device="cuda")
        rot.apply(x, heads, pos=pos, head_stride=hs, out=out)
        heads_of = x.reshape(cols, heads, hs)[..., :hd]
        y, r = rotated(heads_of, np.arange(pos, pos + cols), f, m, layout)
        check(out[:, :heads * hd], y, r)
        assert torch.all(out[:, heads * hd:] == 7.0)
        if tin == tout:
            assert torch.equal(out[:, :heads * hd].reshape(cols, heads, hd)[..., n_rot:], heads_of[..., n_rot:])      # copied as they are


@pytest.mark.parametrize("scaling,factor,original,kw", [
    ("none", 1.0, 0, {}), ("linear", 4.0, 0, {}), ("ntk", 8.0, 0, {}), ("yarn", 4.0, 8192, {}), ("yarn", 0.5, 300, dict(beta_fast=4.0, beta_slow=2.0)),
    ("yarn", 16.0, 40, {}), ("bands", 8.0, 8192, {}), ("bands", 32.0, 100, dict(high=3.0, low=0.5))])
@pytest.mark.parametrize("n_rot,theta", [(64, 1e7), (128, 1e6), (4, 1e4)])
def test_scalings(scaling, factor, original, kw, n_rot, theta):
    eng = engine(act=F32)
    rot = eng.rotary(n_rot=n_rot, theta=theta, scaling=scaling, factor=factor, original=original, **kw)
    f, m = frequencies(n_rot, theta, scaling, factor, original, kw.get("beta_fast", kw.get("high", 0.0)), kw.get("beta_slow", kw.get("low", 0.0)))
    gf, gm = rot.freqs()
    assert np.allclose(gf, f, rtol=1e-14, atol=0) and abs(gm - m) <= 1e-15 * m
    x = torch.randn((50, 4 * 128), device="cuda")
    y, r = rotated(x.view(50, 4, 128), np.arange(50) + 12345, np.array(gf), gm, "half")
    check(rot.apply(x, 4, pos=12345), y, r)
    twice = eng.rotary(n_rot=n_rot, theta=theta, scaling=scaling, factor=factor, original=original, mscale=2.0, **kw)
    y, r = rotated(x.view(50, 4, 128), np.arange(50) + 12345, np.array(gf), 2.0, "half")
    check(twice.apply(x, 4, pos=12345), y, r)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_of_the_device(layout):
    eng = engine(act=F32, hd=64)
    rot = eng.rotary(theta=1e4, layout=layout)
    places = [0, 1, -1, 131071, -131072, 2 ** 31 - 1, -2 ** 31, 5, 5, 1 << 20]
    x = torch.randn((len(places), 3 * 64), device="cuda")
    p = torch.tensor(places, dtype=torch.int32, device="cuda")
    y, r = rotated(x.view(-1, 3, 64), places, *frequencies(64, 1e4), layout)
    # the far angles: two roundings of turns in float64 here, one of radians there, 2^-53 each, of 2^31 radians
    far = np.where(np.abs(np.array(places, dtype=float)) > 1 << 21, 2.0 ** 31 * 2.0 ** -51, 0.0)[:, None, None]
    got = rot.apply(x, 3, positions=p)
    check(got, y, r, far)
    # turning back: the error of both ways, the second's on the first's result
    back = rot.apply(got[:5], 3, positions=-p[:5])
    assert torch.all((back - x[:5]).abs().view(5, 3, 64) <= 2.0 ** -19 * torch.from_numpy(r[:5]).cuda().float())


def test_in_place_and_strided_targets():
    eng = engine(hd=256, act=F16, nH=8)
    rot = eng.rotary(n_rot=64, layout="interleaved")
    x = torch.randn((19, 8 * 512), device="cuda").half()
    want = rot.apply(x, 8, pos=3, head_stride=512)
    gates = x.view(19, 8, 512)[..., 256:].clone()
    assert rot.apply(x, 8, pos=3, head_stride=512, out=x) is x
    assert torch.equal(x.view(19, 8, 512)[..., :256].reshape(19, -1), want) and torch.equal(x.view(19, 8, 512)[..., 256:], gates)
    odd = torch.randn((5, 8 * 257 + 1), device="cuda")[:, 1:]              # no vector fits: odd strides, four-byte alignment
    y, r = rotated(torch.stack([odd[:, h * 257:h * 257 + 256] for h in range(8)], 1), np.arange(5), *frequencies(64, 1e6), "interleaved")
    check(rot.apply(odd, 8, head_stride=257), y, r)


def test_as_the_engines_own_rotation():
    eng = engine(act=F32)
    x = torch.randn((33, 4 * 128), device="cuda")
    own, new = eng.rope(x, 4, 1000), eng.rotary().apply(x, 4, pos=1000)
    length = torch.hypot(x.view(33, 4, 2, 64)[:, :, 0], x.view(33, 4, 2, 64)[:, :, 1]).repeat(1, 1, 2).view(33, -1)
    assert torch.all((own - new).abs() <= (2.0 ** -21 + 2.0 ** -24) * length)


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("nH,nKV,hd,n_rot,layout", [(16, 2, 256, 64, "interleaved"), (16, 8, 128, 128, "half"), (6, 2, 64, 10, "half"), (24, 4, 256, 64, "half")])
@pytest.mark.parametrize("q_dtype", [F16, F32])
def test_append(act, nH, nKV, hd, n_rot, layout, q_dtype):
    n_seqs, max_seq = 5, 300
    eng = engine(nH=nH, nKV=nKV, hd=hd, act=act, max_seq=max_seq, n_seqs=n_seqs, max_cols=512)
    rot = eng.rotary(n_rot=n_rot, theta=1e6, layout=layout, scaling="linear", factor=2.0)
    f, m = frequencies(n_rot, 1e6, "linear", 2.0)
    for items, rows in [([(3, 9, 1)], None), ([(0, 100000, 1), (4, 7, 1), (1, 2 ** 31 - 2, 1)], [17, 299, 0]), ([(2, 40, 200)], None), ([(0, 5, 3), (1, 60, 1), (0, 70, 90)], [10, 20, 13]),
                        ([(4, 1000, 130)], [170])]:
        n = sum(c for _, _, c in items)
        for w in "kv":
            eng.cache(0, w).fill_(0x5a5a)
        q = torch.randn((n, nH * 2 * hd), device="cuda").to(act)
        k, v = [torch.randn((n, nKV * hd + 8), device="cuda").to(act)[:, :nKV * hd] for _ in "kv"]
        v[0, :4] = torch.tensor([math.nan, -math.inf, 65504.0, 1e-8])
        got = eng.rotary_append(0, rot, items, q, k, v, rows=rows, q_head_stride=2 * hd, q_dtype=q_dtype)
        places = np.concatenate([np.arange(p, p + c) for _, p, c in items])
        far = 2.0 ** 31 * 2.0 ** -51 if places.max() > 1 << 21 else 0.0
        y, r = rotated(q.view(n, nH, 2 * hd)[..., :hd], places, f, m, layout)
        check(got, y, r, far)
        yk, rk = rotated(k.reshape(n, nKV, hd), places, f, m, layout)
        at, touched = 0, torch.zeros((n_seqs, max_seq), dtype=torch.bool)
        for (s, p, c), row in zip(items, rows if rows is not None else [p for _, p, _ in items]):
            check(eng.cache(0, "k")[s, row:row + c].view(F16), yk[at:at + c].reshape(c, -1), rk[at:at + c].reshape(c, -1), far)
            gv, wv = eng.cache(0, "v")[s, row:row + c], v[at:at + c].half().contiguous().view(torch.int16)
            nan = torch.isnan(v[at:at + c].float())
            assert torch.equal(gv[~nan], wv[~nan]) and torch.all((gv[nan] & 0x7fff) == 0x7e00)
            touched[s, row:row + c] = True
            at += c
        for w in "kv":
            assert torch.all(eng.cache(0, w).cpu()[~touched] == 0x5a5a)


def test_append_without_q_and_then_decode():
    # the rows are there when a decode follows at once, and every early fetch of the decode kernels respects them
    eng = engine(nH=16, nKV=2, hd=256, max_seq=600, act=F32, rope_mode="none")
    rot = eng.rotary(n_rot=64)
    k, v = [torch.randn((599, 512), device="cuda") for _ in "kv"]
    q = torch.randn((1, 4096), device="cuda")
    for _ in range(20):
        eng.cache(0, "k").zero_(); eng.cache(0, "v").zero_()
        assert eng.rotary_append(0, rot, [(0, 300, 256)], None, k[300:556], v[300:556]) is None
        eng.rotary_append(0, rot, [(0, 44, 256)], None, k[44:300], v[44:300])
        eng.rotary_append(0, rot, [(0, 0, 44)], None, k[:44], v[:44])  # the lower rows last: what follows must not fetch them early
        got = eng.decode(0, [(0, 555, 1)], q)
        kc, vc = [eng.cache(0, w)[0, :556].view(F16).double().view(556, 2, 256) for w in "kv"]
        p = torch.softmax(torch.einsum("gd,rd->gr", q.double().view(16, 256)[:8], kc[:, 0]) / 16, -1)
        assert torch.allclose(got.view(16, 256)[:8].double(), p @ vc[:, 0], rtol=0, atol=2e-5)


def test_streams_and_graphs():
    eng = engine(act=F32, max_seq=128)
    rot = eng.rotary(layout="interleaved")
    x, k, v = [torch.randn((40, w * 128), device="cuda") for w in (4, 2, 2)]
    p = torch.arange(40, dtype=torch.int32, device="cuda")
    want, want_q = rot.apply(x, 4, positions=p), eng.rotary_append(0, rot, [(0, 30, 40)], x, k, v)
    rows = eng.cache(0, "k").clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rot.apply(x, 4, positions=p)
    side.synchronize()
    assert torch.equal(got, want)
    out, q_out = torch.empty_like(want), torch.empty_like(want_q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rot.apply(x, 4, positions=p, out=out)
        eng.rotary_append(0, rot, [(0, 30, 40)], x, k, v, q_out=q_out)
    eng.cache(0, "k").zero_()
    p += 7                                                             # positions are read when the kernel runs
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, rot.apply(x, 4, positions=p)) and torch.equal(q_out, want_q) and torch.equal(eng.cache(0, "k")[0, 30:70], rows[0, 30:70])


@pytest.mark.parametrize("kw", [dict(n_rot=3), dict(n_rot=0), dict(n_rot=130), dict(theta=1.0), dict(theta=math.nan), dict(theta=math.inf), dict(scaling="linear", factor=0.0),
                                dict(scaling="linear", factor=math.nan), dict(scaling="ntk", factor=2.0, n_rot=2), dict(scaling="yarn", factor=2.0),
                                dict(scaling="yarn", factor=2.0, original=10, beta_fast=1.0, beta_slow=2.0), dict(scaling="bands", factor=2.0),
                                dict(scaling="bands", factor=2.0, original=9, low=-1.0), dict(mscale=math.inf)])
def test_refused_configurations(kw):
    with pytest.raises(PaError) as e:
        engine().rotary(**kw)
    assert e.value.code == -1


def test_refused_calls():
    eng, other = engine(max_seq=64, n_seqs=2, max_cols=32), engine()
    rot = eng.rotary()
    x, kv = torch.zeros((4, 512), dtype=F16, device="cuda"), torch.zeros((4, 256), dtype=F16, device="cuda")

    def refused(f, code=-1):
        with pytest.raises(PaError) as e:
            f()
        assert e.value.code == code

    refused(lambda: rot.apply(x.cpu(), 4))
    refused(lambda: rot.apply(x, 5))
    refused(lambda: rot.apply(x.to(torch.bfloat16), 4))
    refused(lambda: rot.apply(x, 4, positions=torch.zeros(4, dtype=torch.int64, device="cuda")))
    refused(lambda: rot.apply(x, 4, positions=torch.zeros(3, dtype=torch.int32, device="cuda")))
    refused(lambda: rot.apply(x, 4, pos=2 ** 31 - 3))
    refused(lambda: rot.apply(x, 4, out=torch.zeros((3, 512), dtype=F16, device="cuda")))
    refused(lambda: rot.apply(x[:, ::2], 2))
    refused(lambda: rot.apply(x, 2, head_stride=256, out=x, out_head_stride=128))
    append = lambda items, rows=None, q=x, k=kv, v=kv, r=rot, **kw: lambda: eng.rotary_append(0, r, items, q, k, v, rows=rows, **kw)
    refused(append([(2, 0, 4)]))
    refused(append([(0, 61, 4)]))
    refused(append([(0, 61, 4)], rows=[61]))
    refused(append([(0, 0, 2), (0, 1, 2)]))
    refused(append([(0, 0, 2), (0, 9, 2)], rows=[5, 6]))
    refused(append([(0, 0, 0), (0, 9, 4)]))
    refused(append([(0, 0, 3)]))
    refused(append([(0, 0, 4)], q=x.float()))
    refused(append([(0, 0, 4)], r=other.rotary()))
    refused(append([(0, 0, 4)], q_dtype=torch.float64))
    refused(lambda: eng.rotary_append(0, rot, [], x[:0], kv[:0], kv[:0]))
    with pytest.raises(ValueError):
        append([(0, 0, 4)], rows=[1, 2])()
    big = torch.zeros((33, 512), dtype=F16, device="cuda")
    refused(lambda: eng.rotary_append(0, rot, [(0, 0, 33)], big, big[:, :256], big[:, :256]))
    q8 = engine(kv_format="q8")
    refused(lambda: q8.rotary_append(0, q8.rotary(), [(0, 0, 4)], x, kv, kv), -2)
    eng.rotary_append(0, rot, [(0, 0, 4)], x, kv, kv)                 # nothing of the above has latched the context
    eng.sync()


def test_columns_that_would_overlap_are_refused():
    # one stride at a time each layout below looks possible; heads of one column and of another are the same addresses
    eng = engine()
    rot = eng.rotary()
    x = torch.randn((3, 4 * 128), device="cuda").half()
    room = torch.zeros(8192, dtype=F16, device="cuda")
    y, r = rotated(x.view(3, 4, 128), np.arange(7, 10), *frequencies(128, 1e6), "half")
    for col, head in [(128, 128), (128, 256), (256, 128), (511, 128), (128, 383), (130, 256), (512, 513), (300, 200)]:
        with pytest.raises(PaError) as e:
            rot.apply(x, 4, pos=7, out=room.as_strided((3, 3 * head + 128), (col, 1)), out_head_stride=head)
        assert e.value.code == -1 and not room.any()
    # columns outermost, heads outermost, and heads of a column on both sides of the next column's first
    for cols, heads, col, head in [(3, 4, 512, 128), (3, 4, 128, 384), (3, 4, 130, 400), (3, 4, 1000, 200), (3, 4, 384, 1152), (2, 2, 256, 384)]:
        room.zero_()
        rot.apply(x[:cols], heads, pos=7, out=room.as_strided((cols, (heads - 1) * head + 128), (col, 1)), out_head_stride=head)
        check(torch.as_strided(room, (cols, heads, 128), (col, head, 1)), y[:cols, :heads], r[:cols, :heads])
        assert int((room != 0).sum()) <= cols * heads * 128


@pytest.mark.parametrize("act", [F16, F32])
def test_append_rotates_q_in_place_with_its_own_layout_only(act):
    eng = engine(nH=16, nKV=2, hd=256, act=act, max_seq=64, max_cols=64)
    rot = eng.rotary(n_rot=64, layout="interleaved")
    full = torch.randn((40, 16 * 512), device="cuda").to(act)                # q and gate of a head side by side
    k, v = [torch.randn((40, 512), device="cuda").to(act) for _ in "kv"]
    other = F32 if act == F16 else F16
    before = full.clone()
    for cols, bad in [(40, dict(q=full, q_head_stride=512, q_out=full)), (40, dict(q=full[:, :4096], q_out=full.view(-1)[:40 * 4096].view(40, 4096))),
                      (1, dict(q=full[:1], q_head_stride=512, q_out=full[:1])), (1, dict(q=full[:1, :4096], q_out=full.view(other).view(-1)[:4096].view(1, 4096)))]:
        with pytest.raises(PaError) as e:
            eng.rotary_append(0, rot, [(0, 3, cols)], bad.pop("q"), k[:cols], v[:cols], **bad)
        assert e.value.code == -1 and torch.equal(full, before)
    for q in (full[:, :4096], full[:1, 4096:]):
        n = q.shape[0]
        want = eng.rotary_append(0, rot, [(0, 3, n)], q, k[:n], v[:n], q_dtype=act)
        assert eng.rotary_append(0, rot, [(0, 3, n)], q, k[:n], v[:n], q_out=q) is q
        assert torch.equal(q, want)


@pytest.mark.parametrize("kw", [dict(scaling="ntk", factor=1e-320), dict(scaling="ntk", factor=1e-300, n_rot=4), dict(scaling="linear", factor=5e-324), dict(scaling="yarn", factor=1e-310, original=10),
                                dict(scaling="bands", factor=1e-310, original=10), dict(mscale=1e39), dict(scaling="yarn", factor=4.0, original=100, mscale=-1e300)])
def test_scalings_past_the_range_of_numbers_are_refused(kw):
    eng = engine()
    with pytest.raises(PaError) as e:
        eng.rotary(**kw)
    assert e.value.code == -1
    rot = eng.rotary(scaling="linear", factor=1e-30, mscale=1e30)              # far, but numbers
    assert all(math.isfinite(f) for f in rot.freqs()[0])
    assert torch.isfinite(rot.apply(torch.full((3, 128), 1e-3, device="cuda"), 1, pos=2 ** 31 - 4)).all()


def test_a_rotation_of_another_engine_is_named_in_the_layers_own_error():
    eng, other = engine(max_cols=32), engine(max_cols=32)
    x, kv = torch.zeros((4, 512), dtype=F16, device="cuda"), torch.zeros((4, 256), dtype=F16, device="cuda")
    with pytest.raises(PaError, match="another context"):
        eng.rotary_append(0, other.rotary(), [(0, 0, 4)], x, kv, kv)
