"""pa_decode_tree: trees of drafted tokens behind the committed rows of their sequences, against softmax attention in 64 bits."""
import math
import random

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
POISON = [math.nan, math.inf, -math.inf, 65504.0]


def engine(nH, nKV, hd, rows, n_seqs, act, max_cols=8, **kw):
    return AttnEngine(AttnConfig(n_heads=nH, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e6, max_seq=rows, n_seqs=n_seqs, act_dtype=act, max_cols=max_cols,
                                 rope_mode="none", **kw))


def fill(eng, seed):
    """Every row of the caches normal values, keys with a few large channels; returns K and V as f16 [n_seqs, max_seq, nKV, hd]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = eng.cfg
    kv = [torch.empty((c.n_seqs, c.max_seq, c.n_kv_heads, c.head_dim), dtype=F16, device="cuda").normal_(generator=g) for _ in "kv"]
    kv[0][..., 3::61] *= 3.0
    for w, x in zip("kv", kv):
        eng.cache(0, w).copy_(x.view(c.n_seqs, c.max_seq, -1).view(torch.int16))
    return kv


def poison(eng, seq, row0):
    """What no call may read: NaN, infinities and the largest numbers in the rows from row0 on."""
    c = eng.cfg
    n = c.max_seq - row0
    if n > 0:
        bad = torch.tensor(POISON, dtype=F16).repeat(n * c.kv_dim // 4 + 1)[:n * c.kv_dim].view(n, c.kv_dim).cuda()
        for w in "kv":
            eng.cache(0, w)[seq, row0:] = bad.view(torch.int16)


def tree(r, n, reach):
    return [-1 if c == 0 or r.random() < 0.05 else r.randint(max(0, c - reach), c - 1) for c in range(n)]


def mask_of(parents, base):
    """[n, base + n]: what every token attends."""
    n = len(parents)
    m = torch.zeros((n, base + n), dtype=torch.bool)
    m[:, :base] = True
    for c in range(n):
        a = c
        while a >= 0:
            m[c, base + a] = True
            a = parents[a]
    return m.cuda()


def attend(q, k, v, mask, gate=None):
    """q [n, nH, hd], k and v [rows, nKV, hd] -> out [n, nH, hd] in float64, and how far a row's scores may be off [n, nH]."""
    n, nH, hd = q.shape
    G = nH // k.shape[1]
    qd, kd, vd = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("nhd,rhd->nhr", qd, kd) / math.sqrt(hd)
    p = torch.softmax(torch.where(mask[:, None], s, -math.inf), -1)
    o = torch.einsum("nhr,rhd->nhd", p, vd)
    # a score: f32 queries as two f16 values (2^-22 of |q|), hd / 16 accumulations of the tensor core and the sum of its two rows (2^-23 of the sum of
    # absolute products each)
    delta = (torch.einsum("nhd,rhd->nhr", qd.abs(), kd.abs()) / math.sqrt(hd)).amax(-1) * (2.0 ** -22 + (hd / 16 + 2) * 2.0 ** -23)
    return (o if gate is None else o * torch.sigmoid(gate.double())), delta


def close(got, want, v, delta, rows):
    # weights: twice the score's error, the exponential's and the f16 pairs' 2^-22 each, and 2^-25 a row of weights that underflow f16, of which the
    # sum is at least 1; sums over the rows by 16 and over at most 512 records; then the gate (its exponential 2^-21) and the store
    big = v.double().abs().amax()
    tol = big * (2 * delta + 2.0 ** -20 + rows * 2.0 ** -25 + (rows / 16 + 64) * 2.0 ** -23)
    if got.dtype == F16:
        tol = tol + 2.0 ** -11 * want.abs().amax(-1) + 2.0 ** -25
    err = (got.double().view(want.shape) - want).abs().amax(-1)
    assert torch.isfinite(got).all()
    assert torch.all(err <= tol), f"{float((err / tol).max())} of the tolerance"


def check(eng, k, v, items, trees, q, gate, got, q_hs=None, gate_hs=None):
    c = eng.cfg
    nH, hd, col = c.n_heads, c.head_dim, 0
    for (s, base, n), t in zip(items, trees):
        rows = base + n
        qq = q[col:col + n].reshape(n, -1)
        qq = torch.stack([qq[:, h * (q_hs or hd):h * (q_hs or hd) + hd] for h in range(nH)], 1)
        gg = None
        if gate is not None:
            gg = torch.stack([gate[col:col + n, h * (gate_hs or hd):h * (gate_hs or hd) + hd] for h in range(nH)], 1)
        want, delta = attend(qq, k[s, :rows], v[s, :rows], mask_of(t, base), gg)
        close(got[col:col + n, :nH * hd], want, v[s, :rows], delta, rows)
        col += n


SHAPES = [(16, 8, 128), (16, 2, 256), (24, 4, 256), (4, 4, 64), (10, 2, 128), (64, 1, 64)]
SETS = [[(0, 1)], [(0, 17), (63, 2)], [(64, 64), (1, 1), (130, 33)], [(301, 8)], [(700, 256)], [(65, 60), (2000, 9), (0, 64), (64, 1), (127, 130)]]


@pytest.mark.parametrize("nH,nKV,hd", SHAPES)
@pytest.mark.parametrize("act,q_dtype,gated", [(F16, F16, True), (F32, F32, False), (F32, F16, True), (F16, F32, False)])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: "+".join(f"{b}.{n}" for b, n in s))
def test_against_64_bits(nH, nKV, hd, act, q_dtype, gated, sizes):
    r = random.Random(len(sizes) * 7 + nH)
    m = len(sizes)
    eng = engine(nH, nKV, hd, max(b + n for b, n in sizes) + 70, m, act)
    k, v = fill(eng, 1)
    seqs = r.sample(range(m), m)                                          # items in another order than their sequences
    items = [(s, b, n) for s, (b, n) in zip(seqs, sizes)]
    for s, b, n in items:
        poison(eng, s, b + n)
    trees = [tree(r, n, r.choice([1, 4, 20])) for _, _, n in items]
    total = sum(n for _, _, n in items)
    q = torch.randn((total, nH * 2 * hd), device="cuda").to(q_dtype)
    gate = torch.randn((total, nH * hd + 16), device="cuda").to(act) if gated else None
    out = torch.full((total, nH * hd + 8), 9.0, dtype=act, device="cuda")
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda")
    eng.decode_tree(0, items, q, parents=parents, gate=gate, out=out, q_head_stride=2 * hd)
    eng.sync()
    assert torch.all(out[:, nH * hd:] == 9.0)
    check(eng, k, v, items, trees, q, gate, out, q_hs=2 * hd)


@pytest.mark.parametrize("wide", ["0", "1"])
@pytest.mark.parametrize("nH,nKV", [(16, 2), (24, 4)])
@pytest.mark.parametrize("sizes", [[(5000, 64)], [(0, 100), (1030, 63), (200, 17)], [(12000, 33)]])
def test_wide_and_narrow_row_tiles(monkeypatch, wide, nH, nKV, sizes):
    monkeypatch.setenv("POOLED_ATTN_SHARED_WIDE", wide)
    r = random.Random(5)
    eng = engine(nH, nKV, 256, max(b + n for b, n in sizes), len(sizes), F16)
    k, v = fill(eng, 2)
    items = [(s, b, n) for s, (b, n) in enumerate(sizes)]
    trees = [tree(r, n, 6) for _, _, n in items]
    total = sum(n for _, _, n in items)
    q, gate = [torch.randn((total, nH * 256), device="cuda").half() for _ in "qg"]
    got = eng.decode_tree(0, items, q, parents=torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda"), gate=gate)
    check(eng, k, v, items, trees, q, gate, got)


@pytest.mark.parametrize("nH,nKV,hd,act", [(64, 1, 64, F32), (128, 8, 64, F16), (32, 4, 256, F32), (32, 4, 256, F16), (48, 8, 128, F32)])
def test_more_columns_than_one_launch_has_records_for(nH, nKV, hd, act):
    # trees are parted, and runs added up in their records
    r = random.Random(9)
    sizes = [(3000, 256), (700, 200), (4500, 150)]
    eng = engine(nH, nKV, hd, 4700, 3, act)
    k, v = fill(eng, 3)
    items = [(s, b, n) for s, (b, n) in enumerate(sizes)]
    trees = [tree(r, n, 9) for _, _, n in items]
    q = torch.randn((606, nH * hd), device="cuda").to(act)
    got = eng.decode_tree(0, items, q, parents=torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda"))
    check(eng, k, v, items, trees, q, None, got)


@pytest.mark.parametrize("nH,nKV,hd", [(16, 8, 128), (16, 2, 256), (16, 2, 64)])
@pytest.mark.parametrize("act", [F16, F32])
def test_a_long_context(nH, nKV, hd, act):
    r = random.Random(4)
    eng = engine(nH, nKV, hd, 33100, 1, act)
    k, v = fill(eng, 4)
    trees = [tree(r, 61, 7)]
    q = torch.randn((61, nH * hd), device="cuda").to(act)
    got = eng.decode_tree(0, [(0, 33001, 61)], q, parents=torch.tensor(trees[0], dtype=torch.int32, device="cuda"))
    check(eng, k, v, [(0, 33001, 61)], trees, q, None, got)


def test_rows_past_four_gigabytes():
    # the last of eight sequences of 300000 rows of 2 KB
    eng = engine(16, 8, 128, 300000, 8, F16)
    r, n, base = random.Random(2), 30, 200
    k, v = [torch.randn((1, base + n, 8, 128), device="cuda").half() for _ in "kv"]
    v[0, base + 3] = math.inf                                             # looked up again for those that attend it
    for w, x in zip("kv", (k, v)):
        eng.cache(0, w)[7, :base + n] = x.view(base + n, -1).view(torch.int16)
    poison_rows = eng.cache(0, "v")[7, base + n:base + n + 64]
    poison_rows[:] = torch.tensor(POISON, dtype=F16).repeat(256).view(torch.int16).cuda()
    parents = tree(r, n, 4)
    parents[3], parents[5] = 2, 3
    q = torch.randn((n, 16 * 128), device="cuda").half()
    got = eng.decode_tree(0, [(7, base, n)], q, parents=torch.tensor(parents, dtype=torch.int32, device="cuda"))
    eng.sync()
    mask = mask_of(parents, base)
    of = mask[:, base + 3]
    assert torch.all(got[of.cuda()] == math.inf) and of.any() and not of.all()
    v[0, base + 3] = 0.0
    want, delta = attend(q.view(n, 16, 128), k[0], v[0], mask)
    keep = ~of.cuda()
    close(got[keep], want[keep], v[0], delta[keep], base + n)


@pytest.mark.parametrize("nH,nKV,hd", [(16, 8, 128), (16, 2, 256), (8, 8, 64)])
def test_chains_and_single_tokens_are_what_the_other_decode_gives(nH, nKV, hd):
    eng = engine(nH, nKV, hd, 1100, 3, F32, max_cols=64)
    fill(eng, 5)
    n = 64 // (nH // nKV)
    q = torch.randn((n, nH * hd), device="cuda")
    chain = eng.decode_tree(0, [(1, 1000, n)], q)
    said = eng.decode_tree(0, [(1, 1000, n)], q, parents=torch.arange(-1, n - 1, dtype=torch.int32, device="cuda"))
    assert torch.equal(chain, said)
    ref = eng.decode(0, [(1, 1000, n)], q)
    assert (chain - ref).abs().max() <= 2e-5 * ref.abs().max()
    one = eng.decode_tree(0, [(2, 700, 1), (0, 0, 1)], q[:2])
    ref = eng.decode(0, [(2, 700, 1), (0, 0, 1)], q[:2])
    assert (one - ref).abs().max() <= 2e-5 * ref.abs().max()


@pytest.mark.parametrize("hd,act", [(256, F16), (256, F32), (128, F16), (64, F32)])
@pytest.mark.parametrize("base,n", [(0, 40), (100, 64), (63, 200)])
def test_other_tokens_may_hold_anything(hd, act, base, n):
    # a token that is no ancestor: NaN, infinities and the largest numbers in its K and V change no bit; one that is: its values arrive
    r = random.Random(base + n)
    eng = engine(8, 2, hd, base + n, 1, act)
    k, v = fill(eng, 6)
    t = tree(r, n, 12)
    parents = torch.tensor(t, dtype=torch.int32, device="cuda")
    q = torch.randn((n, 8 * hd), device="cuda").to(act)
    items = [(0, base, n)]
    clean = eng.decode_tree(0, items, q, parents=parents)
    sees = mask_of(t, base)
    for bad_tokens in ([n - 1], [0], [n // 2, n // 3], list(range(0, n, 3))):
        for w, x in zip("kv", (k, v)):
            eng.cache(0, w).copy_(x.view(1, base + n, -1).view(torch.int16))
            for b in bad_tokens:
                eng.cache(0, w)[0, base + b] = torch.tensor(POISON, dtype=F16).repeat(2 * hd // 4).cuda().view(torch.int16)
        got = eng.decode_tree(0, items, q, parents=parents)
        hit = sees[:, [base + b for b in bad_tokens]].any(1)
        assert torch.equal(got[~hit], clean[~hit]) and torch.isnan(got[hit]).all(1).all()
    # V alone, some values: the same values that are not finite, and where
    for w, x in zip("kv", (k, v)):
        eng.cache(0, w).copy_(x.view(1, base + n, -1).view(torch.int16))
    b, vv = n // 3, v.clone()
    vv[0, base + b, 0, 5], vv[0, base + b, 1, 17], vv[0, base + b, 1, hd - 1] = math.inf, math.nan, -math.inf
    eng.cache(0, "v").copy_(vv.view(1, base + n, -1).view(torch.int16))
    got = eng.decode_tree(0, items, q, parents=parents).view(n, 8, hd).float()
    want = clean.view(n, 8, hd).float().clone()
    hit = sees[:, base + b]
    want[hit, :4, 5], want[hit, 4:, 17], want[hit, 4:, hd - 1] = math.inf, math.nan, -math.inf
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]) and torch.equal(got.isnan(), want.isnan())
    assert (got[fine] - want[fine]).abs().max() <= 2e-2


def test_parents_that_are_no_earlier_token_are_none():
    eng = engine(16, 2, 256, 200, 1, F32)
    k, v = fill(eng, 7)
    q = torch.randn((6, 4096), device="cuda")
    got = eng.decode_tree(0, [(0, 150, 6)], q, parents=torch.tensor([0, 1, 5, -7, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda"))
    check(eng, k, v, [(0, 150, 6)], [[-1] * 6], q, None, got)


def test_equal_bits_and_graphs_on_other_streams():
    eng = engine(24, 4, 256, 3100, 4, F16)
    k, v = fill(eng, 8)
    r = random.Random(3)
    items = [(2, 3000, 40), (0, 77, 12), (2, 1000, 3)]                    # a sequence twice, at two lengths
    trees = [tree(r, n, 5) for _, _, n in items]
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda")
    q, gate = [torch.randn((55, 24 * 256), device="cuda").half() for _ in "qg"]
    ref = eng.decode_tree(0, items, q, parents=parents, gate=gate)
    check(eng, k, v, items, trees, q, gate, ref)
    out = torch.empty_like(ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(eng.decode_tree(0, items, q, parents=parents, gate=gate), ref)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        eng.decode_tree(0, items, q, parents=parents, gate=gate, out=out)
        eng.decode_tree(0, items, q, parents=parents, gate=gate, out=out)
    g.replay()
    assert torch.equal(out, ref)
    trees = [tree(r, n, 5) for _, _, n in items]                          # other trees and queries of the same sizes
    parents.copy_(torch.tensor(sum(trees, []), dtype=torch.int32))
    q.copy_(torch.randn_like(q))
    g.replay()
    check(eng, k, v, items, trees, q, gate, out)


def test_refusals():
    eng = engine(16, 2, 256, 300, 2, F16)
    fill(eng, 9)
    q = torch.zeros((4, 4096), device="cuda", dtype=F16)
    par = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    ok = eng.decode_tree(0, [(0, 100, 4)], q, parents=par)
    assert torch.isfinite(ok).all()
    for items in ([], [(2, 0, 4)], [(0, 297, 4)], [(0, 2 ** 32 - 1, 4)], [(0, 100, 0), (0, 100, 4)], [(0, 0, 257)], [(0, 0, 1)] * 33):
        n = sum(i[2] for i in items)
        with pytest.raises(PaError):
            eng.decode_tree(0, items, torch.zeros((n, 4096), device="cuda", dtype=F16))
    for kw in (dict(parents=par[:3]), dict(parents=par.long()), dict(parents=par.cpu()), dict(gate=q.float()), dict(out=q.float()), dict(out=q[:3]), dict(q_head_stride=-256)):
        with pytest.raises(PaError):
            eng.decode_tree(0, [(0, 100, 4)], q, **kw)
    with pytest.raises(PaError):
        eng.decode_tree(0, [(0, 100, 4)], torch.zeros((4, 4100), device="cuda", dtype=F16)[:, 1:4097])
    with pytest.raises(PaError):
        eng.decode_tree(0, [(0, 100, 4)], torch.zeros((4, 4100), device="cuda", dtype=F16)[:, :4096])
    for kv in ("q8", "f32"):
        with pytest.raises(PaError) as e:
            engine(16, 2, 256, 300, 2, F16, kv_format=kv).decode_tree(0, [(0, 100, 4)], q, parents=par)
        assert e.value.code == -2
    eng.set_origin(0, 5)
    with pytest.raises(PaError):
        eng.decode_tree(0, [(0, 100, 4)], q, parents=par)
    eng.set_origin(0, 0)
    assert torch.equal(eng.decode_tree(0, [(0, 100, 4)], q, parents=par), ok)
