"""pa_decode_shared: single tokens of many sequences behind one prefix, against softmax attention in 64 bits."""
import math

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
POISON = [math.nan, math.inf, -math.inf, 65504.0]


def engine(nH, nKV, hd, rows, n_seqs, act, max_cols=8, **kw):
    return AttnEngine(AttnConfig(n_heads=nH, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e6, max_seq=rows, n_seqs=n_seqs, act_dtype=act, max_cols=max_cols,
                                 rope_mode="none", **kw))


def fill(eng, seed, scale=1.0):
    """Every row of the caches normal values, keys with a few large channels; returns K and V as f16 [n_seqs, max_seq, nKV, hd]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = eng.cfg
    kv = [torch.empty((c.n_seqs, c.max_seq, c.n_kv_heads, c.head_dim), dtype=F16, device="cuda").normal_(generator=g) * scale for _ in "kv"]
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


def attend(q, k, v, gate=None):
    """q [nH, hd], k and v [rows, nKV, hd] -> out [nH, hd] in float64, the weights [nH, rows], and how far scores may be off."""
    nH, hd = q.shape
    G = nH // k.shape[1]
    qd, kd, vd = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("hd,rhd->hr", qd, kd) / math.sqrt(hd)
    p = torch.softmax(s, -1)
    o = torch.einsum("hr,rhd->hd", p, vd)
    # a score: f32 queries as two f16 values (2^-22 of |q|), hd / 16 accumulations of the tensor core and the sum of its two rows (2^-23 of the sum of
    # absolute products each)
    delta = (torch.einsum("hd,rhd->hr", qd.abs(), kd.abs()) / math.sqrt(hd)).amax(-1) * (2.0 ** -22 + (hd / 16 + 2) * 2.0 ** -23)
    if gate is not None:
        o = o * torch.sigmoid(gate.double())
    return o, p, delta


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


SHAPES = [(16, 8, 128), (16, 2, 256), (24, 4, 256), (4, 4, 64), (10, 2, 128), (64, 1, 64)]


@pytest.mark.parametrize("nH,nKV,hd", SHAPES)
@pytest.mark.parametrize("act,q_dtype,gated", [(F16, F16, True), (F32, F32, False), (F32, F16, True), (F16, F32, False)])
@pytest.mark.parametrize("prefix_len,own", [(0, [1, 64, 65, 130]), (1, [0]), (63, [1, 2, 0]), (64, [64] * 7), (65, [0, 0, 0, 17, 200]), (700, list(range(33))), (1000, [1])])
def test_against_64_bits(nH, nKV, hd, act, q_dtype, gated, prefix_len, own):
    n = len(own)
    eng, first = engine(nH, nKV, hd, max(own) + 70, n + 1, act), engine(nH, nKV, hd, prefix_len + 70, 2, act)
    k, v = fill(eng, 1)
    pk, pv = fill(first, 2)
    order = [(5 * i + 3) % n if n % 5 else n - 1 - i for i in range(n)]      # items in another order than their sequences
    for s in range(n):
        poison(eng, s, own[s])
    poison(eng, n, 0)
    poison(first, 1, prefix_len)
    poison(first, 0, 0)
    q = torch.randn((n, nH * 2 * hd), device="cuda").to(q_dtype)
    gate = torch.randn((n, nH * hd + 16), device="cuda").to(act) if gated else None
    out = torch.full((n, nH * hd + 8), 9.0, dtype=act, device="cuda")
    eng.decode_shared(0, first, 1, prefix_len, [(s, prefix_len + own[s] - 1) for s in order], q, gate, out=out, own_base=prefix_len, q_head_stride=2 * hd)
    eng.sync()
    assert torch.all(out[:, nH * hd:] == 9.0)
    for i, s in enumerate(order):
        rows = prefix_len + own[s]
        kk, vv = torch.cat([pk[1, :prefix_len], k[s, :own[s]]]), torch.cat([pv[1, :prefix_len], v[s, :own[s]]])
        want, _, delta = attend(q[i].view(nH, 2 * hd)[:, :hd], kk, vv, gate[i, :nH * hd].view(nH, hd) if gated else None)
        close(out[i, :nH * hd], want, vv, delta, rows)


def test_prefix_in_the_same_layer_at_its_positions():
    eng = engine(16, 2, 256, 900, 4, F32)
    k, v = fill(eng, 3)
    q = torch.randn((4, 4096), device="cuda")
    seqs_pos = [(1, 640), (3, 899), (2, 599), (2, 610)]                     # a sequence twice, at two lengths
    got = eng.decode_shared(0, None, 0, 600, seqs_pos, q)
    for i, (s, pos) in enumerate(seqs_pos):
        kk, vv = torch.cat([k[0, :600], k[s, 600:pos + 1]]), torch.cat([v[0, :600], v[s, 600:pos + 1]])
        want, _, delta = attend(q[i].view(16, 256), kk, vv)
        close(got[i], want, vv, delta, pos + 1)
    # the same rows in one sequence: the decode that reads them there, to both calls' tolerance
    for w in "kv":
        eng.cache(0, w)[1, :600] = eng.cache(0, w)[0, :600]
    ref = eng.decode(0, [(1, 640, 1)], q[:1])
    assert (got[:1] - ref).abs().max() <= 2e-5 * ref.abs().max()


@pytest.mark.parametrize("nH,nKV,hd,n", [(16, 2, 256, 128), (128, 8, 64, 128), (8, 8, 128, 100)])
def test_many_items(nH, nKV, hd, n):
    # 128 heads of 128 items are more rows than one launch has records for
    eng, first = engine(nH, nKV, hd, 40, n, F16), engine(nH, nKV, hd, 200, 1, F16)
    k, v = fill(eng, 4)
    pk, pv = fill(first, 5)
    q, gate = [torch.randn((n, nH * hd), device="cuda").half() for _ in "qg"]
    own = [i % 41 for i in range(n)]
    got = eng.decode_shared(0, first, 0, 200, [(i, 199 + own[i]) for i in range(n)], q, gate, own_base=200)
    for i in range(0, n, 9):
        kk, vv = torch.cat([pk[0], k[i, :own[i]]]), torch.cat([pv[0], v[i, :own[i]]])
        want, _, delta = attend(q[i].view(nH, hd), kk, vv, gate[i].view(nH, hd))
        close(got[i], want, vv, delta, 200 + own[i])


@pytest.mark.parametrize("nH,nKV,hd", [(16, 8, 128), (16, 2, 256), (128, 8, 64)])
@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("prefix_len,own", [(60, [4000, 1, 0, 2501]), (130, [3001])])
def test_long_conversations_behind_a_short_prefix(nH, nKV, hd, act, prefix_len, own):
    eng, first = engine(nH, nKV, hd, 4001, len(own), act), engine(nH, nKV, hd, prefix_len, 1, act)
    k, v = fill(eng, 15)
    pk, pv = fill(first, 16)
    for s, rows in enumerate(own):
        poison(eng, s, rows)
    q = torch.randn((len(own), nH * hd), device="cuda").to(act)
    got = eng.decode_shared(0, first, 0, prefix_len, [(s, prefix_len + rows - 1) for s, rows in enumerate(own)], q, own_base=prefix_len)
    eng.sync()
    for s, rows in enumerate(own):
        kk, vv = torch.cat([pk[0], k[s, :rows]]), torch.cat([pv[0], v[s, :rows]])
        want, _, delta = attend(q[s].view(nH, hd), kk, vv)
        close(got[s], want, vv, delta, prefix_len + rows)


def test_long_prefix_in_many_splits():
    eng, first = engine(16, 2, 256, 300, 3, F16), engine(16, 2, 256, 20011, 1, F16)
    k, v = fill(eng, 6)
    pk, pv = fill(first, 7)
    q = torch.randn((3, 4096), device="cuda").half() * 3          # peaked weights
    got = eng.decode_shared(0, first, 0, 20011, [(0, 20011), (1, 20310), (2, 20010)], q, own_base=20011)
    for i, n in enumerate((1, 300, 0)):
        kk, vv = torch.cat([pk[0], k[i, :n]]), torch.cat([pv[0], v[i, :n]])
        want, _, delta = attend(q[i].view(16, 256), kk, vv)
        close(got[i], want, vv, delta, 20011 + n)


@pytest.mark.parametrize("nH,nKV,hd,n,prefix_len", [(24, 4, 256, 11, 9001), (24, 4, 256, 13, 11633), (24, 4, 256, 45, 4878), (16, 2, 256, 5, 16000), (16, 8, 128, 40, 5000), (8, 8, 64, 70, 7000)])
def test_f32_records_of_a_few_tiles(nH, nKV, hd, n, prefix_len):
    # f32 outputs: a unit of many tiles leaves several records, whatever its last one holds.  What the tensor cores' sums lose by rounding
    # towards zero stays below that of 16 tiles: 2^-24 of the running sum at each of 64 additions, half of them at half of it
    eng, first = engine(nH, nKV, hd, 1300, n, F32), engine(nH, nKV, hd, prefix_len, 1, F32)
    k, v = fill(eng, 13)
    pk, pv = fill(first, 14)
    own = [(97 * i * i) % 1301 for i in range(n)]
    q = torch.randn((n, nH * hd), device="cuda")
    got = eng.decode_shared(0, first, 0, prefix_len, [(i, prefix_len - 1 + own[i]) for i in range(n)], q, own_base=prefix_len)
    for i in range(0, n, 3):
        kk, vv = torch.cat([pk[0], k[i, :own[i]]]), torch.cat([pv[0], v[i, :own[i]]])
        want, _, delta = attend(q[i].view(nH, hd), kk, vv)
        close(got[i], want, vv, delta, prefix_len + own[i])
        assert (got[i].double().view(want.shape) - want).norm() <= 3e-6 * want.norm()


def test_rising_scores_move_the_reference_maximum():
    # every tile's maximum passes the last one's by far: each tile rescales what is summed so far
    eng = engine(2, 1, 128, 1000, 1, F32)
    fill(eng, 8, 0.1)
    k = eng.cache(0, "k").view(F16)
    k[0, :, 0] = torch.linspace(-60, 60, 1000, device="cuda").half()
    q = torch.zeros((1, 256), device="cuda")
    q[0, 0], q[0, 128] = 40.0, -40.0
    kk, vv = k[0].view(1000, 1, 128), eng.cache(0, "v").view(F16)[0].view(1000, 1, 128)
    got = eng.decode_shared(0, None, 0, 0, [(0, 999)], q)
    want, _, delta = attend(q.view(2, 128), kk, vv)
    close(got[0], want, vv, delta, 1000)


def test_rows_appended_just_before():
    eng, first = engine(16, 2, 256, 64, 2, F16, max_cols=64), engine(16, 2, 256, 500, 1, F16)
    rot = eng.rotary(n_rot=64, layout="interleaved")
    pk, pv = fill(first, 9)
    x = [torch.randn((2, w), device="cuda").half() for w in (4096, 512, 512)]
    for step in range(30):
        items = [(0, 500 + step, 1), (1, 500 + 2 * step, 1)]
        q = eng.rotary_append(0, rot, items, x[0], x[1] * (step % 7 - 3), x[2] * (step % 5 - 2), rows=[step, 2 * step], q_dtype=F16)
        got = eng.decode_shared(0, first, 0, 500, [(0, 500 + step), (1, 500 + 2 * step)], q, own_base=500)
        n = step + 1
        kk, vv = torch.cat([pk[0], eng.cache(0, "k").view(F16)[0, :n].view(n, 2, 256)]), torch.cat([pv[0], eng.cache(0, "v").view(F16)[0, :n].view(n, 2, 256)])
        want, _, delta = attend(q[0].view(16, 256), kk, vv)
        close(got[0], want, vv, delta, 500 + n)


def test_prefix_appended_just_before():
    # the prefix's own context, and a layer of the same one, write rows that the next call attends
    eng = engine(16, 8, 128, 400, 3, F32, max_cols=512)
    other = engine(16, 8, 128, 400, 1, F32, max_cols=512)
    rot = [e.rotary(n_rot=64) for e in (eng, other)]
    fill(eng, 20)
    q = torch.randn((2, 2048), device="cuda")
    for turn in range(8):
        k, v = [torch.randn((300, 1024), device="cuda") for _ in "kv"]
        for e, r, pre in ((eng, rot[0], None), (other, rot[1], other)):
            e.rotary_append(0, r, [(0, 0, 300)], None, k, v)
            got = eng.decode_shared(0, pre, 0, 300, [(1, 320), (2, 299)], q)
            pk, pv = [e.cache(0, w)[0, :300].view(F16).view(300, 8, 128) for w in "kv"]
            for i, (s, n) in enumerate(((1, 21), (2, 0))):
                ok, ov = [eng.cache(0, w)[s, 300:300 + n].view(F16).view(n, 8, 128) for w in "kv"]
                vv = torch.cat([pv, ov])
                want, _, delta = attend(q[i].view(16, 128), torch.cat([pk, ok]), vv)
                close(got[i], want, vv, delta, 300 + n)


def test_streams_graphs_and_repeats():
    eng, first = engine(24, 4, 256, 300, 3, F32), engine(24, 4, 256, 3000, 1, F32)
    fill(eng, 10); fill(first, 11)
    q = torch.randn((3, 6144), device="cuda")
    call = lambda out=None: eng.decode_shared(0, first, 0, 3000, [(0, 3100), (1, 3299), (2, 2999)], q, out=out, own_base=3000)
    want = call()
    assert all(torch.equal(call(), want) for _ in range(20))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
        call(out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, call()) and not torch.equal(out, want)


def test_refused_calls():
    eng, first = engine(16, 2, 256, 64, 2, F16), engine(16, 2, 256, 100, 2, F16)
    for e in (eng, first):
        fill(e, 12)
    q = torch.zeros((1, 4096), dtype=F16, device="cuda")

    def refused(code=-1, prefix=first, prefix_seq=0, prefix_len=100, items=((0, 100),), q=q, base=100, e=eng, **kw):
        with pytest.raises(PaError) as err:
            e.decode_shared(0, prefix, prefix_seq, prefix_len, list(items), q, own_base=base, **kw)
        assert err.value.code == code

    refused(prefix_seq=2)
    refused(prefix_len=101, items=[(0, 101)], base=101)
    refused(items=[(2, 100)])
    refused(items=[(0, 98)])                                       # inside the prefix
    refused(items=[(0, 164)])                                      # past the layer's rows
    refused(items=[(0, 100)], base=0)                              # ... where rows are positions
    refused(items=[(0, 100)], base=50)
    refused(items=[(0, 2 ** 31 - 1)])
    refused(items=[(0, 100)] * 129, q=torch.zeros((129, 4096), dtype=F16, device="cuda"))
    refused(items=[], q=q[:0])
    refused(q=q.cpu())
    refused(q=q.to(torch.bfloat16))
    refused(q=torch.zeros((1, 4100), dtype=F16, device="cuda")[:, 4:])      # 8-byte alignment
    refused(q=torch.zeros((2, 4096), dtype=F16, device="cuda"))
    refused(q=q, q_head_stride=512)
    refused(gate=torch.zeros((1, 4096), device="cuda"))
    refused(out=torch.zeros((1, 4000), dtype=F16, device="cuda"))
    refused(prefix=engine(16, 8, 256, 100, 1, F16))
    refused(prefix=engine(16, 2, 128, 100, 1, F16))
    refused(-2, prefix=engine(16, 2, 256, 100, 1, F16, kv_format="q8"))
    refused(-2, e=engine(16, 2, 256, 100, 1, F16, kv_format="f32"))
    refused(-2, e=engine(65, 1, 64, 100, 1, F16), prefix=None, prefix_len=0, base=0, q=torch.zeros((1, 65 * 64), dtype=F16, device="cuda"))
    shard = engine(16, 2, 256, 64, 1, F16)
    shard.set_origin(0, 64)
    refused(-2, e=shard)
    eng.decode_shared(0, first, 0, 100, [(0, 100)], q, own_base=100)
    eng.sync()


@pytest.mark.parametrize("nH,nKV,hd,n,prefix_len,own_len", [(16, 8, 128, 128, 33001, 70), (64, 8, 64, 128, 33001, 1), (24, 4, 256, 100, 20000, 300), (16, 2, 256, 128, 200, 9000), (64, 4, 64, 1, 133000, 0),
                                                            (64, 64, 64, 1, 90001, 5)])
def test_f32_sums_stay_short_where_records_run_short(nH, nKV, hd, n, prefix_len, own_len):
    # More rows of more tiles than there are records of 16 or 4 tiles for: what the tensor cores' sums lose by rounding towards zero is still that of
    # at most 24, whatever the length.  At each of 96 additions at most an f32 unit of the running sum, 2^-24 to 2^-23 of it and half of that on
    # average, the running sum 3/4 of the last on average: 96 * 0.75 * (2^-25 to 2^-24), at 1.4 units 2^-24.5 = 3.0e-6
    eng, first = engine(nH, nKV, hd, max(1, own_len), n, F32), engine(nH, nKV, hd, prefix_len, 1, F32)
    k, v = fill(eng, 21)
    pk, pv = fill(first, 22)
    own = [own_len - (i % 7) * (own_len // 9) for i in range(n)]
    g = torch.Generator(device="cuda").manual_seed(23)
    q = torch.empty((n, nH * hd), device="cuda").normal_(generator=g)
    got = eng.decode_shared(0, first, 0, prefix_len, [(i, prefix_len - 1 + own[i]) for i in range(n)], q, own_base=prefix_len)
    for i in sorted({0, n // 3, n // 2, n - 1}):
        kk, vv = torch.cat([pk[0], k[i, :own[i]]]), torch.cat([pv[0], v[i, :own[i]]])
        for h0 in range(0, nH, nH // nKV):                                     # a kv head at a time: the 64-bit values of all of them would take too much room
            h1 = h0 + nH // nKV
            want, _, delta = attend(q[i].view(nH, hd)[h0:h1], kk[:, h0 * nKV // nH:h1 * nKV // nH], vv[:, h0 * nKV // nH:h1 * nKV // nH])
            close(got[i].view(nH, hd)[h0:h1], want, vv, delta, prefix_len + own[i])
            assert (got[i].view(nH, hd)[h0:h1].double() - want).norm() <= 3e-6 * want.norm()


@pytest.mark.parametrize("nH,nKV,hd,n,prefix_len,own_len", [(64, 1, 64, 128, 131072, 0), (64, 1, 64, 128, 300, 60000), (128, 4, 128, 64, 150000, 3), (32, 2, 256, 128, 100003, 0), (24, 4, 256, 128, 66001, 1)])
def test_f16_results_do_not_shrink_with_the_length(nH, nKV, hd, n, prefix_len, own_len):
    # What rounding towards zero takes from every value alike, over the heads of an item so that the roundings to f16 average out: 2^-24 of the running
    # sum at each of 4 additions a tile, 128 tiles (wide units: 8 a tile): at most 2^-15 (2^-14); with the roundings' share, 2^-12 / sqrt(nH * hd) of the
    # norm, four times over
    eng, first = engine(nH, nKV, hd, max(1, own_len), n if own_len else 1, F16), engine(nH, nKV, hd, prefix_len, 1, F16)
    k, v = fill(eng, 26)
    pk, pv = fill(first, 27)
    g = torch.Generator(device="cuda").manual_seed(28)
    q = torch.empty((n, nH * hd), device="cuda").normal_(generator=g).half()
    got = eng.decode_shared(0, first, 0, prefix_len, [(i if own_len else 0, prefix_len - 1 + own_len) for i in range(n)], q, own_base=prefix_len)
    for i in (0, n // 2, n - 1):
        s = i if own_len else 0
        wants = []
        for h0 in range(0, nH, nH // nKV):
            c = h0 * nKV // nH
            kk, vv = torch.cat([pk[0, :, c:c + 1], k[s, :own_len, c:c + 1]]), torch.cat([pv[0, :, c:c + 1], v[s, :own_len, c:c + 1]])
            want, _, delta = attend(q[i].view(nH, hd)[h0:h0 + nH // nKV], kk, vv)
            close(got[i].view(nH, hd)[h0:h0 + nH // nKV], want, vv, delta, prefix_len + own_len)
            wants.append(want)
        want = torch.cat(wants)
        shrunk = 1 - float((got[i].double().view(want.shape) * want).sum() / (want * want).sum())
        assert abs(shrunk) <= (2.0 ** -14 if hd == 256 else 2.0 ** -15) + 4 * 2.0 ** -12 / math.sqrt(nH * hd), shrunk


WIDE = [(16, 2, 17), (16, 2, 32), (16, 2, 100), (24, 4, 22), (24, 4, 43), (64, 1, 3), (10, 2, 33)]      # G = 8, 6, 64 and 5; the last row tile full and not


@pytest.mark.parametrize("nH,nKV,n", WIDE)
@pytest.mark.parametrize("prefix_len", [1, 64, 65, 777, 20011])
@pytest.mark.parametrize("scale", [1.0, 5.0])
def test_wide_units(monkeypatch, nH, nKV, n, prefix_len, scale):
    # 128 query rows a tile wherever they can be, and nowhere: one tile to many splits of many (the rings wrap), a ragged end, flat and peaked weights
    hd, g = 256, torch.Generator(device="cuda").manual_seed(30)
    q, gate = [torch.empty((n, nH * hd), device="cuda").normal_(generator=g).half() * s for s in (scale, 1.0)]
    own = [(37 * i * i) % 130 for i in range(n)]
    got = []
    for wide in "01":
        monkeypatch.setenv("POOLED_ATTN_SHARED_WIDE", wide)
        eng, first = engine(nH, nKV, hd, 131, n, F16), engine(nH, nKV, hd, prefix_len + 70, 2, F16)
        k, v = fill(eng, 31)
        pk, pv = fill(first, 32)
        for s in range(n):
            poison(eng, s, own[s])
        poison(first, 1, prefix_len)
        poison(first, 0, 0)
        out = torch.full((n, nH * hd + 8), 9.0, dtype=F16, device="cuda")
        call = lambda: eng.decode_shared(0, first, 1, prefix_len, [(i, prefix_len - 1 + own[i]) for i in range(n)], q, gate, out=out, own_base=prefix_len)
        call()
        eng.sync()
        assert torch.all(out[:, nH * hd:] == 9.0)
        got.append(out.clone())
        assert all(torch.equal(call(), got[-1]) for _ in range(5))
        for i in range(0, n, 1 if n < 20 else 7):
            kk, vv = torch.cat([pk[1, :prefix_len], k[i, :own[i]]]), torch.cat([pv[1, :prefix_len], v[i, :own[i]]])
            want, _, delta = attend(q[i].view(nH, hd), kk, vv, gate[i].view(nH, hd))
            close(got[-1][i, :nH * hd], want, vv, delta, prefix_len + own[i])
    if prefix_len >= 777:
        assert not torch.equal(*got)                                  # (two ways of summing: both ran)


@pytest.mark.parametrize("nH,nKV,n", [(16, 2, 128), (24, 4, 85)])
def test_wide_units_of_many_tiles_whose_scores_rise(monkeypatch, nH, nKV, n):
    # few records for many rows: units of dozens of tiles, whose every tile passes the last one's maximum by far, for some heads, and falls for others
    monkeypatch.setenv("POOLED_ATTN_SHARED_WIDE", "1")
    hd, rows = 256, 20011
    eng, first = engine(nH, nKV, hd, 64, n, F16), engine(nH, nKV, hd, rows, 1, F16)
    fill(eng, 33)
    pk, pv = fill(first, 34, 0.1)
    first.cache(0, "k").view(F16)[0].view(rows, nKV, hd)[:, :, 0] = torch.linspace(-900, 900, rows, device="cuda").half()[:, None]
    pk[0, :, :, 0] = torch.linspace(-900, 900, rows, device="cuda").half()[:, None]
    q = torch.zeros((n, nH, hd), dtype=F16, device="cuda")
    q[:, 0::3, 0], q[:, 1::3, 0], q[:, :, 1] = 20.0, -20.0, 1.0
    got = eng.decode_shared(0, first, 0, rows, [(i, rows - 1) for i in range(n)], q.view(n, -1), own_base=rows)
    for i in range(0, n, 13):
        want, _, delta = attend(q[i], pk[0], pv[0])
        close(got[i], want, pv[0], delta, rows)


@pytest.mark.parametrize("nH,nKV,n,rows", [(16, 2, 128, 70003), (24, 4, 128, 131075), (64, 2, 128, 40001)])
def test_wide_units_of_several_runs(monkeypatch, nH, nKV, n, rows):
    # units of more than 128 tiles: runs added up in one record, or one after another, under a reference that moves
    monkeypatch.setenv("POOLED_ATTN_SHARED_WIDE", "1")
    hd = 256
    eng, first = engine(nH, nKV, hd, 200, 2, F16), engine(nH, nKV, hd, rows, 1, F16)
    k, v = fill(eng, 35)
    pk, pv = fill(first, 36, 0.1)
    for c in (first.cache(0, "k").view(F16)[0].view(rows, nKV, hd), pk[0]):
        c[:, :, 0] = torch.linspace(-900, 900, rows, device="cuda").half()[:, None]
    g = torch.Generator(device="cuda").manual_seed(37)
    q = torch.empty((n, nH, hd), device="cuda").normal_(generator=g).half()
    q[:, 0::3], q[:, 1::3], q[:, 2::3, 0] = 0.0, 0.0, 0.0
    q[:, 0::3, 0], q[:, 1::3, 0], q[:, :, 1] = 20.0, -20.0, 1.0
    got = eng.decode_shared(0, first, 0, rows, [(i % 2, rows - 1 + (0, 130)[i % 2]) for i in range(n)], q.view(n, -1), own_base=rows)
    for i in range(0, n, 31):
        m = (0, 130)[i % 2]
        for h0 in range(0, nH, nH // nKV):
            c, h1 = h0 * nKV // nH, h0 + nH // nKV
            vv = torch.cat([pv[0, :, c:c + 1], v[i % 2, :m, c:c + 1]])
            want, _, delta = attend(q[i, h0:h1], torch.cat([pk[0, :, c:c + 1], k[i % 2, :m, c:c + 1]]), vv)
            close(got[i].view(nH, hd)[h0:h1], want, vv, delta, rows + m)
            flat = (torch.arange(h0, h1) % 3 == 2).to(want.device)              # weights of all rows alike: the bound of test_f16_results_do_not_shrink_with_the_length
            w, o = want[flat], got[i].view(nH, hd)[h0:h1][flat].double()
            if rows > 60000:
                assert abs(1 - float((o * w).sum() / (w * w).sum())) <= 2.0 ** -14 + 4 * 2.0 ** -12 / math.sqrt(w.numel())
