"""Sums of attention weights (pa_decode_weights) and the eviction by them (pa_evict), against their definitions in 64 bits; and a
cache kept to a budget with a rotation of its own, as an engine would use them together."""
import math

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError
from tests.test_gpu_rotary import frequencies, rotated
from tests.test_gpu_shared import F16, F32, SHAPES, attend, close, engine, fill, poison

pytestmark = pytest.mark.gpu


def tracked(*a, **kw):
    eng = engine(*a, **kw)
    eng.track_weights(0)
    return eng


def check_sums(got, before, adds, delta):
    # a weight: e to the power of a score twice delta off, its exponential and the division by the sum 2^-20; adding: a rounding per term
    want = before.double() + adds
    tol = adds * (2 * delta + 2.0 ** -20) + 2.0 ** -22 * want
    assert torch.all((got.double() - want).abs() <= tol), float(((got.double() - want).abs() / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("nH,nKV,hd", SHAPES)
@pytest.mark.parametrize("act,q_dtype", [(F16, F16), (F32, F32)])
@pytest.mark.parametrize("lens", [[1], [63, 64, 65], [1025, 1, 500], [2000], list(range(1, 40))])
def test_weights_against_64_bits(nH, nKV, hd, act, q_dtype, lens):
    n, G = len(lens), nH // nKV
    eng = tracked(nH, nKV, hd, max(lens) + 5, n + 1, act)
    k, v = fill(eng, 1)
    for s, m in enumerate(lens):
        poison(eng, s + 1, m)
    w0 = torch.rand((n + 1, nKV, max(lens) + 5), device="cuda") * 0.01
    eng.weights(0).copy_(w0)
    q, gate = torch.randn((n, nH * hd), device="cuda").to(q_dtype), torch.randn((n, nH * hd), device="cuda").to(act)
    got = eng.decode_weights(0, [(s + 1, m - 1) for s, m in enumerate(lens)], q, gate)
    eng.sync()
    assert torch.equal(eng.weights(0)[0], w0[0])
    for s, m in enumerate(lens):
        want, p, delta = attend(q[s].view(nH, hd), k[s + 1, :m], v[s + 1, :m], gate[s].view(nH, hd))
        close(got[s], want, v[s + 1, :m], delta, m)
        check_sums(eng.weights(0)[s + 1, :, :m], w0[s + 1, :, :m], p.view(nKV, G, m).sum(1), delta.max())
        assert torch.equal(eng.weights(0)[s + 1, :, m:], w0[s + 1, :, m:])


def test_weights_of_a_prompts_last_tokens():
    # many tokens of one sequence, each with the rows it sees: more scores than the context has room for, and always the same bits
    eng = tracked(16, 2, 256, 1500, 1, F32)
    k, v = fill(eng, 2)
    lens = [1500 - 3 * i for i in range(20)]
    q = torch.randn((20, 4096), device="cuda")
    call = lambda: (eng.clear_weights(0, 0), eng.decode_weights(0, [(0, m - 1) for m in lens], q), eng.weights(0).clone())[1:]
    got, sums = call()
    adds, worst = torch.zeros((2, 1500), dtype=torch.float64, device="cuda"), 0.0
    for i, m in enumerate(lens):
        want, p, delta = attend(q[i].view(16, 256), k[0, :m], v[0, :m])
        close(got[i], want, v[0, :m], delta, m)
        adds[:, :m] += p.view(2, 8, m).sum(1)
        worst = max(worst, float(delta.max()))
    check_sums(sums[0], torch.zeros_like(sums[0]), adds * (1 + 20 * 2.0 ** -24), worst)
    for _ in range(5):
        again = call()
        assert torch.equal(again[0], got) and torch.equal(again[1], sums)


def test_weights_of_repeated_sequences_in_one_launch():
    eng = tracked(24, 4, 256, 400, 5, F16)
    k, v = fill(eng, 3)
    items = [(2, 300), (0, 17), (2, 399), (4, 64), (0, 399), (2, 0)]
    q = torch.randn((6, 6144), device="cuda").half()
    eng.decode_weights(0, items, q)
    adds, worst = torch.zeros((5, 4, 400), dtype=torch.float64, device="cuda"), 0.0
    for i, (s, pos) in enumerate(items):
        _, p, delta = attend(q[i].view(24, 256), k[s, :pos + 1], v[s, :pos + 1])
        adds[s, :, :pos + 1] += p.view(4, 6, pos + 1).sum(1)
        worst = max(worst, float(delta.max()))
    check_sums(eng.weights(0), torch.zeros_like(eng.weights(0)), adds, worst)


def reference_rows(w, n, keep, first, recent):
    """The rows that stay of n, by one kv head's sums w (a list of floats)."""
    if n <= keep:
        return list(range(n))
    order = sorted(range(first, n - recent), key=lambda r: (-math.inf if math.isnan(w[r]) else -w[r], 0 if math.isnan(w[r]) else 1, r))
    return sorted(list(range(first)) + order[:keep - first - recent] + list(range(n - recent, n)))


def check_eviction(eng, items, keep, first, recent):
    """Runs the call and compares caches, sums and lists with the definition, every other row included."""
    c = eng.cfg
    before = [eng.cache(0, w).clone() for w in "kv"]
    w0 = eng.weights(0).clone()
    kept = eng.evict(0, items, keep, n_first=first, n_recent=recent)
    eng.sync()
    want, ws = [b.clone().view(c.n_seqs, c.max_seq, c.n_kv_heads, c.head_dim) for b in before], w0.clone()
    for i, (src, dst, n) in enumerate(items):
        for h in range(c.n_kv_heads):
            rows = reference_rows(w0[src, h, :n].tolist(), n, keep, first, recent)
            assert kept[i, h].tolist() == rows + [-1] * (keep - len(rows)), (i, h)
            at = torch.tensor(rows, dtype=torch.int64, device="cuda")
            for x, b in zip(want, before):
                x[dst, :len(rows), h] = b.view(x.shape)[src, at, h]
            ws[dst, h, :len(rows)] = w0[src, h, at]
            ws[dst, h, len(rows):] = 0.0
    for w, x in zip("kv", want):
        assert torch.equal(eng.cache(0, w), x.view(c.n_seqs, c.max_seq, -1))
    assert torch.equal(torch.nan_to_num(eng.weights(0), 77.0), torch.nan_to_num(ws, 77.0))


@pytest.mark.parametrize("nKV,hd", [(2, 256), (8, 128), (1, 64)])
@pytest.mark.parametrize("rows,keep,first,recent", [(300, 299, 0, 0), (300, 1, 0, 0), (300, 100, 4, 50), (301, 128, 0, 128), (1111, 700, 700, 0), (1111, 64, 32, 32), (2, 1, 0, 1),
                                                    (2500, 2000, 4, 256), (9000, 1024, 16, 100), (8192, 5000, 0, 9), (8193, 8000, 3, 0), (17001, 3000, 1, 1), (40000, 39000, 5, 7)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(nKV, hd, rows, keep, first, recent, in_place):
    eng = tracked(nKV, nKV, hd, rows + 3, 3, F16)
    fill(eng, rows)
    g = torch.Generator(device="cuda").manual_seed(keep)
    eng.weights(0).normal_(generator=g).mul_(2).exp_()
    check_eviction(eng, [(2, 2 if in_place else 0, rows), (1, 1, max(1, rows // 2))], keep, first, recent)


@pytest.mark.parametrize("kind", ["equal", "few_values", "specials", "small_differences"])
@pytest.mark.parametrize("rows", [700, 10000, 33000])
def test_evict_ties_and_odd_values(kind, rows):
    eng = tracked(2, 2, 64, rows, 2, F16)
    fill(eng, 5)
    w = eng.weights(0)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few_values":
        w.copy_(torch.randint(0, 5, w.shape, device="cuda").float())
    elif kind == "specials":
        w.copy_(torch.tensor([0.0, -0.0, math.inf, math.nan, 1e-45, -1.0, -math.inf, 3e38])[torch.randint(0, 8, w.shape)].cuda())
        w.view(torch.int32)[0, 0, 5::50] = -1                          # a NaN of the other sign
    else:
        w.copy_((torch.randint(0, 3000, w.shape, device="cuda") + 0x3f800000).int().view(torch.float32))
    check_eviction(eng, [(0, 0, rows), (1, 1, rows - 31)], rows // 3, 3, 40)


def test_evict_short_sequences_keep_all_and_forks():
    eng = tracked(4, 4, 128, 256, 8, F16)
    fill(eng, 6)
    eng.weights(0).uniform_()
    check_eviction(eng, [(0, 0, 100), (1, 2, 100), (3, 4, 0), (3, 5, 256), (3, 6, 101), (7, 7, 256)], 100, 10, 20)
    check_eviction(eng, [(0, 1, 256)], 256, 0, 0)
    check_eviction(eng, [(0, 0, 256)], 256, 100, 156)
    assert eng.evict(0, [(0, 0, 10)], 5).shape == (1, 4, 5)


@pytest.mark.parametrize("n", [500, 9000])
def test_evict_without_lists(n):
    # without `kept` the lists live in the context's room
    eng = tracked(2, 2, 128, n, 2, F16)
    fill(eng, 7)
    eng.weights(0).uniform_()
    rows = [reference_rows(eng.weights(0)[0, h].tolist(), n, 200, 0, 0) for h in (0, 1)]
    want = torch.stack([eng.cache(0, "k")[0].view(n, 2, 128)[rows[h], h] for h in (0, 1)], 1)
    rc = eng._call.evict(eng._f_evict, eng.layers[0].value, [(0, 1, n)], 200, 0, 0, None, eng._raw_st())
    assert rc == 0 and torch.equal(eng.cache(0, "k")[1, :200].view(200, 2, 128), want)


def test_decode_right_behind_an_eviction():
    # no kernel may fetch rows ahead of the eviction's end: the library's own decode, the shared one and a whole layer call
    eng = tracked(16, 2, 256, 4200, 1, F32)
    q, kv = torch.randn((1, 4096), device="cuda"), torch.randn((1, 512), device="cuda")
    for how in ("decode", "weights", "layer", "append"):
        k, v = fill(eng, 8)
        eng.weights(0).uniform_()
        kept = eng.evict(0, [(0, 0, 4200)], 3900, n_first=1)
        if how == "decode":
            got = eng.decode(0, [(0, 3899, 1)], q)
        elif how == "weights":
            got = eng.decode_weights(0, [(0, 3899)], q)
        elif how == "layer":
            got = eng.encode_layer(0, 3900, q, kv, kv)
        else:
            eng.kv_append(0, 0, 3900, kv, kv)
            got = eng.decode(0, [(0, 3900, 1)], q)
        at = kept[0].long().t()[..., None].expand(-1, -1, 256)
        kk, vv = k[0].gather(0, at), v[0].gather(0, at)
        if how in ("layer", "append"):
            kk, vv = torch.cat([kk, kv.half().view(1, 2, 256)]), torch.cat([vv, kv.half().view(1, 2, 256)])
        want, _, delta = attend(q.view(16, 256), kk, vv)
        close(got[0], want, vv, delta, len(kk))


@pytest.mark.parametrize("act", [F16, F32])
def test_layers_in_turn_behind_evictions_and_turned_caches(act):
    # two layers of one context, each given up rows, its remaining keys turned back by what the rows have moved (in place, in the cache), then
    # whole layer calls: the fused token fetches rows ahead of its own wait, and none of them may be of before
    eng = AttnEngine(AttnConfig(n_heads=16, n_kv_heads=2, head_dim=256, n_rot=64, rope_theta=1e7, max_seq=2100, n_layers=2, act_dtype=act, max_cols=64))
    rot = eng.rotary()
    g = torch.Generator(device="cuda").manual_seed(7)
    new = lambda *s: torch.empty(s, device="cuda").normal_(generator=g)
    for _ in range(6):
        for li in (0, 1):
            for w in "kv":
                eng.cache(li, w).view(F16).copy_(new(1, 2100, 512))
            eng.track_weights(li)
            eng.weights(li).copy_(new(1, 2, 2100).abs())
        before = [[eng.cache(li, w)[0].view(F16).clone().view(2100, 2, 256) for w in "kv"] for li in (0, 1)]
        kept = [eng.evict(li, [(0, 0, 2000)], 1500, n_first=2, n_recent=30) for li in (0, 1)]
        back = torch.full((1500,), -500, dtype=torch.int32, device="cuda")
        q, k, v = new(1, 4096).to(act), new(1, 512).to(act), new(1, 512).to(act)
        for li in (0, 1):
            rows = eng.cache(li, "k")[0, :1500].view(F16)
            rot.apply(rows, 2, positions=back, out=rows)
            got = eng.encode_layer(li, 1500, q, k, v)
            eng.sync()
            at = kept[li][0].long().t()[..., None].expand(-1, -1, 256)
            kk, vv = [x.gather(0, at) for x in before[li]]
            turned, _ = rotated(kk, [-500] * 1500, *frequencies(64, 1e7), "half")
            kk = torch.from_numpy(turned).cuda()
            held = eng.cache(li, "k")[0, :1501].view(F16).view(1501, 2, 256)
            assert torch.all((held[:1500].double() - kk).abs() <= 2.0 ** -10 * kk.abs() + 2.0 ** -18)
            qr, _ = rotated(q.view(1, 16, 256), [1500], *frequencies(64, 1e7), "half")
            want, _, delta = attend(torch.from_numpy(qr[0]).cuda(), held, torch.cat([vv, v.half().view(1, 2, 256)]))
            close(got[0], want, vv, delta, 1501)


def test_streams_and_graphs():
    eng = tracked(16, 8, 128, 1000, 2, F16)
    fill(eng, 9)
    q = torch.randn((2, 2048), device="cuda").half()
    state = [eng.cache(0, "k").clone(), eng.cache(0, "v").clone()]

    def restore():
        eng.cache(0, "k").copy_(state[0]); eng.cache(0, "v").copy_(state[1]); eng.weights(0).zero_()

    def step(out=None):
        o = eng.decode_weights(0, [(0, 999), (1, 700)], q, out=out)
        return o, eng.evict(0, [(0, 0, 1000), (1, 1, 701)], 600, n_first=4, n_recent=64)

    restore()
    want, kept = step()
    caches = [eng.cache(0, w).clone() for w in "kv"]
    side = torch.cuda.Stream()
    restore()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, kept2 = step()
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(kept, kept2) and all(torch.equal(eng.cache(0, w), x) for w, x in zip("kv", caches))
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, kept3 = step(out)
    for _ in range(3):
        restore()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kept, kept3) and all(torch.equal(eng.cache(0, w), x) for w, x in zip("kv", caches))


def test_room_grows_without_moving_what_graphs_use():
    small = AttnEngine(AttnConfig(n_heads=4, n_kv_heads=2, head_dim=128, n_rot=128, rope_theta=1e6, max_seq=64, n_layers=2, act_dtype=F32, rope_mode="none"))
    small.track_weights(0)
    small.track_weights(0)                                             # a second time: nothing
    fill(small, 10)
    q = torch.randn((1, 512), device="cuda")
    out = torch.empty_like(q)
    small.decode_weights(0, [(0, 63)], q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        small.decode_weights(0, [(0, 63)], q, out=out)
    lib, h = small.L, __import__("ctypes").c_void_p()
    small._ck(lib.pa_layer_create(small.ctx, 4, 5000, __import__("ctypes").byref(h)))
    small._ck(lib.pa_layer_track_weights(h))
    small.clear_weights(0, 0)
    graph.replay()
    torch.cuda.synchronize()
    want, p, delta = attend(q.view(4, 128), *[small.cache(0, w)[0].view(F16).view(64, 2, 128) for w in "kv"])
    close(out[0], want, small.cache(0, "v")[0].view(F16), delta, 64)
    check_sums(small.weights(0)[0], torch.zeros((2, 64), device="cuda"), p.view(2, 2, 64).sum(1), delta.max())
    lib.pa_layer_destroy(h)


@pytest.mark.parametrize("act", [F16, F32])
def test_a_cache_kept_to_a_budget(act):
    # a server's loop: a shared prefix elsewhere is not needed here; every conversation appends at its next row, turned to its position by a
    # scaled rotation, sums its weights, and gives up rows whenever the budget is full.  A plain model of the same caches runs along in 64 bits.
    nH, nKV, hd, budget, slack = 8, 2, 128, 40, 9
    eng = AttnEngine(AttnConfig(n_heads=nH, n_kv_heads=nKV, head_dim=hd, n_rot=hd, rope_theta=1e6, max_seq=budget + slack, n_seqs=2, act_dtype=act, max_cols=8))
    eng.track_weights(0)
    scale = dict(scaling="yarn", factor=8.0, original=32)
    rot = eng.rotary(n_rot=64, theta=1e4, layout="interleaved", **scale)
    f, m = frequencies(64, 1e4, "yarn", 8.0, 32)
    K, V = [[torch.zeros((0, nKV, hd), dtype=torch.float64, device="cuda") for _ in range(2)] for _ in "kv"]
    W = [torch.zeros((nKV, 0), dtype=torch.float64, device="cuda") for _ in range(2)]
    used, evictions = [0, 0], 0
    g = torch.Generator(device="cuda").manual_seed(4)
    for step in range(150):
        pos = [step, 1000 + 3 * step]
        x = [torch.empty((2, w * hd), device="cuda").normal_(generator=g).to(act) for w in (nH, nKV, nKV)]
        q = eng.rotary_append(0, rot, [(s, pos[s], 1) for s in (0, 1)], *x, rows=used, q_dtype=act)
        out = eng.decode_weights(0, [(s, used[s]) for s in (0, 1)], q)
        for s in (0, 1):
            # what the caches hold now, in f16, is the plain model's too: its own rotation agrees with it to f16's rounding
            yk, _ = rotated(x[1][s:s + 1].view(1, nKV, hd), pos[s:s + 1], f, m, "interleaved")
            row = eng.cache(0, "k")[s, used[s]].view(F16).view(nKV, hd).double()
            assert torch.all((row - torch.from_numpy(yk[0]).cuda()).abs() <= 2.0 ** -10 * torch.from_numpy(abs(yk[0])).cuda() + 2.0 ** -17)
            K[s], V[s] = torch.cat([K[s], row[None]]), torch.cat([V[s], x[2][s].half().double().view(1, nKV, hd)])
            W[s] = torch.cat([W[s], torch.zeros((nKV, 1), dtype=torch.float64, device="cuda")], 1)
            want, p, delta = attend(q[s].view(nH, hd), K[s], V[s])
            close(out[s], want, V[s], delta, used[s] + 1)
            W[s] += p.view(nKV, nH // nKV, -1).sum(1)
            assert torch.allclose(eng.weights(0)[s, :, :used[s] + 1].double(), W[s], rtol=1e-3, atol=1e-6)
            used[s] += 1
        if used[0] == budget + slack:
            evictions += 1
            rows = [[reference_rows(eng.weights(0)[s, h, :used[s]].tolist(), used[s], budget, 2, 8) for h in range(nKV)] for s in (0, 1)]
            kept = eng.evict(0, [(s, s, used[s]) for s in (0, 1)], budget, n_first=2, n_recent=8)
            assert kept.tolist() == rows
            for s in (0, 1):
                at = torch.tensor(rows[s], device="cuda")
                pick = at.t()[..., None].expand(-1, -1, hd)
                K[s], V[s], W[s] = K[s].gather(0, pick), V[s].gather(0, pick), W[s].gather(1, at)
                assert torch.equal(eng.cache(0, "k")[s, :budget].view(F16).double().view(budget, nKV, hd), K[s])
                used[s] = budget
    assert evictions == 12


def test_refused_calls():
    eng, plain = tracked(16, 2, 256, 64, 4, F16), engine(16, 2, 256, 64, 4, F16)
    fill(eng, 11)
    q = torch.zeros((1, 4096), dtype=F16, device="cuda")

    def refused(f, code=-1):
        with pytest.raises(PaError) as e:
            f()
        assert e.value.code == code

    refused(lambda: plain.decode_weights(0, [(0, 5)], q))
    refused(lambda: plain.weights(0))
    refused(lambda: plain.clear_weights(0, 0))
    refused(lambda: plain.evict(0, [(0, 0, 10)], 5))
    refused(lambda: eng.decode_weights(0, [(0, 64)], q))
    refused(lambda: eng.decode_weights(0, [(4, 5)], q))
    refused(lambda: eng.decode_weights(0, [], q[:0]))
    refused(lambda: eng.decode_weights(0, [(0, 5)], q.float()[:, :4000]))
    refused(lambda: eng.clear_weights(0, 4))
    for items, keep, first, recent in [([(0, 0, 65)], 5, 0, 0), ([(4, 0, 5)], 5, 0, 0), ([(0, 4, 5)], 5, 0, 0), ([(0, 0, 10)], 0, 0, 0), ([(0, 0, 10)], 65, 0, 0), ([(0, 0, 10)], 5, 3, 3),
                                       ([(0, 0, 10)], 5, 2 ** 32 - 1, 2), ([(0, 1, 10), (2, 1, 10)], 5, 0, 0), ([(0, 1, 10), (1, 2, 10)], 5, 0, 0), ([(1, 2, 10), (0, 1, 10)], 5, 0, 0),
                                       ([(0, 0, 10), (0, 1, 10)], 5, 0, 0), ([], 5, 0, 0), ([(0, 0, 10)] * 33, 5, 0, 0)]:
        refused(lambda: eng.evict(0, items, keep, first, recent))
    refused(lambda: engine(16, 2, 256, 64, 1, F16, kv_format="q8").track_weights(0), -2)
    shard = tracked(16, 2, 256, 64, 1, F16)
    shard.set_origin(0, 64)
    refused(lambda: shard.evict(0, [(0, 0, 10)], 5), -2)
    refused(lambda: shard.decode_weights(0, [(0, 70)], q), -2)
    eng.decode_weights(0, [(0, 63)], q)
    eng.sync()


def test_a_budget_past_the_layer_is_refused_ahead_of_its_list():
    eng = tracked(2, 1, 64, 64, 1, F16)
    for keep in (65, 2 ** 31, 2 ** 32 - 1):
        with pytest.raises(PaError) as e:
            eng.evict(0, [(0, 0, 10)] * 32, keep)
        assert e.value.code == -1


def test_layer_call_right_behind_keys_rotated_into_its_cache():
    # keys kept unrotated elsewhere, rotated into the cache of one layer of two at their new places
    eng = AttnEngine(AttnConfig(n_heads=16, n_kv_heads=2, head_dim=256, n_rot=64, rope_theta=1e7, max_seq=1501, n_layers=2, act_dtype=F16, max_cols=64))
    rot = eng.rotary()
    g = torch.Generator(device="cuda").manual_seed(8)
    new = lambda *s: torch.empty(s, device="cuda").normal_(generator=g).half()
    for turn in range(12):
        li = turn % 2
        raw, q, k, v = new(1500, 512), new(1, 4096), new(1, 512), new(1, 512)
        for w in "kv":
            eng.cache(li, w).view(F16).copy_(new(1, 1501, 512))
        rot.apply(raw, 2, pos=0, out=eng.cache(li, "k")[0, :1500].view(F16))
        got = eng.encode_layer(li, 1500, q, k, v)
        eng.sync()
        kk, vv = [eng.cache(li, w)[0].view(F16).view(1501, 2, 256) for w in "kv"]
        assert torch.equal(kk[:1500].reshape(1500, 512), rot.apply(raw, 2))
        qr, _ = rotated(q.view(1, 16, 256), [1500], *frequencies(64, 1e7), "half")
        want, _, delta = attend(torch.from_numpy(qr[0]).cuda(), kk, vv)
        close(got[0], want, vv, delta, 1501)


@pytest.mark.parametrize("nH,nKV,hd,n,rows", [(64, 1, 64, 128, 20000), (24, 4, 256, 60, 9000)])
def test_f32_sums_stay_short_where_records_run_short(nH, nKV, hd, n, rows):
    # as in test_gpu_shared: no more than 24 tiles by the tensor cores alone, in batches that have no room for as many records
    eng = tracked(nH, nKV, hd, rows, n, F32)
    k, v = fill(eng, 24)
    g = torch.Generator(device="cuda").manual_seed(25)
    q = torch.empty((n, nH * hd), device="cuda").normal_(generator=g)
    lens = [rows - 61 * i for i in range(n)]
    got = eng.decode_weights(0, [(i, m - 1) for i, m in enumerate(lens)], q)
    for i in (0, n // 2, n - 1):
        m = lens[i]
        want, p, delta = attend(q[i].view(nH, hd), k[i, :m], v[i, :m])
        close(got[i], want, v[i, :m], delta, m)
        check_sums(eng.weights(0)[i, :, :m], torch.zeros((nKV, m), device="cuda"), p.view(nKV, nH // nKV, m).sum(1), delta.max())
        assert (got[i].double().view(want.shape) - want).norm() <= 3e-6 * want.norm()
