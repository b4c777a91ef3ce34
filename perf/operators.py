"""Performance cases of the operators around long and many conversations: rotary positions of other layouts and scalings,
attention of a batch behind one shared prefix, and caches that keep the rows attention used most.

A case is one pass through one operator, as an engine calls it for one layer:

  rotate   q (or k) of some columns turned to their positions (`Rotary.apply`)
  append   the front of a layer call: q rotated, k rotated and v converted into the f16 caches (`rotary_append`)
  shared   one token of each of several conversations that begin with the same rows (`decode_shared`)
  weigh    one token of each of several conversations, and how much every cached row was attended (`decode_weights`)
  evict    the rows with the largest sums kept and moved together (`evict`)

Model shapes are the repository's own: "small" 16 q / 8 kv heads x 128, rotated in full; "moe" 16 / 2 x 256 with 64
rotated dims; "hybrid" 24 / 4 x 256 with 64 rotated dims.  The two last have a sigmoid output gate, which their q
projection delivers interleaved with q.
"""
from __future__ import annotations

import math

import torch

own = False     # False: plain torch operations in 32 bits; True: the library's calls

SHAPES = {
    "small": dict(nH=16, nKV=8, hd=128, n_rot=128, theta=1e6, gated=False),
    "moe": dict(nH=16, nKV=2, hd=256, n_rot=64, theta=1e7, gated=True),
    "hybrid": dict(nH=24, nKV=4, hd=256, n_rot=64, theta=1e7, gated=True),
}
ACT = {"f16": torch.float16, "f32": torch.float32}
ORIGINAL, FACTOR = 8192, 4.0                    # a model trained at 8192 positions, stretched to 32768
BETA_FAST, BETA_SLOW, HIGH, LOW = 32.0, 1.0, 4.0, 1.0


def listed():
    return [
        # one token's q in a decode loop: a launch with next to nothing to do
        dict(name="rotate_token", kind="rotate", model="moe", cols=1, top=20000, act="f16", layout="half", scaling="yarn", ragged=False),
        # q of a long prompt, neighbouring dims paired, an eighth of the heads' dims rotated: all of q is read and written
        dict(name="rotate_prompt_8k", kind="rotate", model="hybrid", cols=8192, top=8192, act="f16", layout="interleaved", scaling="linear", ragged=False),
        # tokens of many conversations packed into one buffer, each at a position of its own
        dict(name="rotate_packed_999", kind="rotate", model="small", cols=999, top=131072, act="f32", layout="half", scaling="ntk", ragged=True),
        # thirteen conversations, a token each, into caches that no longer hold every position
        dict(name="append_batch_13", kind="append", model="moe", seqs=13, cols=1, top=65536, act="f16", layout="interleaved", scaling="yarn"),
        # a document of no round length
        dict(name="append_prompt_3k", kind="append", model="small", seqs=1, cols=2999, top=2999, act="f16", layout="half", scaling="bands"),
        # two answers sampled from one short question
        dict(name="shared_2_short", kind="shared", model="small", seqs=2, prefix=301, own=17, act="f16"),
        # a server's long system prompt, 32 users with little of their own yet
        dict(name="shared_32_32k", kind="shared", model="moe", seqs=32, prefix=32768, own=777, act="f16"),
        # a document that eleven questions are asked of, f32 activations
        dict(name="shared_11_9k", kind="shared", model="hybrid", seqs=11, prefix=9001, own=2100, act="f32"),
        # a token of one conversation, its weights summed for the next eviction
        dict(name="weigh_1_4k", kind="weigh", model="moe", seqs=1, ctx=4099, act="f16"),
        # a batch of conversations of every length under a cache budget
        dict(name="weigh_8_16k", kind="weigh", model="hybrid", seqs=8, ctx=16384, act="f32"),
        # a conversation that has filled its budget gives up a fifth of its rows
        dict(name="evict_1_2500", kind="evict", model="small", seqs=1, rows=2500, keep=2000, first=4, recent=256),
        # long prompts of four conversations brought down to an eighth each
        dict(name="evict_4_32k", kind="evict", model="moe", seqs=4, rows=32768, keep=4096, first=16, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "shared", "shared", "weigh", "evict"])
    model = rng.choice(["small", "moe", "hybrid"])
    turn = dict(act=rng.choice(["f16", "f32"]), layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]))
    if kind == "rotate":
        cols = _log(rng, 1, 4096)
        return dict(kind=kind, model=model, cols=cols, top=max(cols, _log(rng, 64, 131072)), ragged=rng.random() < 0.5, **turn)
    if kind == "append":
        seqs = rng.choice([1, rng.randint(2, 32)])
        cols = _log(rng, 1, 4096) if seqs == 1 else 1
        return dict(kind=kind, model=model, seqs=seqs, cols=cols, top=max(cols, _log(rng, 64, 131072)), **turn)
    if kind == "shared":
        seqs = _log(rng, 1, 48)
        prefix = _log(rng, 60, min(65536, 1048576 // seqs) if model == "moe" else min(32768, 524288 // seqs))
        return dict(kind=kind, model=model, seqs=seqs, prefix=prefix, own=_log(rng, 1, max(2, min(4096, 24576 // seqs))), act=turn["act"])
    if kind == "weigh":
        seqs = _log(rng, 1, 16)
        return dict(kind=kind, model=model, seqs=seqs, ctx=_log(rng, 16, min(32768, 65536 // seqs)), act=turn["act"])
    seqs = _log(rng, 1, 6)
    rows = _log(rng, 200, 32768 // seqs)
    keep = max(32, int(rows * rng.uniform(0.1, 0.95)))
    return dict(kind=kind, model=model, seqs=seqs, rows=rows, keep=keep, first=rng.choice([0, 1, 4, 16]), recent=rng.choice([0, 1, keep // 8, keep // 3]))


# ---- sizes ----

def _lengths(n, top, share=16.0):
    """Lengths of n conversations, spread over a factor of `share` below the longest, in no order."""
    return [top if i == 0 else max(1, int(top * share ** -math.modf(0.6180339887 * i)[0])) for i in range(n)]


def _rows(case):
    """Rows of each conversation before an eviction: the last one may be short of the budget."""
    return _lengths(case["seqs"], case["rows"], 4.0)


def work(case):
    s = SHAPES[case["model"]]
    nH, nKV, hd = s["nH"], s["nKV"], s["hd"]
    q_dim, kv_dim, es = nH * hd, nKV * hd, 2 if case.get("act") == "f16" else 4
    row = 4 * kv_dim                                                     # K and V of one cached row
    if case["kind"] == "rotate":
        return {"bytes": 2 * case["cols"] * q_dim * es, "flops": 3 * case["cols"] * nH * s["n_rot"]}
    if case["kind"] == "append":
        n = case["seqs"] * case["cols"]
        return {"bytes": n * (2 * q_dim * es + 2 * kv_dim * es + row), "flops": 3 * n * (nH + nKV) * s["n_rot"]}
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in _rows(case))
        sums = 4 * nKV * (sum(_rows(case)) + case["seqs"] * case["rows"])    # read of the old rows, written of the new ones
        return {"bytes": sums + kept * (2 * row + 4 * nKV), "flops": nKV * sum(_rows(case))}
    acts = case["seqs"] * q_dim * es * (3 if s["gated"] else 2)
    if case["kind"] == "shared":
        own_rows = sum(_lengths(case["seqs"], case["own"]))
        return {"bytes": (case["prefix"] + own_rows) * row + acts, "flops": 4 * q_dim * (case["seqs"] * case["prefix"] + own_rows)}
    rows = sum(_lengths(case["seqs"], case["ctx"]))
    return {"bytes": rows * (row + 8 * nKV) + acts, "flops": (4 * q_dim + 2 * nH) * rows}


# ---- state ----

def _cache(g, dev, s, seqs, rows):
    """K and V of `seqs` caches of `rows` rows: keys with a few outlier channels per head, as real ones have, and normal values."""
    kv = [torch.empty((seqs, rows, s["nKV"], s["hd"]), dtype=torch.float16, device=dev).normal_(generator=g) for _ in "kv"]
    kv[0][..., 5::61] *= 3.0
    return [x.view(seqs, rows, -1) for x in kv]


def _engine(s, act, seqs, rows, cols, kv=None):
    """The handle that an engine keeps for a layer, with these rows in its caches."""
    from pooled_b200 import AttnConfig, AttnEngine
    dev = torch.cuda.current_device()
    eng = AttnEngine(AttnConfig(n_heads=s["nH"], n_kv_heads=s["nKV"], head_dim=s["hd"], n_rot=s["n_rot"], rope_theta=s["theta"], max_seq=rows, n_seqs=seqs,
                                act_dtype=act, max_cols=max(8, cols)), device=dev)
    for which, x in zip("kv", kv or ()):
        eng.cache(0, which).copy_(x.view(torch.int16))
    return eng


def _rotary(eng, case):
    s = SHAPES[case["model"]]
    more = {"yarn": dict(beta_fast=BETA_FAST, beta_slow=BETA_SLOW), "bands": dict(high=HIGH, low=LOW)}.get(case["scaling"], {})
    return eng.rotary(n_rot=s["n_rot"], theta=s["theta"], layout=case["layout"], scaling=case["scaling"], factor=FACTOR, original=ORIGINAL, **more)


def _view(eng, which, *at):
    """Rows of a cache as f16, with the engine that owns them."""
    t = eng.cache(0, which)[at].view(torch.float16)
    t.engine = eng
    return t


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    s, kind = SHAPES[case["model"]], case["kind"]
    nH, nKV, hd = s["nH"], s["nKV"], s["hd"]
    act = ACT[case.get("act", "f16")]
    new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev).normal_(generator=g).to(act)
    wide = 2 * hd if s["gated"] else hd                                  # gated: [q of a head, gate of a head] per head
    st = {"case": case, "s": s, "wide": wide}
    if kind in ("rotate", "append"):
        cols = case["cols"] * case.get("seqs", 1)
        st["q"] = new(cols, nH * wide)
        start = int(torch.randint(0, case["top"] - case["cols"] + 1, (1,), generator=g, device=dev))
        if kind == "rotate":
            st["pos"] = start
            st["positions"] = torch.randint(0, case["top"], (cols,), generator=g, device=dev, dtype=torch.int32) if case["ragged"] else None
            st["columns"] = st["positions"] if case["ragged"] else torch.arange(start, start + cols, device=dev, dtype=torch.int32)
            if own:
                st["eng"] = _engine(s, act, 1, 8, cols)
                st["rot"] = _rotary(st["eng"], case)
            return st
        st["k"], st["v"] = new(cols, nKV * hd), new(cols, nKV * hd)
        places = torch.randint(0, case["top"], (case["seqs"],), generator=g, device=dev).tolist() if case["seqs"] > 1 else [start]
        st["items"] = [(i, p, case["cols"]) for i, p in enumerate(places)]
        st["rows"] = [(3 * i) % 8 for i in range(case["seqs"])]          # rows and positions have parted: the caches keep what was used
        st["columns"] = torch.tensor([p + c for _, p, n in st["items"] for c in range(n)], dtype=torch.int32, device=dev)
        st["at"] = torch.tensor([i * (case["cols"] + 8) + r + c for (i, _, n), r in zip(st["items"], st["rows"]) for c in range(n)], device=dev)
        st["kv"] = [torch.zeros((case["seqs"], case["cols"] + 8, nKV * hd), dtype=torch.float16, device=dev) for _ in "kv"]
        if own:
            st["eng"] = _engine(s, act, case["seqs"], case["cols"] + 8, cols, st["kv"])
            st["rot"] = _rotary(st["eng"], case)
        return st
    if kind == "evict":
        n, rows = case["seqs"], _rows(case)
        st["kv"] = _cache(g, dev, s, 2 * n, case["rows"])                # the second half receives what is kept: the conversations stay
        # sums as softmax weights leave them: most rows little, a few much, the first rows most
        w = torch.empty((2 * n, nKV, case["rows"]), dtype=torch.float32, device=dev).normal_(generator=g).mul_(1.7).exp_()
        w[:, :, :4] *= 50.0
        st["w"] = w
        st["items"] = [(i, n + i, r) for i, r in enumerate(rows)]
        st["n_rows"] = torch.tensor(rows, device=dev)
        if own:
            st["eng"] = _engine(s, act, 2 * n, case["rows"], 1, st["kv"])
            st["eng"].track_weights(0)
            st["eng"].weights(0).copy_(w)
        return st
    st["q"] = new(case["seqs"], nH * wide)
    st["gate"] = st["q"][:, hd:] if s["gated"] else None
    if kind == "shared":
        lens = _lengths(case["seqs"], case["own"])
        st["prefix"] = _cache(g, dev, s, 1, case["prefix"])
        st["kv"] = _cache(g, dev, s, case["seqs"], max(lens))
        st["items"] = [(i, case["prefix"] + n - 1) for i, n in enumerate(lens)]
        if own:
            st["eng"] = _engine(s, act, case["seqs"], max(lens), case["seqs"], st["kv"])
            st["first"] = _engine(s, act, 1, case["prefix"], 8, st["prefix"])
    else:
        lens = _lengths(case["seqs"], case["ctx"])
        st["kv"] = _cache(g, dev, s, case["seqs"], max(lens))
        st["items"] = [(i, n - 1) for i, n in enumerate(lens)]
        st["w"] = torch.rand((case["seqs"], nKV, max(lens)), generator=g, device=dev) * (8.0 / max(lens))     # of a few tokens before
        if own:
            st["eng"] = _engine(s, act, case["seqs"], max(lens), case["seqs"], st["kv"])
            st["eng"].track_weights(0)
            st["eng"].weights(0).copy_(st["w"])
    st["lens"] = torch.tensor(lens, device=dev)
    return st


# ---- the plain forms ----

def _frequencies(case, dev):
    """Turns of each rotated pair per position (float64), and the factor on cos and sin."""
    s = SHAPES[case["model"]]
    n, theta, kind = s["n_rot"], s["theta"], case["scaling"]
    if kind == "ntk":
        theta = theta * FACTOR ** (n / (n - 2))
    i = torch.arange(n // 2, dtype=torch.float64, device=dev)
    f = theta ** (-2.0 * i / n)
    if kind == "linear":
        return f / FACTOR, 1.0
    if kind == "yarn":
        at = lambda turns: n * math.log(ORIGINAL / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))
        lo, hi = max(math.floor(at(BETA_FAST)), 0), min(math.ceil(at(BETA_SLOW)), n - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f * (1.0 - ramp) + f / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1.0
    if kind == "bands":
        turns = ORIGINAL * f / (2.0 * math.pi)                           # turns of a pair over the trained length
        mix = ((turns - LOW) / (HIGH - LOW)).clamp(0.0, 1.0)
        return f * mix + f / FACTOR * (1.0 - mix), 1.0
    return f, 1.0


def _turn(case, x, heads, columns, wide):
    """x [cols, heads * wide] -> [cols, heads, hd] in 32 bits, rotated."""
    s = SHAPES[case["model"]]
    n = s["n_rot"]
    f, m = _frequencies(case, x.device)
    angle = columns.double()[:, None] * f
    cos, sin = [(m * t).float()[:, None] for t in (angle.cos(), angle.sin())]
    x = x.view(x.shape[0], heads, wide)[..., :s["hd"]].float()
    if case["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., n:]], -1)


def _heads(st, x):
    return x.view(*x.shape[:-1], st["s"]["nKV"], st["s"]["hd"]).float()


def _finish(st, o, act):
    """[seqs, nKV, G, hd] -> gated, [seqs, nH * hd] of the activations' type."""
    n = o.shape[0]
    o = o.reshape(n, st["s"]["nH"], st["s"]["hd"])
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["q"].view(n, st["s"]["nH"], -1)[..., st["s"]["hd"]:].float())
    return o.reshape(n, -1).to(act)


def _plain(st):
    case, s, kind = st["case"], st["s"], st["case"]["kind"]
    nH, nKV, hd = s["nH"], s["nKV"], s["hd"]
    act = ACT[case.get("act", "f16")]
    if kind == "rotate":
        return _turn(case, st["q"], nH, st["columns"], st["wide"]).flatten(1).to(act)
    if kind == "append":
        q = _turn(case, st["q"], nH, st["columns"], st["wide"]).flatten(1).to(act)
        st["kv"][0].view(-1, nKV * hd)[st["at"]] = _turn(case, st["k"], nKV, st["columns"], hd).flatten(1).half()
        st["kv"][1].view(-1, nKV * hd)[st["at"]] = st["v"].half()
        return q, st["kv"][0], st["kv"][1]
    if kind == "evict":
        n, keep, first, recent = case["seqs"], case["keep"], case["first"], case["recent"]
        r = torch.arange(case["rows"], device=st["w"].device)
        rows = st["n_rows"][:, None, None]
        w = st["w"][:n]
        always = (r < first) | (r >= rows - recent)
        key = torch.where(r < rows, torch.where(always, math.inf, w), -1.0)      # sums are not negative
        order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
        order = torch.where(order < rows, order, case["rows"]).sort(-1).values   # the rows that stay, in their order; none last
        kept = torch.where(order < rows, order, -1).to(torch.int32)
        at = order.clamp(max=case["rows"] - 1)
        live = kept >= 0
        st["w"][n:, :, :] = 0.0
        st["w"][n:, :, :keep] = torch.where(live, w.gather(-1, at), 0.0)
        for x in st["kv"]:
            head = x.view(2 * n, case["rows"], nKV, hd)
            move = head[:n].gather(1, at.transpose(1, 2)[..., None].expand(-1, -1, -1, hd))
            head[n:, :keep] = torch.where(live.transpose(1, 2)[..., None], move, head[n:, :keep])
        return kept, st["kv"][0][n:, :keep], st["kv"][1][n:, :keep], st["w"][n:]
    q = st["q"].view(case["seqs"], nKV, nH // nKV, -1)[..., :hd].float() / math.sqrt(hd)
    k, v = _heads(st, st["kv"][0]), _heads(st, st["kv"][1])
    seen = torch.arange(k.shape[1], device=k.device) < st["lens"][:, None]
    sc = torch.einsum("bkgd,brkd->bkgr", q, k).masked_fill_(~seen[:, None, None], -math.inf)
    if kind == "shared":
        pk, pv = _heads(st, st["prefix"][0][0]), _heads(st, st["prefix"][1][0])
        sp = torch.einsum("bkgd,rkd->bkgr", q, pk)
        m = torch.maximum(sc.amax(-1), sp.amax(-1))[..., None]
        e, ep = (sc - m).exp_(), (sp - m).exp_()
        o = torch.einsum("bkgr,brkd->bkgd", e, v) + torch.einsum("bkgr,rkd->bkgd", ep, pv)
        return _finish(st, o / (e.sum(-1) + ep.sum(-1))[..., None], act)
    e = (sc - sc.amax(-1, keepdim=True)).exp_()
    p = e / e.sum(-1, keepdim=True)
    st["w"] += p.sum(2)
    return _finish(st, torch.einsum("bkgr,brkd->bkgd", p, v), act), st["w"]


# ---- the library's calls ----

def run(st):
    if not own:
        return _plain(st)
    case, s, kind, eng = st["case"], st["s"], st["case"]["kind"], st["eng"]
    if kind == "rotate":
        return st["rot"].apply(st["q"], s["nH"], pos=st["pos"], positions=st["positions"], head_stride=st["wide"])
    if kind == "append":
        q = eng.rotary_append(0, st["rot"], st["items"], st["q"], st["k"], st["v"], rows=st["rows"], q_head_stride=st["wide"], q_dtype=st["q"].dtype)
        return q, _view(eng, "k", slice(None)), _view(eng, "v", slice(None))
    if kind == "shared":
        return eng.decode_shared(0, st["first"], 0, case["prefix"], st["items"], st["q"], st["gate"], own_base=case["prefix"], q_head_stride=st["wide"],
                                 gate_head_stride=st["wide"])
    if kind == "weigh":
        o = eng.decode_weights(0, st["items"], st["q"], st["gate"], q_head_stride=st["wide"], gate_head_stride=st["wide"])
        w = eng.weights(0)
        w.engine = eng
        return o, w
    n, keep = case["seqs"], case["keep"]
    kept = eng.evict(0, st["items"], keep, n_first=case["first"], n_recent=case["recent"])
    w = eng.weights(0)[n:]
    w.engine = eng
    return kept, _view(eng, "k", slice(n, None), slice(None, keep)), _view(eng, "v", slice(n, None), slice(None, keep)), w


# ---- the definitions in 64 bits ----

def _exact_rotation(case, x, heads, wide, positions):
    s = SHAPES[case["model"]]
    n, hd, base, m = s["n_rot"], s["hd"], s["theta"], 1.0
    freq = []
    if case["scaling"] == "ntk":
        base *= math.exp(math.log(FACTOR) * n / (n - 2))
    dim_of = lambda turns: 0.5 * n * math.log(ORIGINAL / (2.0 * math.pi * turns)) / math.log(base)
    for i in range(n // 2):
        f = math.pow(base, -2.0 * i / n)
        wave = 2.0 * math.pi / f
        if case["scaling"] == "linear":
            f = f / FACTOR
        elif case["scaling"] == "yarn":
            lo, hi = max(0, math.floor(dim_of(BETA_FAST))), min(n - 1, math.ceil(dim_of(BETA_SLOW)))
            t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f, m = (1.0 - t) * f + t * f / FACTOR, 1.0 + 0.1 * math.log(FACTOR)
        elif case["scaling"] == "bands":
            if wave > ORIGINAL / LOW:
                f = f / FACTOR
            elif wave >= ORIGINAL / HIGH:
                t = (ORIGINAL / wave - LOW) / (HIGH - LOW)
                f = (1.0 - t) * f / FACTOR + t * f
        freq.append(f)
    z = torch.polar(torch.full((len(positions), 1, n // 2), m, dtype=torch.float64, device=x.device),
                    positions.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device))
    y = x.double().view(len(positions), heads, wide)[:, :, :hd].clone()
    pair = [slice(0, n // 2), slice(n // 2, n)] if case["layout"] == "half" else [slice(0, n, 2), slice(1, n, 2)]
    turned = torch.complex(y[..., pair[0]].contiguous(), y[..., pair[1]].contiguous()) * z
    y[..., pair[0]], y[..., pair[1]] = turned.real, turned.imag
    return y.reshape(len(positions), heads * hd)


def exact(case, seed):
    st = prepare(case, seed)
    s, kind = st["s"], case["kind"]
    nH, nKV, hd, G = s["nH"], s["nKV"], s["hd"], s["nH"] // s["nKV"]
    if kind == "rotate":
        return _exact_rotation(case, st["q"], nH, st["wide"], st["columns"])
    if kind == "append":
        kv = [x.double() for x in st["kv"]]
        kv[0].view(-1, nKV * hd)[st["at"]] = _exact_rotation(case, st["k"], nKV, hd, st["columns"])
        kv[1].view(-1, nKV * hd)[st["at"]] = st["v"].double()
        return _exact_rotation(case, st["q"], nH, st["wide"], st["columns"]), kv[0], kv[1]
    if kind == "evict":
        return None                                                      # whole values and copies: nothing is computed
    out = torch.empty((case["seqs"], nH, hd), dtype=torch.float64, device=st["q"].device)
    sums = st["w"].double() if kind == "weigh" else None
    q = st["q"].view(case["seqs"], nH, st["wide"])
    for i, n in enumerate(st["lens"].tolist()):                          # one conversation and head after another
        for h in range(nH):
            cut = slice(h // G * hd, (h // G + 1) * hd)
            k, v = [x[i, :n, cut] for x in st["kv"]]
            if kind == "shared":
                k, v = [torch.cat([a[0, :, cut], b]) for a, b in zip(st["prefix"], (k, v))]
            p = torch.softmax(k.double() @ q[i, h, :hd].double() / math.sqrt(hd), 0)
            out[i, h] = p @ v.double()
            if sums is not None:
                sums[i, h // G, :n] += p
            if s["gated"]:
                out[i, h] /= 1.0 + torch.exp(-q[i, h, hd:].double())
    out = out.reshape(case["seqs"], nH * hd)
    return out if sums is None else (out, sums)
