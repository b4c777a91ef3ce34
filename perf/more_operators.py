"""Performance cases of the operators around drafted trees, images and moved caches: attention for trees of drafted tokens,
rotary positions with several axes, and rows of caches copied, forked and moved together.

A case is one pass through one operator, as an engine calls it:

  tree   the tokens of a drafted tree of each of several conversations against the cache and their ancestors (`decode_tree`)
  turn   q of some columns turned to positions of several axes (`Rotary.apply`)
  lay    the front of a layer call at positions that the device holds: q rotated, k rotated and v converted into the f16
         caches (`rotary_append`)
  move   rows of the K and V caches of several layers moved in one call (`move`): the accepted path of drafted trees ("accept"),
         one prompt given to many conversations ("fork"), the middle of a conversation given up ("slide"), conversations
         copied ("copy")

Model shapes are the repository's own: "small" 16 q / 8 kv heads x 128, rotated in full; "moe" 16 / 2 x 256 with 64
rotated dims; "hybrid" 24 / 4 x 256 with 64 rotated dims.  The two last have a sigmoid output gate, which their q
projection delivers interleaved with q.
"""
from __future__ import annotations

import math
import random

import torch

own = False     # False: plain torch operations in 32 bits; True: the library's calls

SHAPES = {
    "small": dict(nH=16, nKV=8, hd=128, n_rot=128, theta=1e6, gated=False),
    "moe": dict(nH=16, nKV=2, hd=256, n_rot=64, theta=1e7, gated=True),
    "hybrid": dict(nH=24, nKV=4, hd=256, n_rot=64, theta=1e7, gated=True),
}
ACT = {"f16": torch.float16, "f32": torch.float32}
#: pairs of every axis: time, height and width share out the rotated pairs, height and width halve them
PAIRS = {("small", 3): (24, 20, 20), ("moe", 3): (12, 10, 10), ("hybrid", 3): (12, 10, 10), ("small", 2): (32, 32), ("moe", 2): (16, 16), ("hybrid", 2): (16, 16)}


def listed():
    return [
        # eight drafts behind a short question, small model: latency is all there is
        dict(name="tree_8_short", kind="tree", model="small", seqs=1, nodes=8, reach=4, ctx=301, act="f16"),
        # a wide tree of drafts deep in a long conversation
        dict(name="tree_64_32k", kind="tree", model="moe", seqs=1, nodes=64, reach=12, ctx=32768, act="f16"),
        # six conversations of every length, a tree each, f32 activations
        dict(name="tree_6x26_9k", kind="tree", model="hybrid", seqs=6, nodes=26, reach=8, ctx=9001, act="f32"),
        # a server's batch of drafted trees
        dict(name="tree_16x60_4k", kind="tree", model="small", seqs=16, nodes=60, reach=10, ctx=4003, act="f16"),
        # one token's q at its time, height and width
        dict(name="turn_token", kind="turn", model="moe", cols=1, axes=3, order="cycled", act="f16"),
        # the patches of a picture at their height and width, each axis with frequencies of its own, f32
        dict(name="turn_patches_4k", kind="turn", model="small", cols=4001, axes=2, order="own", act="f32"),
        # a prompt that is mostly pictures: time, height and width
        dict(name="lay_pictures_8k", kind="lay", model="hybrid", seqs=1, cols=8192, axes=3, order="cycled", act="f16"),
        # drafted trees of a batch into the cache: every node at its depth
        dict(name="lay_trees_16x60", kind="lay", model="small", seqs=16, cols=60, axes=1, order="blocks", act="f16"),
        # the accepted paths of eight trees moved together in every layer
        dict(name="move_accept_8", kind="move", form="accept", model="small", kv="f16", layers=8, seqs=8, rows=400, nodes=60),
        # a prompt that seven answers are drawn from
        dict(name="move_fork_7", kind="move", form="fork", model="moe", kv="f16", layers=2, seqs=7, rows=8000, nodes=0),
        # the oldest part of two long conversations given up behind their first rows: what follows moves down over it
        dict(name="move_slide_2", kind="move", form="slide", model="hybrid", kv="f16", layers=1, seqs=2, rows=16001, nodes=0),
        # conversations of every length copied, int8 caches and their scales
        dict(name="move_copy_q8", kind="move", form="copy", model="moe", kv="q8", layers=4, seqs=3, rows=12345, nodes=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "turn", "lay", "move", "move"])
    model, act = rng.choice(["small", "moe", "hybrid"]), rng.choice(["f16", "f32"])
    if kind == "tree":
        seqs, nodes = _log(rng, 1, 16), _log(rng, 1, 64)
        ctx = _log(rng, 1, max(300, min(32768, 2097152 // (seqs * nodes))))
        return dict(kind=kind, model=model, seqs=seqs, nodes=nodes, reach=rng.choice([1, 3, 8, 20]), ctx=ctx, act=act)
    if kind == "turn":
        axes = rng.choice([2, 3])
        return dict(kind=kind, model=model, cols=_log(rng, 1, 4096), axes=axes, order=rng.choice(["blocks", "cycled"] if axes == 3 else ["blocks", "own"]), act=act)
    if kind == "lay":
        axes = rng.choice([1, 3])
        seqs = rng.choice([1, rng.randint(2, 16)])
        return dict(kind=kind, model=model, seqs=seqs, cols=_log(rng, 1, 4096 if seqs == 1 else 64), axes=axes,
                    order=rng.choice(["blocks", "cycled"]) if axes == 3 else "blocks", act=act)
    form = rng.choice(["accept", "fork", "slide", "copy"])
    kv, layers, seqs = rng.choice(["f16", "f16", "q8", "f32"]), rng.choice([1, 2, 8]), _log(rng, 1, 8)
    rows = _log(rng, 70, max(200, min(16384, 65536 // (seqs * layers))))
    return dict(kind=kind, form=form, model=model, kv=kv, layers=layers, seqs=seqs, rows=rows, nodes=min(64, rows // 2) if form == "accept" else 0)


# ---- sizes ----

def _lengths(n, top, share=16.0):
    """Lengths of n conversations, spread over a factor of `share` below the longest, in no order."""
    return [top if i == 0 else max(1, int(top * share ** -math.modf(0.6180339887 * i)[0])) for i in range(n)]


def _slide(rows):
    """First row that stays behind, the row from which on everything moves there, and how many rows that are."""
    keep, at = min(64, rows // 4), min(64, rows // 4) + max(1, rows // 8)
    return keep, at, rows - at


def work(case):
    s = SHAPES[case["model"]]
    nH, nKV, hd = s["nH"], s["nKV"], s["hd"]
    q_dim, kv_dim, es = nH * hd, nKV * hd, 2 if case.get("act") == "f16" else 4
    if case["kind"] == "tree":
        n = case["nodes"]
        lens = _lengths(case["seqs"], case["ctx"])
        seen = n * sum(lens) + case["seqs"] * n * (1 + n / (case["reach"] + 1))      # rows that the tokens attend, their ancestors about
        return {"bytes": (sum(lens) + case["seqs"] * n) * 4 * kv_dim + case["seqs"] * n * (q_dim * es * (3 if s["gated"] else 2) + 4), "flops": 4 * q_dim * seen}
    if case["kind"] == "turn":
        return {"bytes": case["cols"] * (2 * q_dim * es + 4 * case["axes"]), "flops": 3 * case["cols"] * nH * s["n_rot"]}
    if case["kind"] == "lay":
        n = case["seqs"] * case["cols"]
        return {"bytes": n * (2 * q_dim * es + 2 * kv_dim * es + 4 * kv_dim + 4 * case["axes"]), "flops": 3 * n * (nH + nKV) * s["n_rot"]}
    row = 2 * kv_dim * {"f16": 2, "q8": 1, "f32": 4}[case["kv"]] + (kv_dim // 4 if case["kv"] == "q8" else 0)      # K and V of one row, scales too
    n, r = case["seqs"], case["rows"]
    moved = {"accept": (2 * n * (1 + case["nodes"] // 8)), "fork": r + n * r, "slide": 2 * n * _slide(r)[2], "copy": 2 * sum(_lengths(n, r, 4.0))}[case["form"]]
    return {"bytes": case["layers"] * row * moved, "flops": 0}


# ---- state ----

def _engine(s, act, seqs, rows, cols, layers=1, kv="f16"):
    """The handle that an engine keeps."""
    from pooled_b200 import AttnConfig, AttnEngine
    return AttnEngine(AttnConfig(n_heads=s["nH"], n_kv_heads=s["nKV"], head_dim=s["hd"], n_rot=s["n_rot"], rope_theta=s["theta"], max_seq=rows, n_seqs=seqs, n_layers=layers,
                                 act_dtype=act, max_cols=max(8, cols), kv_format=kv), device=torch.cuda.current_device())


def _kept(eng, t):
    """A view of the engine's memory with the engine that owns it."""
    t.engine = eng
    return t


def _tree(r, n, reach):
    """Parents of a drafted tree: every token hangs on one of the last `reach` before it, the first on the conversation."""
    return [-1 if c == 0 else r.randint(max(0, c - reach), c - 1) for c in range(n)]


def _path(r, parents):
    """The accepted path: down from the first token, child after child, for as long as the model agrees."""
    at, path = 0, [0]
    while r.random() < 0.8:
        children = [c for c, p in enumerate(parents) if p == at]
        if not children:
            break
        at = r.choice(children)
        path.append(at)
    return path


def _positions(case, g, r, dev):
    """int32 [axes, columns]: text runs through all axes alike; of a picture the time stands still while height and width run."""
    cols, axes = case["cols"] * case.get("seqs", 1), case["axes"]
    start = r.randint(0, 20000)
    c = torch.arange(cols, device=dev)
    if axes == 1:                                                        # trees: the tokens' depths
        depth = []
        for _ in range(case["seqs"]):
            base, d = r.randint(0, 32000), []
            for p in _tree(r, case["cols"], 8):
                d.append(base if p < 0 else d[p] + 1)
            depth += d
        return torch.tensor([depth], dtype=torch.int32, device=dev)
    width = max(1, int(math.sqrt(cols) * 1.3))
    hw = [start + c // width, start + c % width]
    return torch.stack(([torch.full_like(c, start)] if axes == 3 else []) + hw).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    r = random.Random(int(seed))
    s, kind = SHAPES[case["model"]], case["kind"]
    nH, nKV, hd = s["nH"], s["nKV"], s["hd"]
    act = ACT[case.get("act", "f16")]
    new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev).normal_(generator=g).to(act)
    wide = 2 * hd if s["gated"] else hd                                  # gated: [q of a head, gate of a head] per head
    st = {"case": case, "s": s, "wide": wide}
    if kind == "tree":
        n, lens = case["nodes"], _lengths(case["seqs"], case["ctx"])
        rows = max(lens) + n
        # keys with a few outlier channels per head, as real ones have, and normal values
        kv = [torch.empty((case["seqs"], rows, nKV, hd), dtype=torch.float16, device=dev).normal_(generator=g) for _ in "kv"]
        kv[0][..., 5::61] *= 3.0
        st["kv"] = [x.view(case["seqs"], rows, -1) for x in kv]
        st["q"] = new(case["seqs"] * n, nH * wide)
        st["gate"] = st["q"][:, hd:] if s["gated"] else None
        st["trees"] = [_tree(r, n, case["reach"]) for _ in lens]
        st["parents"] = torch.tensor(sum(st["trees"], []), dtype=torch.int32, device=dev)
        st["items"] = [(i, m, n) for i, m in enumerate(lens)]
        st["lens"] = torch.tensor(lens, device=dev)
        if own:
            st["eng"] = _engine(s, act, case["seqs"], rows, case["seqs"] * n)
            for which, x in zip("kv", st["kv"]):
                st["eng"].cache(0, which).copy_(x.view(torch.int16))
        return st
    if kind in ("turn", "lay"):
        cols = case["cols"] * case.get("seqs", 1)
        st["q"] = new(cols, nH * wide)
        st["positions"] = _positions(case, g, r, dev)
        if kind == "lay":
            st["k"], st["v"] = new(cols, nKV * hd), new(cols, nKV * hd)
            st["items"] = [(i, (5 * i) % 8, case["cols"]) for i in range(case["seqs"])]      # rows of the caches: the positions are the device's
            st["at"] = torch.tensor([i * (case["cols"] + 8) + row + c for i, row, n in st["items"] for c in range(n)], device=dev)
            st["kv"] = [torch.zeros((case["seqs"], case["cols"] + 8, nKV * hd), dtype=torch.float16, device=dev) for _ in "kv"]
        if own:
            eng = st["eng"] = _engine(s, act, case.get("seqs", 1), case["cols"] + 8, cols)
            many = dict(axes=PAIRS[case["model"], case["axes"]], axes_order=case["order"]) if case["axes"] > 1 else {}
            st["rot"] = eng.rotary(n_rot=s["n_rot"], theta=s["theta"], **many)
            if kind == "lay":
                for which, x in zip("kv", st["kv"]):
                    eng.cache(0, which).copy_(x.view(torch.int16))
                st["out"] = [_kept(eng, eng.cache(0, w).view(torch.float16)) for w in "kv"]
        return st
    # the caches' words, whatever they stand for: [layers, 2, seqs, rows, values]; int8 caches with their scales
    form, n, rows, layers = case["form"], case["seqs"], case["rows"], case["layers"]
    seqs = {"accept": n, "fork": n + 1, "slide": n, "copy": 2 * n}[form]
    words = {"f16": torch.int16, "q8": torch.int8, "f32": torch.int32}[case["kv"]]
    some = lambda dtype, width: torch.randint(-100, 100, (layers, 2, seqs, rows, width), generator=g, device=dev, dtype=dtype)
    st["kv"] = [some(words, nKV * hd)] + ([some(torch.int32, nKV * hd // 32)] if case["kv"] == "q8" else [])
    if form == "accept":
        trees = [_tree(r, case["nodes"], 8) for _ in range(n)]
        paths = [_path(r, t) for t in trees]
        base = [m - case["nodes"] for m in _lengths(n, rows, 2.0)] if rows // 2 > case["nodes"] else [rows - case["nodes"]] * n
        st["lists"] = torch.tensor([[len(p), *p, *[0] * (case["nodes"] - len(p))] for p in paths], dtype=torch.int32, device=dev)
        st["base"] = torch.tensor(base, device=dev)
        st["items"] = [(i, b, i, b, case["nodes"]) for i, b in enumerate(base)]
    elif form == "fork":
        st["items"] = [(0, 0, i + 1, 0, rows) for i in range(n)]
    elif form == "slide":
        keep, at, m = _slide(rows)
        st["items"] = [(i, at, i, keep, m) for i in range(n)]
    else:
        lens = _lengths(n, rows, 4.0)
        st["items"] = [(i, 0, n + i, 0, m) for i, m in enumerate(lens)]
        st["lens"] = torch.tensor(lens, device=dev)
    if own:
        eng = st["eng"] = _engine(s, torch.float16, seqs, rows, 1, layers, case["kv"])
        st["out"] = []
        for li in range(layers):
            for k, w in enumerate("kv"):
                views = [eng.cache(li, w)] + ([eng.cache_scales(li, w)] if case["kv"] == "q8" else [])
                for x, t in zip(st["kv"], views):
                    t = t.view(x.dtype)
                    t.copy_(x[li, k])
                    st["out"].append(_kept(eng, t))
    return st


# ---- the plain forms ----

def _angles(case, positions, dev):
    """Angle of every pair (float64) [columns, pairs] at positions [axes, columns]."""
    s = SHAPES[case["model"]]
    half = s["n_rot"] // 2
    i = torch.arange(half, device=dev)
    if case["axes"] == 1:
        return positions[0].double()[:, None] * s["theta"] ** (-2.0 * i.double() / s["n_rot"])
    pairs = torch.tensor(PAIRS[case["model"], case["axes"]], device=dev)
    ends = pairs.cumsum(0)
    block = (i[:, None] >= ends).sum(1)
    axis, f = block, s["theta"] ** (-2.0 * i.double() / s["n_rot"])
    if case["order"] == "cycled":
        axis = i % len(pairs)
        axis = torch.where(i < len(pairs) * pairs[axis], axis, 0)
    if case["order"] == "own":
        f = s["theta"] ** (-(i - (ends - pairs)[block]).double() / pairs[block])
    return positions.double()[axis].T * f


def _turned(st, x, heads, wide):
    """x [cols, heads * wide] -> [cols, heads * hd] in 32 bits, rotated in halves."""
    s = st["s"]
    n = s["n_rot"]
    angle = _angles(st["case"], st["positions"], x.device)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.view(x.shape[0], heads, wide)[..., :s["hd"]].float()
    a, b = x[..., :n // 2], x[..., n // 2:n]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., n:]], -1).flatten(1)


def _plain(st):
    case, s, kind = st["case"], st["s"], st["case"]["kind"]
    nH, nKV, hd = s["nH"], s["nKV"], s["hd"]
    act = ACT[case.get("act", "f16")]
    if kind == "turn":
        return _turned(st, st["q"], nH, st["wide"]).to(act)
    if kind == "lay":
        q = _turned(st, st["q"], nH, st["wide"]).to(act)
        st["kv"][0].view(-1, nKV * hd)[st["at"]] = _turned(st, st["k"], nKV, hd).half()
        st["kv"][1].view(-1, nKV * hd)[st["at"]] = st["v"].half()
        return q, st["kv"][0], st["kv"][1]
    if kind == "tree":
        B, n = case["seqs"], case["nodes"]
        k, v = [x.view(B, -1, nKV, hd).float() for x in st["kv"]]
        # ancestors: the parents' matrix and itself, squared until paths of every length are in it
        p = st["parents"].view(B, n).long()
        seen = torch.eye(n, device=p.device) + torch.zeros((B, n, n + 1), device=p.device).scatter_(2, torch.where(p < 0, n, p)[..., None], 1.0)[..., :n]
        for _ in range(max(1, (n - 1).bit_length())):
            seen = (seen @ seen).clamp_(max=1.0)
        r = torch.arange(k.shape[1], device=k.device)
        at = r - st["lens"][:, None]                                     # a row's place in its tree
        own_rows = seen.gather(2, at.clamp(0, n - 1)[:, None].expand(-1, n, -1)) > 0
        mask = (at < 0)[:, None] | ((at < n)[:, None] & own_rows)        # [B, n, rows]
        q = st["q"].view(B, n, nKV, nH // nKV, st["wide"])[..., :hd].float() / math.sqrt(hd)
        sc = torch.einsum("bnkgd,brkd->bkgnr", q, k).masked_fill_(~mask[:, None, None], -math.inf)
        e = (sc - sc.amax(-1, keepdim=True)).exp_()
        o = torch.einsum("bkgnr,brkd->bnkgd", e / e.sum(-1, keepdim=True), v).reshape(B * n, nH, hd)
        if st["gate"] is not None:
            o = o * torch.sigmoid(st["q"].view(B * n, nH, -1)[..., hd:].float())
        return o.flatten(1).to(act)
    form, n = case["form"], case["seqs"]
    for x in st["kv"]:
        if form == "accept":
            j = torch.arange(case["nodes"], device=x.device)
            b, to = torch.arange(n, device=x.device)[:, None], st["base"][:, None] + j
            path = x[:, :, b, st["base"][:, None] + st["lists"][:, 1:].long()]
            x[:, :, b, to] = torch.where((j < st["lists"][:, :1])[..., None], path, x[:, :, b, to])
        elif form == "fork":
            x[:, :, 1:] = x[:, :, :1]
        elif form == "slide":
            keep, at, m = _slide(case["rows"])
            x[:, :, :, keep:keep + m] = x[:, :, :, at:].clone()
        else:
            live = torch.arange(case["rows"], device=x.device) < st["lens"][:, None]
            x[:, :, n:] = torch.where(live[..., None], x[:, :, :n], x[:, :, n:])
    return [x[li, k] for li in range(case["layers"]) for k in range(2) for x in st["kv"]]


# ---- the library's calls ----

def run(st):
    if not own:
        return _plain(st)
    case, s, kind, eng = st["case"], st["s"], st["case"]["kind"], st["eng"]
    if kind == "tree":
        return eng.decode_tree(0, st["items"], st["q"], parents=st["parents"], gate=st["gate"], q_head_stride=st["wide"], gate_head_stride=st["wide"])
    if kind == "turn":
        return st["rot"].apply(st["q"], s["nH"], positions=st["positions"], head_stride=st["wide"])
    if kind == "lay":
        q = eng.rotary_append(0, st["rot"], st["items"], st["q"], st["k"], st["v"], q_head_stride=st["wide"], q_dtype=st["q"].dtype, positions=st["positions"])
        return q, *st["out"]
    eng.move(st["items"], lists=st.get("lists"))
    return st["out"]


# ---- the definitions in 64 bits ----

def _exact_turn(case, x, heads, wide, positions):
    s = SHAPES[case["model"]]
    half, hd, axes = s["n_rot"] // 2, s["hd"], case["axes"]
    which, freq = [], []
    if axes == 1:
        which, freq = [0] * half, [math.pow(s["theta"], -i / half) for i in range(half)]
    elif case["order"] == "cycled":
        pairs = PAIRS[case["model"], axes]
        left = list(pairs)
        for i in range(half):
            a = i % axes
            if a and not left[a]:
                a = 0
            left[a] -= 1
            which.append(a)
            freq.append(math.pow(s["theta"], -i / half))
    else:
        for a, n in enumerate(PAIRS[case["model"], axes]):
            freq += [math.pow(s["theta"], -j / n if case["order"] == "own" else -(len(which) + j) / half) for j in range(n)]
            which += [a] * n
    turn = positions.double()[which].t() * torch.tensor(freq, dtype=torch.float64, device=x.device)
    z = torch.polar(torch.ones_like(turn), turn)[:, None]
    y = x.double().view(x.shape[0], heads, wide)[:, :, :hd].clone()
    t = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * z
    y[..., :half], y[..., half:2 * half] = t.real, t.imag
    return y.reshape(x.shape[0], heads * hd)


def exact(case, seed):
    if case["kind"] == "move":
        return None                                                      # copies: nothing is computed
    st = prepare(case, seed)
    s = st["s"]
    nH, nKV, hd, G = s["nH"], s["nKV"], s["hd"], s["nH"] // s["nKV"]
    if case["kind"] == "turn":
        return _exact_turn(case, st["q"], nH, st["wide"], st["positions"])
    if case["kind"] == "lay":
        kv = [x.double() for x in st["kv"]]
        kv[0].view(-1, nKV * hd)[st["at"]] = _exact_turn(case, st["k"], nKV, hd, st["positions"])
        kv[1].view(-1, nKV * hd)[st["at"]] = st["v"].double()
        return _exact_turn(case, st["q"], nH, st["wide"], st["positions"]), kv[0], kv[1]
    n = case["nodes"]
    q = st["q"].view(case["seqs"], n, nH, st["wide"])
    out = torch.empty((case["seqs"], n, nH, hd), dtype=torch.float64, device=q.device)
    for i, m in enumerate(st["lens"].tolist()):                          # one conversation and head after another
        rows = torch.zeros((n, m + n), dtype=torch.bool)
        rows[:, :m] = True
        for c in range(n):
            a = c
            while a >= 0:
                rows[c, m + a] = True
                a = st["trees"][i][a]
        rows = rows.to(q.device)
        for h in range(nH):
            cut = slice(h // G * hd, (h // G + 1) * hd)
            k, v = [x[i, :m + n, cut].double() for x in st["kv"]]
            score = q[i, :, h, :hd].double() @ k.t() / math.sqrt(hd)
            out[i, :, h] = torch.softmax(torch.where(rows, score, -math.inf), -1) @ v
            if s["gated"]:
                out[i, :, h] /= 1.0 + torch.exp(-q[i, :, h, hd:].double())
    return out.reshape(case["seqs"] * n, nH * hd)
