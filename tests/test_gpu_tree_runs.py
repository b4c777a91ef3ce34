"""pa_decode_tree over long runs of tiles: several runs of a unit in wide and narrow row tiles, added up in one record or left in records of their own,
with an error that a lost tile, or a lost low part of a query or weight, is far above.  Which kernel and which runs the sizes reach is worked out
from the plan by test_tree_plan.py."""
import math
import random

import pytest
import torch

from tests.test_gpu_tree import F16, F32, engine, fill, mask_of, tree

pytestmark = pytest.mark.gpu

# name: q heads, kv heads, head_dim, f16 activations and queries, columns of the context, trees (rows, tokens); then what the plan makes of it: wide row
# tiles, several runs of a unit (WIDE and FOLD of the kernel), the longest run in tiles
CASES = {
    "wide_128_own_records": (16, 8, 128, True, 1056, [(8400, 33)] * 32, True, True, 66),
    "wide_128_added_up": (16, 8, 128, True, 960, [(32768, 60)] * 16, True, True, 65),
    "wide_256_added_up": (16, 2, 256, True, 2048, [(16700, 64)] * 32, True, True, 67),
    "wide_64_added_up": (16, 2, 64, True, 2048, [(16700, 64)] * 32, True, True, 66),
    "f32_128_long": (16, 8, 128, False, 64, [(33001, 61)], False, True, 15),
    "f32_256_long": (16, 2, 256, False, 64, [(33001, 61)], False, False, 20),
    "f32_64_long": (16, 2, 64, False, 64, [(33001, 61)], False, True, 15),
    "f32_256_batch": (24, 4, 256, False, 156, [(9001, 26), (5000, 26), (2000, 26), (800, 26), (800, 26), (800, 26)], False, False, 8),
    "f32_128_parts": (48, 8, 128, False, 606, [(3000, 256), (700, 200), (4500, 150)], False, True, 13),
    "f32_64_parts": (64, 1, 64, False, 606, [(3000, 256), (700, 200), (4500, 150)], False, True, 13),
    "f32_256_parts": (32, 4, 256, False, 606, [(3000, 256), (700, 200), (4500, 150)], False, True, 13),
    "f32_128_few_columns": (16, 8, 128, False, 8, [(33001, 8)], False, False, 4),
}


def reference(q, k, v, mask):
    """q [n, nH, hd], k, v [rows, nKV, hd] in float64, a kv head after another: out [n, nH, hd], the scores' root mean square, the largest sum of absolute
    products of one (over sqrt(hd)), and the most weights of a row below 2^-20 of its largest."""
    n, nH, hd = q.shape
    G, out, squares, largest, small = nH // k.shape[1], [], [], 0.0, 0
    for g in range(k.shape[1]):
        qg, kg = q[:, g * G:(g + 1) * G].double(), k[:, g].double()
        s = (qg.reshape(-1, hd) @ kg.t() / math.sqrt(hd)).view(n, G, -1)
        squares.append((s * s).mean())
        largest = max(largest, float((qg.abs().reshape(-1, hd) @ kg.abs().t()).amax()) / math.sqrt(hd))
        p = torch.softmax(torch.where(mask[:, None], s, -math.inf), -1)
        small = max(small, int(((p > 0) & (p < p.amax(-1, keepdim=True) * 2.0 ** -20)).sum(-1).amax()))
        out.append(p @ v[:, g].double())
    return torch.cat(out, 1), math.sqrt(float(sum(squares)) / len(squares)), largest, small


def calls(name):
    nH, nKV, hd, f16, cols, sizes, wide, _, run = CASES[name]
    r = random.Random(len(name))
    act = F16 if f16 else F32
    eng = engine(nH, nKV, hd, max(b + n for b, n in sizes), len(sizes), act, max_cols=cols)
    items = [(s, b, n) for s, (b, n) in enumerate(sizes)]
    trees = [tree(r, n, 9) for _, _, n in items]
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1000 + len(sizes))       # (other numbers than the caches': a query that is a key attends little else)
    q = torch.empty((len(parents), nH, hd), device="cuda").normal_(generator=g).to(act)
    return eng, items, trees, parents, q, (8 if wide else 4) * run


@pytest.mark.parametrize("name", CASES)
def test_relative_error(name):
    eng, items, trees, parents, q, steps = calls(name)
    hd = q.shape[-1]
    k, v = fill(eng, 1)
    got = eng.decode_tree(0, items, q.flatten(1), parents=parents).view(q.shape)
    eng.sync()
    off = size = score = 0.0
    small = col = 0
    for (s, base, n), t in zip(items, trees):
        want, rms, _, few = reference(q[col:col + n], k[s, :base + n], v[s, :base + n], mask_of(t, base))
        off, size = off + float((got[col:col + n].double() - want).square().sum()), size + float(want.square().sum())
        score, small = max(score, rms), max(small, few)
        col += n
    # Of the norm, the errors of single weights and values being independent of the values they meet: the tensor cores cut what they add off, by
    # up to 2^-23 at each of a run's `steps` additions of 16 keys; of a score (hd / 16 of them, and the sum of its two rows) what that makes of its root
    # mean square, which is an error of its weight; f32 queries and weights as two f16 values and the exponential 2^-22 each, records added up 2^-24
    # each (some 64).  f16 outputs: half a step of 2^-10.
    # (Queries rounded to f16 are off by some 2e-4, one tile of the longest case left out by 4e-2.)
    tol = 2.0 ** -23 * (steps + (hd / 16 + 2) * score) + 3 * 2.0 ** -22 + 64 * 2.0 ** -24 + small * 2.0 ** -31
    if got.dtype == F16:
        tol += 2.0 ** -11 + 2.0 ** -25 / math.sqrt(size / got.numel())
    assert torch.isfinite(got).all()
    assert math.sqrt(off / size) <= tol, f"{math.sqrt(off / size):.3g} for {tol:.3g}"


@pytest.mark.parametrize("name", CASES)
def test_every_tile_arrives(name):
    # V holds a one in the dim that a tile's number names: an output is the weight of the tiles of that number, none of them negligible
    eng, items, trees, parents, q, steps = calls(name)
    hd = q.shape[-1]
    k, v = fill(eng, 2)
    rows = torch.arange(v.shape[1], device="cuda")
    v.zero_()
    v[:, rows, :, rows // 64 % hd] = 1.0
    eng.cache(0, "v").copy_(v.view(v.shape[0], v.shape[1], -1).view(torch.int16))
    got = eng.decode_tree(0, items, q.flatten(1), parents=parents).view(q.shape)
    eng.sync()
    col = 0
    for (s, base, n), t in zip(items, trees):
        want, _, largest, small = reference(q[col:col + n], k[s, :base + n], v[s, :base + n], mask_of(t, base))
        # Nothing cancels, so each output has the error of its sum and of its weights, the largest that a score's may be: queries as two f16 values,
        # hd / 16 additions and one of the two rows; the sum below the line has it, too.  Weights below 2^-14 (2^-21 of the largest) lose up to 2^-24 each.
        delta = largest * (2.0 ** -22 + (hd / 16 + 2) * 2.0 ** -23)
        tol = want * (2 * delta + steps * 2.0 ** -23 + 2.0 ** -20 + 128 * 2.0 ** -24) + small * 2.0 ** -31
        if got.dtype == F16:
            tol = tol + want * 2.0 ** -11 + 2.0 ** -25
        err = (got[col:col + n].double() - want).abs()
        assert torch.all(err <= tol), f"item of {base} + {n}: {float((err - tol).amax())} past the tolerance"
        col += n


@pytest.mark.parametrize("hd,act", [(256, F16), (256, F32), (128, F16), (64, F32)])
@pytest.mark.parametrize("base,n", [(0, 40), (100, 64), (63, 200)])
def test_values_that_are_finite_keep_their_bits(hd, act, base, n):
    # infinities and NaN in some V values of one token: every output that none of them reaches has the bits that it has without them
    r = random.Random(base + n)
    eng = engine(8, 2, hd, base + n, 1, act)
    k, v = fill(eng, 6)
    t = tree(r, n, 12)
    parents = torch.tensor(t, dtype=torch.int32, device="cuda")
    q = torch.randn((n, 8 * hd), device="cuda").to(act)
    clean = eng.decode_tree(0, [(0, base, n)], q, parents=parents).view(n, 8, hd)
    b, vv = n // 3, v.clone()
    bad = torch.zeros((8, hd), dtype=torch.bool, device="cuda")
    for head, d, x in ((0, 5, math.inf), (1, 17, math.nan), (1, hd - 1, -math.inf)):
        vv[0, base + b, head, d] = x
        bad[4 * head:4 * head + 4, d] = True
    eng.cache(0, "v").copy_(vv.view(1, base + n, -1).view(torch.int16))
    got = eng.decode_tree(0, [(0, base, n)], q, parents=parents).view(n, 8, hd)
    reached = mask_of(t, base)[:, base + b][:, None, None] & bad
    assert reached.any() and torch.equal(got[~reached], clean[~reached]) and not torch.isfinite(got[reached]).any()
