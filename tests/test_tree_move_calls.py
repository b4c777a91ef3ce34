"""The calls of trees of drafted tokens, positions of several axes and moved rows without a GPU: the CPython module and ctypes make the
same ones, null handles and integers past their width are refused, and the host refuses tensors that do not fit before anything is called."""
import ctypes as C
import os
import re

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError, Rotary
from pooled_b200 import lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I32 = torch.int32


@pytest.fixture(scope="module")
def pa():
    from pooled_b200 import build
    build.build()
    return L.load()


class NoCalls:
    def __getattr__(self, name):
        return lambda *a: pytest.fail(f"{name} was called")


@pytest.fixture
def detached():
    """An engine of 4/2 heads of 64 with two layers and a rotation of two axes, without a device: nothing may reach the library."""
    eng = object.__new__(AttnEngine)
    eng.cfg = AttnConfig(n_heads=4, n_kv_heads=2, head_dim=64, n_rot=64, rope_theta=1e4, max_seq=32, act_dtype=torch.float32)
    eng.device, eng.layers, eng._call, eng.ctx, eng.slots, eng._xc_keep, eng._q_dim, eng._kv_dim = -1, [C.c_void_p(8), C.c_void_p(16)], NoCalls(), None, {}, None, 256, 128
    eng._f_rot_append = eng._f_rot_at = eng._f_tree = eng._f_move = 0
    eng._all_layers, eng._dev = None, torch.device("cpu")
    eng._raw_st = lambda: 0
    rot = object.__new__(Rotary)
    rot.eng, rot.handle, rot._h, rot._apply, rot._f_apply, rot.n_axes = eng, C.c_void_p(8), 8, NoCalls(), 0, 2
    yield eng, rot
    eng.layers = []


def test_struct_layouts_match_the_header():
    assert C.sizeof(L.PaRotaryAxes) == 32 and L.PaRotaryAxes.pairs.offset == 8 and L.PaRotaryAxes.reserved.offset == 24
    assert C.sizeof(L.PaMoveItem) == 24 and L.PaMoveItem.n_rows.offset == 16
    header = open(os.path.join(ROOT, "include", "pooled_attn.h")).read()
    for struct, cls in (("pa_rotary_axes", L.PaRotaryAxes), ("pa_move_item", L.PaMoveItem)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"struct %s \{(.*?)\}" % struct, header, re.S).group(1), flags=re.S)
        assert re.findall(r"(\w+)(?:\[\d+\])?\s*[,;]", body) == [name for name, _ in cls._fields_]


def test_call_module_calls_as_ctypes_does(pa):
    seen = []

    def items(a, i, n, struct):
        it = C.cast(a[i], C.POINTER(struct))
        return [tuple(getattr(it[j], f) for f, _ in struct._fields_) for j in range(a[n])]

    def fake(name):
        res, args = L.SYMBOLS[name]

        def record(*a):
            a = list(a)
            if name == "pa_rotary_append_at":
                rows = C.cast(a[4], C.POINTER(C.c_uint32))
                a[4] = a[4] and [rows[j] for j in range(a[3])]
                a[2] = items(a, 2, 3, L.PaItem)
            elif name == "pa_decode_tree":
                a[1] = items(a, 1, 2, L.PaItem)
            else:
                a[2] = items(a, 2, 3, L.PaMoveItem)
            seen.append((name, *a))
            return len(seen)
        return C.CFUNCTYPE(res, *args)(record)

    class FakeLib:
        pass
    lib, names = FakeLib(), ["pa_rotary_append_at", "pa_decode_tree", "pa_cache_move"]
    for name in names:
        setattr(lib, name, fake(name))
    by_ctypes = L.CtypesCalls(lib)
    entry = {name: C.cast(getattr(lib, name), C.c_void_p).value for name in names}
    q, k, v, g, o = (torch.zeros((3, n + 2 * i))[:, :n] for i, n in enumerate((64, 16, 16, 64, 64)))
    p, lists = torch.zeros((2, 3), dtype=I32), torch.zeros((2, 9), dtype=I32)
    triples, fives = [(3, 7, 1), (0, 2 ** 31, 2)], [(0, 1, 2, 3, 4), (2 ** 32 - 1, 0, 5, 2 ** 31, 0)]
    calls = [("rotary_append_at", (4096, 8192, triples, rows, p, qq, 16, k, v, qo, 1, 7)) for rows in (None, [9, 2 ** 32 - 1]) for qq, qo in ((q, o), (None, None))]
    calls += [("decode_tree", (4096, triples, ps, q, 1, 16, gate, 32, o, 7)) for ps in (None, p[0]) for gate in (None, g)]
    calls += [("cache_move", (4096, 5, it, lp, 9, 7)) for it in (fives, fives[:1], []) for lp in (None, lists)]
    for method, args in calls:
        seen.clear()
        name = "pa_" + method
        assert getattr(pa.call, method)(entry[name], *args) == 1 and getattr(by_ctypes, method)(entry[name], *args) == 2
        assert seen[0] == seen[1] and seen[0][0] == name, method
    for bad in ([(1,)], [3], [(1, 2, 3, 4)], [(1, "a", 2)], [(1, 2, 3, 4, 5, 6)]):
        for method, args in (("rotary_append_at", (4096, 8192, bad, None, p, q, 16, k, v, o, 1, 7)), ("decode_tree", (4096, bad, None, q, 1, 16, None, 32, o, 7)),
                             ("cache_move", (4096, 1, bad, None, 0, 7))):
            with pytest.raises((TypeError, ValueError)):
                getattr(pa.call, method)(entry["pa_" + method], *args)
        with pytest.raises((TypeError, ValueError)):
            by_ctypes.cache_move(0, 4096, 1, bad, None, 0, 7)
    with pytest.raises(ValueError):
        pa.call.rotary_append_at(entry["pa_rotary_append_at"], 4096, 8192, triples, [1], p, q, 16, k, v, o, 1, 7)


@pytest.mark.parametrize("by_module", [True, False])
def test_integers_past_their_width_are_refused(pa, by_module):
    calls = pa.call if by_module else L.CtypesCalls(NoCalls())
    never = C.CFUNCTYPE(C.c_int)(lambda: pytest.fail("the library was called"))
    fn = C.cast(never, C.c_void_p).value
    q, k, o, p = torch.zeros((3, 64)), torch.zeros((3, 16)), torch.zeros((3, 64)), torch.zeros(3, dtype=I32)
    triples = [(3, 7, 1), (0, 9, 2)]
    good = {"rotary_append_at": (4096, 8192, triples, [1, 2], p, q, 16, k, k, o, 1, 7), "decode_tree": (4096, triples, p, q, 1, 16, q, 32, o, 7),
            "cache_move": (4096, 2, [(0, 1, 2, 3, 4)], p, 9, 7)}
    wide = {"rotary_append_at": (6,), "decode_tree": (5, 7), "cache_move": ()}              # places of head strides, 64 bits,
    narrow = {"rotary_append_at": (), "decode_tree": (), "cache_move": (1, 4)}             # of counts, 32 bits,
    places = {"rotary_append_at": 2, "decode_tree": 1, "cache_move": 2}                    # and of the items

    def refused(method, args):
        with pytest.raises(PaError) as e:
            getattr(calls, method)(fn, *args)
        assert e.value.code == -1

    for method, args in good.items():
        for places_of, values in ((wide, (-1, -64, 2 ** 64, 2 ** 64 + 16)), (narrow, (-1, 2 ** 32, 2 ** 32 + 5, -2 ** 40, 2 ** 70))):
            for i in places_of[method]:
                for bad in values:
                    refused(method, (*args[:i], bad, *args[i + 1:]))
        i = places[method]
        for j in range(len(args[i][0])):
            for bad in (-1, 2 ** 32, 2 ** 32 + 1):
                item = list(args[i][0])
                item[j] = bad
                refused(method, (*args[:i], [tuple(item), *args[i][1:]], *args[i + 1:]))
    for bad in ([1, 2 ** 32], [-1, 2]):
        refused("rotary_append_at", (4096, 8192, triples, bad, p, q, 16, k, k, o, 1, 7))


def test_null_handles_are_refused(pa):
    h = C.c_void_p()
    assert pa.pa_rotary_create_axes(None, None, None, C.byref(h)) == -1
    assert pa.pa_rotary_append_at(None, None, None, 0, None, None, None, 0, 0, None, None, 0, None, 0, 0, None) == -1
    assert pa.pa_decode_tree(None, None, 0, None, None, 0, 0, 0, None, 0, 0, None, 0, None) == -1
    assert pa.pa_cache_move(None, 0, None, 0, None, 0, None) == -1 and pa.pa_cache_move(None, 1, None, 0, None, 0, None) == -1
    none = (C.c_void_p * 1)(None)
    assert pa.pa_cache_move(C.addressof(none), 1, None, 0, None, 0, None) == -1


@pytest.mark.parametrize("parents", [torch.zeros(3, dtype=I32), torch.zeros(2, dtype=torch.int64), torch.zeros(2), torch.zeros((1, 2), dtype=I32), torch.zeros((2, 1), dtype=I32),
                                     torch.zeros(4, dtype=I32)[::2], torch.zeros(0, dtype=I32)])
def test_parents_that_are_not_one_per_token_are_refused(detached, parents):
    q = torch.zeros((2, 256))
    with pytest.raises(PaError):
        detached[0].decode_tree(0, [(0, 0, 2)], q, parents, out=torch.zeros((2, 256)))


def test_a_tree_of_tensors_that_do_not_fit_is_refused(detached):
    eng, _ = detached
    q, out, z = torch.zeros((2, 256)), torch.zeros((2, 256)), torch.zeros
    two = [(0, 0, 2)]
    for items, args in ((two, dict(q=z(3, 256))), (two, dict(q=z(2, 255))), (two, dict(q=q, out=z(2, 128))), (two, dict(q=q, out=z(3, 256))), (two, dict(q=q, out=out.half())),
                        (two, dict(q=q, gate=z(1, 256))), (two, dict(q=q, gate=q.half())), (two, dict(q=q, q_head_stride=128)), (two, dict(q=q, q_head_stride=-64)),
                        (two, dict(q=q, gate=q, gate_head_stride=-64)), ([(0, 0, 1)], dict(q=q)), ([(0, 0, 1), (1, 0, 2)], dict(q=q)), (two, dict(q=z(256, 2).t()))):
        args.setdefault("out", out)
        with pytest.raises(PaError):
            eng.decode_tree(0, items, args.pop("q"), **args)
    eng.device = 0                                                    # tensors of another device than the engine's
    for parents in (None, z(2, dtype=I32)):
        with pytest.raises(PaError):
            eng.decode_tree(0, two, q, parents, out=out)


@pytest.mark.parametrize("lists", [torch.zeros((1, 4), dtype=torch.int64), torch.zeros(4, dtype=I32), torch.zeros((2, 4), dtype=I32), torch.zeros((1, 8), dtype=I32)[:, ::2],
                                   torch.zeros((1, 1, 4), dtype=I32)])
def test_lists_that_are_not_one_row_per_item_are_refused(detached, lists):
    with pytest.raises(PaError):
        detached[0].move([(0, 0, 1, 0, 4)], lists)


def test_lists_of_another_device_and_layers_that_are_not_there_are_refused(detached):
    eng, _ = detached
    with pytest.raises(IndexError):
        eng.move([(0, 0, 1, 0, 4)], layers=[2])
    eng.device = 0
    with pytest.raises(PaError):
        eng.move([(0, 0, 1, 0, 4)], torch.zeros((1, 4), dtype=I32))


@pytest.mark.parametrize("positions", [torch.zeros(2, dtype=I32), torch.zeros((1, 2), dtype=I32), torch.zeros((3, 2), dtype=I32), torch.zeros((2, 3), dtype=I32),
                                       torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 2), dtype=I32).t(), torch.zeros((2, 4), dtype=I32)[:, ::2],
                                       torch.zeros((2, 2, 1), dtype=I32)])
def test_positions_that_are_not_one_per_axis_and_column_are_refused(detached, positions):
    eng, rot = detached
    q, kv = torch.zeros((2, 256)), torch.zeros((2, 128))
    with pytest.raises(PaError):
        rot.apply(q, 4, positions=positions, out=q)
    with pytest.raises(PaError):
        eng.rotary_append(0, rot, [(0, 0, 2)], q, kv, kv, q_out=q, positions=positions)


def test_positions_of_one_axis_may_be_flat_or_a_row(detached):
    eng, rot = detached
    rot.n_axes = 1
    rot._places(torch.zeros(2, dtype=I32), 2)
    rot._places(torch.zeros((1, 2), dtype=I32), 2)
    for bad in (torch.zeros((2, 1), dtype=I32), torch.zeros((2, 2), dtype=I32), torch.zeros(4, dtype=I32)[::2]):
        with pytest.raises(PaError):
            rot._places(bad, 2)


def test_axes_past_four_and_unknown_orders_are_refused(detached):
    eng, _ = detached
    eng.L = NoCalls()
    for axes in ([], [8] * 5, [2 ** 32], [-1, 33]):
        with pytest.raises(PaError):
            eng.rotary(axes=axes)
    with pytest.raises(KeyError):
        eng.rotary(axes=[16, 16], axes_order="spiral")


def _arguments(text):
    out, depth, at = [], 0, 1
    for i, c in enumerate(text):
        depth += c in "([{"
        depth -= c in ")]}"
        if (c == "," and depth == 1) or depth == 0:
            out.append(text[at:i].strip())
            at = i + 1
        if depth == 0:
            return [a for a in out if a]


def test_js_methods_lay_out_what_the_header_says():
    js = open(os.path.join(ROOT, "js", "pooled_attn.js")).read()
    method = lambda name: re.search(r"^  %s\(.*?^  }" % name, js, re.M | re.S).group(0)
    call = lambda text, sym: _arguments(text[text.index(sym + "(") + len(sym):])
    axes = method("rotary")
    assert "[axes.length, axesOrder, ...axes, ...Array(6 - axes.length).fill(0)]" in axes           # 2 + n + 6 - n words of pa_rotary_axes
    assert call(axes, "pa_rotary_create_axes")[2] == "new Uint8Array(many.buffer)"
    at = call(method("rotaryAppendAt"), "pa_rotary_append_at")
    assert at[5] == "positions" and at[7:9] == ["BigInt(m * qDim)", "BigInt(m * hd)"]
    tree = call(method("decodeTree"), "pa_decode_tree")
    assert tree[3] == "parents" and tree[8:11] == ["g", "gs", "gh"] and "this._gate(gate, qFull)" in method("decodeTree")
    assert "6 * items.length" in method("move") and call(method("move"), "pa_cache_move")[4:6] == ["lists", "listStride"]


def test_the_quick_look_at_tensors_agrees_with_the_checks_one_by_one(pa, detached):
    eng, rot = detached
    fits, exact = pa.call.fits, pa.call.exact
    z = torch.zeros
    base = z((6, 512))
    matrices = [z((2, 256)), z((2, 256)).half(), z((3, 256)), z((2, 255)), z((2, 300))[:, :256], z((256, 2)).t(), base[::3, :256], base[:2, ::2], z((1, 256)), z((256,)), z((2, 2, 256)),
                z((2, 256), dtype=torch.bfloat16), z((0, 256)), z((2, 1))]
    for q in matrices:
        for gate in (None, *matrices):
            for out in (None, *matrices):
                try:
                    eng._batch(2, q, None, gate, None, out)
                    slow = True
                except (PaError, ValueError):
                    slow = False
                assert fits(-1, 2, q, 256, None, gate, 256, torch.float32, out, 256, torch.float32) == slow, (q.shape, gate is not None and gate.shape, out is not None and out.shape)
    for k in matrices:
        try:
            eng._columns(2, None, None, k[..., :128], z((2, 128)), None)
            slow = True
        except (PaError, ValueError):
            slow = False
        assert fits(-1, 2, None, 256, torch.float32, k[..., :128], 128, torch.float32, z((2, 128)), 128, torch.float32, None, 256, None) == slow, k.shape
    assert not fits(0, 2, matrices[0], 256, None) and fits(-1, -1, matrices[2], 256, None) and fits(0, 2, None, 1, None)          # of another device; any number of columns
    for p in [z((2, 3), dtype=I32), z((2, 3)), z((3, 2), dtype=I32), z((3, 2), dtype=I32).t(), z(3, dtype=I32), z((2, 6), dtype=I32)[:, ::2], z((1, 2, 3), dtype=I32)]:
        try:
            rot._places(p, 3)
            slow = True
        except PaError:
            slow = False
        assert exact(-1, p, I32, 2, 3) == slow, p.shape
        assert exact(-1, p, I32, None, 3) == (tuple(p.shape) == (3,)) and not exact(0, p, I32, 2, 3)
        rot.n_axes = 1
        try:
            rot._places(p, 3)
            slow = True
        except PaError:
            slow = False
        assert exact(-1, p, I32, 1, 3) == slow, p.shape
        rot.n_axes = 2
    assert exact(-1, z((1, 3), dtype=I32), I32, 1, 3) and not exact(-1, z((1, 3), dtype=I32), I32, None, 3)
    for call in (lambda: fits(-1), lambda: fits(-1, 2, base), lambda: fits(-1, 2, base, "x", None), lambda: fits(-1, 2, 3, 4, None), lambda: exact(-1, base, None, 2), lambda: exact(-1, 5, None, 2, 3)):
        with pytest.raises((TypeError, AttributeError)):
            call()


def test_engines_without_the_module_check_one_by_one(detached):
    eng, rot = detached
    assert eng._fits is None and eng._exact is None
    calls = []
    eng._call = type("Calls", (), {"decode_tree": lambda self, *a: calls.append(a) or 0, "rotary_append_at": lambda self, *a: calls.append(a) or 0})()
    rot._apply = lambda *a: calls.append(a) or 0
    q, kv = torch.zeros((2, 256)), torch.zeros((2, 128))
    for fast in (False, True):
        if fast:
            eng._fits, eng._exact = L.load().call.fits, L.load().call.exact
        calls.clear()
        assert eng.decode_tree(0, [(0, 0, 2)], q, torch.zeros(2, dtype=I32), out=q) is q
        assert eng.rotary_append(0, rot, [(0, 0, 2)], q, kv, kv, q_out=q, positions=torch.zeros((2, 2), dtype=I32)) is q
        assert rot.apply(q, 4, positions=torch.zeros((2, 2), dtype=I32), out=q) is q
        assert len(calls) == 3
