"""The calls of the rotary, shared-prefix, weighing and evicting operators without a GPU: the CPython module and ctypes make the same
ones, null handles are refused, and the host refuses tensors that do not fit before anything is called."""
import ctypes as C

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError, Rotary
from pooled_b200 import lib as L


@pytest.fixture(scope="module")
def pa():
    from pooled_b200 import build
    build.build()
    return L.load()


def test_struct_layouts_match_the_header():
    assert C.sizeof(L.PaRotaryConfig) == 72 and L.PaRotaryConfig.theta.offset == 16 and L.PaRotaryConfig.mscale.offset == 48
    assert C.sizeof(L.PaEvictItem) == 16


def test_call_module_calls_as_ctypes_does(pa):
    seen = []

    def items(a, i, n, struct):
        it = C.cast(a[i], C.POINTER(struct))
        return tuple(tuple(getattr(it[j], f) for f, _ in struct._fields_) for j in range(a[n]))

    def fake(name):
        res, args = L.SYMBOLS[name]

        def record(*a):
            a = list(a)
            if name == "pa_rotary_append":
                rows = C.cast(a[4], C.POINTER(C.c_uint32))
                a[4] = a[4] and [rows[j] for j in range(a[3])]
                a[2] = items(a, 2, 3, L.PaItem)
            elif name == "pa_decode_shared":
                a[5] = items(a, 5, 6, L.PaItem)
            elif name == "pa_decode_weights":
                a[1] = items(a, 1, 2, L.PaItem)
            elif name == "pa_evict":
                a[1] = items(a, 1, 2, L.PaEvictItem)
            seen.append((name, *a))
            return len(seen)
        return C.CFUNCTYPE(res, *args)(record)

    class FakeLib:
        pass
    lib = FakeLib()
    names = ["pa_rotary_apply", "pa_rotary_append", "pa_decode_shared", "pa_decode_weights", "pa_evict"]
    for name in names:
        setattr(lib, name, fake(name))
    by_ctypes = L.CtypesCalls(lib)
    entry = {name: C.cast(getattr(lib, name), C.c_void_p).value for name in names}
    q, k, v, g, o = (torch.zeros((3, n + 2 * i))[:, :n] for i, n in enumerate((64, 16, 16, 64, 64)))
    p, kept = torch.zeros(3, dtype=torch.int32), torch.zeros((2, 2, 5), dtype=torch.int32)
    pairs, triples = [(0, 5), (2, 2 ** 32 - 1), (1, 0)], [(3, 7, 1), (0, 2 ** 31, 2)]
    calls = [("rotary_apply", (4096, q, 0, 16, 4, ps, pos, o, 1, 32, 7)) for ps in (None, p) for pos in (0, -5, 2 ** 31 - 1)]
    calls += [("rotary_append", (4096, 8192, triples, rows, qq, 16, k, v, qo, 1, 7)) for rows in (None, [9, 2 ** 32 - 1]) for qq, qo in ((q, o), (None, None))]
    calls += [("decode_shared", (4096, 8192, 2, 100, 50, pairs, q, 1, 16, gate, 32, o, 7)) for gate in (None, g)]
    calls += [("decode_weights", (4096, pairs, q, 1, 16, gate, 32, o, 7)) for gate in (None, g)]
    calls += [("evict", (4096, triples, 5, 1, 2, kp, 7)) for kp in (None, kept)]
    for method, args in calls:
        seen.clear()
        name = "pa_" + method
        assert getattr(pa.call, method)(entry[name], *args) == 1 and getattr(by_ctypes, method)(entry[name], *args) == 2
        assert seen[0] == seen[1] and seen[0][0] == name, method
    for bad in ([(1,)], [3], [(1, 2, 3, 4)], [(1, "a", 2)]):
        for method, args in (("rotary_append", (4096, 8192, bad, None, q, 16, k, v, o, 1, 7)), ("decode_shared", (4096, 8192, 2, 100, 50, bad, q, 1, 16, None, 32, o, 7)),
                             ("decode_weights", (4096, bad, q, 1, 16, None, 32, o, 7)), ("evict", (4096, bad, 5, 1, 2, None, 7))):
            with pytest.raises((TypeError, ValueError)):
                getattr(pa.call, method)(entry["pa_" + method], *args)
    with pytest.raises(ValueError):
        pa.call.rotary_append(entry["pa_rotary_append"], 4096, 8192, triples, [1], q, 16, k, v, o, 1, 7)


def test_null_handles_are_refused(pa):
    h = C.c_void_p()
    assert pa.pa_rotary_create(None, None, C.byref(h)) == -1 and pa.pa_rotary_freqs(None, None, None) == -1
    assert pa.pa_rotary_destroy(None) == 0
    assert pa.pa_rotary_apply(None, None, 0, 0, 0, 0, None, 0, 0, None, 0, 0, 0, None) == -1
    assert pa.pa_rotary_append(None, None, None, 0, None, None, 0, 0, None, None, 0, None, 0, 0, None) == -1
    assert pa.pa_decode_shared(None, None, 0, 0, 0, None, 0, None, 0, 0, 0, None, 0, 0, None, 0, None) == -1
    assert pa.pa_decode_weights(None, None, 0, None, 0, 0, 0, None, 0, 0, None, 0, None) == -1
    assert pa.pa_layer_track_weights(None) == -1 and pa.pa_weights_ptr(None) is None and pa.pa_weights_clear(None, 0, None) == -1
    assert pa.pa_evict(None, None, 0, 0, 0, 0, None, None) == -1


def test_the_host_refuses_what_does_not_fit():
    class Calls:
        def __getattr__(self, name):
            return lambda *a: pytest.fail(f"{name} was called")

    eng = object.__new__(AttnEngine)                                  # an engine without a device: nothing may reach the library
    eng.cfg = AttnConfig(n_heads=4, n_kv_heads=2, head_dim=64, n_rot=64, rope_theta=1e4, max_seq=32, act_dtype=torch.float32)
    eng.device, eng.layers, eng._call, eng.ctx, eng.slots, eng._xc_keep = 0, [C.c_void_p(8)], Calls(), None, {}, None
    eng._f_rot_append = eng._f_shared = eng._f_weights = 0
    rot = object.__new__(Rotary)
    rot.eng, rot.handle, rot._h, rot._apply, rot._f_apply = eng, C.c_void_p(8), 8, Calls(), 0
    q, kv = torch.zeros((2, 256)), torch.zeros((2, 128))             # of another device than the engine's
    for call in (lambda: rot.apply(q, 4), lambda: eng.rotary_append(0, rot, [(0, 0, 2)], q, kv, kv, q_out=q), lambda: eng.decode_shared(0, None, 0, 0, [(0, 1), (0, 2)], q, out=q),
                 lambda: eng.decode_weights(0, [(0, 1), (0, 2)], q, out=q)):
        with pytest.raises(PaError):
            call()
    eng._q_dim, eng._kv_dim, eng.device = 256, 128, -1                                                 # ... of the same: the shapes
    meta = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt)
    for call in (lambda: rot.apply(q, 5, out=meta(2, 320)), lambda: rot.apply(q, 4, out=meta(1, 256)), lambda: rot.apply(q, 4, positions=meta(2), out=q),
                 lambda: rot.apply(q, 4, positions=meta(3, dt=torch.int32), out=q), lambda: rot.apply(q.t(), 4, out=q),
                 lambda: eng.rotary_append(0, rot, [(0, 0, 1)], q, kv, kv, q_out=q), lambda: eng.rotary_append(0, rot, [(0, 0, 2)], q.half(), kv, kv, q_out=q),
                 lambda: eng.rotary_append(0, rot, [(0, 0, 2)], q, kv, meta(2, 136)[:, :128], q_out=q), lambda: eng.rotary_append(0, rot, [(0, 0, 2)], q, kv[:, :64], kv, q_out=q),
                 lambda: eng.decode_shared(0, None, 0, 0, [(0, 1)], q, out=q), lambda: eng.decode_shared(0, None, 0, 0, [(0, 1), (0, 2)], q, out=q[:, :128]),
                 lambda: eng.decode_weights(0, [(0, 1), (0, 2)], q, gate=q.half(), out=q), lambda: eng.decode_weights(0, [(0, 1), (0, 2)], q, out=q.half()),
                 lambda: eng.decode_weights(0, [(0, 1), (0, 2)], q, q_head_stride=128, out=q)):
        with pytest.raises(PaError):
            call()
    eng.layers = []


class NoCalls:
    def __getattr__(self, name):
        return lambda *a: pytest.fail(f"{name} was called")


@pytest.fixture
def detached():
    """An engine of 4/2 heads of 64 and a rotation that have no device (tensors of the host pass for the engine's): nothing may reach the library."""
    eng = object.__new__(AttnEngine)
    eng.cfg = AttnConfig(n_heads=4, n_kv_heads=2, head_dim=64, n_rot=64, rope_theta=1e4, max_seq=32, act_dtype=torch.float32)
    eng.device, eng.layers, eng._call, eng.ctx, eng.slots, eng._xc_keep, eng._q_dim, eng._kv_dim = -1, [C.c_void_p(8)], NoCalls(), None, {}, None, 256, 128
    eng._f_rot_append = eng._f_shared = eng._f_weights = eng._f_evict = 0
    eng._raw_st = lambda: 0
    rot = object.__new__(Rotary)
    rot.eng, rot.handle, rot._h, rot._apply, rot._f_apply = eng, C.c_void_p(8), 8, NoCalls(), 0
    yield eng, rot
    eng.layers = []


@pytest.mark.parametrize("width,head_stride", [(64, None), (128, None), (255, None), (256, 128), (447, 128)])
def test_a_q_that_does_not_hold_its_heads_is_refused_ahead_of_an_append(detached, width, head_stride):
    eng, rot = detached
    kv, out = torch.zeros((2, 128)), torch.zeros((2, 256))
    with pytest.raises(PaError):
        eng.rotary_append(0, rot, [(0, 0, 2)], torch.zeros((2, width)), kv, kv, q_head_stride=head_stride, q_out=out)


@pytest.mark.parametrize("stride", [-1, -64, -2 ** 40])
def test_heads_ahead_of_their_column_are_refused(detached, stride):
    # a negative stride would pass for one that fits and become an address ahead of the tensor
    eng, rot = detached
    q, kv, out = torch.zeros((2, 256)), torch.zeros((2, 128)), torch.zeros((2, 256))
    pairs = [(0, 1), (0, 2)]
    for call in (lambda: rot.apply(q, 4, head_stride=stride, out=out), lambda: rot.apply(q, 4, out=out, out_head_stride=stride), lambda: rot.apply(q, 4, head_stride=stride, out=q),
                 lambda: eng.rotary_append(0, rot, [(0, 0, 2)], q, kv, kv, q_head_stride=stride, q_out=out), lambda: eng.decode_shared(0, None, 0, 0, pairs, q, out=out, q_head_stride=stride),
                 lambda: eng.decode_shared(0, None, 0, 0, pairs, q, gate=q, out=out, gate_head_stride=stride), lambda: eng.decode_weights(0, pairs, q, out=out, q_head_stride=stride),
                 lambda: eng.decode_weights(0, pairs, q, gate=q, out=out, gate_head_stride=stride)):
        with pytest.raises(PaError):
            call()


@pytest.mark.parametrize("by_module", [True, False])
def test_integers_past_their_width_are_refused(pa, by_module):
    # wrapped, 2^32 + 5 rows to keep would be 5, position 2^31 would turn the other way
    calls = pa.call if by_module else L.CtypesCalls(NoCalls())
    never = C.CFUNCTYPE(C.c_int)(lambda: pytest.fail("the library was called"))
    fn = C.cast(never, C.c_void_p).value
    q, k, o, p = torch.zeros((3, 64)), torch.zeros((3, 16)), torch.zeros((3, 64)), torch.zeros((2, 2, 5), dtype=torch.int32)
    pairs, triples = [(0, 5), (2, 6), (1, 0)], [(3, 7, 1), (0, 9, 2)]
    good = {
        "rotary_apply": (4096, q, 0, 16, 4, None, 0, o, 1, 16, 7), "rotary_append": (4096, 8192, triples, [1, 2], q, 16, k, k, o, 1, 7),
        "decode_shared": (4096, 8192, 2, 100, 50, pairs, q, 1, 16, q, 32, o, 7), "decode_weights": (4096, pairs, q, 1, 16, q, 32, o, 7),
        "evict": (4096, triples, 5, 1, 2, p, 7), "attn_layer": (4096, 1, 77, 2, q, 32, k, k, q, 32, None, o, 5), "attn_items": (4096, pairs, q, 32, k, k, q, 64, o, 0, 5),
        "rope_append": (4096, 1, 77, q, 32, k, k, None, o, 5), "decode_gather": (4096, 1, p, 9, q, 1, 32, q, 64, o, 5)}
    wide = {"rotary_apply": (3, 8 + 1), "rotary_append": (5,), "decode_shared": (8, 10), "decode_weights": (4, 6), "evict": (), "attn_layer": (5, 9), "attn_items": (3, 7), "rope_append": (4,),
            "decode_gather": (6, 8)}                               # places of head strides, 64 bits
    narrow = {"rotary_apply": (4,), "rotary_append": (), "decode_shared": (2, 3, 4), "decode_weights": (), "evict": (2, 3, 4), "attn_layer": (1, 2, 3), "attn_items": (),
              "rope_append": (1, 2), "decode_gather": (1, 3)}
    places = {"rotary_append": 2, "decode_shared": 5, "decode_weights": 1, "evict": 1, "attn_items": 1}       # of the items

    def refused(method, args):
        with pytest.raises(L.PaError) as e:
            getattr(calls, method)(fn, *args)
        assert e.value.code == -1

    for method, args in good.items():
        for places_of, values in ((wide, (-1, -64, 2 ** 64, 2 ** 64 + 16)), (narrow, (-1, 2 ** 32, 2 ** 32 + 5, -2 ** 40, 2 ** 70))):
            for i in places_of[method]:
                for bad in values:
                    refused(method, (*args[:i], bad, *args[i + 1:]))
        if method in places:
            i = places[method]
            for k_ in range(len(args[i][0])):
                for bad in (-1, 2 ** 32, 2 ** 32 + 1):
                    item = list(args[i][0])
                    item[k_] = bad
                    refused(method, (*args[:i], [tuple(item), *args[i][1:]], *args[i + 1:]))
    for bad in (2 ** 31, -2 ** 31 - 1, 2 ** 32, 2 ** 64):
        refused("rotary_apply", (*good["rotary_apply"][:6], bad, *good["rotary_apply"][7:]))
    for bad in ([1, 2 ** 32], [-1, 2]):
        refused("rotary_append", (4096, 8192, triples, bad, q, 16, k, k, o, 1, 7))


def test_integers_of_the_other_calls_are_refused_too(detached):
    eng, _ = detached
    eng.L = NoCalls()
    for call in (lambda: eng.clear_weights(0, 2 ** 32), lambda: eng.clear_weights(0, -1), lambda: eng.rotary(n_rot=2 ** 32 + 64), lambda: eng.rotary(original=-1),
                 lambda: eng.decode(0, [(0, 2 ** 32 + 5, 1)], torch.zeros((1, 256)), out=torch.zeros((1, 256)))):
        with pytest.raises(PaError):
            call()
