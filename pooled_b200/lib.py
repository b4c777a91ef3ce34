"""ctypes binding of libpooled_attn.so (include/pooled_attn.h).  Fails loudly when the library is missing."""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import operator
import os
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
SO_PATH = os.path.join(HERE, "libpooled_attn.so")
CALL_PATH = os.path.join(HERE, "_pa_call" + sysconfig.get_config_var("EXT_SUFFIX"))   # of this interpreter's ABI only

PA_F32, PA_F16 = 0, 1
PA_ROPE_NONE, PA_ROPE_F64, PA_ROPE_TABLE = 0, 1, 2
PA_KV_F16, PA_KV_Q8, PA_KV_F32 = 0, 1, 2
PA_FLAG_FAST = 1
PA_ROPE_HALF, PA_ROPE_INTERLEAVED = 0, 1
PA_ROPE_SCALE_NONE, PA_ROPE_SCALE_LINEAR, PA_ROPE_SCALE_NTK, PA_ROPE_SCALE_YARN, PA_ROPE_SCALE_BANDS = 0, 1, 2, 3, 4
PA_ROPE_AXES_BLOCKS, PA_ROPE_AXES_CYCLED, PA_ROPE_AXES_OWN = 0, 1, 2
PA_MODE_AUTO, PA_MODE_DECODE, PA_MODE_PREFILL = 0, 1, 2
STATUS = {0: "PA_OK", -1: "PA_EINVAL", -2: "PA_EUNSUPPORTED", -3: "PA_ENOMEM", -4: "PA_ECUDA", -5: "PA_ETIMEOUT", -6: "PA_ESTATE"}


class PaError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{STATUS.get(code, code)}: {msg}")
        self.code = code


class PaConfig(C.Structure):
    _fields_ = [("n_heads", C.c_uint32), ("n_kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("n_rot", C.c_uint32),
                ("rope_theta", C.c_double), ("rope_mode", C.c_uint32), ("act_dtype", C.c_uint32), ("max_cols", C.c_uint32),
                ("splits", C.c_uint32), ("flags", C.c_uint32), ("reserved", C.c_uint32 * 5)]


class PaItem(C.Structure):
    _fields_ = [("seq", C.c_uint32), ("pos", C.c_uint32), ("n_cols", C.c_uint32), ("reserved", C.c_uint32)]


class PaRotaryConfig(C.Structure):
    _fields_ = [("n_rot", C.c_uint32), ("layout", C.c_uint32), ("scaling", C.c_uint32), ("original", C.c_uint32), ("theta", C.c_double),
                ("factor", C.c_double), ("fast", C.c_double), ("slow", C.c_double), ("mscale", C.c_double), ("reserved", C.c_uint32 * 4)]


class PaRotaryAxes(C.Structure):
    _fields_ = [("n_axes", C.c_uint32), ("order", C.c_uint32), ("pairs", C.c_uint32 * 4), ("reserved", C.c_uint32 * 2)]


class PaMoveItem(C.Structure):
    _fields_ = [("src_seq", C.c_uint32), ("src_row", C.c_uint32), ("dst_seq", C.c_uint32), ("dst_row", C.c_uint32), ("n_rows", C.c_uint32), ("reserved", C.c_uint32)]


class PaEvictItem(C.Structure):
    _fields_ = [("src_seq", C.c_uint32), ("dst_seq", C.c_uint32), ("n_rows", C.c_uint32), ("reserved", C.c_uint32)]


class PaStats(C.Structure):
    _fields_ = [("kernel_launches", C.c_uint64), ("kv_bytes_streamed", C.c_uint64), ("calls", C.c_uint64)]


# name -> (restype, argtypes): every symbol include/pooled_attn.h declares
_vp, _u32, _u64, _i, _sz = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int, C.c_size_t
SYMBOLS = {
    "pa_create": (_i, [_i, C.POINTER(PaConfig), C.POINTER(_vp)]),
    "pa_destroy": (_i, [_vp]),
    "pa_layer_create": (_i, [_vp, _u32, _u32, C.POINTER(_vp)]),
    "pa_layer_create_fmt": (_i, [_vp, _u32, _u32, _i, C.POINTER(_vp)]),
    "pa_layer_destroy": (_i, [_vp]),
    "pa_layer_set_origin": (_i, [_vp, _u32]),
    "pa_layer_set_next": (_i, [_vp, _vp]),
    "pa_cache_ptr": (_vp, [_vp, _i]),
    "pa_cache_export": (_i, [_vp, _u32, _u32, _u32, _i, _vp, C.POINTER(_u32), _vp]),
    "pa_cache_import": (_i, [_vp, _u32, _u32, _u32, _i, _vp, C.POINTER(_u32), _vp]),
    "pa_slot_save": (_i, [_vp, _u32, _u32, C.POINTER(_vp), _vp]),
    "pa_slot_load": (_i, [_vp, _u32, _vp, C.POINTER(_u32), _vp]),
    "pa_slot_export": (_i, [_vp, _i, _vp, _vp]),
    "pa_slot_info": (_i, [_vp, C.POINTER(_u32), C.POINTER(_u32), C.POINTER(_u32)]),
    "pa_slot_drop": (_i, [_vp]),
    "pa_last_error": (C.c_char_p, [_vp]),
    "pa_version": (C.c_char_p, []),
    "pa_sync": (_i, [_vp, _vp]),
    "pa_reset": (_i, [_vp]),
    "pa_alloc": (_i, [_vp, _sz, C.POINTER(_vp)]),
    "pa_free": (_i, [_vp, _vp]),
    "pa_alloc_host": (_i, [_vp, _sz, C.POINTER(_vp)]),
    "pa_free_host": (_i, [_vp, _vp]),
    "pa_upload": (_i, [_vp, _vp, _vp, _sz, _vp]),
    "pa_download": (_i, [_vp, _vp, _vp, _sz, _vp]),
    "pa_dec_config": (_u32, [_u32, _u32, _u32, _u32]),
    "pa_dec_split_len": (_u32, [_u32, _u32]),
    "pa_dec_splits": (_u32, [_u32, _u32]),
    "pa_tile_split_len": (_u32, [_u32, _u32, _u32, _u32]),
    "pa_plan_splits": (_u32, [_vp, _u32, _u32]),
    "pa_rope": (_i, [_vp, _vp, _u64, _u64, _u32, _u32, _u32, _vp, _vp, _u64, _vp]),
    "pa_kv_append": (_i, [_vp, _u32, _u32, _u32, _vp, _vp, _u64, _i, _vp]),
    "pa_rope_append": (_i, [_vp, _u32, _u32, _u32, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _vp, _vp]),
    "pa_rope_append_items": (_i, [_vp, _vp, _u32, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _vp]),
    "pa_decode": (_i, [_vp, C.POINTER(PaItem), _u32, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_decode_gather": (_i, [_vp, _u32, _u32, _vp, _u32, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_decode_partial": (_i, [_vp, C.POINTER(PaItem), _u32, _vp, _i, _u64, _u64, _vp, _vp]),
    "pa_merge": (_i, [_vp, _vp, _u32, _u32, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_exchange_bytes": (_sz, [_vp, _u32, _u32]),
    "pa_shared_alloc": (_i, [_vp, _sz, C.POINTER(_vp), _vp]),
    "pa_shared_open": (_i, [_vp, _vp, C.POINTER(_vp)]),
    "pa_shared_close": (_i, [_vp, _vp]),
    "pa_exchange_init": (_i, [_vp, _u32, _u32, C.POINTER(_vp), _u32]),
    "pa_decode_exchange": (_i, [_vp, C.POINTER(PaItem), _u32, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_attn_items": (_i, [_vp, _vp, _u32, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _u64, _u64, _vp, _u64, C.c_int, _vp]),
    "pa_attn_layer_sharded": (_i, [_vp, _u32, _u32, _u32, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _u64, _u64, _vp, _vp, _u64, _vp]),
    "pa_prefill": (_i, [_vp, _u32, _u32, _u32, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_sigmoid_mul": (_i, [_vp, _vp, _u64, _vp, _u64, _u64, _u32, _vp]),
    "pa_layer_set_head_norm": (_i, [_vp, _vp, _vp, C.c_double]),
    "pa_head_norm": (_i, [_vp, _vp, _u64, _u64, _u32, _u32, _vp, C.c_double, _vp, _u64, _u64, _vp]),
    "pa_attn_layer": (_i, [_vp, _u32, _u32, _u32, _i, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _u64, _u64, _vp, _vp, _u64, _vp]),
    "pa_attn_layer_host": (_i, [_vp, _u32, _u32, _u32, _i, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _u64, _u64, _vp, _vp, _u64, _vp]),
    "pa_attn_step_host": (_i, [C.POINTER(_vp), _u32, _u32, _u32, _u32, _i, _vp, _u64, _u64, _u64, _vp, _vp, _u64, _u64, _vp, _u64, _u64, _u64, _vp, _u64, _u64, _vp]),
    "pa_decode_static": (_i, [_i, _vp, _vp, _u32, _u32, _u32, _u32, _u32, _u32, _vp, _vp, _vp, _vp, C.c_char_p, _sz]),
    "pa_decode_static_status": (_i, [_i, _vp, C.POINTER(_u32)]),
    "pa_rotary_create": (_i, [_vp, C.POINTER(PaRotaryConfig), C.POINTER(_vp)]),
    "pa_rotary_create_axes": (_i, [_vp, C.POINTER(PaRotaryConfig), C.POINTER(PaRotaryAxes), C.POINTER(_vp)]),
    "pa_rotary_destroy": (_i, [_vp]),
    "pa_rotary_freqs": (_i, [_vp, C.POINTER(C.c_double), C.POINTER(C.c_double)]),
    "pa_rotary_apply": (_i, [_vp, _vp, _i, _u64, _u64, _u32, _vp, C.c_int32, _u32, _vp, _i, _u64, _u64, _vp]),
    "pa_rotary_append": (_i, [_vp, _vp, _vp, _u32, _vp, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _i, _u64, _vp]),
    "pa_rotary_append_at": (_i, [_vp, _vp, _vp, _u32, _vp, _vp, _vp, _u64, _u64, _vp, _vp, _u64, _vp, _i, _u64, _vp]),
    "pa_decode_tree": (_i, [_vp, _vp, _u32, _vp, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_cache_move": (_i, [_vp, _u32, _vp, _u32, _vp, _u32, _vp]),
    "pa_decode_shared": (_i, [_vp, _vp, _u32, _u32, _u32, _vp, _u32, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_layer_track_weights": (_i, [_vp]),
    "pa_weights_ptr": (_vp, [_vp]),
    "pa_weights_clear": (_i, [_vp, _u32, _vp]),
    "pa_decode_weights": (_i, [_vp, _vp, _u32, _vp, _i, _u64, _u64, _vp, _u64, _u64, _vp, _u64, _vp]),
    "pa_evict": (_i, [_vp, _vp, _u32, _u32, _u32, _u32, _vp, _vp]),
    "pa_set_wait_limit": (_i, [_vp, _u32]),
    "pa_get_stats": (_i, [_vp, C.POINTER(PaStats)]),
    "pa_timing_begin": (_i, [_vp, _u32]),
    "pa_set_core_only": (_i, [_vp, _i]),
    "pa_timing_end": (_i, [_vp, C.POINTER(C.c_double), C.POINTER(_u64)]),
}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fit(v, lo, hi, what):
    v = operator.index(v)
    if not lo <= v <= hi:
        raise PaError(-1, f"{v} is no {what}")
    return v


def u32(v) -> int:
    """v as a parameter of 32 bits: ctypes would wrap what does not fit."""
    return v if type(v) is int and 0 <= v <= 0xffffffff else _fit(v, 0, 0xffffffff, "unsigned 32-bit integer")


def i32(v) -> int:
    return _fit(v, -2 ** 31, 2 ** 31 - 1, "32-bit integer")


def u64(v) -> int:
    return _fit(v, 0, 2 ** 64 - 1, "unsigned 64-bit integer")


def _gate(t, head_stride):
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), u64(head_stride))


class CtypesCalls:
    """What csrc/pa_call.c does, by ctypes (`entry` is not needed: the functions are the library's)."""

    def __init__(self, lib):
        self.lib = lib

    def attn_layer(self, entry, layer, seq, pos, mode, q, q_head_stride, k, v, gate, gate_head_stride, cs_table, out, stream):
        return self.lib.pa_attn_layer(layer, u32(seq), u32(pos), u32(q.shape[0]), u32(mode), _ptr(q), q.stride(0), u64(q_head_stride), _ptr(k), _ptr(v), k.stride(0),
                                      *_gate(gate, gate_head_stride), _ptr(cs_table), _ptr(out), out.stride(0), stream)

    def attn_items(self, entry, layer, seqs_pos, q, q_head_stride, k, v, gate, gate_head_stride, out, exchange, stream):
        return self.lib.pa_attn_items(layer, self._items(seqs_pos, False), len(seqs_pos), _ptr(q), q.stride(0), u64(q_head_stride), _ptr(k), _ptr(v), k.stride(0),
                                      *_gate(gate, gate_head_stride), _ptr(out), out.stride(0), exchange, stream)

    def rope_append(self, entry, layer, seq, pos, q, q_head_stride, k, v, cs_table, q_rot, stream):
        return self.lib.pa_rope_append(layer, u32(seq), u32(pos), u32(q.shape[0]), _ptr(q), q.stride(0), u64(q_head_stride), _ptr(k), _ptr(v), k.stride(0), _ptr(cs_table),
                                       _ptr(q_rot), stream)

    def decode_gather(self, entry, layer, seq, lists, list_stride, q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream):
        return self.lib.pa_decode_gather(layer, u32(seq), u32(q.shape[0]), _ptr(lists), u32(list_stride), _ptr(q), q_dtype, q.stride(0), u64(q_head_stride),
                                         *_gate(gate, gate_head_stride), _ptr(out), out.stride(0), stream)

    def _items(self, items, n_cols=True):
        return (PaItem * max(1, len(items)))(*[PaItem(*map(u32, it), 0) if n_cols else PaItem(*map(u32, it), 1, 0) for it in items])

    def rotary_apply(self, entry, rotary, x, x_dtype, head_stride, n_heads, positions, pos, y, y_dtype, y_head_stride, stream):
        return self.lib.pa_rotary_apply(rotary, _ptr(x), x_dtype, x.stride(0), u64(head_stride), u32(n_heads), _ptr(positions), i32(pos), u32(x.shape[0]), _ptr(y), y_dtype,
                                        y.stride(0), u64(y_head_stride), stream)

    def rotary_append(self, entry, rotary, layer, items, rows, q, q_head_stride, k, v, q_out, q_out_dtype, stream):
        if rows is not None and len(rows) != len(items):
            raise ValueError("one row per item")
        r = None if rows is None else (C.c_uint32 * max(1, len(rows)))(*map(u32, rows))
        return self.lib.pa_rotary_append(rotary, layer, self._items(items), len(items), r, *_gate(q, q_head_stride), _ptr(k), _ptr(v), k.stride(0), _ptr(q_out),
                                         q_out_dtype, 0 if q_out is None else q_out.stride(0), stream)

    def rotary_append_at(self, entry, rotary, layer, items, rows, positions, q, q_head_stride, k, v, q_out, q_out_dtype, stream):
        if rows is not None and len(rows) != len(items):
            raise ValueError("one row per item")
        r = None if rows is None else (C.c_uint32 * max(1, len(rows)))(*map(u32, rows))
        return self.lib.pa_rotary_append_at(rotary, layer, self._items(items), len(items), r, _ptr(positions), *_gate(q, q_head_stride), _ptr(k), _ptr(v), k.stride(0),
                                            _ptr(q_out), q_out_dtype, 0 if q_out is None else q_out.stride(0), stream)

    def decode_tree(self, entry, layer, items, parents, q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream):
        return self.lib.pa_decode_tree(layer, self._items(items), len(items), _ptr(parents), _ptr(q), q_dtype, q.stride(0), u64(q_head_stride), *_gate(gate, gate_head_stride),
                                       _ptr(out), out.stride(0), stream)

    def cache_move(self, entry, layers, n_layers, items, lists, list_stride, stream):
        if any(len(it) != 5 for it in items):
            raise ValueError("the items are a sequence of (src_seq, src_row, dst_seq, dst_row, n_rows)")
        arr = (PaMoveItem * max(1, len(items)))(*[PaMoveItem(*map(u32, it), 0) for it in items])
        return self.lib.pa_cache_move(layers, u32(n_layers), arr, len(items), _ptr(lists), u32(list_stride), stream)

    def decode_shared(self, entry, layer, prefix_layer, prefix_seq, prefix_len, own_base, seqs_pos, q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream):
        return self.lib.pa_decode_shared(layer, prefix_layer, u32(prefix_seq), u32(prefix_len), u32(own_base), self._items(seqs_pos, False), len(seqs_pos), _ptr(q), q_dtype,
                                         q.stride(0), u64(q_head_stride), *_gate(gate, gate_head_stride), _ptr(out), out.stride(0), stream)

    def decode_weights(self, entry, layer, seqs_pos, q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream):
        return self.lib.pa_decode_weights(layer, self._items(seqs_pos, False), len(seqs_pos), _ptr(q), q_dtype, q.stride(0), u64(q_head_stride),
                                          *_gate(gate, gate_head_stride), _ptr(out), out.stride(0), stream)

    def evict(self, entry, layer, items, n_keep, n_first, n_recent, kept, stream):
        arr = (PaEvictItem * max(1, len(items)))(*[PaEvictItem(*map(u32, it), 0) for it in items])
        return self.lib.pa_evict(layer, arr, len(items), u32(n_keep), u32(n_first), u32(n_recent), _ptr(kept), stream)


class Lib:
    """The loaded shared library with typed entry points."""

    def __init__(self, path: str = SO_PATH):
        if not os.path.exists(path):
            raise PaError(-4, f"{path} is missing: build it with `python -m pooled_b200.build` (nvcc, sm_100a). "
                              "There is no CPU or PyTorch fallback for the attention path.")
        self.path = path
        self.dll = C.CDLL(path)
        for name, (res, args) in SYMBOLS.items():
            fn = getattr(self.dll, name)   # AttributeError when the library lacks a declared symbol
            fn.restype, fn.argtypes = res, args
            setattr(self, name, fn)
        self.call = self._load_call()

    def _load_call(self):
        """The CPython module with the per-layer calls (csrc/pa_call.c), which takes their addresses in this library from
        `entry`; the same calls through ctypes where it was not built for this interpreter."""
        self.entry = {n: C.cast(getattr(self.dll, n), C.c_void_p).value for n in
                      ("pa_attn_layer", "pa_attn_items", "pa_rope_append", "pa_decode_gather", "pa_rotary_apply", "pa_rotary_append", "pa_decode_shared",
                       "pa_decode_weights", "pa_evict", "pa_rotary_append_at", "pa_decode_tree", "pa_cache_move")}
        if not os.path.exists(CALL_PATH):
            return CtypesCalls(self)
        loader = importlib.machinery.ExtensionFileLoader("_pa_call", CALL_PATH)
        mod = importlib.util.module_from_spec(importlib.util.spec_from_file_location("_pa_call", CALL_PATH, loader=loader))
        loader.exec_module(mod)
        return mod

    def check(self, rc: int, ctx=None):
        if rc != 0:
            msg = self.pa_last_error(ctx)
            raise PaError(rc, msg.decode() if msg else "")


_lib: Lib | None = None


def load() -> Lib:
    global _lib
    if _lib is None:
        _lib = Lib()
    return _lib
