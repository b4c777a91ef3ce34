"""Lists of AttnEngine.move that hold no word, without a GPU: an empty tensor has no address, and a call without lists moves whole items."""
import ctypes as C

import pytest
import torch

from pooled_b200 import AttnConfig, AttnEngine, PaError


class NoCalls:
    def __getattr__(self, name):
        return lambda *a: pytest.fail(f"{name} was called")


@pytest.mark.parametrize("n", [1, 2])
def test_lists_without_words_are_refused(n):
    eng = object.__new__(AttnEngine)
    eng.cfg = AttnConfig(n_heads=4, n_kv_heads=2, head_dim=64, n_rot=64, rope_theta=1e4, max_seq=32, act_dtype=torch.float32)
    eng.device, eng.layers, eng._call, eng.ctx, eng.slots, eng._xc_keep = -1, [C.c_void_p(8), C.c_void_p(16)], NoCalls(), None, {}, None
    eng._f_move, eng._all_layers = 0, None
    eng._raw_st = lambda: 0
    try:
        lists = torch.zeros((n, 0), dtype=torch.int32)
        assert lists.data_ptr() == 0
        with pytest.raises(PaError):
            eng.move([(0, 0, 1, 8 * i, 4) for i in range(n)], lists)
    finally:
        eng.layers = []
