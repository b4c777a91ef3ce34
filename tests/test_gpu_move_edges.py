"""pa_cache_move at its edges: items and lists that move no row, wherever their rows would lie, and an order of tiles whose wait runs out."""
import pytest
import torch

from pooled_b200 import PaError
from tests.test_gpu_move import arrays, engine, expected, fill, same

pytestmark = pytest.mark.gpu

FORMATS = [("f16", 2, 256, True), ("q8", 2, 64, False), ("f32", 1, 128, False)]


@pytest.mark.parametrize("kv,nKV,hd,track", FORMATS)
@pytest.mark.parametrize("items", [
    [(0, 0, 1, 0, 100), (1, 50, 2, 0, 0)],                                # its source inside another's destination,
    [(0, 0, 1, 0, 100), (2, 50, 1, 50, 0)],                               # its destination,
    [(0, 0, 1, 0, 100), (2, 0, 0, 50, 0)],                                # its destination inside another's source
    [(1, 50, 2, 0, 0), (2, 50, 1, 60, 0), (0, 0, 1, 0, 100), (2, 0, 0, 50, 0), (0, 40, 0, 70, 0)],
    [(0, 20, 0, 10, 700), (0, 30, 0, 40, 0)],                             # among rows that move over one another
    [(0, 10, 0, 10, 0), (0, 5, 0, 15, 40)],
    [(0, 5, 1, 5, 0), (0, 5, 1, 5, 0)]])
def test_items_without_rows_meet_nothing(kv, nKV, hd, track, items):
    eng = engine(nKV, hd, 800, 3, kv, layers=2)
    if track:
        eng.track_weights(0)
    fill(eng, 1)
    want = expected(eng, items)
    eng.move(items)
    assert same(eng, want)


@pytest.mark.parametrize("items", [[(0, 0, 1, 0, 100), (0, 0, 1, 50, 100)], [(0, 0, 1, 0, 100), (1, 50, 0, 20, 60)], [(0, 10, 0, 30, 60)]])
def test_lists_without_room_for_a_row_move_nothing(items):
    # one word a list: its count, of rows that it has no offsets for.  Sources and destinations may then lie anywhere
    eng = engine(2, 256, 200, 2)
    fill(eng, 2)
    want = expected(eng, [])
    eng.move(items, lists=torch.full((len(items), 1), 7, dtype=torch.int32, device="cuda"))
    assert same(eng, want)


def test_spans_that_do_meet_are_refused_beside_items_without_rows():
    eng = engine(2, 256, 200, 3)
    fill(eng, 3)
    want = expected(eng, [])
    empty = (0, 50, 1, 50, 0)
    for items in ([(0, 0, 1, 0, 100), (1, 99, 2, 0, 1)], [(0, 0, 1, 0, 100), (2, 0, 1, 99, 1)], [(0, 0, 1, 0, 100), (2, 0, 0, 0, 1)], [(0, 0, 1, 0, 100), (2, 0, 0, 99, 1)],
                  [(0, 0, 1, 0, 1), (2, 0, 1, 0, 1)]):
        for at in range(3):
            with pytest.raises(PaError):
                eng.move(items[:at] + [empty] + items[at:])
    for bad in ((0, 201, 1, 0, 0), (0, 0, 1, 201, 0), (3, 0, 1, 0, 0), (0, 0, 3, 0, 0)):
        with pytest.raises(PaError):
            eng.move([(0, 0, 1, 0, 10), bad])
    assert same(eng, want)
    items = [(0, 0, 1, 0, 100), (1, 100, 2, 0, 1), (2, 10, 1, 101, 20), empty]         # neighbours do not meet
    want = expected(eng, items)
    eng.move(items)
    assert same(eng, want)


def test_lists_without_words_are_refused():
    # (an empty tensor has no address: without the check the call would be one without lists, which moves whole items)
    eng = engine(2, 256, 100, 2)
    fill(eng, 4)
    want = expected(eng, [])
    with pytest.raises(PaError):
        eng.move([(0, 0, 1, 0, 50)], lists=torch.empty((1, 0), dtype=torch.int32, device="cuda"))
    assert same(eng, want)


@pytest.mark.parametrize("up,listed", [(False, False), (True, False), (False, True)])
def test_a_wait_that_runs_out_overwrites_no_row_that_was_not_read(up, listed):
    # one look for the neighbour's tile: the call comes back by itself with a status, every word is the one that was there or the one that belongs
    # there, and after a reset moves are right again
    eng = engine(4, 256, 20000, 1)
    n = 19999
    if listed:
        kept = [i for i in range(20000) if i % 3]
        items, lists = [(0, 0, 0, 0, 20000)], [[len(kept), *kept]]
        on_device = torch.tensor(lists, dtype=torch.int32, device="cuda")
    else:
        items, lists, on_device = [(0, 0, 0, 1, n) if up else (0, 1, 0, 0, n)], None, None
    ran_out = 0
    for trial in range(40):
        fill(eng, trial)
        was, want = expected(eng, []), expected(eng, items, lists)
        eng.set_wait_limit(1)
        eng.move(items, lists=on_device)
        try:
            eng.sync()
        except PaError as e:
            assert e.code == -5                                            # PA_ETIMEOUT
            ran_out += 1
            with pytest.raises(PaError) as latched:
                eng.move(items, lists=on_device)
            assert latched.value.code == -6                                # PA_ESTATE
            eng.reset()
            for layer, b, w in zip(arrays(eng), was, want):
                for x, y, z in zip(layer, b, w):
                    assert torch.all((x == y) | (x == z))
        else:
            assert same(eng, want)
        eng.set_wait_limit(0)
        if ran_out == 3:
            break
    assert ran_out
    fill(eng, 99)
    for _ in range(2):
        want = expected(eng, items, lists)
        eng.move(items, lists=on_device)
        assert same(eng, want)
