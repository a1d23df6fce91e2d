"""Places of the batch are served in order; how a server goes on behind one that has to wait."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def step(kv, dev, n_new, rows=400):
    s = kv.new_step(rows)
    kv.plan(torch.tensor(n_new, dtype=torch.int32, device=dev), s)
    return kv.state.tolist(), s.kv_len.tolist()


def test_a_prompt_that_waits_lets_others_go_on_when_it_is_planned_with_nothing(sqa, dev):
    kv = sqa.PagedKvCache(1, 256, 1, 10, 16, 4, 20, device=dev)
    state, lens = step(kv, dev, [0, 16, 15, 100])        # 1 + 1 + 7 of 10 pages
    assert state[1:3] == [1, 0] and lens == [0, 16, 15, 100]
    state, lens = step(kv, dev, [90, 1, 1, 1])            # 6 pages wanted at place 0, 1 free
    assert state[1:3] == [1, 2] and lens == [0, 0, 16, 101]  # place 1 is at a page's end, 2 and 3 are not
    state, lens = step(kv, dev, [90, 1, 0, 0])            # asked again: refused again
    assert state[1:3] == [1, 2] and lens == [0, 0, 16, 101]
    state, lens = step(kv, dev, [0, 1, 0, -1])            # place 0 waits: 1 goes on, 3 ends
    assert state[1:3] == [7, 0] and lens == [0, 17, 16, 0]
    state, lens = step(kv, dev, [90, 1, 0, 0])            # 7 free pages cover its 6
    assert state[1:3] == [1, 0] and lens == [90, 18, 16, 0]


def test_places_behind_one_that_passes_the_rows(sqa, dev):
    kv = sqa.PagedKvCache(1, 256, 1, 40, 16, 4, 20, device=dev)
    assert step(kv, dev, [3, 3, 3, 3])[1] == [3, 3, 3, 3]
    state, lens = step(kv, dev, [5, 30, 0, 1], rows=32)   # 5, 35, 35 and 36 rows of 32
    assert state[2] == 3 and lens == [8, 0, 0, 0]
    assert kv.n_past.tolist() == [8, 3, 3, 3]
    state, lens = step(kv, dev, [5, 26, 0, 1], rows=32)
    assert state[2] == 0 and lens == [13, 29, 3, 4]
