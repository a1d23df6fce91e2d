"""PagedKvCache's calls run on its own device, whatever the current one is (no GPU needed)."""
import contextlib

import pytest
import torch


@pytest.mark.parametrize("method", ["plan", "append", "attend"])
def test_calls_switch_to_the_device_of_the_cache(sqa, monkeypatch, method):
    kv = sqa.PagedKvCache(1, 256, 2, 4, 16, 2, 2, device="cpu")
    step = kv.new_step(3)
    inside, seen = [], []

    @contextlib.contextmanager
    def device(d):
        inside.append(torch.device(d))
        yield
        inside.pop()

    def call(*args, **kw):
        seen.append(list(inside))
        return step

    monkeypatch.setattr(torch.cuda, "device", device)
    if method == "plan":
        monkeypatch.setattr(sqa, "paged_plan", call)
        kv.plan(torch.zeros(2, dtype=torch.int32), step)
    elif method == "append":
        monkeypatch.setattr(sqa, "set_rows_q4_0", call)
        kv.append(0, torch.zeros(3, 512), torch.zeros(3, 512), step)
    else:
        with pytest.raises(sqa.SqaError):  # paged_attn takes care of it by itself, and refuses the CPU's tensors
            kv.attend(0, torch.zeros(3, 16, 256), step, 1)
        return
    assert seen and all(s == [torch.device("cpu")] for s in seen)
