"""A plan's device tensors are recorded once with each stream that a run uses them on."""
from types import SimpleNamespace

import torch


def test_every_stream_of_a_run_is_recorded_once(monkeypatch):
    from atflash import _runtime
    now, seen = {"raw": 7}, []
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda idx: now["raw"], raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda idx: ("stream", idx, now["raw"]))
    tensors = [SimpleNamespace(record_stream=lambda s, i=i: seen.append((i, s))) for i in range(3)]
    held = _runtime.PlanTensors(torch.device("cuda", 2), *tensors)
    held.use()
    held.use()
    assert seen == [(i, ("stream", 2, 7)) for i in range(3)]
    now["raw"] = 9
    held.use()
    now["raw"] = 7
    held.use()
    assert seen[3:] == [(i, ("stream", 2, 9)) for i in range(3)]
