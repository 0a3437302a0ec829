"""The paged prefill's wrapper between threads: a run keeps the plan that it began with
until its call has returned, whatever plan() another thread makes meanwhile."""
import gc
import types
import weakref

import torch

from test_serving_cpu import _lib


class Held:
    """Stands for a plan's device tensors."""

    def __init__(self, *tensors):
        self.used = 0

    def use(self):
        self.used += 1


def test_a_run_keeps_its_plan_while_another_thread_plans(monkeypatch):
    ffi, _ = _lib()
    from atflash import _runtime, paged
    monkeypatch.setattr(_runtime, "PlanTensors", Held)
    monkeypatch.setattr(_runtime, "error_flag", lambda dev: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda dev: types.SimpleNamespace(multi_processor_count=148))
    w = object.__new__(paged.BatchPrefillWithPagedKVCacheWrapper)
    w._ws, w._dev, w._kv_layout = torch.empty(1 << 20, dtype=torch.uint8), torch.device("cpu"), "NHD"
    w._plan = w._planned = None
    plan = lambda tokens: w.plan([0, tokens], [0, 1], [0], [5], 4, 2, 128, 16)
    seen = []

    def paged_run(address, *args):
        first = weakref.ref(w._plan)
        plan(3)  # what another thread does between the plan's address and the end of the call
        gc.collect()
        # the address still leads to the plan that the run began with
        assert first() is not None
        seen.append(ffi.AtfPrefillPagedParams.from_address(address).total_q)
        return "out"

    monkeypatch.setattr(ffi, "binding", lambda: types.SimpleNamespace(paged_run=paged_run))
    plan(2)
    kv = torch.zeros(1)
    assert w.run(kv, (kv, kv)) == "out" and w.run(kv, (kv, kv)) == "out"
    assert seen == [2, 3]
