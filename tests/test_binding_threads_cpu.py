"""The compiled binding is set up once, however many threads ask for it first."""
import threading
import time
import types

import torch

from test_serving_cpu import _lib


def test_threads_set_the_binding_up_once(monkeypatch, tmp_path):
    import sys

    import atflash
    ffi, _ = _lib()
    inits = []

    def init(*args):
        inits.append(args)
        time.sleep(0.05)  # another thread's turn

    fake = types.SimpleNamespace(torch_version=torch.__version__, version=ffi.ATF_VERSION, init=init)
    (tmp_path / "there").write_text("")
    monkeypatch.setattr(ffi, "_bind", None)
    monkeypatch.setattr(ffi, "_BINDING_PATH", str(tmp_path / "there"))
    monkeypatch.setitem(sys.modules, "atflash._binding", fake)
    monkeypatch.setattr(atflash, "_binding", fake, raising=False)
    got, start = [], threading.Barrier(8)

    def ask():
        start.wait()
        got.append(ffi.binding())

    threads = [threading.Thread(target=ask) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(inits) == 1 and got == [fake] * 8
