"""The native calls' signatures are declared before any thread makes a call (an undeclared one would pass a 64-bit stream handle as 32 bits)."""
import threading
import time

from deeplearning4j_amd.native import lib as L
from deeplearning4j_amd.ops import vocab_loss as VL


class _Function:
    def __init__(self):
        self._argtypes = None

    @property
    def argtypes(self):
        return self._argtypes

    @argtypes.setter
    def argtypes(self, types):
        time.sleep(0.05)                                                   # (wide open for another thread)
        self._argtypes = types


class _Library:
    def __init__(self):
        for name in ("dl4j_linear_loss_fwd", "dl4j_linear_loss_bwd", "dl4j_topk_distill", "dl4j_linear_loss_bytes"):
            setattr(self, name, _Function())


def test_no_thread_gets_the_library_with_undeclared_calls(monkeypatch):
    stub = _Library()
    monkeypatch.setattr(L, "hip", lambda: stub)
    monkeypatch.setattr(VL, "_LIB", None, raising=False)
    seen = []

    def call(delay):
        time.sleep(delay)
        lib = VL._lib()
        seen.append([f.argtypes is not None for f in vars(lib).values()])
    threads = [threading.Thread(target=call, args=(0.02 * k,)) for k in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen) == 6 and all(all(s) for s in seen)
