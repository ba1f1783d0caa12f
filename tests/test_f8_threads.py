"""Two threads' first products with one weight."""
import ctypes
import threading
import time

import torch

from litellmengine_b200.csrc import ops


def test_a_weight_is_described_once(monkeypatch):
    """What the kernels' launches read is on the host, at the address that `described` gives: it has to outlive the call, whoever else asks for it meanwhile."""
    made = []

    def describe(room, *rest):
        made.append(room)
        time.sleep(0.2)                                           # the other thread gets here, as it does while a library call is under way
        ctypes.memset(room, 7, 64)
        return 0

    monkeypatch.setattr(ops, "_mx_call", lambda name: (lambda: 64) if name == "llm_f8_weight_size" else describe)
    w, got = ops.F8Weight((32, 64), False, torch.device("cpu")), []
    threads = [threading.Thread(target=lambda: got.append(w.described())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and got == made * 4 and w.described() == made[0]
    assert ctypes.string_at(made[0], 64) == b"\x07" * 64
    w.buffer = w.buffer.clone()                                   # at another address: described again
    assert w.described() == made[1] and len(made) == 2
