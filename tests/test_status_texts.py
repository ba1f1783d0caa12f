"""Every code that a kernel writes into a status word has words, and `check_status` says them."""
import os
import re
from types import SimpleNamespace

import pytest
import torch

from litellmengine_b200.csrc import ops
from litellmengine_b200.engine import runner as engine_runner

CSRC = os.path.dirname(ops.__file__)


def codes_written():
    text = {n: open(os.path.join(CSRC, n), encoding="utf-8").read() for n in sorted(os.listdir(CSRC)) if n.endswith((".cu", ".cuh", ".h"))}
    found = {}
    for name, t in text.items():
        for code in re.findall(r"atomicCAS\(status, 0, (\w+)\)", t):
            if not code.isdigit():
                code, = re.findall(rf"^#define {code} (\d+)$", t, re.M)
            found.setdefault(int(code), name)
    return found


def test_every_code_has_words():
    found = codes_written()
    assert {1, 4, 8, 9, 10, 11} <= set(found)
    for code, name in found.items():
        assert engine_runner.STATUS_TEXT.get(code) or ops.STREAM_STATUS_TEXT.get(code), (code, name)
    assert not set(engine_runner.STATUS_TEXT) & set(ops.STREAM_STATUS_TEXT)


@pytest.mark.parametrize("code", sorted(engine_runner.STATUS_TEXT) + [10])
def test_a_runner_says_them(monkeypatch, code):
    """Words on the host; nothing runs on a device."""
    step, products = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    monkeypatch.setattr(ops, "stream_status", lambda device: products)
    runner = engine_runner.ModelRunner.__new__(engine_runner.ModelRunner)
    runner.buffers, runner.device = SimpleNamespace(status=step), torch.device("cpu")
    for word in (step, products):
        word.copy_(torch.tensor([code, 123], dtype=torch.int32))
        with pytest.raises(RuntimeError, match=rf"device status {code}: \w.* \(at index 123\)") as said:
            runner.check_status()
        assert "unknown" not in str(said.value)
        runner.check_status()                                     # cleared by the raise
