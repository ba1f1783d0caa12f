"""The status word of the matrix products: one a device, however the device is named."""
import torch

from litellmengine_b200.csrc import ops


def test_a_device_without_an_index_has_the_current_ones_word(monkeypatch):
    made = []
    zeros = torch.zeros

    def on_the_host(*size, dtype=None, device=None):
        made.append(str(device))
        return zeros(*size, dtype=dtype)

    monkeypatch.setattr(ops, "_stream_status", {})
    monkeypatch.setattr(torch, "zeros", on_the_host)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    a = ops.stream_status("cuda")
    assert a is ops.stream_status(torch.device("cuda", 1)) and a is ops.stream_status("cuda:1") and a is ops.stream_status(torch.device("cuda"))
    assert a is not ops.stream_status("cuda:0")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    assert ops.stream_status("cuda") is ops.stream_status("cuda:0")
    assert made == ["cuda:1", "cuda:0"]
