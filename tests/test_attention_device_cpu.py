"""On which device the library is asked and called (no GPU: the device calls are stubbed)."""
import contextlib

import pytest
import torch

from flashdiffusion_b200 import attention, native


class Head:
    """What the call looks at of a tensor of heads on device 1."""
    device = torch.device("cuda", 1)


@pytest.mark.parametrize("start", [0, 1])
def test_workspaces_are_sized_on_the_device_of_the_heads(monkeypatch, start):
    """Their size depends on the number of SMs of the current device, which need not be the heads'."""
    state, seen = {"device": start}, []

    @contextlib.contextmanager
    def device(d):
        before, state["device"] = state["device"], d.index
        yield
        state["device"] = before

    class Library:
        def fd_attention_workspace_bytes(self, args, backward):
            seen.append(("size", state["device"]))
            return 0

    monkeypatch.setattr(native, "load", lambda: Library())
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["device"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)

    def entry(*args):
        seen.append(("call", state["device"]))
        return native.FD_OK

    attention._call(entry, b"", 0, Head())
    assert seen == [("size", 1), ("call", 1)] and state["device"] == start
