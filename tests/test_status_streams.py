"""The device's status word is ready for every stream once it has been made."""
import importlib

import pytest
import torch


@pytest.mark.gpu
def test_a_report_of_another_stream_than_the_first_calls_is_kept(monkeypatch):
    """The first call's stream is still busy when a kernel on another one reports that its sizes do not fit."""
    common = importlib.import_module("iris_testing_b200.ops._common")
    from iris_testing_b200 import ops
    from iris_testing_b200._native import NativeError
    x = torch.ones(20, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(2, 256, 64, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([10, 11], dtype=torch.int32, device="cuda")
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        del_later = torch.zeros(4, dtype=torch.int32, device="cuda")       # memory of each stream's own, so that nothing below
    with torch.cuda.stream(second):
        ops.linear(x, w, group_rows=rows - 1)                              # waits for the device to get some
    torch.cuda.synchronize()
    del del_later
    ops.check_default_status()
    monkeypatch.setattr(common, "_DEFAULT_STATUS", {})
    with torch.cuda.stream(first):
        torch.cuda._sleep(400_000_000)               # some 200 ms
        ops.default_status(x.device)
    with torch.cuda.stream(second):
        ops.linear(x, w, group_rows=rows)
    torch.cuda.synchronize()
    with pytest.raises(NativeError, match="overflow"):
        ops.check_default_status()
