"""The operators run on the device that their tensors lie on, whichever is current: every entry point that pay_sparse_attention and linear_mxfp4 reach is called through the
helper that makes it so.  (CPU: tensors without memory that claim to lie on a second GPU; nothing is launched.)"""
import pytest
import torch
from torch._subclasses import FakeTensor, FakeTensorMode

from wan2gp_amd import ops

BF = torch.bfloat16


class Entry:
    def __init__(self, name):
        self.__name__ = name

    def __call__(self, *args):
        assert self.__name__.endswith("_bytes"), f"{self.__name__} is called past _call"
        return 0


class Library:
    def __getattr__(self, name):
        return Entry(name)


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(ops._L, "load", Library)
    monkeypatch.setattr(ops, "_call", lambda device, fn, *args: seen.append((fn.__name__, device)))
    monkeypatch.setattr(FakeTensor, "data_ptr", lambda self: 4096, raising=False)
    monkeypatch.setattr(torch.UntypedStorage, "data_ptr", lambda self: id(self))
    monkeypatch.setattr(ops, "ptr", lambda t: None)
    monkeypatch.setattr(ops, "stream_ptr", lambda: None)
    with FakeTensorMode():
        yield seen


def test_pay_sparse_attention_on_another_device(calls):
    q, k, v = (torch.empty(1, n, 2, 128, dtype=BF, device="cuda:1") for n in (200, 300, 300))
    o = ops.pay_sparse_attention([q, k, v], 2)
    assert o.device == q.device
    assert [n for n, _ in calls] == ["wan_block_mean", "wan_block_mean", "wan_select_blocks", "wan_transpose_v", "wan_sparse_attention"]
    assert all(d == q.device for _, d in calls), calls


def test_linear_mxfp4_on_another_device(calls):
    x, w = torch.empty(20, 64, dtype=BF, device="cuda:1"), torch.empty(96, 64, dtype=BF, device="cuda:1")
    codes, scales = ops.mxfp4_quantize(w)
    ops.mxfp4_dequantize(codes, scales)
    y = ops.linear_mxfp4(x, codes, scales)
    ops.linear_mxfp4(None, codes, scales, x_mx=ops.mxfp4_quantize(x))
    assert y.device == x.device
    assert [n for n, _ in calls] == ["wan_mxfp4_quantize", "wan_mxfp4_dequantize", "wan_linear_mxfp4", "wan_mxfp4_quantize", "wan_gemm_mxfp4"]
    assert all(d == x.device for _, d in calls), calls
