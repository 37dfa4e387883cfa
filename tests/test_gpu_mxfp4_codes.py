"""Codes that a program's own arithmetic left in a wider integer type, a byte in each: the same results as from bytes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from wan2gp_amd import ops
    return ops


@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("M,N,K", [(3, 200, 288), (130, 264, 544), (9001, 1160, 1056)])
def test_widened_codes(ops, dtype, M, N, K):
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    x, w = torch.randn(M, K, generator=g, device="cuda").to(BF), torch.randn(N, K, generator=g, device="cuda").to(BF)
    (xc, xs), (wc, ws) = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    ref = ops.linear_mxfp4(x, wc, ws)
    assert torch.equal(ops.linear_mxfp4(x, wc.to(dtype), ws), ref)
    assert torch.equal(ops.linear_mxfp4(None, wc.to(dtype), ws, x_mx=(xc.to(dtype), xs)), ref)
    assert torch.equal(ops.mxfp4_dequantize(wc.to(dtype), ws), ops.mxfp4_dequantize(wc, ws))
    low, high = wc & 15, wc >> 4                                         # put together again as a program would
    both = low.to(dtype) + 16 * high.to(dtype)
    assert torch.equal(ops.linear_mxfp4(x, both, ws), ref)


def test_other_types_are_refused(ops):
    from wan2gp_amd.lib import WanHipError
    w = torch.randn(64, 96, device="cuda").to(BF)
    codes, scales = ops.mxfp4_quantize(w)
    for bad in (codes.float(), codes.to(BF), codes.bool()):
        with pytest.raises(WanHipError, match="uint8"):
            ops.mxfp4_dequantize(bad, scales)
    with pytest.raises(WanHipError, match="uint8"):                      # scales are never widened: a byte's place in their tiles counts
        ops.mxfp4_dequantize(codes, scales.int())
