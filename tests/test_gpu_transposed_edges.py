"""The transposed epilogue of the bf16 and of the scaled-fp8 Linears where a row of the output holds fewer than 256 tokens: exact results (small whole numbers), and nothing in
front of the output, behind it or between tokens and ldc touched."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
GUARD = 64


@pytest.fixture(scope="module")
def ops():
    from wan2gp_amd import ops
    return ops


def operands(M, N, K):
    g = torch.Generator(device="cuda")
    g.manual_seed(M + N + K)
    draw = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, device="cuda").to(BF)
    x, w, b = draw(-2, 3, M, K), draw(-2, 3, N, K), draw(-8, 9, N)
    return x, w, b


def guarded(N, ldc):
    buf = torch.full((N + 2 * GUARD, ldc), 7.0, dtype=BF, device="cuda")
    return buf, buf[GUARD : GUARD + N]


def held(buf, out, M, ref):
    assert torch.equal(out[:, :M], ref)
    assert (buf[:GUARD] == 7).all() and (buf[GUARD + len(out):] == 7).all() and (buf[:, M:] == 7).all()


@pytest.mark.parametrize("M,N,K,ldc", [(104, 40000, 64, 128), (64, 33000, 128, 64), (248, 20600, 64, 248), (8, 40010, 64, 64), (200, 70001, 128, 200), (130, 30000, 64, 192), (512, 20600, 64, 512),
                                       (104, 300, 64, 128), (64, 384, 128, 64)])
def test_bf16(ops, M, N, K, ldc):
    x, w, b = operands(M, N, K)
    buf, out = guarded(N, ldc)
    ops.linear(x, w, b, epilogue=ops.EPI_TRANSPOSED, out=out, ldc=ldc)
    held(buf, out, M, (w.float() @ x.float().t() + b.float()[:, None]).to(BF))


@pytest.mark.parametrize("vector", [False, True])
@pytest.mark.parametrize("M,N,K,ldc", [(64, 384, 128, 64), (104, 300, 256, 128), (8, 1000, 256, 8), (248, 520, 384, 248), (200, 40000, 128, 200), (512, 384, 256, 512), (130, 384, 256, 192)])
def test_scaled_fp8(ops, M, N, K, ldc, vector):
    x, w, _ = operands(M, N, K)
    x[0, 0] = 448                                                         # the tensor's maximum: its scale is 1
    w[:, 0] = 0
    scale = torch.ones(N if vector else 1, dtype=torch.float32, device="cuda")
    buf, out = guarded(N, ldc)
    ops.linear_fp8(x, w.to(torch.float8_e4m3fn), scale, epilogue=ops.EPI_TRANSPOSED, out=out, ldc=ldc)
    held(buf, out, M, (w.float() @ x.float().t()).to(BF))
