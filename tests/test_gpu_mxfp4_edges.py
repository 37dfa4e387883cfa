"""linear_mxfp4 at the edges of its 256 x 256 tiles: outputs and residuals whose rows are narrower than a tile, rows and columns left over at a tile's end, rows further
apart than they are long -- every result exact (small whole numbers: below 2^24 fp32 holds every sum in any order), and nothing in front of the output, behind it
or between its rows touched."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
GUARD = 64          # rows (or, in a transposed output, rows of ldc) in front of and behind what is written


@pytest.fixture(scope="module")
def ops():
    from wan2gp_amd import ops
    return ops


def whole(M, N, K):
    """Operands whose blocks all have the scale 1, a bias, a residual, a modulation table, and x w^T + bias in fp32, exact"""
    g = torch.Generator(device="cuda")
    g.manual_seed(M + 3 * N + K)
    draw = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, device="cuda").to(BF)
    x, w = draw(-1, 2, M, K) * 2, draw(-1, 2, N, K) * 2
    x[:, ::32] = 4
    w[:, ::32] = 4
    b, r, mod = draw(-8, 9, N), draw(-8, 9, M, N), draw(0, 3, 6, N)
    return x, w, b, r, mod, x.float() @ w.float().t() + b.float()


def guarded(M, N):
    buf = torch.full((M + 2 * GUARD, N), 7.0, dtype=BF, device="cuda")
    return buf, buf[GUARD : GUARD + M]


def untouched(buf, rows, what):
    assert (buf[:GUARD] == 7).all() and (buf[GUARD + rows :] == 7).all(), what


# a partial last row tile in front of rows of 8 .. 248 columns, with and without stages left over at K's end; two column tiles, the second partial; one row in the last tile
SHAPES = [(65520, 64, 1536), (20000, 200, 1536), (40000, 8, 1536), (40000, 64, 256), (17000, 136, 256), (33001, 128, 1536), (50001, 72, 800), (16500, 248, 512), (16897, 248, 288), (17001, 264, 256),
          (8300, 520, 288), (16385, 256, 256), (75600, 192, 5120)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_nothing_behind_the_output_is_written(ops, M, N, K):
    x, w, b, r, mod, y = whole(M, N, K)
    xm, wm = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    buf, out = guarded(M, N)
    ops.linear_mxfp4(None, *wm, b, x_mx=xm, out=out)
    assert torch.equal(out, y.to(BF))
    untouched(buf, M, "none")
    buf, out = guarded(M, N)
    ops.linear_mxfp4(None, *wm, b, epilogue=ops.EPI_GATE_RES, residual=r, mod=mod, e=mod * 0 + 1, gate_idx=3, x_mx=xm, out=out)
    gated = (r.float() + y * (mod[3].float() + 1)).to(BF)
    assert torch.equal(out, gated)
    untouched(buf, M, "gated")
    buf, out = guarded(M, N)                                             # in place
    out.copy_(r)
    ops.linear_mxfp4(None, *wm, b, epilogue=ops.EPI_GATE_RES, residual=out, mod=mod, e=mod * 0 + 1, gate_idx=3, x_mx=xm, out=out)
    assert torch.equal(out, gated)
    untouched(buf, M, "gated, in place")
    buf, out = guarded(M, N)
    ops.linear_mxfp4(x, *wm, b, epilogue=ops.EPI_GELU_TANH, out=out)
    untouched(buf, M, "gelu")
    y = y.double()
    gelu = torch.nn.functional.gelu(y, approximate="tanh")
    bound = 2.0 ** -18 * y.abs()                                         # (hardware exp2 and reciprocal)
    assert ((out.double() - gelu).abs() <= bound + 2.0 ** -8 * (gelu.abs() + bound) + 1e-30).all()


@pytest.mark.parametrize("M,N,K,ldc", [(104, 40000, 1536, 128), (104, 40000, 512, 104), (200, 20000, 1536, 200), (8, 40000, 256, 64), (248, 16900, 288, 256), (264, 17001, 256, 264), (136, 17000, 256, 192),
                                       (104, 40000, 1536, 1000)])
def test_nothing_around_a_transposed_output_is_written(ops, M, N, K, ldc):
    x, w, b, _, _, y = whole(M, N, K)
    buf = torch.full((N + 2 * GUARD, ldc), 7.0, dtype=BF, device="cuda")
    ops.linear_mxfp4(x, *ops.mxfp4_quantize(w), b, epilogue=ops.EPI_TRANSPOSED, out=buf[GUARD : GUARD + N], ldc=ldc)
    assert torch.equal(buf[GUARD : GUARD + N, :M], y.to(BF).t())
    untouched(buf, N, "transposed")
    assert (buf[:, M:] == 7).all()                                       # the places between M and ldc


@pytest.mark.parametrize("M,N,K,ldc", [(20000, 200, 512, 208), (40000, 64, 256, 1024), (17001, 264, 256, 520), (300, 72, 512, 80), (12, 72, 512, 96), (257, 1000, 768, 1024)])
def test_rows_further_apart_than_they_are_long(ops, M, N, K, ldc):
    """A column slice of a wider buffer as output and residual (the C entry takes the pitch): its neighbours stay as they were."""
    from wan2gp_amd import lib
    x, w, b, r, mod, y = whole(M, N, K)
    (a, sa), (c, sc) = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    L = lib.load()
    need = L.wan_gemm_mxfp4_scratch_bytes(M, N, K)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    e = mod * 0 + 1
    wide = torch.full((M, ldc), 7.0, dtype=BF, device="cuda")
    wide[:, :N] = r
    res = wide.clone()
    for epi, out in ((lib.EPI_GATE_RES, torch.full_like(wide, 7.0)), (lib.EPI_GATE_RES, res), (lib.EPI_NONE, torch.full_like(wide, 7.0))):
        src = res if out is res else wide
        lib.check(L.wan_gemm_mxfp4(a.data_ptr(), sa.data_ptr(), c.data_ptr(), sc.data_ptr(), b.data_ptr(), out.data_ptr(), ldc, M, N, K, epi, src.data_ptr(), mod.data_ptr(), e.data_ptr(), 6, 3, M,
                                   ws.data_ptr(), need, lib.stream_ptr()), "wan_gemm_mxfp4")
        ref = (r.float() + y * (mod[3].float() + 1)).to(BF) if epi == lib.EPI_GATE_RES else y.to(BF)
        assert torch.equal(out[:, :N], ref) and (out[:, N:] == 7).all()


@pytest.mark.parametrize("M,N,K,shape", [(300, 520, 512, (520, 384)), (104, 256, 64, (1, 256, 256)), (20, 72, 96, (72, 20)), (9000, 1160, 256, (2, 580, 9000))])
def test_a_transposed_output_is_written_by_its_own_rows(ops, M, N, K, shape):
    x, w, b, _, _, y = whole(M, N, K)
    out = torch.full(shape, 7.0, dtype=BF, device="cuda")
    assert ops.linear_mxfp4(x, *ops.mxfp4_quantize(w), b, epilogue=ops.EPI_TRANSPOSED, out=out) is out
    rows = out.view(N, -1)
    assert torch.equal(rows[:, :M], y.to(BF).t()) and (rows[:, M:] == 7).all()


def test_a_transposed_output_that_is_too_small_is_refused(ops):
    from wan2gp_amd.lib import WanHipError
    x, w, b, _, _, _ = whole(100, 64, 64)
    wm = ops.mxfp4_quantize(w)
    for out, ldc in ((torch.zeros(64, 96, dtype=BF, device="cuda"), None), (torch.zeros(63, 128, dtype=BF, device="cuda"), None), (torch.zeros(64, 128, dtype=BF, device="cuda"), 96)):
        with pytest.raises(WanHipError, match="does not hold"):
            ops.linear_mxfp4(x, *wm, b, epilogue=ops.EPI_TRANSPOSED, out=out, ldc=ldc)
