"""MXFP4 on the GPU against plain 64-bit forms: mxfp4_quantize / mxfp4_dequantize (codes, scales and values: equal) and linear_mxfp4.

linear_mxfp4's tolerance, from its roundings: K products summed in fp32 (each addition off by at most 2^-23 of the running magnitude -- the matrix
instruction may truncate), then the epilogue in fp32 (GELU: slope at most 1.13, its hardware exp2 and reciprocal 2^-18 of the value) and one rounding to
bf16 (2^-8)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


@pytest.fixture(scope="module")
def ops():
    from wan2gp_amd import ops
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def quant_ref(x):
    """-> (codes [M, K] one to a byte, exponents [M, K / 32], values [M, K] in 64 bits) by distance to the grid; ties to the even code"""
    x = x.cpu().to(F64)
    M, K = x.shape
    v = x.view(M, K // 32, 32)
    top = v.abs().amax(2)
    m, p = torch.frexp(top)
    e = torch.where(top > 0, (p - 3 + (m >= 0.875)).clamp(-127, 125), torch.full_like(p, -127))
    y = v / torch.pow(torch.tensor(2.0, dtype=F64), e.to(F64)).unsqueeze(2)
    grid = torch.tensor(GRID, dtype=F64)
    d = (y.abs().unsqueeze(3) - grid).abs()
    near = d.amin(3, keepdim=True)
    tie = d == near
    even = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0], dtype=torch.bool)
    code = torch.where((tie.sum(3) > 1), (tie & even).int().argmax(3), tie.int().argmax(3))
    val = torch.where(y < 0, -grid[code], grid[code]) * torch.pow(torch.tensor(2.0, dtype=F64), e.to(F64)).unsqueeze(2)
    code = code + 8 * torch.signbit(y).int()
    return code.view(M, K), e + 127, val.view(M, K)


def untile(scales, M, K):
    P, S = (M + 127) // 128, (K + 255) // 256
    full = scales.cpu().view(P, S, 4, 16, 2, 8).permute(0, 3, 5, 1, 4, 2).reshape(P * 128, S * 8)
    return full[:M, : K // 32], full


def rows(g, M, K):
    return (torch.randn(M, K, generator=g, device="cuda") * torch.exp(2.0 * torch.randn(K, generator=g, device="cuda"))).to(BF)


# ---- quantisation ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,K", [(1, 32), (1, 256), (3, 96), (127, 288), (128, 512), (129, 5120), (300, 1536), (1000, 64)])
def test_quantize(ops, M, K):
    x = rows(gen(M * K), M, K)
    codes, scales = ops.mxfp4_quantize(x)
    c, e, v = quant_ref(x)
    got = torch.stack([codes.cpu() & 15, codes.cpu() >> 4], 2).view(M, K)
    mine, full = untile(scales, M, K)
    assert torch.equal(mine.int(), e.int())
    assert torch.equal(got.int(), c.int())
    full = full.clone(); full[:M, : K // 32] = 0
    assert (full == 0).all()                                                   # the padding of the last tiles
    assert torch.equal(ops.mxfp4_dequantize(codes, scales).cpu().to(F64), v)


def test_quantize_every_bf16_against_every_scale(ops):
    """All finite bf16 values, each beside a block maximum of several magnitudes: borders, ties, subnormals and the ends of the exponent range."""
    bits = torch.arange(1 << 16, dtype=torch.int32)
    every = bits.to(torch.int16).view(BF)
    every = every[torch.isfinite(every.float())]
    for top in (0.0, 1.0, 1.75, 1.7421875, 3.0, 6.0, 7.0, 2.0 ** -120, 2.0 ** 126, 3.3895313892515355e38):
        x = torch.zeros(len(every), 32, dtype=BF)
        x[:, 5] = every
        x[:, 17] = top
        codes, scales = ops.mxfp4_quantize(x.cuda())
        c, e, v = quant_ref(x)
        mine, _ = untile(scales, len(x), 32)
        assert torch.equal(mine.int(), e.int()), top
        got = torch.stack([codes.cpu() & 15, codes.cpu() >> 4], 2).view(len(x), 32)
        assert torch.equal(got.int(), c.int()), top
        assert torch.equal(ops.mxfp4_dequantize(codes, scales).cpu().to(F64), v.to(BF).to(F64)), top


def test_quantize_nonfinite_blocks_are_nan(ops):
    x = torch.ones(2, 96, dtype=BF, device="cuda")
    x[0, 3] = float("inf"); x[1, 40] = float("nan"); x[1, 90] = -float("inf")
    v = ops.mxfp4_dequantize(*ops.mxfp4_quantize(x))
    nan = torch.isnan(v)
    assert nan[0, :32].all() and nan[1, 32:].all() and not nan[0, 32:].any() and not nan[1, :32].any()
    w = torch.ones(64, 96, dtype=BF, device="cuda")
    y = ops.linear_mxfp4(x, *ops.mxfp4_quantize(w))
    assert torch.isnan(y).all()
    clean = torch.ones(5, 96, dtype=BF, device="cuda")
    w[7, 0] = float("nan")
    y = ops.linear_mxfp4(clean, *ops.mxfp4_quantize(w))
    assert torch.isnan(y[:, 7]).all() and (y[:, :7] == 96).all() and (y[:, 8:] == 96).all()


def test_quantize_strided_rows_and_shapes(ops):
    x = rows(gen(4), 70, 640)
    a = ops.mxfp4_quantize(x[:, 128:384])
    b = ops.mxfp4_quantize(x[:, 128:384].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = ops.mxfp4_quantize(x.view(7, 10, 640))
    assert c[0].shape == (7, 10, 320) and ops.mxfp4_dequantize(*c).shape == (7, 10, 640)
    codes, scales = ops.mxfp4_quantize(x[:0])
    assert codes.shape == (0, 320) and ops.mxfp4_dequantize(codes, scales).shape == (0, 640)


# ---- the product -----------------------------------------------------------------------------------------------------------------------
def operands(ops, g, M, N, K):
    x = rows(g, M, K)
    w = (torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)).to(BF)
    xm, wm = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    xd, wd = ops.mxfp4_dequantize(*xm).to(F64), ops.mxfp4_dequantize(*wm).to(F64)     # (held to the plain form above)
    return x, xm, wm, xd, wd


def linear_ref(xd, wd, bias):
    y = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if bias is not None:
        y, mag = y + bias.to(F64), mag + bias.to(F64).abs()
    err = (xd.shape[1] + 2) * 2.0 ** -23 * mag                                        # in fp32, in front of any rounding
    return y, err


def close(got, ref, err):
    d = (got.to(F64) - ref).abs()
    assert (d <= err + 1e-30).all(), ((d / (err + 1e-30)).max().item(), (d > err + 1e-30).sum().item())


SHAPES = [(1, 8, 32), (1, 5120, 512), (2, 64, 64), (5, 200, 96), (16, 256, 256), (33, 1000, 320), (128, 128, 256), (130, 264, 544), (257, 513, 768), (300, 1536, 1536), (1000, 640, 2080),
          (1024, 2048, 512), (4097, 4096, 768), (20000, 1024, 1280), (9001, 1160, 1056), (40000, 264, 32), (5000, 2056, 2848), (1, 30720, 5120), (64, 5120, 13824)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_every_epilogue(ops, M, N, K):
    g = gen(M + N + K)
    x, xm, wm, xd, wd = operands(ops, g, M, N, K)
    bias = torch.randn(N, generator=g, device="cuda").to(BF)
    y, err = linear_ref(xd, wd, bias)
    got = ops.linear_mxfp4(x, *wm, bias)
    assert got.shape == (M, N)
    close(got, y, err + 2.0 ** -8 * (y.abs() + err))
    assert torch.equal(got, ops.linear_mxfp4(None, *wm, bias, x_mx=xm))
    y0, err0 = linear_ref(xd, wd, None)
    close(ops.linear_mxfp4(x, *wm), y0, err0 + 2.0 ** -8 * (y0.abs() + err0))
    gelu = torch.nn.functional.gelu(y, approximate="tanh")
    bound = 1.13 * err + 2.0 ** -18 * y.abs()
    close(ops.linear_mxfp4(x, *wm, bias, epilogue=1), gelu, bound + 2.0 ** -8 * (gelu.abs() + bound))
    r = torch.randn(M, N, generator=g, device="cuda").to(BF)
    nb = 2 if M % 2 == 0 else 1
    mod, e = torch.randn(6, N, generator=g, device="cuda").to(BF), torch.randn(nb, 6, N, generator=g, device="cuda").to(BF)
    gate = (mod[4].to(F64) + e[:, 4].to(F64)).repeat_interleave(M // nb, 0)
    out = r.to(F64) + y * gate
    bound = err * gate.abs() + 2.0 ** -22 * (r.to(F64).abs() + (y * gate).abs())
    got = ops.linear_mxfp4(x, *wm, bias, epilogue=2, residual=r, mod=mod, e=e, gate_idx=4)
    close(got, out, bound + 2.0 ** -8 * (out.abs() + bound))
    out = r.to(F64) + y
    got = ops.linear_mxfp4(x, *wm, bias, epilogue=2, residual=r)
    bound = err + 2.0 ** -22 * (r.to(F64).abs() + y.abs())
    close(got, out, bound + 2.0 ** -8 * (out.abs() + bound))
    inplace = r.clone()
    assert torch.equal(ops.linear_mxfp4(x, *wm, bias, epilogue=2, residual=inplace, out=inplace), got)
    vt = ops.linear_mxfp4(x, *wm, bias, epilogue=3)
    assert vt.shape == (N, (M + 63) // 64 * 64) and (vt[:, M:] == 0).all()
    close(vt[:, :M], y.t(), (err + 2.0 ** -8 * (y.abs() + err)).t())


def test_gate_rows_of_many_batches(ops):
    """Batches shorter than a tile, and of a tile's size and a little more: every row takes its own batch's gate."""
    g = gen(9)
    for nb, rpb, N, K in ((50, 100, 2048, 256), (19, 257, 2304, 320), (1, 5000, 2304, 256)):
        M = nb * rpb
        x, xm, wm, xd, wd = operands(ops, g, M, N, K)
        y, err = linear_ref(xd, wd, None)
        r = torch.randn(M, N, generator=g, device="cuda").to(BF)
        mod, e = torch.randn(6, N, generator=g, device="cuda").to(BF), torch.randn(nb, 6, N, generator=g, device="cuda").to(BF)
        gate = (mod[2].to(F64) + e[:, 2].to(F64)).repeat_interleave(rpb, 0)
        out = r.to(F64) + y * gate
        bound = err * gate.abs() + 2.0 ** -22 * (r.to(F64).abs() + (y * gate).abs())
        close(ops.linear_mxfp4(None, *wm, epilogue=2, residual=r, mod=mod, e=e, gate_idx=2, x_mx=xm), out, bound + 2.0 ** -8 * (out.abs() + bound))


def test_linear_leaves_what_lies_past_the_result(ops):
    g = gen(5)
    x, xm, wm, xd, wd = operands(ops, g, 300, 520, 512)
    buf = torch.full((400, 520), 7.0, dtype=BF, device="cuda")
    ops.linear_mxfp4(x, *wm, out=buf[:300])
    assert (buf[300:] == 7).all()
    vt = torch.full((521, 384), 7.0, dtype=BF, device="cuda")
    ops.linear_mxfp4(x, *wm, epilogue=3, out=vt[:520], ldc=384)
    assert (vt[520:] == 7).all() and (vt[:520, 300:] == 7).all()


def test_linear_is_exact_where_fp32_is(ops):
    """Small integers: every product and sum is exact, so the result is, at every place of a tile."""
    g = gen(6)
    for M, N, K in ((256, 256, 256), (300, 700, 288), (4096, 4096, 512), (3, 100, 640)):
        x = torch.randint(-1, 2, (M, K), generator=g, device="cuda").to(BF) * 2
        w = torch.randint(-1, 2, (N, K), generator=g, device="cuda").to(BF) * 2
        x[:, ::32] = 4; w[:, ::32] = 4                                          # (every block's scale is one)
        y = x.to(F64) @ w.to(F64).t()
        assert torch.equal(ops.linear_mxfp4(x, *ops.mxfp4_quantize(w)).to(F64), y.to(BF).to(F64)), (M, N, K)


@pytest.mark.parametrize("M,N,K", [(40000, 1288, 32), (40001, 1288, 288), (33000, 2000, 512), (30720, 2304, 800), (25000, 2312, 1312), (70000, 520, 1600)])
def test_several_tiles_a_workgroup(ops, M, N, K):
    """Small integers again, so that every place of every tile of a workgroup's run is held to the exact result: stages left over at a tile's end, edges in both
    directions, all four epilogues."""
    g = gen(M)
    x = torch.randint(-1, 2, (M, K), generator=g, device="cuda").to(BF) * 2
    w = torch.randint(-1, 2, (N, K), generator=g, device="cuda").to(BF) * 2
    x[:, ::32] = 4; w[:, ::32] = 4
    b = torch.randint(-8, 9, (N,), generator=g, device="cuda").to(BF)
    r = torch.randint(-8, 9, (M, N), generator=g, device="cuda").to(BF)
    mod = torch.randint(0, 3, (6, N), generator=g, device="cuda").to(BF)
    xm, wm = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    y = (x.float() @ w.float().t()).to(torch.float32) + b.float()                   # (whole numbers below 2^24: exact in any order)
    assert torch.equal(ops.linear_mxfp4(None, *wm, b, x_mx=xm), y.to(BF))
    assert torch.equal(ops.linear_mxfp4(None, *wm, b, epilogue=2, residual=r, mod=mod, e=mod * 0 + 1, gate_idx=3, x_mx=xm), (r.float() + y * (mod[3].float() + 1)).to(BF))
    assert torch.equal(ops.linear_mxfp4(None, *wm, b, epilogue=3, x_mx=xm)[:, :M], y.to(BF).t())
    gelu = torch.nn.functional.gelu(y.double(), approximate="tanh")
    bound = 2.0 ** -18 * y.double().abs()
    close(ops.linear_mxfp4(None, *wm, b, epilogue=1, x_mx=xm), gelu, bound + 2.0 ** -8 * (gelu.abs() + bound))


def test_linears_on_streams_beside_each_other(ops):
    g = gen(8)
    cases = []
    for M, N, K in ((3, 2048, 5120), (600, 1536, 1536), (9000, 2304, 512)):
        x, xm, wm, xd, wd = operands(ops, g, M, N, K)
        cases.append((x, wm, ops.linear_mxfp4(x, *wm)))
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([ops.linear_mxfp4(x, *wm) for x, wm, _ in cases for _ in range(3)])
    torch.cuda.synchronize()
    for per in outs:
        assert all(torch.equal(o, cases[i // 3][2]) for i, o in enumerate(per))


@pytest.mark.parametrize("M,N,K", [(1, 128, 5120), (1, 7, 32), (3, 1536, 13824), (16, 5120, 5120), (16, 1160, 1056), (17, 1160, 1056), (7, 257, 288), (15, 1000, 8960), (16, 640, 17000 // 32 * 32),
                                   (16, 640, 20000), (2, 30720, 1536), (16, 700, 2560), (16, 700, 2592), (8, 12300, 4800), (9, 12300, 4800), (1, 640, 4480), (1, 640, 4512), (1, 12288, 64000)])
def test_linear_of_few_rows(ops, M, N, K):
    """Both sides of the limits of the kernel for up to 16 rows: every epilogue, strided rows, rows quantised inside and in front."""
    g = gen(M * N + K)
    wide = rows(g, M, K + 64)
    x = wide[:, 32 : K + 32] if M > 1 else wide[:, 32 : K + 32].contiguous()
    w = (torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)).to(BF)
    xm, wm = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    xd, wd = ops.mxfp4_dequantize(*xm).to(F64), ops.mxfp4_dequantize(*wm).to(F64)
    bias = torch.randn(N, generator=g, device="cuda").to(BF)
    y, err = linear_ref(xd, wd, bias)
    got = ops.linear_mxfp4(x, *wm, bias)
    close(got, y, err + 2.0 ** -8 * (y.abs() + err))
    assert torch.equal(got, ops.linear_mxfp4(None, *wm, bias, x_mx=xm))
    gelu = torch.nn.functional.gelu(y, approximate="tanh")
    bound = 1.13 * err + 2.0 ** -18 * y.abs()
    close(ops.linear_mxfp4(x, *wm, bias, epilogue=1), gelu, bound + 2.0 ** -8 * (gelu.abs() + bound))
    r = torch.randn(M, N, generator=g, device="cuda").to(BF)
    mod, e = torch.randn(6, N, generator=g, device="cuda").to(BF), torch.randn(M, 6, N, generator=g, device="cuda").to(BF)   # (a gate a row)
    gate = mod[1].to(F64) + e[:, 1].to(F64)
    out = r.to(F64) + y * gate
    bound = err * gate.abs() + 2.0 ** -22 * (r.to(F64).abs() + (y * gate).abs())
    inplace = r.clone()
    close(ops.linear_mxfp4(x, *wm, bias, epilogue=2, residual=inplace, out=inplace, mod=mod, e=e, gate_idx=1), out, bound + 2.0 ** -8 * (out.abs() + bound))
    vt = torch.full((N + 1, 64), 7.0, dtype=BF, device="cuda")
    ops.linear_mxfp4(x, *wm, bias, epilogue=3, out=vt[:N], ldc=64)
    close(vt[:N, :M], y.t(), (err + 2.0 ** -8 * (y.abs() + err)).t())
    assert (vt[N:] == 7).all() and (vt[:, M:] == 7).all()


def test_output_over_the_input_is_refused(ops):
    from wan2gp_amd.lib import WanHipError
    g = gen(32)
    w = ops.mxfp4_quantize((torch.randn(512, 512, generator=g, device="cuda") / 22).to(BF))
    for M in (3, 40):
        buf = rows(g, 2 * M, 512)
        x = buf[:M]
        ref = ops.linear_mxfp4(x, *w)
        with pytest.raises(WanHipError, match="overlap"):
            ops.linear_mxfp4(x, *w, out=x)
        with pytest.raises(WanHipError, match="overlap"):
            ops.linear_mxfp4(x, *w, out=buf[1 : M + 1])
        assert torch.equal(ops.linear_mxfp4(x, *w, out=buf[M:]), ref) and torch.equal(buf[M:], ref)


def test_few_rows_with_nonfinite_blocks(ops):
    """A row with an infinity or a NaN is NaN, its neighbours are not touched."""
    g = gen(31)
    x = rows(g, 5, 512)
    x[1, 40], x[3, 511] = float("nan"), float("inf")
    w = (torch.randn(300, 512, generator=g, device="cuda") / 20).to(BF)
    wm = ops.mxfp4_quantize(w)
    got = ops.linear_mxfp4(x, *wm)
    assert torch.isnan(got[[1, 3]]).all()
    x[[1, 3]] = 0
    assert torch.equal(got[[0, 2, 4]], ops.linear_mxfp4(x, *wm)[[0, 2, 4]])


def test_captured_linears_of_two_graphs(ops):
    g = gen(7)
    state = []
    for n in range(2):
        x, xm, wm, xd, wd = operands(ops, g, 3, 1024, 5120)
        ops.linear_mxfp4(x, *wm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_mxfp4(x, *wm)
        state.append((graph, x, wm, out))
    for turn in range(3):
        for graph, x, wm, out in state:
            x.copy_(rows(g, 3, 5120))
        for graph, *_ in state:
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, wm, out in state:
            assert torch.equal(out, ops.linear_mxfp4(x, *wm))


# ---- a block's attention on both -------------------------------------------------------------------------------------------------------
def test_sparse_attention_between_mxfp4_linears(ops):
    """The attention half of a block as it would run: q, k and V^T from 4-bit Linears of one quantised input, RMSNorm + RoPE, block lists, sparse attention, the
    output projection with its residual -- against the same steps in 64 bits on the tensors that the step before left."""
    import sys, os
    sys.path.insert(0, os.path.dirname(__file__))
    from test_gpu_sparse_attention import attend_ref, check, select_ref
    g = gen(8)
    B, L, H = 1, 900, 4
    d = H * 128
    x = rows(g, L, d)
    wq, wk, wv, wo = [ops.mxfp4_quantize((torch.randn(d, d, generator=g, device="cuda") / math.sqrt(d)).to(BF)) for _ in range(4)]
    bias = (0.1 * torch.randn(d, generator=g, device="cuda")).to(BF)
    gq = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(BF)
    xm = ops.mxfp4_quantize(x)
    q = ops.linear_mxfp4(None, *wq, bias, x_mx=xm).view(B, L, H, 128)
    k = ops.linear_mxfp4(None, *wk, bias, x_mx=xm).view(B, L, H, 128)
    vt = ops.linear_mxfp4(None, *wv, bias, x_mx=xm, epilogue=3).view(B, d, -1)
    ang = torch.rand(L, 128, generator=g, device="cuda") * 6.28
    ops.rmsnorm_rope_(q, k, gq, gq, (torch.cos(ang), torch.sin(ang)))
    qm, km = ops.block_mean(q, 128), ops.block_mean(k, 64)
    index, count = ops.select_blocks(qm, km, 5)
    ri, rc = select_ref(qm, km, 5)
    assert torch.equal(index, ri) and torch.equal(count, rc)
    o = ops.sparse_attention(q, k, vt, index, count)
    check(o, *attend_ref(q, k, vt, index, count))
    got = ops.linear_mxfp4(o.view(L, d), *wo, bias, epilogue=2, residual=x)
    y, err = linear_ref(ops.mxfp4_dequantize(*ops.mxfp4_quantize(o.view(L, d))).to(F64), ops.mxfp4_dequantize(*wo).to(F64), bias)
    out = x.to(F64) + y
    bound = err + 2.0 ** -22 * (x.to(F64).abs() + y.abs())
    close(got, out, bound + 2.0 ** -8 * (out.abs() + bound))
