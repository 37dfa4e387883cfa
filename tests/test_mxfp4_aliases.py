"""An output that shares memory with an operand: refused in front of the first launch, whichever kernel would run (on the CPU: addresses alone are compared, every call is
refused), unless it is the residual itself."""
import ctypes

import pytest

from wan2gp_amd import lib

P = ctypes.c_void_p
BASE = 1 << 30            # the output
FAR = {n: (1 << 32) + (i << 30) for i, n in enumerate(("x", "As", "W", "Ws", "bias", "R", "mod", "e", "ws"))}

# rows that stay in one kernel, tiles in parts, small tiles, large ones
SIZES = [(3, 64, 64), (300, 128, 5120), (512, 1024, 512), (40000, 264, 256)]


def call(entry, M, N, K, epi, ldc=None, **at):
    a = {n: P(v) for n, v in FAR.items()} | {n: P(v) for n, v in at.items()}
    L = lib.load()
    ldc = ldc or ((M + 63) // 64 * 64 if epi == lib.EPI_TRANSPOSED else N)
    x = (a["x"], a["As"]) if entry == "gemm" else (a["x"], K)
    rc = getattr(L, f"wan_{entry}_mxfp4")(*x, a["W"], a["Ws"], a["bias"], P(BASE), ldc, M, N, K, epi, a["R"], a["mod"], a["e"], 6, 2, (M + 1) // 2, a["ws"], 1 << 40, None)
    assert rc == 1, "not refused"
    return L.wan_last_error().decode()


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("entry", ["linear", "gemm"])
def test_operands_under_the_output(entry, M, N, K):
    size = M * N * 2
    for epi in (lib.EPI_NONE, lib.EPI_GELU_TANH, lib.EPI_GATE_RES, lib.EPI_TRANSPOSED):
        last = N * ((M + 63) // 64 * 64) * 2 - ((-M) % 64) * 2 if epi == lib.EPI_TRANSPOSED else size
        for name, length in (("W", N * K // 2), ("Ws", 1024), ("bias", 2 * N), ("x", M * K * 2 if entry == "linear" else M * K // 2)):
            for at in (BASE, BASE + (last - 1) // 16 * 16, BASE - (length - 1) // 16 * 16):
                if at % 16 == 0:
                    assert "overlap" in call(entry, M, N, K, epi, **{name: at}), (epi, name, at - BASE)
    for name, length in (("mod", 12 * N), ("e", 24 * N)):
        for at in (BASE, BASE + size - 16, BASE - (length - 16)):
            assert "gate" in call(entry, M, N, K, lib.EPI_GATE_RES, **{name: at})
    if entry == "gemm":
        assert "quantised rows" in call(entry, M, N, K, lib.EPI_NONE, As=BASE + size - 16)


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("entry", ["linear", "gemm"])
def test_a_residual_under_part_of_the_output(entry, M, N, K):
    for off in (16, -16, 2 * N, -2 * N, (M - 1) * N * 2, -(M - 1) * N * 2):
        assert "must be the residual" in call(entry, M, N, K, lib.EPI_GATE_RES, R=BASE + off), off
    wide = 2 * N + 16                                                     # rows side by side in a wider buffer, not far enough apart
    for off in (2 * N - 16, -2 * N + 16, 2 * (wide + N) - 16):
        assert "must be the residual" in call(entry, M, N, K, lib.EPI_GATE_RES, ldc=wide, R=BASE + off), off


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SIZES)
def test_neighbours_that_share_nothing_are_taken(M, N, K):
    """Output and residual side by side in one buffer, and a residual that is the output: the results of buffers apart."""
    import torch
    from wan2gp_amd import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    draw = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)
    x, w, r, mod, e = draw(M, K), draw(N, K), draw(M, N), draw(6, N), draw(1, 6, N)
    (a, sa), (c, sc) = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    ref = ops.linear_mxfp4(x, c, sc, epilogue=lib.EPI_GATE_RES, residual=r, mod=mod, e=e, gate_idx=2)
    L = lib.load()
    need = L.wan_gemm_mxfp4_scratch_bytes(M, N, K)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    both = torch.cat([r, torch.zeros_like(r)], 1)
    out = both.data_ptr() + 2 * N
    lib.check(L.wan_gemm_mxfp4(a.data_ptr(), sa.data_ptr(), c.data_ptr(), sc.data_ptr(), None, out, 2 * N, M, N, K, lib.EPI_GATE_RES, both.data_ptr(), mod.data_ptr(), e.data_ptr(), 6, 2, M,
                               ws.data_ptr(), need, lib.stream_ptr()), "wan_gemm_mxfp4")
    assert torch.equal(both[:, N:], ref) and torch.equal(both[:, :N], r)
    assert torch.equal(ops.linear_mxfp4(x, c, sc, epilogue=lib.EPI_GATE_RES, residual=r, mod=mod, e=e, gate_idx=2, out=r), ref)
