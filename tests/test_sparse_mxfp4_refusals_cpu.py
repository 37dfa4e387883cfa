"""What the block-sparse attention and MXFP4 entry points refuse (CPU: every check comes in front of the first launch).  The C entries are called with
aligned addresses that nothing may read."""
import ctypes

import pytest
import torch

from wan2gp_amd import lib, ops

P = ctypes.c_void_p
A = P(1 << 20)           # 16-byte aligned
ODD = P((1 << 20) + 8)   # 8-byte aligned only


def refuse(rc, word):
    assert rc == 1
    msg = lib.load().wan_last_error().decode()
    assert word in msg, msg


def mean(so, **kw):
    a = dict(x=A, row=512, batch=5120, lens=None, out=A, B=1, L=10, H=4, block=64) | kw
    return so.wan_block_mean(a["x"], a["row"], a["batch"], a["lens"], a["out"], a["B"], a["L"], a["H"], a["block"], None)


def select(so, **kw):
    a = dict(q=A, k=A, lens=None, index=A, count=A, B=2, Bk=2, H=4, Hk=2, nq=3, nk=5, keep=2, ws=A, n=1 << 20) | kw
    return so.wan_select_blocks(a["q"], a["k"], a["lens"], a["index"], a["count"], a["B"], a["Bk"], a["H"], a["Hk"], a["nq"], a["nk"], a["keep"], a["ws"], a["n"], None)


def attend(so, **kw):
    a = dict(q=A, qr=512, qb=51200, k=A, kr=256, kb=25600, vt=A, o=A, index=A, count=None, lens=None, B=2, Bk=2, Lq=100, Lk=100, ldv=128, H=4, Hk=2, keep=2, ws=A, n=1 << 40) | kw
    return so.wan_sparse_attention(a["q"], a["qr"], a["qb"], a["k"], a["kr"], a["kb"], a["vt"], a["o"], a["index"], a["count"], a["lens"], a["B"], a["Bk"], a["Lq"], a["Lk"],
                                  a["ldv"], a["H"], a["Hk"], a["keep"], 0, a["ws"], a["n"], None)


def gemm(so, **kw):
    a = dict(A=A, As=A, W=A, Ws=A, bias=None, C=A, ldc=64, M=3, N=64, K=64, epi=0, R=None, mod=None, e=None, n_mod=0, gate=-1, rpb=1, ws=A, n=1 << 40) | kw
    return so.wan_gemm_mxfp4(a["A"], a["As"], a["W"], a["Ws"], a["bias"], a["C"], a["ldc"], a["M"], a["N"], a["K"], a["epi"], a["R"], a["mod"], a["e"], a["n_mod"], a["gate"], a["rpb"],
                            a["ws"], a["n"], None)


@pytest.mark.parametrize("call,kw,word", [
    (mean, dict(x=None), "null"), (mean, dict(out=None), "null"), (mean, dict(L=0), "empty"), (mean, dict(block=0), "empty"), (mean, dict(B=0), "empty"), (mean, dict(row=504), "strides"),
    (mean, dict(row=516), "strides"), (mean, dict(batch=5121), "strides"), (mean, dict(x=ODD), "aligned"), (mean, dict(B=70000), "grid"),
    (select, dict(index=None), "null"), (select, dict(k=None), "null"), (select, dict(Bk=3), "Bk must divide"), (select, dict(Hk=3), "heads"), (select, dict(Hk=0), "heads"), (select, dict(keep=0), "empty"),
    (select, dict(nk=0), "empty"), (select, dict(nk=20001, n=1 << 40), "20,000"), (select, dict(nk=257, ws=None), "scratch"), (select, dict(nk=257, n=2 * 4 * 3 * 257 * 8 - 1), "scratch"), (select, dict(nk=257, ws=ODD, n=1 << 30), "scratch"),
    (select, dict(nq=1 << 30, n=1 << 60), "grid"),
    (attend, dict(q=None), "null"), (attend, dict(index=None), "null"), (attend, dict(Bk=4), "Bk must divide"), (attend, dict(Hk=3), "heads"), (attend, dict(Lk=0), "empty"), (attend, dict(keep=0), "empty"),
    (attend, dict(ldv=100), "ldv"), (attend, dict(ldv=64), "ldv"), (attend, dict(qr=504), "strides"), (attend, dict(kr=260), "strides"), (attend, dict(kb=3), "strides"), (attend, dict(vt=ODD), "aligned"),
    (attend, dict(kr=1 << 24), "offsets"), (attend, dict(ldv=1 << 23), "offsets"), (attend, dict(Lq=1 << 40), "grid"),
    (gemm, dict(A=None), "null"), (gemm, dict(Ws=None), "null"), (gemm, dict(M=0), "positive"), (gemm, dict(N=0), "positive"), (gemm, dict(K=48), "multiple of 32"), (gemm, dict(K=0), "multiple of 32"),
    (gemm, dict(C=ODD), "aligned"), (gemm, dict(As=ODD), "aligned"), (gemm, dict(ldc=63), "ldc"), (gemm, dict(epi=3, ldc=2), "ldc"), (gemm, dict(epi=4), "unknown epilogue"), (gemm, dict(epi=2), "residual"),
    (gemm, dict(epi=2, R=A, gate=0), "gate"), (gemm, dict(epi=2, R=A, mod=A, e=A, n_mod=6, gate=6), "gate"), (gemm, dict(epi=2, R=A, mod=A, e=A, n_mod=6, gate=2, rpb=0), "gate")])
def test_c_entries_refuse(call, kw, word):
    refuse(call(lib.load(), **kw), word)


def test_quantiser_entries_refuse():
    L = lib.load()
    for kw, word in ((dict(x=None), "null"), (dict(M=0), "positive"), (dict(K=33), "multiple of 32"), (dict(row=32), "row stride"), (dict(row=68), "row stride"), (dict(x=ODD), "aligned"), (dict(scales=ODD), "aligned")):
        a = dict(x=A, row=64, codes=A, scales=A, M=2, K=64) | kw
        refuse(L.wan_mxfp4_quantize(a["x"], a["row"], a["codes"], a["scales"], a["M"], a["K"], None), word)
    for kw, word in ((dict(out=None), "null"), (dict(M=-1), "positive"), (dict(K=31), "multiple of 32"), (dict(codes=ODD), "aligned")):
        a = dict(codes=A, scales=A, out=A, M=2, K=64) | kw
        refuse(L.wan_mxfp4_dequantize(a["codes"], a["scales"], a["out"], a["M"], a["K"], None), word)


def test_linear_entry_refuses():
    L = lib.load()
    for kw, word in ((dict(x=None), "null"), (dict(W=None), "null"), (dict(M=0), "positive"), (dict(K=40), "multiple of 32"), (dict(M=17, n=100), "scratch"), (dict(M=17, ws=None), "scratch"), (dict(row=32), "row stride"), (dict(M=17, row=68), "row stride"),
                     (dict(epi=2), "residual"), (dict(epi=7), "unknown epilogue"), (dict(ldc=63), "ldc"), (dict(C=ODD), "aligned"), (dict(x=ODD), "aligned")):
        a = dict(x=A, row=64, W=A, Ws=A, C=A, ldc=64, M=3, N=64, K=64, epi=0, ws=A, n=1 << 40) | kw
        refuse(L.wan_linear_mxfp4(a["x"], a["row"], a["W"], a["Ws"], None, a["C"], a["ldc"], a["M"], a["N"], a["K"], a["epi"], None, None, None, 0, -1, 1, a["ws"], a["n"], None), word)
    B = 1 << 24                                                        # (addresses alone are compared; every call here is refused)
    for kw in (dict(x=B, C=B), dict(x=B, C=B + 128), dict(x=B, C=B - 16), dict(x=B, C=B + 16, M=200), dict(x=B, C=B + 64 * 2, row=128, ldc=96, M=200), dict(x=B, C=B + 256, epi=3, row=1024),
               dict(x=B, C=B + 96, row=128, ldc=128)):
        a = dict(x=A, row=64, W=A, Ws=A, C=A, ldc=64, M=3, N=64, K=64, epi=0, ws=A, n=1 << 40) | kw
        if a["epi"] == 3:
            a["ldc"] = 64
        refuse(L.wan_linear_mxfp4(a["x"], a["row"], a["W"], a["Ws"], None, a["C"], a["ldc"], a["M"], a["N"], a["K"], a["epi"], None, None, None, 0, -1, 1, a["ws"], a["n"], None), "overlap")
    need = L.wan_gemm_mxfp4_scratch_bytes(17, 64, 5120)
    assert need > 0
    refuse(gemm(L, M=17, K=5120, n=need - 1), "scratch")
    refuse(gemm(L, M=17, K=5120, ws=None), "scratch")
    assert L.wan_linear_mxfp4_scratch_bytes(16, 64, 2560) == 0 and L.wan_gemm_mxfp4_scratch_bytes(16, 64, 2560) == 0   # (few rows stay in the LDS)
    assert L.wan_linear_mxfp4_scratch_bytes(17, 64, 5120) >= 17 * 2560 + 20 * 1024 + need and L.wan_gemm_mxfp4_scratch_bytes(4096, 5120, 5120) == 0


def test_scratch_and_scale_sizes():
    L = lib.load()
    assert L.wan_mxfp4_scale_bytes(1, 32) == 1024 and L.wan_mxfp4_scale_bytes(129, 257) == 4096 and L.wan_mxfp4_scale_bytes(0, 32) == 0 and L.wan_mxfp4_scale_bytes(75600, 13824) == 591 * 54 * 1024
    assert L.wan_select_blocks_scratch_bytes(2, 4, 3, 256) == 0 and L.wan_select_blocks_scratch_bytes(2, 4, 3, 257) == 2 * 4 * 3 * 257 * 8   # (fewer stay in the LDS)
    assert L.wan_select_blocks_scratch_bytes(0, 1, 1, 1) == 0 and L.wan_select_blocks_scratch_bytes(1, 40, 591, 1182) >= 0


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, 64, 2, 128, dtype=torch.bfloat16)
    m = torch.zeros(1, 2, 1, 128)
    for call in (lambda: ops.block_mean(z, 64), lambda: ops.select_blocks(m, m, 1), lambda: ops.sparse_attention(z, z, torch.zeros(1, 256, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 1, 1, dtype=torch.int32)),
                 lambda: ops.mxfp4_quantize(z), lambda: ops.mxfp4_dequantize(torch.zeros(1, 16, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8)),
                 lambda: ops.linear_mxfp4(z, torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8)), lambda: ops.pay_sparse_attention([z, z, z], 1)):
        with pytest.raises(lib.WanHipError, match="CPU|CUDA"):
            call()
