"""Build-time guard for the block-sparse attention and the MXFP4 GEMM: what their inline-asm MFMAs rest on is visible in the gfx950 ISA that hipcc emits with
the library's own flags (cross-compiled here, no GPU): no scratch, the accumulators in the accumulator file, the instruction mix of a tile / stage, and no
register written straight in front of an MFMA that reads it (hipcc pads no wait state around inline asm)."""
import collections
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    flags = re.search(r"^CXXFLAGS = (.*)$", open(os.path.join(ROOT, "wan2gp_amd", "csrc", "Makefile")).read(), re.M).group(1)
    flags = flags.replace("$(ARCH)", "gfx950").replace("$(EXTRA)", "").split()
    out = tmp_path_factory.mktemp("isa")

    def compile_(name):
        dst = out / (name + ".s")
        if not dst.exists():
            subprocess.run([HIPCC, *flags, "-S", "--cuda-device-only", os.path.join(ROOT, "wan2gp_amd", "csrc", name + ".hip"), "-o", str(dst)], check=True,
                           stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
        return dst.read_text()
    return compile_


def kernels(text, stem):
    """name -> (instruction lines, metadata) of every kernel whose mangled name contains `stem`"""
    res = {}
    for m in re.finditer(r"^(_Z\S*" + stem + r"\S*):", text, re.M):
        end = text.index(".Lfunc_end", m.end())
        lines = [l for l in (x.strip() for x in text[m.end():end].split("\n")) if l and not l.startswith((";", "."))]
        meta = {k: int(v) for k, v in re.findall(r"; (NumVgprs|NumAgprs|ScratchSize|LDSByteSize): (\d+)", text[end:end + 6000])}
        res[m.group(1)] = (lines, meta)
    return res


def _regs(tok):
    m = re.fullmatch(r"([va])\[(\d+):(\d+)\]", tok)
    if m:
        return {(m.group(1), r) for r in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.fullmatch(r"([va])(\d+)", tok)
    return {(m.group(1), int(m.group(2)))} if m else set()


def written_in_front(lines):
    """pairs of a vector-ALU instruction and the MFMA right behind it that reads what it writes"""
    bad = []
    for prev, cur in zip(lines, lines[1:]):
        if not cur.startswith("v_mfma") or not prev.startswith("v_") or prev.startswith("v_mfma"):
            continue
        written = _regs(prev.split(None, 1)[1].split(",")[0].strip())
        read = set().union(*(_regs(t.strip().split()[0]) for t in cur.split(None, 1)[1].split(",")[1:] if t.strip()))
        if written & read:
            bad.append((prev, cur))
    return bad


def spans(lines):
    """instruction counts between consecutive barriers"""
    ops = [l.split()[0] for l in lines]
    bars = [i for i, o in enumerate(ops) if o == "s_barrier"]
    return [collections.Counter(ops[a:b]) for a, b in zip(bars, bars[1:])]


def test_block_sparse_attention(asm):
    ks = kernels(asm("attention_sparse"), "attn_sparse_kernel")
    assert len(ks) == 2
    for name, (lines, meta) in ks.items():
        assert meta["ScratchSize"] == 0 and meta["LDSByteSize"] == 80 * 1024 and meta["NumAgprs"] == 256, (name, meta)
        assert not written_in_front(lines), written_in_front(lines)[:4]
        ops = collections.Counter(l.split()[0] for l in lines)
        # six tiles of 128 MFMAs and 8 for the row sums in the loop (images of K times images of V^T) and the last half's products behind it
        assert ops["v_mfma_f32_16x16x32_bf16"] == 6 * 136 + 36, ops["v_mfma_f32_16x16x32_bf16"]
        assert sum(1 for l in lines if l.startswith("buffer_load_dwordx4") and l.endswith("lds")) == 6 * 16 + 2 * 16
        assert sum(1 for l in lines if l.startswith("s_waitcnt vmcnt(8) lgkmcnt(0)")) == 6


def test_mxfp4_gemm_of_many_tiles(asm):
    ks = kernels(asm("gemm_mxfp4m"), "gemm_mxfp4m_kernel")
    assert len(ks) == 4                                              # none, GELU, gated residual, transposed
    for name, (lines, meta) in ks.items():
        assert meta["ScratchSize"] == 0 and meta["LDSByteSize"] == 160 * 1024 and meta["NumAgprs"] == 256, (name, meta)
        assert not written_in_front(lines), written_in_front(lines)[:4]
        ops = collections.Counter(l.split()[0] for l in lines)
        assert ops["v_mfma_scale_f32_16x16x128_f8f6f4"] == 256, ops   # a tile's first stage and the others
        assert ops["s_barrier"] == 3
        # a tile's first stage waits for nothing younger than the 32 stores of the epilogue in front of it, and hipcc puts no full wait behind them
        assert ops["buffer_store_dwordx4"] == 32
        first = next(i for i, l in enumerate(lines) if l.startswith("s_waitcnt vmcnt(32) lgkmcnt(0)"))
        store = max(i for i, l in enumerate(lines[:first]) if l.startswith("buffer_store"))
        assert not [l for l in lines[store:first] if "vmcnt(0)" in l], name


def test_mxfp4_gemm_of_few_tiles(asm):
    ks = kernels(asm("gemm_mxfp4"), "gemm_mxfp4_kernel")
    assert len(ks) == 8                                              # each epilogue, whole and in parts along K
    for name, (lines, meta) in ks.items():
        assert meta["ScratchSize"] == 0 and meta["NumAgprs"] >= 64, (name, meta)
        assert not written_in_front(lines), written_in_front(lines)[:4]
        ops = collections.Counter(l.split()[0] for l in lines)
        assert ops["v_mfma_scale_f32_16x16x128_f8f6f4"] == 32 and ops["s_barrier"] == 2, ops


@pytest.mark.parametrize("unit", ["attention_sparse", "sparse_select", "gemm_mxfp4", "gemm_mxfp4m", "mxfp4_ops"])
def test_no_packed_fp32_instruction_and_no_scratch(asm, unit):
    text = asm(unit)
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    sizes = re.findall(r"; ScratchSize: (\d+)", text)
    assert sizes and set(sizes) == {"0"}, sizes
