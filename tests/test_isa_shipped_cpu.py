"""The ISA guards on what ships: every translation unit compiled with the Makefile's own flags (cross-compiled here, no GPU).  test_isa_invariants.py compiles with packed
fp32 instructions allowed, which the library is not built with; its checks of the hot kernels are run here on the other setting, and in the whole library no kernel may hold
such an instruction or spill."""
import glob
import os
import re
import shutil
import subprocess

import pytest

import test_isa_invariants as inv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "wan2gp_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
UNITS = sorted(os.path.basename(p)[:-4] for p in glob.glob(os.path.join(CSRC, "*.hip")))


def flags():
    line = re.search(r"^CXXFLAGS = (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1)
    return line.replace("$(ARCH)", "gfx950").replace("$(EXTRA)", "").split()


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    out = tmp_path_factory.mktemp("shipped")

    def of(name, *_, defines=()):
        dst = out / (name + ".s")
        if not dst.exists():
            subprocess.run([HIPCC, *flags(), *defines, "-S", "--cuda-device-only", os.path.join(CSRC, name + ".hip"), "-o", str(dst)], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
        return dst.read_text()
    return of


def test_the_library_is_built_without_packed_fp32():
    f = flags()
    assert ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"] == f[f.index("-Xclang"):][:4]
    line = re.search(r"^SRCS = (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1)
    assert sorted(s[:-4] for s in line.split()) == UNITS                                     # nothing is built otherwise


@pytest.mark.parametrize("unit", UNITS)
def test_no_packed_fp32_instruction_and_no_scratch(asm, unit):
    text = asm(unit)
    spilled, packed = {}, set()
    for m in re.finditer(r"^(_Z\S+):", text, re.M):
        end = text.find(".Lfunc_end", m.end())
        size = re.search(r"; ScratchSize: (\d+)", text[end : end + 6000]) if end > 0 else None
        if size is None:
            continue
        if int(size.group(1)):
            spilled[m.group(1)] = int(size.group(1))
        if re.search(r"\bv_pk_(add|mul|fma)_f32\b", text[m.end() : end]):
            packed.add(m.group(1))
    assert not spilled and not packed, (spilled, packed)


@pytest.mark.parametrize("check", ["test_gemm256k_registers_lds_and_no_scratch", "test_gemm256k_main_loop_instruction_mix", "test_attention_w64q_no_scratch_and_hardware_conversions",
                                   "test_attention_bounded_loop_instruction_mix", "test_attention_bounded_tile_scalar_and_wait_instructions", "test_attention_w16n_tile_instruction_mix",
                                   "test_gemm256m_registers_and_stage_instruction_mix", "test_attention_xkv_stream_has_no_valu_write_in_front_of_an_mfma_that_reads_it"])
def test_hot_kernels_as_they_ship(asm, monkeypatch, check):
    monkeypatch.setattr(inv, "asm_of", asm)
    if "gemm256k" in check:
        getattr(inv, check)(inv.kernels(asm("gemm256k"), "gemm256k_kernel"))
    elif "w64q" in check or "bounded_loop" in check:
        getattr(inv, check)(inv.kernels(asm("attention_w64q"), "attn_w64q_kernel"))
    else:
        getattr(inv, check)(None)
