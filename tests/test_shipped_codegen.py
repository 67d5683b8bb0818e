"""The codegen guards on what ships (CPU only): the GEMM kernels compiled with the library's own flags, asked of its Makefile, and the
matrix instructions' wait states in them too."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_gemm_codegen as gemm
import test_mfma_wait_states as waits

pytestmark = gemm.pytestmark


def _flags():
    return subprocess.run(["make", "-s", "flags"], cwd=gemm.CSRC, check=True, capture_output=True, text=True).stdout.split()


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    """{variant: assembly}, compiled side by side."""
    folder = str(tmp_path_factory.mktemp("asm"))

    def compile_one(variant):
        out = os.path.join(folder, variant + ".s")
        subprocess.run([gemm.HIPCC, *_flags(), "-DTE_GEMM_PART=0", f"-DTE_GEMM_DEV_ONE={variant}", "--cuda-device-only", "-S",
                        "gemm_fp8.hip", "-o", out], cwd=gemm.CSRC, check=True, capture_output=True, timeout=600)
        with open(out) as fh:
            return fh.read()

    with ThreadPoolExecutor(5) as pool:
        return dict(zip(gemm.VARIANTS.values(), pool.map(compile_one, gemm.VARIANTS.values())))


def test_the_flags_are_those_of_the_build():
    flags = _flags()
    assert "-O3" in flags and "--offload-arch=gfx950" in flags and "-packed-fp32-ops" in flags
    build = subprocess.run(["make", "-n", "-B", "build/lora.o"], cwd=gemm.CSRC, check=True, capture_output=True, text=True).stdout
    assert " ".join(flags) in build


def test_the_wait_state_guard_compiles_with_them():
    with open(waits.__file__) as fh:
        guard = fh.read()
    host_only = ("-W", "-fvisibility")
    assert [f for f in _flags() if not f.startswith(host_only) and f'"{f}"' not in guard] == []


@pytest.mark.parametrize("name", list(gemm.VARIANTS))
def test_gemm_k_loops(name, asm, monkeypatch, tmp_path):
    monkeypatch.setattr(gemm, "_asm_of", lambda variant, _: asm[variant])
    gemm.test_k_loop_has_no_compiler_vmem_wait_and_no_scratch(name, tmp_path)
    if "K-major (" in name:
        gemm.test_bare_asm_dma_in_k_loop_sees_no_valu_written_sgpr(name, tmp_path)


@pytest.mark.parametrize("name", list(gemm.VARIANTS))
def test_gemm_results_are_not_read_early(name, asm, monkeypatch):
    """32x32x64, sixteen passes: 20 wait states, the compiler's own smallest distance on straight lines."""
    monkeypatch.setattr(waits, "WAIT_STATES", 20)
    kernels = waits._kernels(asm[gemm.VARIANTS[name]])
    assert sum("v_mfma" in t for blocks in kernels.values() for _, ins in blocks for t in ins) >= 16
    assert not any(waits._early_reads(blocks) for blocks in kernels.values())


@pytest.mark.parametrize("name", list(gemm.VARIANTS))
def test_no_packed_fp32_instruction(name, asm):
    assert not any(i.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32")) for i in gemm._instructions(asm[gemm.VARIANTS[name]]))
