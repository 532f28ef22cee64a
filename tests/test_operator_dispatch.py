"""Every kernel of the operators is launched by some size that the GPU tests run (CPU only: the host code that
chooses the kernels runs with a launch that records them)."""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest
import test_int8_gpu
import test_int8_kernels_gpu
import test_qk_norm_gpu

from stagehand_amd.int8 import DTYPE_CODES

REPO = Path(__file__).resolve().parent.parent
CSRC, NATIVE, CLANG = REPO / "stagehand_amd" / "csrc", REPO / "tests" / "native", Path("/opt/rocm/llvm/bin/clang++")
pytestmark = pytest.mark.skipif(not CLANG.exists() or not (NATIVE / "dispatch.cpp").exists(),
                                reason="needs ROCm's clang and tests/native")

KERNELS = re.findall(r'\{kMod(?:Int8|QkNorm), "(\w+)"\}', (CSRC / "sh_kernels.cpp").read_text())


def parametrised(test, name):
    """The values that a test's parametrize marks give ``name`` (its whole tuple of names)."""
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0] == name)


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    """calls → the kernels that each launches, in order"""
    exe = tmp_path_factory.mktemp("dispatch") / "dispatch"
    subprocess.run([str(CLANG), "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{REPO / 'include'}",
                    f"-I{CSRC}", str(CSRC / "sh_int8.cpp"), str(CSRC / "sh_qk_norm.cpp"), str(NATIVE / "dispatch.cpp"), "-o",
                    str(exe)], check=True)

    def run(calls):
        out = subprocess.run([str(exe)], input="\n".join(calls) + "\n", capture_output=True, text=True)
        assert out.returncode == 0, out.stderr
        return [[KERNELS[int(i)] for i in line.split()] for line in out.stdout.splitlines()]

    return run


def all_of(prefix):
    return {k for k in KERNELS if k.startswith(prefix)}


def test_sizes_of_the_int8_tests_reach_every_kernel(launched):
    calls = [f"quantize {t} {c} {code}" for t, c in parametrised(test_int8_gpu.test_quantize_tokens_is_bit_exact, "tokens,cols")
             for code in DTYPE_CODES.values()]
    for tokens, out, inp in test_int8_gpu.SIZES:  # the type that the test draws for the size
        calls.append(f"linear {tokens} {out} {inp} {DTYPE_CODES[test_int8_gpu.DTYPES[(tokens * 31 + out) % 3]]}")
    calls += [f"linear {t} {o} {i} {code}" for t, o, i in
              parametrised(test_int8_kernels_gpu.test_every_kernel_in_every_type, "tokens,out,inp") for code in DTYPE_CODES.values()]
    got = {k for line in launched(calls) for k in line}
    wanted = all_of("sh_quantize_") | all_of("sh_matmul_i8_") | all_of("sh_linear_i8_")
    assert len(wanted) == 25 and wanted <= got, f"no test reaches {sorted(wanted - got)}"


@pytest.mark.parametrize("sizes,kernels", [("TILE_128", {"sh_matmul_i8_128x128_kernel"}),
                                           ("FEW_WIDE", {f"sh_linear_i8_{t}_16x32_kernel" for t in ("bf16", "f16", "f32")}),
                                           ("FEW_NARROW", {f"sh_linear_i8_{t}_16x16_kernel" for t in ("bf16", "f16", "f32")})])
def test_the_lists_hold_what_they_are_named_for(launched, sizes, kernels):
    for t, o, i in getattr(test_int8_kernels_gpu, sizes):
        lines = launched([f"linear {t} {o} {i} {code}" for code in DTYPE_CODES.values()])
        assert {line[-1] for line in lines} == kernels, (t, o, i, lines)


def test_cases_of_the_norm_tests_reach_every_kernel(launched):
    calls = [f"norm {b} {hq} {hk} {s} {d} {rot} {DTYPE_CODES[dtype]} {int(inter)} {int(back)}"
             for b, hq, hk, s, d, rot in test_qk_norm_gpu.CASES for dtype in test_qk_norm_gpu.DTYPES for inter in (0, 1) for back in (0, 1)]
    got = {k for line in launched(calls) for k in line}
    wanted = all_of("sh_qk_norm_")
    assert len(wanted) == 49 and wanted <= got, f"no test reaches {sorted(wanted - got)}"
