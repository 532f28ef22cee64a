"""Every kernel of the training operators is launched by some size that the GPU tests run, and every size that the calls
take has a launch within the device's limits (CPU only: the host code that chooses the kernels runs with a launch that
records them)."""
from __future__ import annotations

import random
import re
import subprocess
from pathlib import Path

import pytest
import test_act8_gpu
import test_layer_norm_gpu
import test_weight_grad_act8_gpu

from stagehand_amd.int8 import DTYPE_CODES

REPO = Path(__file__).resolve().parent.parent
CSRC, NATIVE, CLANG = REPO / "stagehand_amd" / "csrc", REPO / "tests" / "native", Path("/opt/rocm/llvm/bin/clang++")
pytestmark = pytest.mark.skipif(not CLANG.exists() or not (NATIVE / "dispatch_training.cpp").exists(),
                                reason="needs ROCm's clang and tests/native")

KERNELS = re.findall(r'\{kMod(?:LayerNorm|Act8|WeightGrad), "(\w+)"\}', (CSRC / "sh_kernels.cpp").read_text())


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    """calls → the kernels that each launches, in order"""
    exe = tmp_path_factory.mktemp("dispatch") / "dispatch"
    subprocess.run([str(CLANG), "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{REPO / 'include'}",
                    f"-I{CSRC}", str(CSRC / "sh_layer_norm.cpp"), str(CSRC / "sh_act8.cpp"), str(NATIVE / "dispatch_training.cpp"),
                    "-o", str(exe)], check=True)

    def run(calls):
        out = subprocess.run([str(exe)], input="\n".join(calls) + "\n", capture_output=True, text=True)
        assert out.returncode == 0, out.stderr
        return [[KERNELS[int(i)] for i in line.split()] for line in out.stdout.splitlines()]

    return run


def reached(launched, calls, prefix, count):
    got, wanted = {k for line in launched(calls) for k in line}, {k for k in KERNELS if k.startswith(prefix)}
    assert len(wanted) == count and wanted <= got, f"no test reaches {sorted(wanted - got)}"


def test_cases_of_the_norm_tests_reach_every_kernel(launched):
    reached(launched, [f"norm {b} {s} {n} {code} {mod} {p}" for b, s, n in test_layer_norm_gpu.CASES for code in DTYPE_CODES.values()
                       for mod in (0, 1) for p in (0, 1, 2)], "sh_layer_norm_", 37)


def test_sizes_of_the_act8_tests_reach_every_kernel(launched):
    reached(launched, [f"keep {t} {c} {code} {back}" for t, c in test_act8_gpu.SIZES for code in DTYPE_CODES.values() for back in (0, 1)],
            "sh_act8_", 6)


def test_sizes_of_the_weight_gradient_tests_reach_every_kernel(launched):
    reached(launched, [f"grad {t} {o} {i} {code} 1" for t, o, i in test_weight_grad_act8_gpu.SIZES for code in DTYPE_CODES.values()],
            "sh_weight_grad_", 12)


def test_kernels_are_of_the_type_that_is_asked_for(launched):
    for name, code in zip(("bf16", "f16", "f32"), DTYPE_CODES.values()):
        calls = [f"norm 2 9 {n} {code} 0 {p}" for n in (64, 600, 2000, 9000) for p in (0, 1, 2)]
        calls += [f"keep 5 40 {code} 0", f"keep 5 40 {code} 1", f"grad 5 40 40 {code} 0", f"grad 900 4100 4100 {code} 0"]
        for line in launched(calls):
            assert f"_{name}_" in line[0]
    assert [line[0].split("_kernel")[0] for line in launched(["norm 1 5 100 1 0 0", "norm 1 5 100 1 0 1", "norm 1 5 100 1 0 2"])] == \
        ["sh_layer_norm_bf16_wave1", "sh_layer_norm_backward_bf16_wave1", "sh_layer_norm_backward_kept_bf16_wave1"]


def test_any_size_has_a_launch(launched):
    rng, calls = random.Random(0), []

    def some(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    for _ in range(3000):
        cols = some(1, 16384)
        batch = some(1, 8000000)
        calls.append(f"norm {batch} {some(1, 0x7FFFFFFF // batch)} {cols} {rng.randint(1, 3)} {rng.randint(0, 1)} {rng.randint(0, 2)}")
        cols = some(1, 0xFFFFFF)
        tokens = some(1, max(1, 0xFFFFF000 // (-(-cols // 32) * 4)))
        calls.append(f"keep {tokens} {cols} {rng.randint(1, 3)} {rng.randint(0, 1)}")
        calls.append(f"grad {tokens} {some(1, min(0x3FFFFF, 2 ** 37 // cols))} {cols} {rng.randint(1, 3)} {rng.randint(0, 1)}")
    calls += ["norm 1 2147483647 1 1 0 1", "norm 8388607 255 16384 3 1 1", "norm 8388607 1 5000 1 1 0", "keep 256 16777215 1 0", "grad 256 4194303 32 1 1", "grad 1073741000 1 1 2 1"]
    for line in launched(calls):
        assert line
