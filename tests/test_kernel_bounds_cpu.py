"""What the kernels of the operators around a linear layer read and write, on the CPU: their own sources (rms_norm.hip, global_norm.hip,
gemm_epilogue.hip, gemm_epilogue.hpp, gemm_edge.hip) and entry points (linear_ops.cpp) compiled for the host (tests/fake_hip/emu/), every operand flush
against pages that may not be touched -- at its end, then at its start -- over the shapes at which the kernels change their form.  Inline assembly
is taken out (a wave's wait becomes a meeting of its lanes); nothing else of the sources changes."""
import platform
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC, EMU = ROOT / "cubecl_amd" / "csrc", ROOT / "tests" / "fake_hip" / "emu"
CLANG = "/opt/rocm/llvm/bin/clang++"
KERNELS = ["rms_norm.hip", "global_norm.hip", "gemm_epilogue.hip", "gemm_edge.hip", "linear_ops.cpp"]
HEADERS = ["internal.hpp", "gemm_common.hpp", "rowops.hpp", "gemm_epilogue.hpp", "linear_ops.hpp", "row_span.hpp"]


def for_the_host(text):
    text = text.replace('asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");', "emu_wave_sync();")
    text = text.replace("__builtin_amdgcn_sched_barrier(0);", "emu_wave_sync();")
    text = re.sub(r"^(\s*)asm(?: volatile)?\(.*?\);(?=\s)", r"\1;", text, flags=re.M)
    return text.replace("__attribute__((address_space(4))) ", "")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not Path(CLANG).exists() or platform.machine() != "x86_64":
        pytest.skip("no clang++ with the kernels' vector types, or no x86-64 to switch fibers on")
    d = tmp_path_factory.mktemp("emu")
    src = d / "cubecl_amd" / "csrc"
    src.mkdir(parents=True)
    (d / "include").mkdir()
    shutil.copy(ROOT / "include" / "mi355cube.h", d / "include")
    for name in KERNELS + HEADERS:
        (src / name).write_text(for_the_host((CSRC / name).read_text()))
    jobs = []
    for name in KERNELS + [str(EMU / "bounds.cpp")]:
        f = src / name if name in KERNELS else Path(name)
        obj = d / (f.stem + ".o")
        jobs.append((obj, subprocess.Popen([CLANG, "-std=c++20", "-O2", "-w", "-I", str(EMU), "-I", str(src), "-x", "c++", "-c", str(f), "-o", str(obj)], stderr=subprocess.PIPE, text=True)))
    for obj, job in jobs:
        err = job.communicate()[1]
        assert job.returncode == 0, err[:3000]
    exe = d / "bounds"
    subprocess.run([CLANG, "-o", str(exe)] + [str(o) for o, _ in jobs], check=True)
    runs = {}                                            # both sides at once
    for side in ("end", "front"):
        with open(d / side, "w") as log:
            runs[side] = subprocess.Popen([str(exe), side], stdout=log), d / side
    yield runs
    for run, _ in runs.values():
        run.kill()


@pytest.mark.parametrize("side", ["end", "front"])
def test_nothing_outside_an_operand_is_touched_and_every_output_is_written(program, side):
    run, log = program[side]
    status = run.wait(timeout=900)
    lines = log.read_text().splitlines()
    assert status == 0 and lines[-1] == "clean", (status, lines[-3:], [l for l in lines if "not written" in l or " for " in l][:5])
