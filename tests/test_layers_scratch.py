"""CPU tests of the learned layers' scratch: the size queries against what the passes count
(tests/layer_scratch_check.cpp, linked with the library's objects), the order of its uses against
fakes (tests/scratch_order_check.cpp), and the choice between kernels (tests/few_rows_check.cpp)."""
import importlib.util
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
PKG = ROOT / "alphafold2-webgpu_b200"


def _build_module():
    spec = importlib.util.spec_from_file_location("af2_build", PKG / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_queries_cover_every_part_of_the_gradients(tmp_path):
    mod = _build_module()
    mod.build()
    cuda = Path(mod.nvcc()).resolve().parent.parent
    exe = tmp_path / "layer_scratch_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(PKG / "csrc"), "-I", str(ROOT / "include"), "-isystem",
                    str(cuda / "include"), str(ROOT / "tests" / "layer_scratch_check.cpp"),
                    *map(str, sorted((PKG / "csrc" / "_build").glob("*.o"))), "-o", str(exe),
                    f"-L{cuda / 'lib64'}", "-lcudart_static", "-ldl", "-lrt", "-pthread"], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.strip() == "ok"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_order_between_uses_of_the_scratch(tmp_path):
    exe = tmp_path / "scratch_order_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(PKG / "csrc"), str(ROOT / "tests" / "scratch_order_check.cpp"),
                    "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.strip() == "ok"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_choice_of_the_kernel_for_few_rows(tmp_path):
    cuda = Path(_build_module().nvcc()).resolve().parent.parent
    exe = tmp_path / "few_rows_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(PKG / "csrc"), "-isystem", str(cuda / "include"),
                    str(ROOT / "tests" / "few_rows_check.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.strip() == "ok"
