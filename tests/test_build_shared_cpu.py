"""Registers and spills of the kernels around a cache of shared pages, by the compiler's own count."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = {"pages_shared_kernel": 96, "pages_shared_tc_kernel": 184}       # bytes of stores a thread; none of the others spills
USED = {"pages_shared_kernel": 80, "pages_shared_tc_kernel": 96}        # what their warps' shares add up to
FORMS = """#include "rotary.cuh"
#include "pages_rows.cuh"
#include "pages_shared.cuh"
#include "pages_shared_tc.cuh"
using namespace b200;
""" + "".join(f"template __global__ void b200::rope_kernel<{n}>(const __grid_constant__ RopeParams, int, int);\n" for n in ("true", "false")) + "".join(
    f"template __global__ void b200::pages_write_kernel<{v}, {n}>(const __grid_constant__ PageWrite, int);\n" for v in ("true", "false") for n in (1, 2)) + "".join(
    f"template __global__ void b200::pages_read_kernel<{n}>(const __grid_constant__ PageRead);\n" for n in (0, 1, 2)) + "".join(
    f"template __global__ void b200::pages_shared_join_kernel<{n}>(const __grid_constant__ PageShared);\n" for n in (1, 2, 8))


def test_registers_and_spills(tmp_path):
    spec = importlib.util.spec_from_file_location("bonsai_b200_build_shared", os.path.join(ROOT, "p40-kernel_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    if not shutil.which(b.NVCC):
        pytest.skip("no nvcc")
    (tmp_path / "forms.cu").write_text(FORMS)
    run = subprocess.run([b.NVCC, *[f for f in b.FLAGS if f != "-shared"], "-Xptxas", "-v", f"-I{b.CSRC}", "-c", str(tmp_path / "forms.cu"), "-o", str(tmp_path / "forms.o")],
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]
    found = re.findall(r"properties for \S*?(rope|pages_(?:write|read)|pages_shared(?:_\w+?)?)_kernel\S*\n.*?(\d+) bytes spill stores.*\n.*?Used (\d+) registers", run.stderr)
    names = {f"{n}_kernel" for n, _, _ in found}
    assert {"rope_kernel", "pages_write_kernel", "pages_read_kernel", "pages_shared_plan_kernel", "pages_shared_kernel", "pages_shared_planes_kernel", "pages_shared_tc_kernel",
            "pages_shared_join_kernel"} <= names, names
    over = [(n, int(s)) for n, s, _ in found if int(s) > MOST.get(f"{n}_kernel", 0)]
    assert not over, over
    for n, _, used in found:
        assert int(used) == USED.get(f"{n}_kernel", int(used)), (n, used)
