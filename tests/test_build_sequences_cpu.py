"""What the kernels of the calls for several sequences spill, by the compiler's own count."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = {  # bytes of stores a thread; none of the others spills
    "pages_tc_kernel": 260,             # 96 registers, of which 64 are a row's sums
    "pages_redo_kernel": 12, "gdn_chunk_kernel": 48}
FORMS = """#include "gdn_seqs.cuh"
#include "heads.cuh"
#include "pages.cuh"
#include "pages_tc.cuh"
using namespace b200;
""" + "".join(f"template __global__ void b200::pages_attn_kernel<{n}>(const __grid_constant__ PageAttn, int);\n" for n in (0, 1, 2, 4)) + "".join(
    f"template __global__ void b200::pages_join_kernel<{n}>(const __grid_constant__ PageAttn);\n" for n in (1, 2, 8)) + "".join(
    f"template __global__ void b200::qk_norm_rope_kernel<{n}>(const __grid_constant__ QkNormParams);\n" for n in ("true, 1", "true, 4")) + "".join(
    f"template __global__ void b200::gdn_seqs_step_kernel<{n}>(const __grid_constant__ GdnSeqs, int);\n" for n in (1, 4))


def test_spills(tmp_path):
    spec = importlib.util.spec_from_file_location("bonsai_b200_build_spills_seqs", os.path.join(ROOT, "p40-kernel_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    if not shutil.which(b.NVCC):
        pytest.skip("no nvcc")
    (tmp_path / "forms.cu").write_text(FORMS)
    run = subprocess.run([b.NVCC, *[f for f in b.FLAGS if f != "-shared"], "-Xptxas", "-v", f"-I{b.CSRC}", "-c", str(tmp_path / "forms.cu"), "-o", str(tmp_path / "forms.o")],
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]
    found = re.findall(r"properties for \S*?(qk_norm_rope|pages_\w+?|gdn_\w+?)_kernel\S*\n.*?(\d+) bytes spill stores", run.stderr)
    names = {f"{n}_kernel" for n, _ in found}
    assert {"qk_norm_rope_kernel", "pages_attn_kernel", "pages_join_kernel", "pages_tc_kernel", "pages_redo_kernel", "pages_planes_kernel", "gdn_seqs_step_kernel",
            "gdn_planes_kernel", "gdn_chunk_kernel", "gdn_scan_kernel"} <= names, names
    over = [(n, int(s)) for n, s in found if f"{n}_kernel" != "gdn_step_kernel" and int(s) > MOST.get(f"{n}_kernel", 0)]
    assert not over, over
