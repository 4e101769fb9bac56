"""The kernels of attention over a paged cache keep what they hold in registers: their code objects'
own notes say so (a spill there is a load in the loop over the keys)."""
import os
import re
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
TOOLS = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


def spills(name, tmp_path):
    code = os.path.join(HERE, "..", "llama.rust_amd", name + ".hsaco")
    tools = [os.path.join(TOOLS, t) for t in ("clang-offload-bundler", "llvm-readelf")]
    if not os.path.exists(code) or not all(shutil.which(t) for t in tools):
        pytest.skip("no code object, or no tool to read it")
    obj = str(tmp_path / "k.o")
    subprocess.run([tools[0], "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=" + code, "--output=" + obj], check=True)
    notes = subprocess.run([tools[1], "--notes", obj], check=True, capture_output=True, text=True).stdout
    names, counts = re.findall(r"\.symbol:\s+(\S+)\.kd", notes), re.findall(r"\.vgpr_spill_count:\s+(\d+)", notes)
    assert len(names) == len(counts) > 0
    return {n: int(c) for n, c in zip(names, counts) if int(c)}


def test_paged_attention(tmp_path):
    assert spills("ghip_fap", tmp_path) == {}
