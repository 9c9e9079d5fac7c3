"""The C++ provider over the paged cache (include/mugen_attn_paged.hpp): it compiles as
C++20 and C++23 host code, and tests/cpp/paged_check.cpp (built by
__graft_entry__.build()) drives it on the GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("std", ["c++20", "c++23"])
def test_provider_header_compiles(tmp_path, std):
    cxx = shutil.which("g++")
    if cxx is None or not os.path.isdir("/opt/rocm/include"):
        pytest.skip("no host C++ compiler / ROCm headers")
    src = tmp_path / "paged.cpp"
    src.write_text('#include "mugen_attn_paged.hpp"\n'
                   "int main() { std::unique_ptr<mugen_attn::GqaAttentionPaged> a;\n"
                   "  return mugen_attn::GqaAttentionPaged::create(mugen_attn::GqaPagedShape{}, &a) ? 1 : 0; }\n")
    subprocess.run([cxx, f"-std={std}", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", "-c", str(src), "-I",
                    os.path.join(ROOT, "include"), "-I", "/opt/rocm/include", "-o", str(tmp_path / "paged.o")], check=True)


@pytest.mark.gpu
def test_provider(device):
    exe = os.path.join(ROOT, "tests", "cpp", "paged_check")
    assert os.path.exists(exe), "tests/cpp/paged_check is built by __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout[-4000:], r.stderr[-2000:], flush=True)
    assert r.returncode == 0 and r.stdout.strip().endswith("PASS"), r.stdout[-2000:]
    assert r.stdout.count(" done") == 4
