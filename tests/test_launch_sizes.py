"""The division that launches are sized with, on the CPU, up to INT32_MAX (tests/cpp/launch_sizes.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ceil_div_of_large_bounds(tmp_path):
    exe = str(tmp_path / "launch_sizes")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    os.path.join(ROOT, "atomflow_amd", "csrc"), "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "launch_sizes.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
