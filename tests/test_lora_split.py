"""How the adapters' first product cuts K, on the CPU: tests/cpp/lora_split.cpp walks the arithmetic that the launch
and its kernels share (af_lora_split.h)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_load_within_its_row(tmp_path):
    exe = str(tmp_path / "lora_split")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "atomflow_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "lora_split.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout[-1000:])
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout[:1000]
