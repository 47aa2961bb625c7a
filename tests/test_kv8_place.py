"""Which positions the workgroups of the 8-bit cache's append kernel take (lq_kv8_place.h), on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_new_token_once(tmp_path):
    exe = str(tmp_path / "kv8_place")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-Wall", "-Werror", "-I", os.path.join(ROOT, "latentq_llm_amd", "csrc"),
                    os.path.join(ROOT, "tests", "host", "kv8_place.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
