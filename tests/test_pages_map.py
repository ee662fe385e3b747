"""The bookkeeping of shared KV pages on the CPU (tests/pages_map_check.cpp)."""
import os
import subprocess

from conftest import ROOT


def test_pages_are_mapped_whole_or_not_at_all(tmp_path):
    exe = str(tmp_path / "pages_map_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I",
                    os.path.join(ROOT, "llama3.go_b200", "csrc"),
                    os.path.join(ROOT, "tests", "pages_map_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr
