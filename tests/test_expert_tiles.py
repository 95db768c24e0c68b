"""Builds and runs the host checks of the grouped product's tile sequence (tests/cpp/test_expert_tiles.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tile_sequence(tmp_path):
    out = str(tmp_path / "test_expert_tiles")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "ponni_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "test_expert_tiles.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
