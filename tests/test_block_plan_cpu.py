"""Row ranges and tile counts of grouped block products (csrc/block_plan.h), compiled with g++ and run without a device: offsets
that break the rules give ranges that do not overlap, so a walk never finds more tiles than a launch is sized for."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "vpux_plugin_b200", "csrc")


def compiled(name, tmp_path):
    out = str(tmp_path / name)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-I", os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "cpp", name + ".cpp"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return out


def test_offsets_give_disjoint_rows_and_bounded_tiles(tmp_path):
    r = subprocess.run([compiled("test_block_plan", tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "block plan: 0 failed" in r.stdout, r.stdout[-4000:] + r.stderr
