"""Row ranges, tile counts and forms of block products (csrc/block_plan.h), compiled with g++ and run without a device: offsets that
break the rules give ranges that do not overlap, so a walk never finds more tiles than a launch is sized for; the sizes that the GPU
tests name for a form reach it."""
import functools
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "vpux_plugin_b200", "csrc")


@functools.lru_cache(maxsize=None)
def compiled(name):
    out = os.path.join(tempfile.mkdtemp(), name)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-I", os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "cpp", name + ".cpp"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return out


def test_offsets_give_disjoint_rows_and_bounded_tiles():
    r = subprocess.run([compiled("test_block_plan")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "block plan: 0 failed" in r.stdout, r.stdout[-4000:] + r.stderr


def forms_of(products):
    """The form of every (rows, experts, outputs, multiprocessors)"""
    r = subprocess.run([compiled("block_form")] + [str(v) for p in products for v in p], capture_output=True, text=True, timeout=60)
    return r.stdout.split()


def test_every_form_is_reached_at_its_border():
    want = {(1, 0, 4096, 148): "Swap16", (16, 0, 32000, 148): "Swap16", (17, 0, 4096, 148): "Swap32", (64, 0, 4096, 148): "Swap32",
            (64, 0, 11008, 148): "Wide128", (65, 0, 4096, 148): "Swap128", (512, 0, 1024, 148): "Swap128", (192, 0, 4096, 148): "Wide128",
            (1024, 0, 4096, 148): "Wide256", (1500, 0, 4096, 148): "Wide128", (4096, 0, 11008, 148): "Wide256",
            (32, 64, 1024, 148): "Swap16", (2048, 64, 2048, 148): "Wide256", (901, 7, 1410, 148): "Wide128", (8192, 32, 4096, 148): "Wide256"}
    assert forms_of(want) == list(want.values())
