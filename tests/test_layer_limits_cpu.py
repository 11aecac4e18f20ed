"""What the layer products may reach and what they refuse, without a GPU: the requests of every tile replayed on the host, and
descriptors that the device layer's entry points have to turn down, the plan at the largest sizes, the argument checks with
buffers of any size."""
import os
import shutil
import subprocess

import pytest

from clblast_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "clblast_amd", "csrc")


def compiled(tmp_path, name, sources):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no g++ here")
    binary = tmp_path / name
    done = subprocess.run([compiler, "-std=c++17", "-O2", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC] + sources +
                          ["-o", str(binary), "-lpthread"], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]
    run = subprocess.run([str(binary)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
    assert "violations 0" in run.stdout


def test_no_request_leaves_its_operand(tmp_path):
    """Depths of less than a slab among them: the second team of wavefronts then has nothing, and begins behind the operand"""
    compiled(tmp_path, "requests", [os.path.join(ROOT, "tests", "host", "layer_requests.cpp")])


def test_descriptors_that_are_refused(tmp_path):
    folder = os.path.dirname(_lib.LIB_PATH)
    compiled(tmp_path, "descriptors", [os.path.join(ROOT, "tests", "host", "layer_descriptor.cpp"), "-L" + folder, "-lclblast_hip", "-Wl,-rpath," + folder])


def test_plans_of_the_largest_sizes(tmp_path):
    compiled(tmp_path, "limits", [os.path.join(ROOT, "tests", "host", "layer_limits.cpp")])


def test_calls_that_are_told_apart(tmp_path):
    compiled(tmp_path, "calls", [os.path.join(ROOT, "tests", "host", "layer_calls.cpp")] +
             [os.path.join(CSRC, "routines", name) for name in ("xlayer.cpp", "xgemm.cpp", "routine_common.cpp", "tile_table.cpp")])
