"""The layer products without a GPU: the plan of their launches, the refusals of every entry point (with a device layer of
stubs that checks the reach of every accepted call), the exported templates, the Python calls' own checks and the reference
that the GPU tests compare with, against automatic differentiation and differences."""
import os
import shutil
import subprocess

import pytest
import torch

from clblast_amd import _lib, api
from tests import layer_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "clblast_amd", "csrc")
KINDS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def compiled(tmp_path, name, sources):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no g++ here")
    binary = tmp_path / name
    done = subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC] + sources +
                          ["-o", str(binary), "-lpthread"], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-3000:]
    run = subprocess.run([str(binary)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
    assert "violations 0" in run.stdout


def test_the_plan_of_a_launch(tmp_path):
    compiled(tmp_path, "plan", [os.path.join(ROOT, "tests", "host", "layer_plan_sweep.cpp")])


def test_refusals(tmp_path):
    compiled(tmp_path, "refusals", [os.path.join(ROOT, "tests", "host", "layer_refusals.cpp")] +
             [os.path.join(CSRC, "routines", name) for name in ("xlayer.cpp", "xgemm.cpp", "routine_common.cpp", "tile_table.cpp")])


def test_cpp_templates_are_exported():
    symbols = subprocess.run(["nm", "-D", "--defined-only", "-C", _lib.LIB_PATH], capture_output=True, text=True).stdout
    for routine in ("GemmEpilogue", "GemmActivationGradient", "ActivationGradient", "GemmGrouped", "GemmGroupedGradient"):
        for type_name in ("float", "unsigned short", "clblast::bfloat16"):
            assert "clblast::%s<%s>(" % (routine, type_name) in symbols, (routine, type_name)


def test_python_calls_refuse_what_they_cannot_pass_on():
    a = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU"):
        api.gemmEpilogue(None, 4, 4, 4, a, a, a, 4, 4, 4)
    with pytest.raises(ValueError, match="data-type"):
        api.gemmEpilogue(None, 4, 4, 4, a, a.half(), a, 4, 4, 4)
    with pytest.raises(ValueError, match="unknown activation"):
        api.gemmEpilogue(None, 4, 4, 4, a, a, a, 4, 4, 4, activation="tanh")
    with pytest.raises(ValueError, match="unknown activation"):
        api.activationGradient(None, 4, 4, a, a, a, 4, 4, 4, activation="swish")


@pytest.mark.parametrize("kind", KINDS)
def test_reference_against_differentiation(kind):
    """Values against torch's own functions, slopes against automatic differentiation and central differences (in 64 bits an
    error of h^2 / 6 times the third derivative, below 3 here, plus 2^-52 / h: below 1e-9 for h = 1e-5)"""
    g = torch.Generator().manual_seed(1)
    z = (3 * torch.randn(2000, generator=g, dtype=torch.float64)).requires_grad_()
    theirs = {"none": lambda x: x, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
              "gelu_tanh": lambda x: torch.nn.functional.gelu(x, approximate="tanh"), "silu": torch.nn.functional.silu}[kind](z)
    theirs.sum().backward()
    at = z.detach()
    assert float((ref.act(at, kind) - theirs.detach()).abs().max()) < 1e-14
    assert float((ref.slope(at, kind) - z.grad).abs().max()) < 1e-14
    h = 1e-5
    smooth = at[at.abs() > 2 * h] if kind == "relu" else at
    differences = (ref.act(smooth + h, kind) - ref.act(smooth - h, kind)) / (2 * h)
    assert float((ref.slope(smooth, kind) - differences).abs().max()) < 1e-9
