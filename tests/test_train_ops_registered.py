"""torch.ops.dmb has the training operators' CUDA kernels as soon as the package is imported."""

import subprocess
import sys

import pytest

from dtensor_muon_b200.ops import _ext

OPS = ["qk_norm_rope", "qk_norm_rope_backward", "route", "route_backward", "token_logprobs", "token_logprobs_backward",
       "policy_loss", "preference_loss"]


def _fresh(code):
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    return out.stdout


@pytest.mark.skipif(not _ext.available(), reason="needs the built extension")
def test_the_kernels_are_registered_on_import():
    got = _fresh("import torch, dtensor_muon_b200\n"
                 f"for op in {OPS}: print(op, torch._C._dispatch_has_kernel_for_dispatch_key('dmb::' + op, 'CUDA'))\n"
                 "print(torch.cuda.is_initialized())")
    assert got.split() == [w for op in OPS for w in (op, "True")] + ["False"]


def test_a_package_that_is_not_built_can_be_imported():
    got = _fresh("import importlib.util, sys\n"
                 "find = importlib.util.find_spec\n"
                 "importlib.util.find_spec = lambda name, *a: None if name.endswith('._C') else find(name, *a)\n"
                 "import torch, dtensor_muon_b200\n"
                 "from dtensor_muon_b200.ops import _ext\n"
                 "print(_ext._C is None, _ext._IMPORT_ERROR is None, 'route' in dir(torch.ops.dmb) or bool(torch.ops.dmb.route))")
    assert got.split() == ["True", "True", "True"]


@pytest.mark.gpu
def test_a_kernel_is_the_first_call():
    _fresh("import torch, dtensor_muon_b200\n"
           "x = torch.randn(9, 8, device='cuda', requires_grad=True)\n"
           "r = torch.ops.dmb.route(x, 2, None)\n"
           "r[3].backward()\n"
           "assert x.grad.any()")
