"""The likelihood and distillation operators on CPU tensors: the cases of
likelihood_edge_cases.py, and what needs no device."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import likelihood_edge_cases as E  # noqa: E402

DEV = torch.device("cpu")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_candidates(dtype):
    E.case_candidates(DEV, dtype, 5003, 3)


@pytest.mark.parametrize("v,k", [(700, 1), (30001, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_small_mass(dtype, v, k):
    E.case_small_mass(DEV, dtype, v, k, 4)


@pytest.mark.parametrize("transform", sorted(E.TRANSFORMS))
@pytest.mark.parametrize("call", E.CALLS)
def test_transforms(call, transform):
    E.case_transforms(DEV, call, transform)


def test_beside_forward_mode():
    E.case_beside_forward_mode(DEV)


@pytest.mark.parametrize("transform", ["grad", "jvp", "vmap", "dual"])
@pytest.mark.parametrize("call", ["scores", "loss and grad"])
def test_transforms_while_tracing(call, transform):
    """Inside a compiled function and around one."""
    x, f = E._calls()[call]
    t = E.TRANSFORMS[transform]
    torch._dynamo.reset()
    inside = torch.compile(lambda v: t(lambda u: f(DEV, u), v), backend="eager")
    compiled = torch.compile(lambda v: f(DEV, v), backend="eager")
    assert torch.isfinite(compiled(x)).all()
    for run in (inside, lambda v: t(compiled, v)):
        with pytest.raises(Exception, match="forward-mode"):
            run(x)
    torch._dynamo.reset()


def test_temperature_is_a_number():
    E.case_temperature_is_a_number(DEV)
