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
