"""The likelihood and distillation kernels on the cases of likelihood_edge_cases.py."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import likelihood_edge_cases as E  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# a block to a row, and clusters of two, four and eight
@pytest.mark.parametrize("v,rows", [(4003, 3), (8003, 3), (20011, 30), (70001, 3), (150001, 6)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_candidates(dtype, v, rows):
    E.case_candidates(DEV, dtype, v, rows)
