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


# a warp, blocks of 128 and 256 and a cluster to a row
@pytest.mark.parametrize("v,k,rows", [(300, 1, 9), (1000, 7, 9), (1000, 200, 9), (9001, 5, 9),
                                      (32768, 1, 400), (32768, 64, 400), (200003, 3, 3)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_small_mass(dtype, v, k, rows):
    E.case_small_mass(DEV, dtype, v, k, rows)


@pytest.mark.parametrize("transform", sorted(E.TRANSFORMS))
@pytest.mark.parametrize("call", E.CALLS)
def test_transforms(call, transform):
    E.case_transforms(DEV, call, transform)


def test_beside_forward_mode():
    E.case_beside_forward_mode(DEV)


def test_temperature_is_a_number():
    E.case_temperature_is_a_number(DEV)


# a cluster to a row, and as many rows as give each one block
@pytest.mark.parametrize("dtype,rows,every", [(F32, 3, 0), (F32, 900, 0), (F32, 3, 8),
                                              (F32, 900, 8), (BF16, 900, 0), (BF16, 900, 8)])
def test_long_sums(dtype, rows, every):
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    E.case_long_sums(DEV, dtype, rows, every)


@pytest.mark.parametrize("v", [900, 40000])
def test_one_target(v):
    E.case_one_target(DEV, v)
