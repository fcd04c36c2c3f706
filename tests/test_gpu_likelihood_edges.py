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


@pytest.mark.filterwarnings("ignore:Dynamo detected a call to a .functools.lru_cache")
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled(dynamic):
    E.case_compiled(DEV, dynamic)


def test_custom_ops_check():
    """The three custom ops behind compiled calls: their schemas, fake implementations and
    dispatch, as torch.library checks them."""
    from cherimoya_b200 import ops
    tests = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    g = torch.Generator().manual_seed(3)
    z = torch.randn(4, 3, 50, generator=g).to(DEV)
    t = torch.randint(0, 50, (4, 2, 5), generator=g).to(DEV)
    lp = torch.full((4, 2, 5), -2.0, device=DEV)
    m = torch.rand(4, 3, 50, generator=g).to(DEV) < 0.8
    w, up = torch.rand(4, 2, generator=g).to(DEV), torch.randn((), generator=g).to(DEV)
    for mask in (None, m):
        for stats in (False, True):
            torch.library.opcheck(ops.log_probs, (z, mask, [1, 2], t, 3, 1.5, stats),
                                  test_utils=tests)
        out = ops.log_probs(z, mask, [1, 2], t, 3, 1.5, True)
        torch.library.opcheck(ops.log_probs_backward,
                              (z, mask, [1, 2], t, out[4], out[5], out[1], lp, w, None, None, 1.5),
                              test_utils=tests)
        for weight, upstream, reduce, grad in ((None, None, False, True), (w, up, True, True),
                                               (w, w, False, True), (None, None, True, False)):
            torch.library.opcheck(ops.distill, (z, mask, [1, 2], t, lp, False, weight, 0.25,
                                                upstream, not reduce, reduce, grad, 1.5),
                                  test_utils=tests)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_many_long_rows(dtype, masked):
    E.case_many_long_rows(DEV, dtype, masked, 150)
