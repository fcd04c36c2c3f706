"""The likelihood and distillation operators on CPU tensors: the cases of
likelihood_edge_cases.py, and what needs no device."""

import ctypes
import decimal
import math
import os
import random
import subprocess
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import likelihood_edge_cases as E  # noqa: E402
from cherimoya_b200 import _lib  # noqa: E402

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


def test_exp64(tmp_path):
    """The kernels' 64-bit exponential, compiled for the host, against 40 digits: within 1e-14
    of itself, the bound that its comment derives."""
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    src, so = tmp_path / "e.cc", tmp_path / "e.so"
    src.write_text('#include "chm_exp64.h"\n'
                   'extern "C" double e(double x) { return chm::lk::exp64(x); }\n')
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-I", csrc, str(src), "-o", str(so)],
                   check=True)
    f = ctypes.CDLL(str(so)).e
    f.argtypes, f.restype = [ctypes.c_double], ctypes.c_double
    rng = random.Random(3)
    log2 = math.log(2.0)
    xs = [rng.uniform(-700, 700) for _ in range(4000)] + [rng.uniform(-2, 2) for _ in range(4000)]
    xs += [(n + 0.5) * log2 * (1 + s) for n in range(-1009, 1009) for s in (-1e-15, 0.0, 1e-15)]
    xs += [0.0, -0.0, 5e-324, -5e-324, 1e-300, 700.0, -700.0] + [2.0 ** -i for i in range(60)]
    with decimal.localcontext() as ctx:
        ctx.prec = 40
        off = max(abs(decimal.Decimal(f(x)) / decimal.Decimal(x).exp() - 1) for x in xs)
    assert off < 1e-14
    assert f(-700.1) == f(-math.inf) == 0.0 and f(700.1) == f(math.inf) == math.inf
    assert math.isnan(f(math.nan)) and f(0.0) == 1.0


@pytest.mark.parametrize("every", [0, 8])
def test_long_sums(every):
    E.case_long_sums(DEV, F32, 2, every)


@pytest.mark.parametrize("v", [900, 40000])
def test_one_target(v):
    E.case_one_target(DEV, v)


def test_abi_outputs_that_may_not_be_null():
    """Of chm_log_probs' outputs those of given and top entries are needed where there are such."""
    lib = _lib.load()
    off, size = (ctypes.c_int64 * 1)(0), (ctypes.c_int32 * 1)(10)
    bogus = 64                                   # aligned, never dereferenced
    rows = _lib.Rows(bogus, 0, 1, 2, 10, ctypes.addressof(off), ctypes.addressof(size), None, 0,
                     None, None, 0, None, 1.0)
    for s, k, lp, top, at in ((1, 0, None, None, None), (1, 1, None, bogus, bogus),
                              (0, 1, None, None, bogus), (0, 1, None, bogus, None)):
        assert lib.chm_log_probs(rows, bogus, s, k, lp, None, None, top, at, None, None) == 1


@pytest.mark.filterwarnings("ignore:Dynamo detected a call to a .functools.lru_cache")
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled(dynamic):
    E.case_compiled(DEV, dynamic)


@pytest.mark.parametrize("masked", [False, True])
def test_many_long_rows(masked):
    E.case_many_long_rows(DEV, F32, masked, 1)
