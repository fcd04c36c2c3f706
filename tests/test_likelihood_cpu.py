"""Likelihood and distillation operators on CPU tensors against the 64-bit oracle: the
semantics (masks, empty rows, extremes, repeated and bad indices, layouts), gradients, and
every refusal. The GPU tests run the same cases through the kernels."""

import ctypes
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import likelihood_cases as K  # noqa: E402
from cherimoya_b200 import _lib  # noqa: E402

DEV = torch.device("cpu")


@pytest.mark.parametrize("case", K.SCORE, ids=str)
def test_scores(case):
    K.case_scores(DEV, *case)


@pytest.mark.parametrize("case", K.DISTILL, ids=str)
def test_distill(case):
    K.case_distill(DEV, *case)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [K.F32, K.BF16, K.F16])
def test_odd_values(dtype, masked):
    K.case_odd_values(DEV, dtype, masked)


def test_bad_indices():
    K.case_bad_indices(DEV)


def test_empty():
    K.case_empty(DEV)


def test_layouts():
    K.case_layouts(DEV)


def test_differences():
    K.case_differences(DEV)


def test_teacher_and_student():
    K.case_teacher_student(DEV)


@pytest.mark.parametrize("match,call", K.REFUSED, ids=[str(i) for i in range(len(K.REFUSED))])
def test_refusals(match, call):
    K.case_refused(DEV, match, call)


def test_no_second_derivative():
    K.case_no_second_derivative(DEV)


def test_abi_rejects_before_any_launch():
    """Null pointers, sizes and types that the kernels do not take are refused on the host."""
    lib = _lib.load()
    off = (ctypes.c_int64 * 1)(0)
    size = (ctypes.c_int32 * 1)(10)
    bogus = 64                                   # aligned, never dereferenced

    def rows(**kw):
        d = dict(logits=bogus, dtype=0, n_groups=1, n_examples=2, row_stride=10,
                 group_offset=ctypes.addressof(off), group_size=ctypes.addressof(size), mask=None,
                 mask_row_stride=0, mask_group_offset=None, grad=None, grad_row_stride=0,
                 grad_group_offset=None, temperature=1.0)
        d.update(kw)
        return _lib.Rows(*[d[f] for f, _ in _lib.Rows._fields_])

    def score(r, targets=None, s=0, k=0, lp=None, top=None, at=None):
        return lib.chm_log_probs(r, targets, s, k, lp, None, None, top, at, None, None)

    too_long = (ctypes.c_int32 * 1)((1 << 20) + 1)
    for bad in (dict(logits=None), dict(logits=62 + 1), dict(dtype=3), dict(n_groups=0),
                dict(n_examples=-1), dict(group_offset=None), dict(group_size=None),
                dict(temperature=0.0), dict(temperature=float("nan")), dict(mask=bogus),
                dict(grad=bogus), dict(group_size=ctypes.addressof(too_long))):
        assert score(rows(**bad)) == 1, bad
    assert score(rows(n_examples=1 << 31)) == 2
    assert score(rows(), s=1) == 1 and score(rows(), s=1025, targets=bogus, lp=bogus) == 1
    assert score(rows(), k=1) == 1 and score(rows(), k=129, top=bogus, at=bogus) == 1
    assert score(rows(n_examples=0, logits=None)) == 0
    assert lib.chm_log_probs_backward(rows(), None, 0, None, 0, bogus, None, None, None, None,
                                      None, None) == 1          # no gradient buffer
    g = rows(grad=bogus, grad_group_offset=ctypes.addressof(off))
    assert lib.chm_log_probs_backward(g, None, 0, None, 0, None, None, None, None, None, None,
                                      None) == 1                # no statistics
    assert lib.chm_log_probs_backward(g, None, 0, None, 0, bogus, None, None, bogus, None, None,
                                      None) == 1                # entropy's gradient without it

    def distill(r, i=bogus, p=bogus, k=1, stride=0, row_loss=bogus, loss=None):
        return lib.chm_distill(r, i, p, k, 0, None, 1.0, None, stride, row_loss, loss, None)

    assert distill(rows(), i=None) == 1 and distill(rows(), p=None) == 1
    assert distill(rows(), k=-1) == 1 and distill(rows(), k=1025) == 1
    assert distill(rows(), stride=2) == 1
    assert distill(rows(), row_loss=None, loss=bogus) == 1


@pytest.mark.parametrize("v,k", [(50, 7), (900, 40)])
def test_hard_rows(v, k):
    K.case_hard_rows(DEV, K.F32, v, k)


@pytest.mark.parametrize("v,k", [(60, 20), (70000, 90)])
def test_repeats(v, k):
    K.case_repeats(DEV, v, k, 3)


def test_many_targets():
    K.case_many_targets(DEV, 2000)


@pytest.mark.parametrize("T", [1 / 1024, 1024.0])
@pytest.mark.parametrize("dtype", [K.F32, K.F16])
def test_temperatures(dtype, T):
    K.case_temperatures(DEV, dtype, T)


@pytest.mark.parametrize("current", [0, 1])
def test_launches_on_the_logits_device(monkeypatch, current):
    """The call runs with the logits' device current, on that device's stream, whichever device
    was current, and that one is current again behind it."""
    from cherimoya_b200 import ops
    state = {"current": current}

    class Guard:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, state["current"] = state["current"], self.index

        def __exit__(self, *_):
            state["current"] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    seen = ops._on(torch.device("cuda", 1), lambda *a: (state["current"],) + a, "x")
    assert seen == (1, "x", 101) and state["current"] == current


@pytest.mark.parametrize("dtype", [K.F32, K.BF16])
def test_ends(dtype):
    K.case_ends(DEV, dtype, 131, 40, 5)
