"""CPU tests of the answer operators' argument checks and sizes at their edges."""
import ctypes as ct

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ytm_b200 import _lib, answers


@pytest.mark.parametrize("x", ["YTM_BITS", "YTM_F32", "YTM_F16", "YTM_BF16"])
@pytest.mark.parametrize("c,k", [(33, 2), (2048, 1000), (10000, 10), (65536, 100), (65536, 4000), (1 << 20, 700)])
@pytest.mark.parametrize("group", [32, 128])
def test_votes_workspace_does_not_grow_with_the_samples(x, c, k, group):
    size = lambda n: _lib.load().ytm_q4_votes_workspace_bytes(getattr(_lib, x), n, c, k, group)  # noqa: E731
    sizes = [size(n) for n in (1, 64, 1000, 30000, 250000, 1 << 24, (1 << 31) - 1)]
    assert all(0 < s <= 1 << 30 for s in sizes), sizes


def test_gave_up_needs_a_place_for_the_count():
    assert _lib.load().ytm_q4_votes_gave_up(None, None) == 1


def test_tensors_without_memory_of_their_own_are_refused():
    with FakeTensorMode():
        cs, i = torch.empty((3, 8), device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")
    for f in (lambda: answers.answer(cs), lambda: answers.class_loss(cs, i), lambda: answers.q4_pack(cs),
              lambda: answers.q4_votes(cs, cs.byte(), cs, 32)):
        with pytest.raises(ValueError, match="memory"):
            f()
    with pytest.raises(TypeError, match="strided"):
        answers.answer(torch.zeros((3, 8)).to_sparse())


@pytest.mark.parametrize("k", [4, 1000])
def test_loss_workspaces_off_a_boundary_are_refused(k):
    """Sums of 8 bytes lie at its start."""
    a = _lib.LossArgs(cs=16, cs_stride=k, n=100000, k=k, cs_type=_lib.YTM_I32, target=16, loss=16, temperature_all=1.0)
    for at in (4, 8, 20):
        assert _lib.load().ytm_class_loss(ct.byref(a), ct.c_void_p(at), None) == 1
