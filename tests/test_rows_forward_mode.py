"""Tensors that carry a tangent (forward-mode differentiation) are refused, as those that require gradients are: no kernel
here moves or scales a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from jax_gs_amd import _lib


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    native = _lib.tensors()
    index, x = torch.zeros(6, dtype=torch.int32), torch.zeros(6, 5)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(x, torch.ones(6, 5))
        row = forward_ad.make_dual(torch.zeros(5), torch.ones(5))
        calls = [lambda t: native.take([t], None, 3, -1, "take_rows"), lambda t: native.move([t], None, index, -1, "move_rows_"),
                 lambda t: native.dense([t], -1, "clip_grads_", False), lambda t: native.dense([t], -1, "clip_grads_", True)]
        for call in calls:
            for carries in (dual, dual[:, :]):
                with pytest.raises(RuntimeError, match="tangent"):
                    call(carries)
            call(x)
            call(forward_ad.unpack_dual(dual).primal)
        for call in (lambda: native.take([x], [row], 3, -1, "take_rows"), lambda: native.move([x], [row], index, -1, "move_rows_")):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
    for call in calls:  # beyond the level there is no tangent
        call(dual)
