"""CPU tier: calls of the token-wise operators that torch's transformations make, which are refused before anything reaches a GPU."""
import os

import pytest
import torch


@pytest.fixture(scope="module")
def ops():
    from vae_gan_amd import lib as L
    if not os.path.exists(L.LIB_PATH) or not os.path.exists(os.path.join(os.path.dirname(L.LIB_PATH), "_vgtorch.so")):
        pytest.skip("the libraries are not built")
    from vae_gan_amd import ops
    return ops


def calls(ops):
    """(operator, its floating-point arguments)"""
    tokens = torch.zeros(2, dtype=torch.int64)
    return [(ops.layer_norm, [torch.ones(2, 8), torch.ones(8), torch.ones(8)]),
            (lambda x, w, b, r: ops.linear_act(x, w, b, 3, r), [torch.ones(2, 8), torch.ones(4, 8), torch.ones(4), torch.ones(2, 4)]),
            (lambda x: ops.token_logprobs(x, tokens)[0], [torch.ones(2, 8)])]


def test_tangents_are_refused(ops):
    """Without a gradient wanted the kernels run outside autograd: a dual tensor must not come back without its tangent."""
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        for call, args in calls(ops):
            for i in range(len(args)):
                duals = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*duals)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*duals)


def test_traces_are_refused(ops):
    """A trace would hold the allocation of the result and nothing that writes it."""
    for call, args in calls(ops):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(lambda *a: call(*a), tuple(args))
