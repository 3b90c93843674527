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


def test_other_operators_refuse_the_activations_of_linear_act(ops):
    """GELU and SiLU are linear_act's; a convolution or BatchNorm asked for one must not run without an activation."""
    from vae_gan_amd import lib as L
    lib = L.load()
    desc = None                                        # refused before it is read
    one = 16
    for act in (L.ACT_GELU, L.ACT_SILU, -1):
        for name, rc in (("conv_fwd", lambda: lib.vg_conv_fwd(desc, one, one, None, one, None, act, 0, None)),
                         ("conv_fwd_splitk", lambda: lib.vg_conv_fwd_splitk(desc, one, one, None, one, act, 2, one, None)),
                         ("conv_dgrad", lambda: lib.vg_conv_dgrad(desc, one, one, None, one, None, act, 0, None)),
                         ("thin_conv_fwd", lambda: lib.vg_thin_conv_fwd(desc, one, one, None, one, None, act, one, None)),
                         ("conv1_fwd", lambda: lib.vg_conv1_fwd(desc, one, one, None, one, act, None)),
                         ("bn_act_fwd", lambda: lib.vg_bn_act_fwd(one, None, one, one, one, 4, 64, 64, act, 0, None)),
                         ("bn_bwd_reduce", lambda: lib.vg_bn_bwd_reduce(one, one, one, one, one, one, one, one, 4, 64, 64, 64, act, 0, None)),
                         ("bn_bwd_apply", lambda: lib.vg_bn_bwd_apply(one, one, one, one, one, one, one, one, one, one, None, None, None, 0, None, 4, 4,
                                                                      1.0, 64, 64, 64, act, 0, None)),
                         ("act_bwd", lambda: lib.vg_act_bwd(one, one, one, 64, act, 0, None))):
            assert rc() == -1 and name + ": activation" in L.last_error(), (name, act, L.last_error())


def test_adamw_rounding_refusals(ops):
    from vae_gan_amd import lib as L
    from vae_gan_amd.optim import FlatAdamW
    p = [torch.nn.Parameter(torch.zeros(4, 4))]
    with pytest.raises(ValueError, match="rounding"):
        FlatAdamW(p, state_bits=8, rounding="down")
    with pytest.raises(ValueError, match="rounding"):
        FlatAdamW(p, state_bits=32, rounding="stochastic")
    lib, one = L.load(), 16
    assert lib.vg_adamw8_dithered_step(one, one, one + 1, one, one, one, None, 256, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None) == -1
    assert "adamw8_dithered_step: states must be 4-byte aligned" in L.last_error()
    assert lib.vg_adamw8_dithered_step(one, one, one, one, one, one, None, 255, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None) == -1
    assert "multiple" in L.last_error()


def test_rows_beyond_the_range_of_the_kernels_indexes(ops):
    """A row of 2^32 + 8 elements must not be taken for one of 8."""
    from vae_gan_amd import lib as L
    lib, one, most = L.load(), 16, 1 << 30
    x = torch.empty(1, (1 << 32) + 8, device="meta")
    with pytest.raises(RuntimeError, match="columns in a row"):
        ops.layer_norm(x, torch.ones(8), torch.ones(8), c=8)
    with pytest.raises(RuntimeError, match="logits in a row"):
        ops.token_logprobs(x, torch.zeros(1, dtype=torch.int64))
    assert lib.vg_layer_norm_fwd(one, 2 * most, one, one, one, 2 * most, None, 1, 8, most + 8, 1e-5, 0, None) == -1 and "stored" in L.last_error()


def test_launches_of_too_many_workgroups_are_refused_by_name(ops):
    """2^32 threads or more in one dimension do not launch: the message says which operator's, and nothing is run before it."""
    from vae_gan_amd import lib as L
    lib, one = L.load(), 16

    def refused(rc, name):
        assert rc == -1 and name in L.last_error() and "too many" in L.last_error(), (rc, L.last_error())
    n = (1 << 31) - 1
    refused(lib.vg_token_logprobs_fwd(one, 8, one, -100, n, 8, 0, one, one, None, None, None, None, 1, None), "token_logprobs_fwd")
    refused(lib.vg_token_logprobs_fwd(one, 4096, one, -100, n, 4096, 0, one, one, None, None, None, None, 1, None), "token_logprobs_fwd")
    refused(lib.vg_token_logprobs_bwd(one, 8, one, -100, one, one, one, one, one, 8, n, 8, 1, None), "token_logprobs_bwd")
    refused(lib.vg_layer_norm_fwd(one, 9000, one, one, one, 9000, None, 1 << 24, 9000, 9000, 1e-5, 1, None), "layer_norm_fwd")
    refused(lib.vg_layer_norm_bwd(one, 9000, one, 9000, one, one, one, 9000, one, one, one, 1 << 24, 9000, 9000, 1, None), "layer_norm_bwd")
    refused(lib.vg_linear_act_fwd(one, 64, one, 1, None, 0, None, 0, one, None, None, (1 << 30) - 1, 1024, 64, 0, 1, None), "linear_act")
