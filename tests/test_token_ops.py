"""CPU tier: what the token-wise operators (layer norm, linear_act, token_logprobs, AdamW) refuse, in Python and at the C
entry points, before anything reaches a GPU."""
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


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_layer_norm_refusals(ops):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.layer_norm(z(2, 8), z(8), z(8))
    with pytest.raises(RuntimeError, match="c = 9"):
        ops.layer_norm(z(2, 8), z(9), z(9), c=9)
    with pytest.raises(RuntimeError, match="c = 0"):
        ops.layer_norm(z(2, 8), z(8), z(8), c=0)
    with pytest.raises(RuntimeError, match="weight must be float32"):
        ops.layer_norm(z(2, 8), z(7), z(8))
    with pytest.raises(RuntimeError, match="bias must be float32"):
        ops.layer_norm(z(2, 8), z(8), z(8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no columns"):
        ops.layer_norm(z(2, 0), z(0), z(0))
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(z(2, 8), z(8), z(8), eps=-1.0)
    with pytest.raises(TypeError, match="unsupported"):
        ops.layer_norm(z(2, 8, dtype=torch.float16), z(8), z(8))


def test_linear_act_refusals(ops):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_act(z(2, 8), z(4, 8))
    with pytest.raises(RuntimeError, match="cannot be multiplied"):
        ops.linear_act(z(2, 8), z(4, 7))
    with pytest.raises(RuntimeError, match="cannot be multiplied"):
        ops.linear_act(z(2, 0), z(4, 0))
    with pytest.raises(TypeError, match="weight is"):
        ops.linear_act(z(2, 8), z(4, 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="bias is"):
        ops.linear_act(z(2, 8, dtype=torch.bfloat16), z(4, 8), z(4, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="bias of shape"):
        ops.linear_act(z(2, 8), z(4, 8), z(5))
    with pytest.raises(RuntimeError, match="residual"):
        ops.linear_act(z(2, 8), z(4, 8), residual=z(1, 4))              # no broadcasting
    with pytest.raises(RuntimeError, match="residual"):
        ops.linear_act(z(2, 8), z(4, 8), residual=z(2, 4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="activation"):
        ops.linear_act(z(2, 8), z(4, 8), act=9)
    with pytest.raises(TypeError, match="unsupported"):
        ops.linear_act(z(2, 8, dtype=torch.float64), z(4, 8, dtype=torch.float64))


def test_token_logprobs_refusals(ops):
    t = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.token_logprobs(z(2, 8), t)
    with pytest.raises(RuntimeError, match="tokens must be int64"):
        ops.token_logprobs(z(2, 8), t.int())
    with pytest.raises(RuntimeError, match="tokens must be int64"):
        ops.token_logprobs(z(2, 3, 8), t)
    with pytest.raises(ValueError, match="top"):
        ops.token_logprobs(z(2, 8), t, top=9)
    with pytest.raises(ValueError, match="top"):
        ops.token_logprobs(z(2, 80), t, top=33)
    with pytest.raises(ValueError, match="top"):
        ops.token_logprobs(z(2, 8), t, top=-1)
    with pytest.raises(RuntimeError, match="no logits"):
        ops.token_logprobs(z(2, 0), t)
    with pytest.raises(TypeError, match="unsupported"):
        ops.token_logprobs(z(2, 8, dtype=torch.float16), t)


def test_adamw_refusals():
    from vae_gan_amd.optim import FlatAdamW
    p = [torch.nn.Parameter(z(4, 4))]
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        FlatAdamW(p)
    with pytest.raises(ValueError, match="state_bits"):
        FlatAdamW(p, state_bits=4)
    with pytest.raises(ValueError, match="weight_decay"):
        FlatAdamW(p, weight_decay=-0.1)
    with pytest.raises(ValueError, match="betas"):
        FlatAdamW(p, betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="empty"):
        FlatAdamW([])
    with pytest.raises(RuntimeError, match="float32"):
        FlatAdamW([torch.nn.Parameter(z(4, dtype=torch.bfloat16))])


def test_optimizer_choice_in_the_command_line_and_the_builder():
    from vae_gan_amd import cli
    args = cli.build_parser("vq").parse_args([])
    assert args.optimizer == "adam" and cli.config_from_args("vq", args).optimizer == "adam"
    args = cli.build_parser("beta").parse_args(["--optimizer", "adamw8bit", "--weight_decay", "0.05"])
    cfg = cli.config_from_args("beta", args)
    assert (cfg.optimizer, cfg.weight_decay) == ("adamw8bit", 0.05)
    with pytest.raises(SystemExit):
        cli.build_parser("vq").parse_args(["--optimizer", "sgd"])
    from vae_gan_amd.train import build_optimizers
    cfg.optimizer = "sgd"
    model = torch.nn.Module()
    model.encoder = model.decoder = model.discriminator = torch.nn.Linear(2, 2)
    with pytest.raises(ValueError, match="optimizer"):
        build_optimizers(model, cfg)


def test_c_entry_points_return_an_error_instead_of_launching(ops):
    from vae_gan_amd import lib as L
    lib = L.load()
    one = 16          # never read: every call below is refused on the host

    def refused(rc, text):
        assert rc == -1 and text in L.last_error(), (rc, L.last_error())
    ln = lambda **k: lib.vg_layer_norm_fwd(*[{**dict(x=one, ldx=8, w=one, b=one, y=one, ldy=8, stats=None, rows=1, c=8, cs=8, eps=1e-5,   # noqa: E731
                                                    dtype=0, st=None), **k}[n] for n in "x ldx w b y ldy stats rows c cs eps dtype st".split()])
    refused(ln(x=None), "null")
    refused(ln(dtype=2), "dtype")
    refused(ln(c=9), "columns")
    refused(ln(ldx=7), "row stride")
    refused(ln(rows=1 << 31), "rows")
    assert ln(rows=0, x=None) == 0
    refused(lib.vg_layer_norm_bwd(one, 8, one, 8, one, one, one, 8, one, None, None, 1, 8, 8, 0, None), "workspace")
    la = lambda **k: lib.vg_linear_act_fwd(*[{**dict(x=one, ldx=8, w=one, wdt=0, b=None, bdt=0, r=None, ldr=0, y=one, s=None, ws=None, m=1, n=4,   # noqa: E731
                                                     k=8, act=0, dt=0, st=None), **k}[q] for q in "x ldx w wdt b bdt r ldr y s ws m n k act dt st".split()])
    refused(la(ldx=7), "row stride")
    refused(la(m=0), "0 x 4 x 8")
    refused(la(n=1 << 20), "1048576")
    refused(la(act=7), "activation")
    refused(la(wdt=1), "weight dtype")
    refused(la(r=one, ldr=3), "row stride")
    refused(la(k=7, m=100), "workspace")               # rows that are not whole 16-byte pieces are copied first
    refused(la(ws=one, k=7, m=100), "256")
    refused(lib.vg_linear_act_dz(one, None, one, None, 0, None, 1, 4, 0, None), "null")
    refused(lib.vg_linear_act_dz(one, one, one, one, 0, None, 1, 4, 0, None), "null")
    refused(lib.vg_linear_act_dgrad(one, None, 0, one, None, 1, 4, 8, 0, None), "null")
    refused(lib.vg_linear_act_wgrad(one, one, 7, one, 0, None, 1, 4, 8, 0, None), "row stride")
    refused(lib.vg_token_logprobs_fwd(one, 8, one, -100, 1, 8, 9, one, one, None, one, one, None, 0, None), "alternatives")
    refused(lib.vg_token_logprobs_fwd(one, 7, one, -100, 1, 8, 0, one, one, None, None, None, None, 0, None), "stride")
    refused(lib.vg_token_logprobs_fwd(one, 1 << 20, one, -100, 1, 1 << 20, 0, one, one, None, None, None, None, 0, None), "workspace")
    refused(lib.vg_token_logprobs_bwd(one, 8, one, -100, None, one, one, one, one, 8, 1, 8, 0, None), "null")
    refused(lib.vg_adamw_step(one, one, one, one, None, 255, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None), "multiple")
    refused(lib.vg_adamw_step(one, one, one, one, None, 256, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1.0, None), "step")
    refused(lib.vg_adamw_step(one + 4, one, one, one, None, 256, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None), "aligned")
    refused(lib.vg_adamw8_step(one, one, one + 1, one, one, one, None, 256, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None), "aligned")
