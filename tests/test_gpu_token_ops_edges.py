"""GPU tier: values at which the token-wise operators' arithmetic can lose what the formulas keep, against float64.

Tolerances count roundings as in test_gpu_token_ops.py, whose oracles are used: u = 2^-24 is half a step of f32, h(T) half a step
of the storage type."""
import math

import pytest
import torch

from test_gpu_token_ops import lp_check, within

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------------------------- log probabilities far from zero
# rows in a wave's registers (a part of a wave, a wave), a wave per long row, a block per row, split rows
FAR_SHAPES = [(1, 40), (1, 2048), (130, 2500), (1, 5003), (1, 70001)]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("repeat,v", FAR_SHAPES)
def test_token_logprobs_rows_and_parts_far_from_zero(repeat, v, dt):
    """Finite mask fills and logits of any size: a row's exponents are of the distance to its maximum, wherever that lies.  Rows
    all at the fill, halves and stripes of it (a thread's first accesses may be nothing else), distances of a few steps there."""
    g = gen(v)
    fills = (-1e9, -1e10, -1e12, -1e20, -1e30, 1e10, 1e30, 2.0 ** 20, -2.0 ** 20, 2.0 ** 20 + 64)
    rows = []
    for f in fills:
        n = lambda: torch.randn(v, device="cuda", generator=g)      # noqa: E731
        x = [torch.full((v,), f, device="cuda"), n(), n(), n(), n(), f + torch.randint(-3, 4, (v,), device="cuda", generator=g)]
        x[1][: v // 2] = f
        x[2][v // 2:] = f
        x[3][::2] = f
        x[4][:] = -math.inf
        x[4][: v // 3] = f
        x[4][v - 1] = 1.0
        rows += x
    # the sums of one row about maxima on both sides of where the exponents' form changes
    border = torch.full((v,), 2.0 ** 20 - 6, device="cuda")
    border[v // 2:] += torch.randint(0, 12, (v - v // 2,), device="cuda", generator=g)
    rows += [border, border.flip(0), -border]
    x = torch.stack(rows).to(dt).repeat(repeat if repeat == 1 else repeat // 2, 1)
    if repeat > 1:
        assert x.shape[0] >= 2048
    t = torch.randint(0, v, (x.shape[0],), device="cuda", generator=g)
    lp_check(x, t, top=min(v, 5))


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("v", [3, 2500, 70001])
def test_token_logprobs_distances_near_the_end_of_the_range(v, dt):
    """ln p = x - m - ln s is finite wherever x - m is, although (x - m) log2 e is not."""
    x = torch.full((4, v), -math.inf, device="cuda")
    x[0, :3] = torch.tensor([3e38, 0.0, 1e38])
    x[1, :3] = torch.tensor([1.9e38, -1e38, 1.9e38])
    x[2, :3] = torch.tensor([0.0, -3e38, -2.5e38])
    x[3, :3] = torch.tensor([1.5e38, -1.5e38, 7.0])
    x = x.to(dt)
    lp_check(x, torch.ones(4, dtype=torch.int64, device="cuda"), top=3)
    lp_check(x, torch.full((4,), 2, device="cuda"), top=3)


# ---------------------------------------------------------------------------------------------- layer norm far from zero
# rows of a part of a wave, of a wave, of a block, and too long for its registers
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("c", [3, 41, 127, 1000, 1001, 5003, 8191, 9001])
def test_layer_norm_of_constant_rows_is_the_bias(c, dt):
    """A row of one value has the mean of that value, exactly, and no spread: xh = 0, whatever the width and the value."""
    from vae_gan_amd import ops
    g = gen(c)
    x = torch.tensor([1000.0, 30000.0, 0.1, -1000.123, 3e-5, -7e8, 1 / 3, 0.0], device="cuda").to(dt)[:, None].repeat(1, c)
    w, b = torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    dy = torch.randn(8, c, device="cuda", generator=g).to(dt)
    xg, wg, bg = (t.detach().requires_grad_() for t in (x, w, b))
    y = ops.layer_norm(xg, wg, bg)
    assert torch.equal(y.detach(), b.to(dt).expand(8, c))
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy)
    assert not dw.any()
    gd = dy.double() * w.double()
    r = 1e-5 ** -0.5
    # the mean of c products and the difference: each term passes c / 256 + 64 roundings
    tol = (64 + c / 256) * U * r * (gd.abs() + gd.abs().mean(1, keepdim=True))
    within(dx, r * (gd - gd.mean(1, keepdim=True)), tol + torch.finfo(dt).eps / 2 * (r * (gd - gd.mean(1, keepdim=True))).abs(), "dx")


@pytest.mark.parametrize("c", [41, 127, 1000, 5003, 9001])
def test_layer_norm_of_a_small_spread_on_a_large_mean(c):
    """x - mu is exact here (x and mu within a factor of 2), so xh is off by its own sums' roundings alone: n u of what they hold,
    the spread and what the first mean was off by, n u |mu|; neither is of the size of u |mu| r."""
    from vae_gan_amd import ops
    g = gen(c)
    x = 1000 + 0.01 * torch.randn(16, c, device="cuda", generator=g)
    x[8:] = 30000 + torch.randn(8, c, device="cuda", generator=g)
    w, b = torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    y = ops.layer_norm(x, w, b)
    xd, n = x.double(), 64 + c / 256
    var, mu = torch.var_mean(xd, 1, unbiased=False, keepdim=True)
    r = (var + 1e-5).rsqrt()
    xh = (xd - mu) * r
    slack = (1 + n * U * mu.abs() * r).square()
    ref = xh * w.double() + b.double()
    within(y, ref, 2 * n * U * (xh.abs() + 1) * slack * w.double().abs() + 4 * U * (ref.abs() + b.double().abs()), "y")


# ---------------------------------------------------------------------------------------------- activations at their ends
def act_values(z, act, dt, rows):
    """act(z) and the gradient of its sum, for values z, through a product that is exact (one input, weight 1): few rows, or tiles
    whose other columns repeat the values."""
    from vae_gan_amd import ops
    n = 1 if rows else 64
    x = z.reshape(-1, 1).to(dt).requires_grad_()
    w = torch.ones(n, 1, dtype=dt, device="cuda")
    parts = x.split(60) if rows else (x,)
    y = torch.cat([ops.linear_act(p, w, None, act) for p in parts])
    assert all(torch.equal(y[:, 0], y[:, j]) for j in range(n))
    dy = torch.zeros_like(y)
    dy[:, 0] = 1
    (dx,) = torch.autograd.grad(y, x, dy)
    return y.detach()[:, 0], dx[:, 0]


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_gelu_keeps_its_negative_tail(dt, rows):
    """z Phi(z) and Phi(z) + z phi(z) relative to the size of their terms.  Phi(-|z|) is off by 4.1e-6 (bf16; measured against erfc
    over a grid in f32 arithmetic) or 9 u (f32) and an ulp of the reciprocal; e^(-z^2/2) by 2 u and, beside bf16, by the rounding
    of z^2/2 log2 e: z^2 u.  f32 results below 2^-126 have no full mantissa: an absolute 2^-126 for them."""
    from vae_gan_amd import lib as L
    z = torch.cat([torch.linspace(-12.5, 9, 700, device="cuda"), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 40.0, 1e20], device="cuda")]).to(dt)
    y, dx = act_values(z, L.ACT_GELU, dt, rows)
    zd = z.double()
    phi, pdf = torch.special.erfc(-zd / math.sqrt(2)) / 2, (-zd * zd / 2).exp() / math.sqrt(2 * math.pi)
    own = 4.1e-6 + 8 * U if dt == BF16 else 16 * U
    rel = own + (4 + (zd * zd if dt == BF16 else 0 * zd)) * U
    h = torch.finfo(dt).eps / 2
    within(y, zd * phi, (zd * phi).abs() * (h + rel.clamp_max(1)) + 2.0 ** -126, "y")
    slope, mag = phi + zd * pdf, phi + (zd * pdf).abs()
    if dt == BF16:       # kept in f16 (half a step 2^-11, 2^-25 for its subnormals), rounded to bf16 as dz
        tol = slope.abs() * (2.0 ** -11 + 2.0 ** -8) * 1.001 + 2.0 ** -25
    else:
        tol = slope.abs() * h + 2.0 ** -126
    within(dx, slope, tol + mag * rel.clamp_max(1), "slope")


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_logistic_activations_keep_both_tails(act, dt, rows):
    """Relative to the size of their terms: e^-|z| is off by 2 u (f32), or by 2 u + 2 |z| u (bf16: two roundings of |z| log2 e); the
    quotient and the products by at most 6 u more.  In f32 a slope is kept to where it ends (2^-126)."""
    from vae_gan_amd import lib as L
    z = torch.cat([torch.linspace(-80, 80, 700, device="cuda"), torch.linspace(-9, 9, 300, device="cuda"), torch.tensor([0.0, -0.0, 1e-6], device="cuda")]).to(dt)
    y, dx = act_values(z, L.ACT_SIGMOID if act == "sigmoid" else L.ACT_SILU, dt, rows)
    zd = z.double()
    p, q = 1 / (1 + (-zd).exp()), 1 / (1 + zd.exp())
    h = torch.finfo(dt).eps / 2
    rel = (8 + (2 * zd.abs() if dt == BF16 else 0 * zd)) * U
    value, slope, mag = (p, p * q, p * q) if act == "sigmoid" else (zd * p, p * (1 + zd * q), p * (1 + zd.abs() * q))
    within(y, value, value.abs() * (h + rel) + 2.0 ** -126, "y")
    if dt == BF16:       # kept in f16 (half a step 2^-11, 2^-25 for its subnormals), rounded to bf16 as dz
        tol = slope.abs() * (2.0 ** -11 + 2.0 ** -8) * 1.001 + 2.0 ** -25
    else:
        tol = slope.abs() * h + 2.0 ** -126
    within(dx, slope, tol + mag * 2 * rel, "slope")


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
def test_small_slopes_beside_bf16(act, rows):
    """A slope is kept as 2^14 times itself in f16: half a step of 2^-11 relative down to 2^-28, an absolute 2^-39 below; then one
    rounding of dz to bf16.  (e^-|z| itself: 2 u + 2 |z| u.)"""
    from vae_gan_amd import lib as L
    z = torch.cat([torch.linspace(-27, -8, 400, device="cuda"), torch.linspace(8, 27, 400, device="cuda")]).to(BF16)
    _, dx = act_values(z, {"sigmoid": L.ACT_SIGMOID, "silu": L.ACT_SILU, "gelu": L.ACT_GELU}[act], BF16, rows)
    zd = z.double()
    p, q = 1 / (1 + (-zd).exp()), 1 / (1 + zd.exp())
    phi, pdf = torch.special.erfc(-zd / math.sqrt(2)) / 2, (-zd * zd / 2).exp() / math.sqrt(2 * math.pi)
    slope, rel = {"sigmoid": (p * q, 2 * (8 + 2 * zd.abs()) * U), "silu": (p * (1 + zd * q), 3 * (8 + 2 * zd.abs()) * U),
                  "gelu": (phi + zd * pdf, 5e-6 + (8 + zd * zd) * U)}[act]
    within(dx, slope, slope.abs() * (2.0 ** -11 + 2.0 ** -8 + rel) * 1.001 + 2.0 ** -39, "slope")
    if act == "sigmoid":
        assert bool((dx[z > -26] > 0)[:100].all())


# ---------------------------------------------------------------------------------------------- forward-mode derivatives
def test_tangents_are_refused_on_the_gpu():
    """Also where the gradient that comes into a backward pass carries one."""
    import torch.autograd.forward_ad as fwd
    from vae_gan_amd import ops
    x, w, b = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(8, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    calls = [lambda a: ops.layer_norm(a, w, b), lambda a: ops.linear_act(a, torch.eye(8, device="cuda"), b, 3), lambda a: ops.token_logprobs(a, t)[0]]
    with fwd.dual_level():
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fwd.make_dual(x, torch.ones_like(x)))
            xg = x.clone().requires_grad_()
            y = call(xg)
            dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, xg, dy)
    for call in calls:
        xg = x.clone().requires_grad_()
        y = call(xg)
        assert torch.isfinite(torch.autograd.grad(y, xg, torch.ones_like(y))[0]).all()


# ---------------------------------------------------------------------------------------------- AdamW in 8 bits over many steps
def builder_optimizer():
    """The generator's optimizer of `--optimizer adamw8bit`, over 64 blocks of 256 elements."""
    from types import SimpleNamespace
    from vae_gan_amd.train import build_optimizers
    model = torch.nn.Module()
    model.encoder, model.decoder, model.discriminator = (torch.nn.Linear(256, 64, bias=False).cuda() for _ in range(3))
    model.decoder.weight.requires_grad_(False)
    return build_optimizers(model, SimpleNamespace(optimizer="adamw8bit", lr=1e-4, beta1=0.9, beta2=0.999, weight_decay=0.0))[0]


def test_adamw_8bit_second_moments_follow_inside_a_block():
    """Half of every block's gradients are three times as large as the state that the run starts from.  1000 steps later each half's
    moments are right on average.  A step changes a root by 0.0005 |g^2 / v - 1| of itself, 0.0005 on average, f = 0.004 to 0.008 of
    a code's step of 0.06 to 0.125: rounding adds a variance of f (1 - f) squared steps and the decay of 0.0005 a step takes it
    back, so the deviation is sqrt(f / 0.001) steps, 17 to 25 %, and, the root being what is rounded, half its square, at most
    3 %, too much on average.  The median of 8192 elements is off by 0.25 * 1.25 / 90 = 0.0035, four times that is 0.014; 5 %
    covers both.  Without the changes' share of the rounding the medians are 0.94 and 2.3."""
    opt = builder_optimizer()
    g = gen(7)
    size = torch.exp(0.7 * torch.randn(64, 256, device="cuda", generator=g))
    scale = size.amax(1, keepdim=True) / 448
    opt.root_sq.copy_((size / scale).to(torch.float8_e4m3fn).view(-1))
    opt.root_sq_scale.copy_(scale[:, 0])
    v = (size / scale).to(torch.float8_e4m3fn).double().mul(scale.double()).square()
    size[:, :128] *= 3
    for _ in range(1000):
        grad = size * torch.randn(64, 256, device="cuda", generator=g)
        v = 0.999 * v + 0.001 * grad.double().square()
        opt.flat_g.copy_(grad.view(-1))
        opt.step()
    ratio = opt.root_sq.float().view(64, 256) * opt.root_sq_scale[:, None] / v.sqrt()
    for half in (ratio[:, :128], ratio[:, 128:]):
        assert abs(float(half.median()) - 1) <= 0.05 and float(half.std()) <= 0.3, (float(half.median()), float(half.std()))


def test_adamw_8bit_first_moments_reach_a_steady_gradient():
    """Gradients of 1 beside one of 10 in each block, whose moment is there already and sets the scale: m goes to 1 (rounded to
    nearest it stops at 0.71, where a tenth of what is left is less than half a step).  f = 0.1 (1 - m) steps, at most 0.1 near the
    end: a deviation of sqrt(0.1 / 0.2) steps of 6 to 12 %, below 0.09; the mean of 16320 elements is off by 0.0007, and the two
    sides of 1 have steps of 1/16 and 1/8 in which the same deviation is not the same probability: 2 % covers it."""
    opt = builder_optimizer()
    opt.flat_g.fill_(1.0)
    opt.flat_g[::256] = 10.0
    opt.exp_avg[::256] = 448.0
    opt.exp_avg_scale.fill_(10 / 448)
    for _ in range(300):
        opt.step()
    m = (opt.exp_avg.float().view(64, 256) * opt.exp_avg_scale[:, None])[:, 1:]
    assert abs(float(m.mean()) - 1) <= 0.02 and float(m.std()) <= 0.12, (float(m.mean()), float(m.std()))
    assert float((m.mean(1) - 1).abs().max()) <= 0.02 + 5 * 0.09 / 16      # 255 elements a block


def test_adamw_8bit_stochastic_rounding_takes_either_neighbour():
    """One step: each code is one of the two beside the exact value, and their mean is the exact value (a deviation of at most half a
    step each: five standard errors of n elements, and 2^-16 for the 16 bits of chance).  Scales, parameters and updates are those
    of rounding to nearest; the same step again gives the same bits."""
    from test_gpu_token_ops import SHAPES, make_opt, states
    opt, g = make_opt(8, shapes=SHAPES + [(300, 256)])
    for _ in range(3):
        opt.flat_g.copy_(torch.randn(opt.numel, device="cuda", generator=g) * torch.exp(2 * torch.randn(opt.numel, device="cuda", generator=g)))
        for q, o in zip(opt.params, opt.offsets):
            opt.flat_g[o + q.numel():(o + q.numel() + 255) // 256 * 256] = 0
        opt.step()
    m, v = states(opt)
    sd, grad = opt.state_dict(), opt.flat_g.double()
    two = []
    for _ in range(2):
        o, _ = make_opt(8, shapes=SHAPES + [(300, 256)], rounding="stochastic")
        o.load_state_dict(sd)
        o.flat_p.copy_(opt.flat_p), o.flat_g.copy_(opt.flat_g)
        two.append(o)
    for o in (opt, *two):
        o.step()
    a, b = two
    for name in ("flat_p", "exp_avg_scale", "root_sq_scale"):
        assert torch.equal(getattr(a, name), getattr(opt, name)), name
    for name in ("exp_avg", "root_sq"):
        assert torch.equal(getattr(a, name).view(torch.uint8), getattr(b, name).view(torch.uint8)), name
    b1, b2 = opt.betas
    for codes, scale, exact in ((a.exp_avg, a.exp_avg_scale, b1 * m + (1 - b1) * grad), (a.root_sq, a.root_sq_scale, (b2 * v + (1 - b2) * grad * grad).sqrt())):
        q = (exact.view(-1, 256) / scale.double()[:, None]).view(-1)
        q = torch.where(q.abs() < 2.0 ** -9, torch.zeros_like(q), q) if codes is a.root_sq else q      # raised to 2^-9
        got = torch.where(q == 0, torch.zeros_like(q), codes.double())
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
        off = (got - q) / step
        assert float(off.abs().max()) <= 1 + 2.0 ** -12
        n = int((q != 0).sum())
        assert abs(float(off.sum()) / n) <= 5 * 0.5 / n ** 0.5 + 2.0 ** -15, float(off.sum()) / n
        assert float((off.abs() > 0.55).float().mean()) > 0.1                                          # not to nearest


# ---------------------------------------------------------------------------------------------- gradients that nobody asked for
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("c", [41, 512, 5000, 9001])
def test_layer_norm_without_a_gradient_of_x(c, dt):
    """Parameters alone: the same bits as beside dx, and its memory less (workspaces are the same: up to 768 parts of 8 c bytes)."""
    from vae_gan_amd import ops
    g = gen(c)
    rows = (8 << 20) // c
    x, dy = torch.randn(rows, c, device="cuda", generator=g).to(dt), torch.randn(rows, c, device="cuda", generator=g).to(dt)
    w, b = torch.randn(c, device="cuda", generator=g).requires_grad_(), torch.randn(c, device="cuda", generator=g).requires_grad_()

    def grads(xs, wanted):
        y = ops.layer_norm(xs, w, b)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = torch.autograd.grad(y, wanted, dy)
        return out, torch.cuda.max_memory_allocated() - before
    xg = x.detach().requires_grad_()
    full, more = grads(xg, (xg, w, b))
    (dw, db), less = grads(x, (w, b))
    assert more - less >= x.numel() * x.element_size()
    assert torch.equal(dw, full[1]) and torch.equal(db, full[2])


def test_adamw_8bit_stochastic_rounding_beyond_the_cache():
    """Buffers over 256 MiB take the streaming kernel: the same bits at the same places as in a small buffer."""
    from test_gpu_token_ops import make_opt
    n = 999_936                                                     # whole blocks
    big, g = make_opt(8, shapes=[(17_000_001,)], rounding="stochastic")
    small, _ = make_opt(8, shapes=[(n,)], rounding="stochastic")
    small.flat_p.copy_(big.flat_p[:n])
    for _ in range(3):
        big.zero_grad()
        big.params[0].grad.add_(torch.randn(17_000_001, device="cuda", generator=g) * 1e-3)
        small.flat_g.copy_(big.flat_g[:n])
        big.step(), small.step()
    # one parameter of one dimension in both: neither is decayed
    assert torch.equal(big.flat_p[:n], small.flat_p)
    for name in ("exp_avg", "root_sq"):
        assert torch.equal(getattr(big, name)[:n].view(torch.uint8), getattr(small, name).view(torch.uint8)), name
    for name in ("exp_avg_scale", "root_sq_scale"):
        assert torch.equal(getattr(big, name)[:n // 256], getattr(small, name)), name
    assert torch.isfinite(big.flat_p).all() and not big.flat_p[17_000_001:].any()
