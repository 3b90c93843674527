"""GPU tier: layer norm, linear_act, token_logprobs and FlatAdamW against their definitions in float64.

Tolerances count roundings.  u = 2^-24 is half a step of f32, h(T) half a step of the storage type (bf16 2^-8, f32 2^-24).
A result may be off by h(T) |result| for its own rounding, plus u times the number of f32 operations a term goes through times
the sum of the terms' magnitudes (the usual bound on a sum, |fl(sum) - sum| <= n u sum |terms|)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def half(dt):
    return torch.finfo(dt).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, ref, tol, what):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what + ": NaN in other places"
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), what + ": infinities"
    over = (got - ref).abs() - tol
    over = over[fin.expand_as(over)]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} off, worst by {float(over.max()):.3e}"


# ---------------------------------------------------------------------------------------------- layer norm
def ln_oracle(x, w, b, dy, c, eps, dt):
    """Values and tolerances.  A row's sums pass through at most 32 adds in a lane and 8 levels of joining (c <= 8192; longer
    rows c / 256 in a lane): n = 64 + c / 256 operations a term covers sums, products and the root."""
    n = 64 + c / 256
    xv = x.double()[..., :c]
    mu = xv.mean(-1, keepdim=True)
    r = ((xv - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (xv - mu) * r
    e_xh = n * U * ((xv.abs() + xv.abs().mean(-1, keepdim=True)) * r + xh.abs())
    y = xh * w.double() + b.double()
    out = {"y": (y, half(dt) * y.abs() + e_xh * w.double().abs() + 4 * U * (y.abs() + b.double().abs()))}
    if dy is not None:
        d = dy.double()[..., :c]
        g = d * w.double()
        mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        dx = r * (g - mg - xh * mgx)
        mag = g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)
        e = n * U * mag + e_xh * mgx.abs() + xh.abs() * (g.abs() * e_xh).mean(-1, keepdim=True)
        out["dx"] = (dx, half(dt) * dx.abs() + r * e + 2 * n * U * r * mag)
        rows = d.reshape(-1, c).shape[0]
        m = 256 + rows / 1024      # rows a lane adds up, folds over lanes, waves and at most 1024 parts
        out["dw"] = ((d * xh).reshape(-1, c).sum(0), (d.abs() * (e_xh + m * U * xh.abs())).reshape(-1, c).sum(0))
        out["db"] = (d.reshape(-1, c).sum(0), m * U * d.abs().reshape(-1, c).sum(0))
    return out


def ln_check(x, w, b, dy, c, eps=1e-5):
    from vae_gan_amd import ops
    xg, wg, bg = (t.detach().requires_grad_() for t in (x, w, b))
    y = ops.layer_norm(xg, wg, bg, eps, c)
    assert y.dtype == x.dtype and y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy)
    ref = ln_oracle(x, w, b, dy, c, eps, x.dtype)
    for name, got in (("y", y.detach()[..., :c]), ("dx", dx[..., :c]), ("dw", dw), ("db", db)):
        within(got, *ref[name], name)
    assert not y.detach()[..., c:].any() and not dx[..., c:].any()
    return y.detach(), dx, dw, db


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,c,pad", [(1, 1, 0), (1, 8, 0), (3, 41, 7), (5, 41, 0), (67, 64, 0), (1030, 127, 1), (257, 128, 0), (9, 512, 0),
                                         (4100, 256, 0), (33, 1000, 24), (7, 1001, 0), (5, 2048, 0), (4, 2049, 0), (3, 4096, 0), (6, 5000, 8),
                                         (2, 8192, 0), (3, 8191, 0), (3, 10007, 0), (70, 9000, 8)])
def test_layer_norm(rows, c, pad, dt):
    g = gen(rows * 7 + c)
    x = (torch.randn(rows, c + pad, device="cuda", generator=g) * 2 + torch.randn(c + pad, device="cuda", generator=g)).to(dt)
    w, b = 1 + 0.3 * torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    dy = torch.randn(rows, c + pad, device="cuda", generator=g).to(dt)
    got = ln_check(x, w, b, dy, c)
    again = ln_check(x, w, b, dy, c)
    assert all(torch.equal(p, q) for p, q in zip(got, again))            # no atomics: the same bits


@pytest.mark.parametrize("dt", [BF16, F32])
def test_layer_norm_values_where_it_goes_wrong(dt):
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    g = gen(5)
    x = torch.randn(8, 64, device="cuda", generator=g)
    x[0] = 0                     # no spread: xh = 0, r = eps^-1/2
    x[1] = 1000.0                # a constant far from zero: the centred values are exactly 0
    x[2] = 512 + torch.randint(0, 4, (64,), device="cuda", generator=g)       # a small spread on a large mean (exact in bf16 steps of 4: rounded below)
    x[3] *= 1e-18
    x[4] *= 1e15
    x = x.to(dt)
    dy = torch.randn(8, 64, device="cuda", generator=g).to(dt)
    y, dx, _, _ = ln_check(x, w, b, dy, 64)
    assert not y[0].any() and not y[1].any()
    bad = x.clone()
    bad[5, 3], bad[6, 9] = float("nan"), float("inf")
    from vae_gan_amd import ops
    yb = ops.layer_norm(bad, w, b)
    assert torch.isnan(yb[5]).all() and torch.isnan(yb[6]).all() and torch.equal(yb[:5], y[:5]) and torch.equal(yb[7], y[7])


@pytest.mark.parametrize("dt", [BF16, F32])
def test_layer_norm_strides_and_shapes(dt):
    from vae_gan_amd import ops
    g = gen(11)
    base = torch.randn(6, 10, 96, device="cuda", generator=g).to(dt)
    w, b = torch.randn(64, device="cuda", generator=g), torch.randn(64, device="cuda", generator=g)
    dyb = torch.randn(6, 10, 96, device="cuda", generator=g).to(dt)
    for x, dy in ((base[..., :64], dyb[..., :64]), (base[..., 1:65], dyb[..., 3:67]), (base.transpose(0, 1)[..., :64], dyb.transpose(0, 1)[..., 32:]),
                  (base[:, ::2, :64], dyb[:, ::2, :64]), (base[:1, :1, :64].expand(3, 4, 64), dyb[:3, :4, :64]), (base[0, 0, :64], dyb[0, 0, :64]),
                  (base[:64 // 16, 0].t()[:64].t()[:, :64], dyb[:4, 1, :64])):
        ln_check(x, w, b, dy, 64)
    ln_check(torch.randn(40, 5, device="cuda", generator=g).to(dt).t(), torch.ones(40, device="cuda"), torch.zeros(40, device="cuda"),
             torch.randn(5, 40, device="cuda", generator=g).to(dt), 40)           # columns are not contiguous
    x = torch.zeros(0, 64, dtype=dt, device="cuda", requires_grad=True)
    wg, bg = w.clone().requires_grad_(), b.clone().requires_grad_()
    y = ops.layer_norm(x, wg, bg)
    y.sum().backward()
    assert y.shape == x.shape and x.grad.shape == x.shape and not wg.grad.any() and not bg.grad.any()
    # only some gradients wanted
    x = base[0, :, :64].contiguous()
    wg = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(ops.layer_norm(x, wg, b), (wg,), dyb[0, :, :64])
    full = ln_check(x, w, b, dyb[0, :, :64], 64)
    assert torch.equal(dw, full[2])
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.layer_norm(xg, w, b), (xg,), dyb[0, :, :64])
    assert torch.equal(dx, full[1])
    with pytest.raises(RuntimeError):
        d1 = torch.autograd.grad(ops.layer_norm(xg, w, b).float().sum(), xg, create_graph=True)[0]
        d1.float().sum().backward()


def test_layer_norm_gradient_against_differences():
    """Central differences of the f64 definition, step s: truncation s^2/6 |f'''| and rounding are far below the 1e-6 asked for."""
    g = gen(3)
    c, s = 12, 1e-4
    x = torch.randn(3, c, device="cuda", generator=g)
    w, b = torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    dy = torch.randn(3, c, device="cuda", generator=g)
    got = ln_check(x, w, b, dy, c)

    def f(xd, wd):
        v, m = torch.var_mean(xd, -1, unbiased=False, keepdim=True)
        return float((((xd - m) / torch.sqrt(v + 1e-5) * wd + b.double()) * dy.double()).sum())
    for i in range(c):
        e = torch.zeros(3, c, dtype=torch.float64, device="cuda")
        e[1, i] = s
        num = (f(x.double() + e, w.double()) - f(x.double() - e, w.double())) / (2 * s)
        assert abs(num - float(got[1][1, i])) <= 1e-5 * (1 + abs(num))
        num = (f(x.double(), w.double() + e[1]) - f(x.double(), w.double() - e[1])) / (2 * s)
        assert abs(num - float(got[2][i])) <= 1e-5 * (1 + abs(num))


# ---------------------------------------------------------------------------------------------- linear_act
ACTS = {"none": 0, "lrelu": 1, "sigmoid": 2, "gelu": 3, "silu": 4}
LIP = {"none": 1.0, "lrelu": 1.0, "sigmoid": 0.25, "gelu": 1.13, "silu": 1.1}        # largest |act'|
BEND = {"none": 0.0, "lrelu": 0.0, "sigmoid": 0.1, "gelu": 0.8, "silu": 0.5}         # largest |act''|


def act_oracle(z, act):
    f = torch.nn.functional
    return {"none": lambda a: a * 1, "lrelu": lambda a: f.leaky_relu(a, 0.2), "sigmoid": torch.sigmoid, "gelu": f.gelu, "silu": f.silu}[act](z)


def la_oracle(x, w, b, res, dy, act, dt):
    x, w = x.double().reshape(-1, x.shape[-1]), w.double()
    k, n = w.shape[1], w.shape[0]
    m = x.shape[0]
    z = x @ w.t() + (0 if b is None else b.double())
    ez = (k + 4) * U * (x.abs() @ w.abs().t() + (0 if b is None else b.double().abs()))
    zz = z.detach().requires_grad_()
    a = act_oracle(zz, act)
    y = a.detach()
    ey = LIP[act] * ez + 16 * U * (1 + z.abs())
    if res is not None:
        y = y + res.double().reshape(m, n)
        ey = ey + U * y.abs()
    out = {"y": (y, half(dt) * y.abs() + ey)}
    if dy is not None:
        d = dy.double().reshape(m, n)
        (dz,) = torch.autograd.grad(a, zz, d)
        (slope,) = torch.autograd.grad(act_oracle(zz, act), zz, torch.ones_like(z))
        # act' goes through f16 (half a step 2^-11 relative, 2^-25 for its subnormals) beside bf16 tensors, f32 beside f32
        stored = half(torch.float16) * slope.abs() + 2.0 ** -25 if dt == BF16 else U * slope.abs()
        e_slope = BEND[act] * ez + (stored + 16 * U * (1 + z.abs()) if act != "none" else 0 * z)
        if act == "lrelu":
            e_slope = e_slope + 0.8 * (z.abs() <= ez)                # the sign may flip
        e_dz = d.abs() * e_slope
        r_dz = e_dz + (half(dt) * dz.abs() if act != "none" else 0)  # rounded to the storage type before the products
        dx, dw = dz @ w, dz.t() @ x
        out["dx"] = (dx, half(dt) * dx.abs() + r_dz @ w.abs() + (n + 4) * U * (dz.abs() @ w.abs()))
        out["dw"] = (dw, half(dt) * dw.abs() + r_dz.t() @ x.abs() + (m + 4) * U * (dz.abs().t() @ x.abs()))
        db = dz.sum(0)
        out["db"] = (db, (0 if b is None else half(b.dtype)) * db.abs() + e_dz.sum(0) + (m / 256 + 300) * U * dz.abs().sum(0))
    return out


def la_check(x, w, b, act, res, dy):
    from vae_gan_amd import ops
    names = [n for n, t in (("x", x), ("w", w), ("b", b), ("res", res)) if t is not None]
    t = {n: v.detach().requires_grad_() for n, v in (("x", x), ("w", w), ("b", b), ("res", res)) if v is not None}
    y = ops.linear_act(t["x"], t["w"], t.get("b"), ACTS[act], t.get("res"))
    n = w.shape[0]
    assert y.shape == (*x.shape[:-1], n) and y.dtype == x.dtype
    ref = la_oracle(x, w, b, res, dy, act, x.dtype)
    within(y.detach().reshape(-1, n), *ref["y"], "y")
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, ACTS[act], res), y.detach())
    grads = dict(zip(names, torch.autograd.grad(y, [t[k] for k in names], dy)))
    assert all(grads[k].dtype == t[k].dtype and grads[k].shape == t[k].shape for k in names)
    within(grads["x"].reshape(-1, x.shape[-1]), *ref["dx"], "dx")
    within(grads["w"], *ref["dw"], "dw")
    if b is not None:
        within(grads["b"], *ref["db"], "db")
    if res is not None:
        assert torch.equal(grads["res"], dy)
    return y.detach(), grads


def la_data(m, k, n, dt, seed, scale=1.0):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)      # noqa: E731
    return (r(m, k).to(dt), (r(n, k) * scale / k ** 0.5).to(dt), (0.5 * r(n)).to(dt), r(m, n).to(dt), r(m, n).to(dt))


LA_SHAPES = [(1, 1, 1), (1, 16, 16), (1, 1024, 512), (2, 96, 40), (3, 100, 7), (7, 1031, 65), (16, 512, 2048), (17, 64, 64), (64, 64, 64), (65, 63, 129),
             (127, 128, 128), (128, 256, 128), (130, 520, 257), (255, 72, 264), (256, 256, 256), (300, 264, 520), (515, 33, 128), (1000, 512, 384),
             (1025, 136, 1000), (2048, 64, 512), (4099, 512, 64), (9, 8, 4104), (33, 4104, 8)]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("m,k,n", LA_SHAPES)
def test_linear_act_shapes(m, k, n, dt):
    x, w, b, res, dy = la_data(m, k, n, dt, m + 3 * k + 5 * n)
    act = list(ACTS)[(m + k + n) % 5]
    one = la_check(x, w, b, act, res if (m + k) % 2 else None, dy)
    two = la_check(x, w, b, act, res if (m + k) % 2 else None, dy)
    assert torch.equal(one[0], two[0]) and all(torch.equal(one[1][k], two[1][k]) for k in one[1])


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m,k,n", [(1, 64, 128), (12, 256, 100), (200, 128, 256), (515, 136, 384)])
def test_linear_act_activations(m, k, n, act, dt):
    x, w, b, res, dy = la_data(m, k, n, dt, 17 + m, scale=3.0)
    la_check(x, w, b, act, res, dy)
    la_check(x, w, None, act, None, dy)


@pytest.mark.parametrize("m,k,n", [(1, 128, 64), (5, 100, 77), (384, 256, 512), (700, 65, 130)])
def test_linear_act_master_weights(m, k, n):
    """bf16 activations with f32 weights and bias: the products take the weights rounded to bf16, gradients are f32.  The oracle
    gets the rounded weights; dw's own rounding is then that of f32, which the bf16 tolerance contains."""
    x, w, b, res, dy = la_data(m, k, n, BF16, 23 + m)
    w32, b32 = w.float() * (1 + 2.0 ** -12), b.float() * 1.0001
    from vae_gan_amd import ops
    for act in ("none", "gelu"):
        xg, wg, bg = x.clone().requires_grad_(), w32.clone().requires_grad_(), b32.clone().requires_grad_()
        y = ops.linear_act(xg, wg, bg, ACTS[act], res)
        dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy)
        assert dw.dtype == F32 and db.dtype == F32
        ref = la_oracle(x, w32.to(BF16), b32, res, dy, act, BF16)
        within(y.detach(), *ref["y"], "y")
        within(dx, *ref["dx"], "dx")
        tol = ref["dw"][1] - (half(BF16) - U) * ref["dw"][0].abs()       # not rounded to bf16
        within(dw, ref["dw"][0], tol, "dw")
        within(db, *ref["db"], "db")


@pytest.mark.parametrize("dt", [BF16, F32])
def test_linear_act_strides_shapes_and_partial_gradients(dt):
    from vae_gan_amd import ops
    x, w, b, res, dy = la_data(60, 96, 72, dt, 29)
    wide = torch.randn(60, 200, device="cuda", generator=gen(1)).to(dt)
    la_check(wide[:, :96], w, b, "silu", wide[:, 100:172], dy)              # rows of wider tensors
    la_check(wide[:, 3:99], w, b, "gelu", wide[:, 101:173], dy)             # ... that start between 16-byte boundaries
    la_check(wide[::2, :96].repeat(2, 1), w, b, "none", None, dy)
    la_check(x.view(3, 20, 96), w, b, "gelu", res.view(3, 20, 72), dy.view(3, 20, 72))
    la_check(x.view(3, 20, 96).transpose(0, 1), w, b, "lrelu", res.view(3, 20, 72).transpose(0, 1), dy.view(20, 3, 72))
    la_check(x[0], w, b, "sigmoid", res[0], dy[0])                           # a vector
    la_check(x[:1].expand(60, 96), w, b, "none", None, dy)                   # every row the same storage
    wt = torch.randn(96, 72, device="cuda", generator=gen(2)).to(dt).t()     # a transposed weight
    la_check(x, wt, b, "gelu", None, dy)
    (dyt,) = (torch.randn(72, 60, device="cuda", generator=gen(4)).to(dt).t(),)
    la_check(x, w, b, "gelu", res, dyt)
    e = torch.zeros(0, 96, dtype=dt, device="cuda", requires_grad=True)
    wg, bg = w.clone().requires_grad_(), b.clone().requires_grad_()
    y = ops.linear_act(e, wg, bg, ACTS["gelu"], torch.zeros(0, 72, dtype=dt, device="cuda"))
    y.sum().backward()
    assert y.shape == (0, 72) and e.grad.shape == (0, 96) and not wg.grad.any() and not bg.grad.any()
    full = la_check(x, w, b, "gelu", res, dy)[1]
    for name, i in (("x", 0), ("w", 1), ("b", 2), ("res", 3)):
        t = [v.clone().requires_grad_(j == i) for j, v in enumerate((x, w, b, res))]
        (gr,) = torch.autograd.grad(ops.linear_act(t[0], t[1], t[2], ACTS["gelu"], t[3]), (t[i],), dy)
        assert torch.equal(gr, full[name]), name


@pytest.mark.parametrize("dt", [BF16, F32])
def test_linear_act_nonfinite_values_stay_in_their_rows(dt):
    from vae_gan_amd import ops
    x, w, b, _, _ = la_data(70, 72, 100, dt, 31)
    y0 = ops.linear_act(x, w, b, ACTS["silu"])
    xb = x.clone()
    xb[3, 5], xb[40, 71] = float("nan"), float("inf")
    y = ops.linear_act(xb, w, b, ACTS["silu"])
    rest = [i for i in range(70) if i not in (3, 40)]
    assert torch.isnan(y[3]).all() and torch.equal(y[rest], y0[rest])
    big = ops.linear_act(torch.full((2, 8), 100.0, dtype=dt, device="cuda"), torch.full((3, 8), -100.0, dtype=dt, device="cuda"), None, ACTS["silu"])
    assert not big.isnan().any() and float(big.abs().max()) == 0                # e^80000 overflows: the limit is 0


def test_linear_act_kernel_variants():
    """Every tile size, unsplit and split, in each product's layout, and the few-rows kernels, against f64 through the C ABI."""
    from vae_gan_amd import lib as L
    lib = L.load()
    P = lambda t: t.data_ptr()      # noqa: E731
    seen = set()

    def note(out, ref, tol):
        seen.add(lib.vg_last_linear_act_kernel().decode())
        within(out, ref, tol, lib.vg_last_linear_act_kernel().decode())
    for dt, shapes in ((BF16, [(16384, 1024, 4096), (16300, 1000, 4090), (4096, 256, 4096), (4096, 1024, 256), (4096, 4096, 256), (1024, 512, 512), (300, 4096, 300),
                               (1000, 264, 2000), (4000, 128, 128), (64, 256, 2048), (16, 64, 64), (30, 64, 64), (700, 8192, 1400), (16384, 512, 2048),
                               (2048, 128, 2048), (128, 2048, 2048), (768, 4096, 1536), (768, 1536, 4096), (1536, 8192, 1536), (1536, 1536, 8192)]),
                       (F32, [(4096, 512, 2048), (2048, 2048, 512), (1024, 512, 512), (300, 4096, 300), (4000, 128, 128), (16, 64, 64), (30, 64, 64), (64, 64, 64),
                              (16384, 256, 1024), (300, 300, 4096), (2048, 128, 2048), (2048, 2048, 128), (128, 2048, 2048), (768, 1024, 1536),
                              (768, 1536, 1024), (1024, 768, 1536)])):
        code, e = L.vg_dtype(dt), half(dt)
        for m, k, n in shapes:
            g = gen(m + k + n)
            x, w, dz = (torch.randn(*s_, device="cuda", generator=g).to(dt) for s_ in ((m, k), (n, k), (m, n)))
            X, W, Z = x.double(), w.double(), dz.double()
            y, dx, dw = torch.empty(m, n, dtype=dt, device="cuda"), torch.empty_like(x), torch.empty_like(w)
            ws = torch.empty(max(lib.vg_linear_act_fwd_ws_bytes(P(x), k, P(w), code, m, n, k, code), lib.vg_linear_act_dgrad_ws_bytes(P(dz), P(w), code, m, n, k, code),
                                 lib.vg_linear_act_wgrad_ws_bytes(P(dz), P(x), k, m, n, k, code), 1), dtype=torch.uint8, device="cuda")
            L.check(lib.vg_linear_act_fwd(P(x), k, P(w), code, None, 0, None, 0, P(y), None, P(ws), m, n, k, 0, code, L.stream()))
            ref = X @ W.t()
            note(y, ref, e * ref.abs() + (k + 4) * U * (X.abs() @ W.abs().t()))
            L.check(lib.vg_linear_act_dgrad(P(dz), P(w), code, P(dx), P(ws), m, n, k, code, L.stream()))
            ref = Z @ W
            note(dx, ref, e * ref.abs() + (n + 4) * U * (Z.abs() @ W.abs()))
            L.check(lib.vg_linear_act_wgrad(P(dz), P(x), k, P(dw), code, P(ws), m, n, k, code, L.stream()))
            ref = Z.t() @ X
            note(dw, ref, e * ref.abs() + (m + 4) * U * (Z.t().abs() @ X.abs()))
    want = {f"rows<{t},{r}>" for t in ("bf16", "f32") for r in (16, 32, 64)}
    want |= {f"tile<{t},{size},{layout}>{join}" for t, size in (("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 128))
             for layout in ("nn", "nt", "tt") for join in ("", "+join")}
    assert want <= seen, (sorted(want - seen), sorted(seen))


@pytest.mark.parametrize("dt", [BF16, F32])
def test_linear_act_rows_far_apart(dt):
    """Rows 10 MB and more apart: beyond what a tile's 32-bit offsets cover, so they are copied first."""
    _, w, b, res, dy = la_data(150, 64, 72, dt, 37)
    wide = torch.empty(150, 5_000_000 if dt == BF16 else 2_600_000, dtype=dt, device="cuda")
    wide[:, :64] = torch.randn(150, 64, device="cuda", generator=gen(2)).to(dt)
    la_check(wide[:, :64], w, b, "silu", res, dy)
    la_check(wide[:7, :64], w, b, "none", None, dy[:7])


def test_offsets_beyond_32_bits():
    """More than 2^31 elements and 2^32 bytes in one tensor: the first and the last rows against f64."""
    from vae_gan_amd import lib as L
    from vae_gan_amd import ops
    rows, c = 70000, 32768
    x = torch.empty(rows, c, dtype=BF16, device="cuda")
    ends = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    x[ends] = torch.randn(5, c, device="cuda", generator=gen(6)).to(BF16)
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    with torch.no_grad():
        y = ops.layer_norm(x, w, b)
        ref = ln_oracle(x[ends], w, b, None, c, 1e-5, BF16)
        within(y[ends], *ref["y"], "layer norm")
        del y
        t = torch.randint(0, c, (rows,), device="cuda", generator=gen(7))
        logp, ent, _, _ = ops.token_logprobs(x, t)
        ref, _ = lp_oracle(x[ends].double(), t[ends], None, None, -100, BF16)
        within(logp[ends], *ref["logp"], "logp")
        within(ent[ends], *ref["entropy"], "entropy")
    xg = x.requires_grad_()
    out = ops.token_logprobs(xg, t)
    da, db = torch.randn(rows, device="cuda", generator=gen(8)), torch.randn(rows, device="cuda", generator=gen(9))
    (dx,) = torch.autograd.grad(out[:2], (xg,), (da, db))
    ref, _ = lp_oracle(x[ends].detach().double(), t[ends], da[ends], db[ends], -100, BF16)
    within(dx[ends], *ref["dx"], "dlogits")
    del dx, out, xg, x
    m, k, n = 70000, 16, 32768
    a, wt = torch.randn(m, k, device="cuda", generator=gen(1)).to(BF16), torch.randn(n, k, device="cuda", generator=gen(2)).to(BF16)
    ends = torch.tensor([0, 63, m - 65, m - 1], device="cuda")
    with torch.no_grad():
        y = ops.linear_act(a, wt, None, L.ACT_LRELU)
    ref = la_oracle(a[ends], wt, None, None, None, "lrelu", BF16)
    within(y[ends], *ref["y"], "linear_act")
    # the same tensor as the input of a product: contraction over its 70000 rows, and over its 32768 columns
    with torch.no_grad():
        z = ops.linear_act(y, torch.ones(8, n, dtype=BF16, device="cuda"))
    want = y[ends].double().sum(1, keepdim=True).expand(-1, 8)
    within(z[ends], want, half(BF16) * want.abs() + (n + 4) * U * y[ends].double().abs().sum(1, keepdim=True), "wide rows")
    wg = torch.zeros(8, n, dtype=BF16, device="cuda", requires_grad=True)
    dz = torch.zeros(m, 8, dtype=BF16, device="cuda")
    dz[ends] = 1
    (dw,) = torch.autograd.grad(ops.linear_act(y, wg), (wg,), dz)
    want = y[ends].double().sum(0, keepdim=True).expand(8, -1)
    within(dw, want, half(BF16) * want.abs() + 8 * U * y[ends].double().abs().sum(0, keepdim=True), "long contraction")


def test_linear_act_gradient_against_differences():
    g = gen(8)
    x, w, b = (torch.randn(*s, device="cuda", generator=g) for s in ((3, 9), (5, 9), (5,)))
    dy = torch.randn(3, 5, device="cuda", generator=g)
    s = 1e-4
    for act in ACTS:
        _, gr = la_check(x, w, b, act, None, dy)
        f = lambda xd, wd, bd: float((act_oracle(xd @ wd.t() + bd, act) * dy.double()).sum())      # noqa: E731
        X, W, B = x.double(), w.double(), b.double()
        for t, name, at in ((X, "x", (1, 4)), (W, "w", (2, 3)), (B, "b", (4,))):
            e = torch.zeros_like(t)
            e[at] = s
            args = lambda q: (X + q if t is X else X, W + q if t is W else W, B + q if t is B else B)   # noqa: E731
            num = (f(*args(e)) - f(*args(-e))) / (2 * s)
            assert abs(num - float(gr[name][at])) <= 1e-5 * (1 + abs(num)), (act, name)


# ---------------------------------------------------------------------------------------------- token_logprobs
def lp_oracle(x, t, da, db, ignore, dt):
    """x [rows, vocab] f64.  A row's sum passes through at most 32 adds in a lane, or vocab / 256 of a block's, and a dozen
    joins; an exponential is off by (2 + |d|) u for an exponent d (its own rounding and the product that forms it)."""
    rows, v = x.shape
    empty = (x == -math.inf).all(1, keepdim=True)
    mx = torch.where(empty, torch.zeros_like(x[:, :1]), x.amax(1, keepdim=True))
    ls = (x - mx).exp().sum(1, keepdim=True).log()         # apart from mx: at 3e38 even a double has no room for ln(sum)
    lnp = torch.where(empty, torch.full_like(x, -math.inf), (x - mx) - ls)
    p = lnp.exp()
    used = lnp.clamp_min(-300.0)
    h = -(p * used).sum(1)
    ok = (t != ignore) & (t >= 0) & (t < v)
    pick = lnp.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
    logp = torch.where(ok, pick, torch.where(t == ignore, 0.0, math.nan))
    d = (x - mx).clamp_min(-300.0)
    c = 64 + v / 256
    d1, d2 = (p * d.abs()).sum(1), (p * d * d).sum(1)
    e_ls = U * (c + 2 * d1 + ls[:, 0].abs().nan_to_num(0, 0, 0))
    out = {"logp": (logp, e_ls + 4 * U * (logp.abs().nan_to_num(0, 0, 0) + c / 16)), "entropy": (h, e_ls + U * (c + (c + 4) * d1 + 4 * d2 + 4 * h.abs()))}
    if da is not None:
        a = torch.where(ok & ~empty[:, 0], da.double(), 0.0)[:, None]
        b = db.double()[:, None]
        term = torch.where(p > 0, p * (used + h[:, None]), torch.zeros_like(p))
        dx = -a * p - b * term
        e_lnp = e_ls[:, None] + 4 * U * (d.abs() + used.abs())
        tol = p * (a.abs() + b.abs() * (used + h[:, None]).abs()) * (e_lnp + U * (8 + 2 * used.abs())) + p * b.abs() * (e_lnp + out["entropy"][1][:, None])
        hit = torch.zeros_like(p)
        hit.scatter_(1, t.clamp(0, v - 1)[:, None], 1.0)
        dx = dx + hit * a
        # the exponential instruction has no subnormal results: a p below 2^-126 may be 0
        tol = tol + 2.0 ** -126 * (a.abs() + b.abs() * (used + h[:, None]).abs())
        out["dx"] = (dx, tol + half(dt) * dx.abs() + 4 * U * hit * a.abs() + 2e-45)
    return out, lnp


def ranks(x, k):
    """Places of the k best: by value, equal ones by place (NaN as -inf)."""
    v = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    return torch.sort(v.double(), dim=1, descending=True, stable=True).indices[:, :k]


def lp_check(x, t, top=0, ignore=-100, seed=0):
    from vae_gan_amd import ops
    lead, v = x.shape[:-1], x.shape[-1]
    g = gen(seed)
    da, db = torch.randn(lead, device="cuda", generator=g), torch.randn(lead, device="cuda", generator=g)
    xg = x.detach().requires_grad_()
    logp, ent, tl, ta = ops.token_logprobs(xg, t, top, ignore)
    assert logp.shape == lead and logp.dtype == ent.dtype == F32
    flat = x.double().reshape(-1, v)
    ref, lnp = lp_oracle(flat, t.reshape(-1), da.reshape(-1), db.reshape(-1), ignore, x.dtype)
    within(logp.detach().reshape(-1), *ref["logp"], "logp")
    within(ent.detach().reshape(-1), *ref["entropy"], "entropy")
    if top:
        want = ranks(x.reshape(-1, v), top)
        assert torch.equal(ta.reshape(-1, top), want)
        assert tl.shape == ta.shape == (*lead, top) and not tl.requires_grad
        within(tl.reshape(-1, top), lnp.gather(1, want), ref["logp"][1].max() + 8 * U * lnp.gather(1, want).abs().nan_to_num(0, 0, 0), "top_logp")
    (dx,) = torch.autograd.grad((logp, ent), (xg,), (da, db))
    assert dx.shape == x.shape and dx.dtype == x.dtype
    within(dx.reshape(-1, v), *ref["dx"], "dx")
    return logp.detach(), ent.detach(), tl, ta, dx


LP_SHAPES = [(2100, 2500, 3), (2050, 5001, 0), (2200, 4096, 0), (1, 1, 0), (3, 2, 0), (5, 8, 0), (9, 63, 1), (130, 64, 0), (7, 100, 4), (64, 512, 0), (31, 513, 0), (3, 1000, 24), (17, 2048, 0), (9, 2049, 0),
             (40, 4100, 0), (5, 8192, 0), (600, 2500, 0), (2, 50001, 3), (1, 200003, 5), (1, 262144, 0), (520, 20000, 0)]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,v,pad", LP_SHAPES)
def test_token_logprobs(rows, v, pad, dt):
    g = gen(rows + v)
    x = torch.zeros(rows, v + pad, dtype=dt, device="cuda")[:, :v]
    x.copy_(3 * torch.randn(rows, v, device="cuda", generator=g))
    t = torch.randint(0, v, (rows,), device="cuda", generator=g)
    t[::5] = -100
    one = lp_check(x, t, top=min(v, (0, 1, 5, 32)[(rows + v) % 4]))
    two = lp_check(x, t, top=min(v, (0, 1, 5, 32)[(rows + v) % 4]))
    assert all(p is None or torch.equal(p, q) for p, q in zip(one, two))


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,v,team", [(600, 51200, 256), (2100, 2560, 64), (2, 70400, 256)])
def test_token_logprobs_best_in_few_places(rows, v, team, dt):
    """Rows whose best are all in the hands of a few threads (more than are listed), few ranked logits in masked rows at either
    end, and rows of equal values but for a few."""
    g = gen(v)
    x = torch.randn(rows, v, device="cuda", generator=g)
    stripe = (torch.arange(v, device="cuda") // (16 // torch.tensor([], dtype=dt).element_size())) % team
    x[0] = x[0] + 5 * (stripe % 50 == 3)
    if rows > 2:
        x[1] = -math.inf
        x[1, v - 3:] = 1.0
        x[2] = -math.inf
        x[2, :5] = -2.0
        x[3] = 0.5
        x[3, v // 2: v // 2 + 3] = 0.75
        x[4] = torch.where(stripe % 50 == 3, x[4], torch.full_like(x[4], -math.inf))
        x[5] = 0.5
        x[5, : v - 2] = -1.0
    x = x.to(dt)
    t = torch.randint(0, v, (rows,), device="cuda", generator=g)
    for top in (1, 8, 32):
        lp_check(x, t, top=top)


@pytest.mark.parametrize("rows,v,dt", [(2100, 10007, F32), (4200, 10007, BF16)])
def test_token_logprobs_beyond_the_cache(rows, v, dt):
    """Logits and gradient that take most of the last-level cache: the gradient leaves by other stores."""
    x = (3 * torch.randn(rows, v, device="cuda", generator=gen(12))).to(dt)
    t = torch.randint(0, v, (rows,), device="cuda", generator=gen(13))
    lp_check(x, t, top=0)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_token_logprobs_equal_bests_far_from_the_front(dt):
    """More equal bests than are listed, in the last part of a row, with none or a few better ones."""
    g = gen(8)
    x = torch.randn(520, 20011, device="cuda", generator=g).clamp_(-1, 1).to(dt)
    x[0] = 0.0
    x[0, 12345:] = 1.0
    x[1] = x[0]
    x[1, [20010, 7]] = 2.0
    x[2, 10000:] = 30.0
    x[3] = -math.inf
    x[3, 19000:] = torch.finfo(dt).min
    t = torch.randint(0, 20011, (520,), device="cuda", generator=g)
    for top in (1, 5):
        lp_check(x, t, top=top)
        lp_check(x.repeat(4, 1), t.repeat(4), top=top)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("v", [6, 70, 700, 2050, 5003, 70001])
def test_token_logprobs_masks_and_ties(v, dt):
    g = gen(v)
    low = torch.finfo(dt).min
    x = torch.randn(14, v, device="cuda", generator=g).to(dt)
    t = torch.randint(0, v, (14,), device="cuda", generator=g)
    x[0] = -math.inf                                       # nothing allowed
    x[1] = -math.inf
    x[1, v // 2] = 0.5                                     # one code allowed, and taken
    t[1] = v // 2
    x[2] = -math.inf
    x[2, v - 1] = -3.0                                     # one allowed, another one taken: logp -inf
    t[2] = 0
    x[3] = 0.25                                            # all equal
    x[4] = low                                             # all at the type's lowest value: as good as equal
    x[5, ::2] = low                                        # masked by the lowest value
    x[6, ::3] = -math.inf
    x[7] = (x[7] * 2).round()                              # many ties
    x[8, : v // 2] = 0.0
    x[8, v // 2:] = -0.0                                   # equal values of either sign
    x[9] = x[9].abs() * -1000
    x[10] = x[10] * 1e4                                    # one code takes everything
    t[11] = -100
    lp_check(x, t, top=min(v, 8))
    lp_check(x, t, top=0, ignore=int(t[6]))                # an ignored token inside the vocabulary
    if 2048 < v < 10000:                                   # enough rows for a wave each
        lp_check(x.repeat(150, 1), t.repeat(150), top=5)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("v", [40, 3001, 40000])
def test_token_logprobs_nonfinite_logits_and_foreign_tokens(v, dt):
    from vae_gan_amd import ops
    g = gen(v)
    x = torch.randn(6, v, device="cuda", generator=g).to(dt)
    t = torch.randint(0, v, (6,), device="cuda", generator=g)
    base = ops.token_logprobs(x, t, top=4)
    xb = x.clone()
    xb[1, 2], xb[2, 3], xb[3] = float("nan"), float("inf"), float("nan")
    tb = t.clone()
    tb[4], tb[5] = v, -7
    xg = xb.clone().requires_grad_()
    logp, ent, tl, ta = ops.token_logprobs(xg, tb, top=4)
    assert torch.isnan(logp[1:]).all() and torch.isnan(ent[1:4]).all() and torch.isfinite(ent[4:]).all()
    assert torch.equal(logp[0], base[0][0]) and torch.equal(ent[4:], base[1][4:]) and torch.equal(ta[[0, 4, 5]], base[3][[0, 4, 5]])
    assert torch.equal(ta[[1, 2, 3]], ranks(xb, 4)[[1, 2, 3]]) and torch.isnan(tl[1:4]).all()
    (dx,) = torch.autograd.grad(logp.sum() + 0 * ent.sum(), (xg,))
    assert not dx[4:].any() and torch.isfinite(dx[0]).all() and torch.isnan(dx[1]).all()


@pytest.mark.parametrize("dt", [BF16, F32])
def test_token_logprobs_strides_shapes_and_partial_gradients(dt):
    from vae_gan_amd import ops
    g = gen(2)
    base = torch.randn(4, 6, 640, device="cuda", generator=g).to(dt)
    t = torch.randint(0, 500, (4, 6), device="cuda", generator=g)
    for x in (base[..., :500], base[..., 1:501], base[..., 3:503], base[:, :, 100:600]):
        lp_check(x, t, top=3)
    lp_check(base.transpose(0, 1)[..., :500], t.t(), top=2)
    lp_check(base[:1, :1, :500].expand(4, 6, 500), t, top=1)
    big = torch.randn(3, 6000, device="cuda", generator=g).to(dt)
    lp_check(big[:, 1:5002], t[:3, 0].contiguous(), top=4)
    lp_check(base[0, 0, :500], t[0, 0], top=2)               # a single position: tokens is 0-dimensional
    empty = torch.zeros(0, 9, dtype=dt, device="cuda", requires_grad=True)
    logp, ent, tl, ta = ops.token_logprobs(empty, torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
    (logp.sum() + ent.sum()).backward()
    assert logp.shape == ent.shape == (0,) and ta.shape == (0, 2) and empty.grad.shape == (0, 9)
    # one of the two gradients only: with zero for the other
    x = base[0, :, :500].contiguous()
    for which in (0, 1):
        xg = x.clone().requires_grad_()
        out = ops.token_logprobs(xg, t[0])
        (dx,) = torch.autograd.grad(out[which].sum(), (xg,))
        ones, zero = torch.ones(6, device="cuda"), torch.zeros(6, device="cuda")
        xg2 = x.clone().requires_grad_()
        out = ops.token_logprobs(xg2, t[0])
        (dx2,) = torch.autograd.grad(out[:2], (xg2,), (ones, zero) if which == 0 else (zero, ones))
        assert torch.equal(dx, dx2)


def test_token_logprobs_gradient_against_differences():
    g = gen(4)
    x = torch.randn(2, 11, device="cuda", generator=g)
    t = torch.tensor([3, 10], device="cuda")
    xg = x.clone().requires_grad_()
    from vae_gan_amd import ops
    logp, ent, _, _ = ops.token_logprobs(xg, t)
    (dx,) = torch.autograd.grad((logp * torch.tensor([1.0, -2.0], device="cuda")).sum() + 0.7 * ent.sum(), (xg,))

    def f(v):
        lnp = torch.log_softmax(v, 1)
        return float(lnp[0, 3] - 2 * lnp[1, 10] - 0.7 * (lnp.exp() * lnp).sum())
    for r in range(2):
        for j in range(11):
            e = torch.zeros(2, 11, dtype=torch.float64, device="cuda")
            e[r, j] = 1e-4
            num = (f(x.double() + e) - f(x.double() - e)) / 2e-4
            assert abs(num - float(dx[r, j])) <= 1e-5 * (1 + abs(num))


# ---------------------------------------------------------------------------------------------- AdamW
SHAPES = [(1,), (255,), (256,), (257,), (64, 3, 3, 3), (64,), (100, 37), (5000,), (3, 1, 1), (513, 129)]


def make_opt(bits, seed=0, shapes=SHAPES, **kw):
    from vae_gan_amd.optim import FlatAdamW
    g = gen(seed)
    ps = [torch.nn.Parameter(torch.randn(*s, device="cuda", generator=g)) for s in shapes]
    return FlatAdamW(ps, state_bits=bits, **{**dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1, decay_filter=lambda p: p.dim() > 1), **kw}), g


def states(opt):
    if opt.state_bits == 32:
        return opt.exp_avg.double(), opt.exp_avg_sq.double()
    ex = lambda c, s: (c.view(-1, 256).double() * s.double()[:, None]).view(-1)      # noqa: E731
    return ex(opt.exp_avg, opt.exp_avg_scale), ex(opt.root_sq, opt.root_sq_scale).square()


def adamw_step_check(opt, grad_scale=1.0):
    """One step from the optimizer's present state against the formulas in f64.  m and v take 4 roundings, the update 8."""
    p, g = opt.flat_p.double(), opt.flat_g.double() * grad_scale
    m, v = states(opt)
    opt.step(grad_scale)
    t, (b1, b2) = opt.step_count, opt.betas
    dec = torch.ones(opt.numel, dtype=torch.float64, device="cuda") if opt._decay is None else opt._decay.double().repeat_interleave(256)
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    root = v2.sqrt()
    den = root / math.sqrt(1 - b2 ** t) + opt.eps
    upd = opt.lr / (1 - b1 ** t) * m2 / den
    p2 = p * (1 - opt.lr * opt.weight_decay * dec) - upd
    e_m = 4 * U * (b1 * m.abs() + (1 - b1) * g.abs())
    e_p = 4 * U * (p.abs() + p2.abs()) + opt.lr / (1 - b1 ** t) * e_m / den + 16 * U * upd.abs()
    within(opt.flat_p, p2, e_p, "p")
    if opt.state_bits == 32:
        within(opt.exp_avg, m2, e_m + 2e-45, "m")
        within(opt.exp_avg_sq, v2, 6 * U * v2 + 2e-45, "v")
    else:
        sm, sr = (m2.abs().view(-1, 256).amax(1) / 448).clamp_min(2.0 ** -126), (root.view(-1, 256).amax(1) / 448).clamp_min(2.0 ** -126)
        within(opt.exp_avg_scale, sm, 8 * U * sm, "m scale")
        # v is an f32: its smallest step 2^-149 (two of them here) is 5.3e-23 in the root
        tiny = math.sqrt(2 * 2.0 ** -149)
        within(opt.root_sq_scale, sr, 8 * U * sr + tiny / 448, "r scale")
        # e4m3: half a step of 2^-4 relative, half of 2^-9 (the smallest value) absolute; a nonzero root is at least that smallest value
        gm, gv = states(opt)
        within(gm, m2, m2.abs() * (2.0 ** -4 + 16 * U) + sm.repeat_interleave(256) * 2.0 ** -10 * 1.001 + e_m, "m")
        least = sr.repeat_interleave(256) * 2.0 ** -9 * (1 + 16 * U)        # in the optimizer's own scale, checked to 8 u above
        within(gv.sqrt(), root, root * (2.0 ** -4 + 16 * U) + torch.where(root < least, least, 0.501 * least) + tiny, "r")
        assert torch.equal(gv > 0, (v2 > 0) & (v2 >= 0)) or bool(((gv > 0) | (v2 < 1e-44)).all())
    pad = torch.ones(opt.numel, dtype=torch.bool, device="cuda")
    for q, o in zip(opt.params, opt.offsets):
        pad[o:o + q.numel()] = False
    assert not opt.flat_p[pad].any()


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_steps(bits):
    opt, g = make_opt(bits)
    for i in range(5):
        opt.zero_grad()
        for k, p in enumerate(opt.params):
            p.grad.add_(torch.randn(p.shape, device="cuda", generator=g) * 10.0 ** (k - 5))
        adamw_step_check(opt, 1.0 if i < 3 else 0.5)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_extreme_gradients(bits):
    opt, g = make_opt(bits, shapes=[(256,), (256, 2), (256,), (256,)])
    for i, scale in enumerate((1e-25, 1e-12, 1e12, 0.0, 1.0)):
        opt.zero_grad()
        opt.params[0].grad.add_(torch.randn(256, device="cuda", generator=g) * scale)
        opt.params[1].grad[:, 0] = torch.randn(256, device="cuda", generator=g) * 1e-9       # a wide range inside a block
        opt.params[1].grad[:, 1] = torch.randn(256, device="cuda", generator=g) * 1e3
        adamw_step_check(opt)
        assert torch.isfinite(opt.flat_p).all()


@pytest.mark.parametrize("bits,n", [(32, 10_000_003), (8, 17_000_001)])
def test_adamw_beyond_the_cache(bits, n):
    """Buffers over 256 MiB: four blocks a wave, streaming accesses; the last wave's blocks are not all there."""
    opt, g = make_opt(bits, shapes=[(n,), (77, 3)])
    for _ in range(2):
        opt.zero_grad()
        for p in opt.params:
            p.grad.add_(torch.randn(p.shape, device="cuda", generator=g) * 1e-3)
        adamw_step_check(opt)


def test_adamw_8bit_nonfinite_gradients_stay_with_their_elements():
    opt, g = make_opt(8, shapes=[(300,)])
    other, _ = make_opt(8, shapes=[(300,)])
    grad = torch.randn(300, device="cuda", generator=g)
    for o in (opt, other):
        o.flat_g[:300] = grad
    other.flat_g[7] = 0
    opt.flat_g[7], opt.flat_g[299] = float("nan"), float("inf")
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[7, 299]] = False
    opt.step(), other.step()
    m, v = states(opt)
    assert torch.isnan(opt.flat_p[7]) and torch.isnan(m[7]) and torch.isnan(v[7]) and torch.isnan(m[299])
    assert torch.equal(opt.flat_p[:256][keep[:256]], other.flat_p[:256][keep[:256]])
    assert torch.isfinite(m[:300][keep]).all() and torch.isfinite(opt.exp_avg_scale).all()
    opt.flat_g[:300] = 0.1
    opt.step()
    assert torch.isnan(opt.flat_p[7]) and torch.isfinite(opt.flat_p[:300][keep]).all()


def test_adamw_8bit_moments_follow_the_decay_of_a_block():
    """With no gradient the second moment falls by beta2 a step: the scale carries it although every code rounds to itself."""
    opt, g = make_opt(8, shapes=[(256,)], betas=(0.9, 0.999), lr=0.0)
    opt.flat_g.copy_(torch.randn(256, device="cuda", generator=g))
    opt.step()
    s0 = opt.root_sq_scale.clone()
    opt.flat_g.zero_()
    for _ in range(10):
        opt.step()
    # ten roundings of the largest value, whose code is exactly 448
    assert abs(float(opt.root_sq_scale / s0) - 0.999 ** 5) <= 10 * 8 * U


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_state_dict_and_decay_choice(bits, tmp_path):
    opt, g = make_opt(bits)
    opt.flat_g.copy_(torch.randn(opt.numel, device="cuda", generator=g))
    for q, o in zip(opt.params, opt.offsets):
        opt.flat_g[o + q.numel():(o + q.numel() + 255) // 256 * 256] = 0
    opt.step()
    torch.save(opt.state_dict(), tmp_path / "o.pth")
    sd = torch.load(tmp_path / "o.pth", map_location="cpu", weights_only=True)
    two, _ = make_opt(bits, seed=0, lr=1.0, weight_decay=0.5)
    two.flat_p.copy_(opt.flat_p)
    two.load_state_dict(sd)
    assert two.step_count == 1 and two.lr == 1e-2 and two.weight_decay == 0.1
    for o in (opt, two):
        o.flat_g.mul_(-0.5) if o is opt else o.flat_g.copy_(opt.flat_g)
        o.step()
    assert torch.equal(opt.flat_p, two.flat_p)
    assert sd["param_groups"][0]["weight_decay"] == 0.1
    with pytest.raises(ValueError, match="bit"):
        make_opt(40 - bits)[0].load_state_dict(sd)
    assert opt.decays == [len(s) > 1 for s in SHAPES]


def test_adamw_32bit_matches_torch():
    """torch.optim.AdamW on the same gradients: both are within the roundings of three steps (p is O(1), each step adds 8 u)."""
    opt, g = make_opt(32, decay_filter=None)
    ref = [torch.nn.Parameter(p.detach().clone()) for p in opt.params]
    ta = torch.optim.AdamW(ref, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    for _ in range(3):
        opt.zero_grad()
        for p, r in zip(opt.params, ref):
            p.grad.add_(torch.randn(p.shape, device="cuda", generator=g))
            r.grad = p.grad.clone()
        opt.step()
        ta.step()
    for p, r in zip(opt.params, ref):
        assert float((p - r).abs().max()) <= 3 * 16 * U * (float(r.abs().max()) + 1)


def test_adamw_buckets_and_frozen_parameters():
    """The data-parallel buckets are slices of the flat gradient buffer, whose tensors begin at multiples of 256 here; a
    parameter that needs no gradient is left alone."""
    from vae_gan_amd.optim import FlatAdamW
    from vae_gan_amd.train import DataParallel
    ps = [torch.nn.Parameter(torch.ones(300, device="cuda")), torch.nn.Parameter(torch.ones(5, device="cuda"), requires_grad=False),
          torch.nn.Parameter(torch.ones(256, device="cuda")), torch.nn.Parameter(torch.ones(2, 2, device="cuda"))]
    opt = FlatAdamW(ps, lr=0.1, weight_decay=0.5)
    assert opt.offsets == [0, 512, 768] and opt.numel == 1024 and opt._decay is None
    assert DataParallel.span(opt, [ps[2]]) == (512, 768) and DataParallel.span(opt, [ps[2], ps[3]]) == (512, 1024)
    opt.zero_grad()
    opt.step()
    assert torch.equal(ps[1], torch.ones(5, device="cuda")) and float((ps[0] - 0.95).abs().max()) <= 2 * U


def test_training_step_with_adamw_and_checkpoint(tmp_path):
    """build_optimizers with config.optimizer, one D+G step of the VQ model and its checkpoint."""
    from vae_gan_amd import loop, ops
    from vae_gan_amd.testing import synthetic_images
    from vae_gan_amd.train import build_optimizers, vq_train_step
    from vae_gan_amd.vq_vae_gan.config import Config
    from vae_gan_amd.vq_vae_gan.model import VQVAEGAN
    ops.set_compute_dtype(BF16)
    for kind in ("adamw", "adamw8bit"):
        cfg = Config()
        cfg.optimizer, cfg.weight_decay = kind, 0.05
        model = VQVAEGAN(cfg).cuda().train()
        og, od, sg, sd_ = build_optimizers(model, cfg)
        assert og.state_bits == (8 if kind == "adamw8bit" else 32) and og.weight_decay == 0.05 and od.lr == cfg.lr / 2
        assert [d for d in og.decays] == [p.dim() > 1 for p in og.params]
        before = og.flat_p.clone()
        vq_train_step(model, synthetic_images(2, 64, seed=1).cuda(), og, od)
        assert torch.isfinite(og.flat_p).all() and not torch.equal(before, og.flat_p)
        path = str(tmp_path / (kind + ".pth"))
        loop.save_checkpoint(path, 3, model, og, od, sg, sd_, 1.0)
        model2 = VQVAEGAN(cfg).cuda()
        o2 = build_optimizers(model2, cfg)
        loop.load_checkpoint(path, model2, *o2, full=True)
        assert o2[0].step_count == 1 and all(torch.equal(a, b) for a, b in zip(states(o2[0]), states(og)))


# ---------------------------------------------------------------------------------------------- together
def code_model(k, c, gen_, dt):
    """Two norm / widen / narrow layers and a head over k codes, as parameters (f32 masters)."""
    r = lambda *s, q=1.0: torch.nn.Parameter(q * torch.randn(*s, device="cuda", generator=gen_))      # noqa: E731
    ps = {"table": r(k, c)}
    for i in range(2):
        ps.update({f"n{i}w": torch.nn.Parameter(torch.ones(c, device="cuda")), f"n{i}b": r(c, q=0.1), f"u{i}": r(2 * c, c, q=c ** -0.5), f"ub{i}": r(2 * c, q=0.1),
                   f"d{i}": r(c, 2 * c, q=(2 * c) ** -0.5), f"db{i}": r(c, q=0.1)})
    ps.update({"nw": torch.nn.Parameter(torch.ones(c, device="cuda")), "nb": r(c, q=0.1), "head": r(k, c, q=c ** -0.5)})
    return ps


def code_model_run(ps, idx, target, dt):
    from vae_gan_amd import lib as L
    from vae_gan_amd import ops
    x = ps["table"][idx].to(dt)
    for i in range(2):
        h = ops.layer_norm(x, ps[f"n{i}w"], ps[f"n{i}b"])
        h = ops.linear_act(h, ps[f"u{i}"], ps[f"ub{i}"], L.ACT_GELU)
        x = ops.linear_act(h, ps[f"d{i}"], ps[f"db{i}"], residual=x)
    logits = ops.linear_act(ops.layer_norm(x, ps["nw"], ps["nb"]), ps["head"])
    logp, ent, _, _ = ops.token_logprobs(logits, target)
    return -logp.sum() / (target >= 0).sum() - 0.01 * ent.mean()


def code_model_oracle(ps, idx, target):
    f = torch.nn.functional
    x = ps["table"][idx]
    c = x.shape[-1]
    for i in range(2):
        h = f.layer_norm(x, (c,), ps[f"n{i}w"], ps[f"n{i}b"])
        x = f.gelu(h @ ps[f"u{i}"].t() + ps[f"ub{i}"]) @ ps[f"d{i}"].t() + ps[f"db{i}"] + x
    lnp = torch.log_softmax(f.layer_norm(x, (c,), ps["nw"], ps["nb"]) @ ps["head"].t(), -1)
    used = target >= 0
    pick = lnp.gather(-1, target.clamp_min(0)[..., None])[..., 0]
    return -(pick * used).sum() / used.sum() + 0.01 * (lnp.exp() * lnp).sum(-1).mean()


@pytest.mark.parametrize("dt,tol", [(F32, 2e-5), (BF16, 4e-2)])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_training_step_of_a_code_model(dt, tol, bits):
    """The operators as they are used: loss and every parameter's gradient against f64, then the update.  bf16: about a dozen
    roundings of h = 2^-8 relative lie on a path from a parameter to the loss and back, as many again in the gradient's own
    path; independent ones add up as sqrt(24) h / sqrt(3) = 1.1e-2 of the norm, and 4e-2 is 3.6 times that.  f32: sums of up to
    600 terms, sqrt(600 * 24) u = 7e-6."""
    from vae_gan_amd.optim import FlatAdamW
    k, c = 300, 72
    g = gen(9)
    ps = code_model(k, c, g, dt)
    idx = torch.randint(0, k, (3, 7, 9), device="cuda", generator=g)
    target = torch.randint(0, k, (3, 7, 9), device="cuda", generator=g)
    target[0, 0] = -100
    opt = FlatAdamW(list(ps.values()), lr=1e-3, weight_decay=0.1, decay_filter=lambda p: p.dim() > 1, state_bits=bits)
    ref = {n: p.detach().double().requires_grad_() for n, p in ps.items()}
    want = code_model_oracle(ref, idx, target)
    want.backward()
    opt.zero_grad()
    loss = code_model_run(ps, idx, target, dt)
    loss.backward()
    assert abs(float(loss) - float(want)) <= tol * abs(float(want))
    for n, p in ps.items():
        e = float((p.grad.double() - ref[n].grad).norm() / ref[n].grad.norm())
        assert e <= tol, (n, e)
    adamw_step_check(opt)
    opt.zero_grad()
    code_model_run(ps, idx, target, dt).backward()
    adamw_step_check(opt)


# ---------------------------------------------------------------------------------------------- streams and graphs
@pytest.mark.parametrize("dt", [BF16, F32])
def test_modules(dt):
    """nn.LayerNorm on an NHWC activation with padded channels and nn.LinearAct on token rows with its input as the residual."""
    from vae_gan_amd import lib as L
    from vae_gan_amd import nn as vnn
    g = gen(31)
    norm, lin = vnn.LayerNorm(41).cuda(), vnn.LinearAct(48, 48, act=L.ACT_GELU).cuda()
    x = torch.zeros(2, 5, 7, 48, device="cuda")
    x[..., :41] = torch.randn(2, 5, 7, 41, device="cuda", generator=g)
    x = x.to(dt)
    y = norm(x)
    ref = ln_oracle(x.reshape(-1, 48), norm.weight.detach(), norm.bias.detach(), None, 41, 1e-5, dt)
    assert y.shape == x.shape and not y[..., 41:].any()
    within(y.detach().reshape(-1, 48)[:, :41], *ref["y"], "y")
    tokens = y.detach().reshape(70, 48).requires_grad_()
    dy = torch.randn(70, 48, device="cuda", generator=g).to(dt)
    once = torch.autograd.grad(lin(tokens, tokens), (tokens, lin.weight, lin.bias), dy, retain_graph=True)
    other = tokens.detach().clone().requires_grad_()
    apart = torch.autograd.grad(lin(tokens, other), (tokens, other, lin.weight, lin.bias), dy)
    assert torch.equal(apart[1], dy) and torch.equal(once[1], apart[2]) and torch.equal(once[2], apart[3])
    within(once[0].detach(), apart[0].double() + dy.double(), half(dt) * (apart[0].double() + dy.double()).abs(), "the input's two gradients")


def test_second_derivatives_are_refused_and_a_graph_can_be_walked_twice():
    from vae_gan_amd import ops
    g = gen(32)
    x = torch.randn(9, 40, device="cuda", generator=g, requires_grad=True)
    w, b = torch.randn(40, 40, device="cuda", generator=g), torch.zeros(40, device="cuda")
    t = torch.randint(0, 40, (9,), device="cuda", generator=g)
    for f in (lambda: ops.layer_norm(x, b + 1, b), lambda: ops.linear_act(x, w, b, ACTS["silu"]), lambda: ops.token_logprobs(x, t)[0]):
        out = f().sum()
        first, = torch.autograd.grad(out, x, retain_graph=True)
        assert torch.equal(first, torch.autograd.grad(out, x)[0])
        with pytest.raises(RuntimeError, match="differentiated twice"):
            torch.autograd.grad(f().sum(), x, create_graph=True)


def test_two_streams_at_once():
    """The same operators on two streams, each with its own workspaces, interleaved."""
    from vae_gan_amd import ops
    g = gen(33)
    data = [[torch.randn(*s, device="cuda", generator=g).to(BF16) for s in ((700, 1030), (300, 1030), (300,))] for _ in range(2)]
    t = torch.randint(0, 300, (700,), device="cuda", generator=g)

    def run(x, w, b):
        xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        logp, ent, _, ta = ops.token_logprobs(ops.linear_act(xg, wg, b, ACTS["gelu"]), t, top=4)
        return [logp.detach(), ta] + list(torch.autograd.grad(logp.sum() + ent.sum(), (xg, wg)))
    want = [run(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for out in got[i] for a, b in zip(out, want[i]))


def test_operators_on_another_stream():
    from vae_gan_amd import ops
    x, w, b, res, dy = la_data(300, 256, 128, BF16, 3)
    t = torch.randint(0, 128, (300,), device="cuda", generator=gen(1))
    gam, bet = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")

    def run():
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = ops.layer_norm(ops.linear_act(xg, wg, b, ACTS["gelu"], res), gam, bet)
        logp, ent, tl, ta = ops.token_logprobs(y, t, top=3)
        return (logp, ta) + torch.autograd.grad(logp.sum() + ent.sum(), (xg, wg))
    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    assert all(torch.equal(a, b_) for a, b_ in zip(want, got))


def test_captured_and_replayed_with_new_inputs():
    """Forward, backward and two graphs of the same operators: every replay against the eager result, with eager work between."""
    from vae_gan_amd import ops
    g = gen(21)
    rows, c, k, v = 260, 96, 192, 5000
    w, hw = torch.randn(k, c, device="cuda", generator=g) / c ** 0.5, torch.randn(v, k, device="cuda", generator=g) / k ** 0.5
    gam, bet, bias = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda"), torch.zeros(k, device="cuda")

    def run(x, t):
        leaves = [q.detach().requires_grad_() for q in (x, gam, bet, w, bias, hw)]
        xx, ga, be, ww, bb, hh = leaves
        y = ops.linear_act(ops.linear_act(ops.layer_norm(xx, ga, be), ww, bb, ACTS["silu"]), hh)
        logp, ent, tl, ta = ops.token_logprobs(y, t, top=2)
        return [logp.detach(), tl, ta] + list(torch.autograd.grad(-logp.mean() - 0.1 * ent.mean(), leaves))
    made = []
    for dt in (BF16, F32):
        x = torch.randn(rows, c, device="cuda", generator=g).to(dt)
        t = torch.randint(0, v, (rows,), device="cuda", generator=g)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run(x, t)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(x, t)
        made.append((graph, x, t, out))
    for i in range(4):
        for graph, x, t, out in made:
            x.copy_(torch.randn(rows, c, device="cuda", generator=g))
            t.random_(0, v, generator=g)
            graph.replay()
            if i % 2:
                torch.cuda.synchronize()
            want = run(x, t)
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_step_captured(bits):
    """A captured step repeats its learning rate and bias correction; the states advance on every replay."""
    from vae_gan_amd import lib as L
    one, g = make_opt(bits)
    two, _ = make_opt(bits)
    grads = [torch.randn(one.numel, device="cuda", generator=g) * 0.1 for _ in range(3)]
    for o in (one, two):
        o.step_count = 50
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        one.step_count = 51
        one._update(1.0)
    for gr in grads:
        one.flat_g.copy_(gr)
        two.flat_g.copy_(gr)
        graph.replay()
        two.step_count = 51
        two._update(1.0)
    assert torch.equal(one.flat_p, two.flat_p) and all(torch.equal(a, b) for a, b in zip(states(one), states(two)))
