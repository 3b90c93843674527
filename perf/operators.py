"""Cases of the token-wise operators that a model of the codebook indices is trained with, in their plain form and through
the framework: layer norm, the matrix product with bias / activation / residual, the log probabilities of given codes, and
the AdamW step over many tensors.

``own`` False: elementary torch operations in 32 bits, each result rounded once.  ``own`` True: the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5                    # layer norm
LR, BETAS, ADAM_EPS = 1e-4, (0.9, 0.999), 1e-8
BLOCK = 256                   # elements of one tensor that share a scale of the 8-bit states


# ----------------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------------
def listed():
    return [
        # one position of a 512-wide code model, as when codes are drawn one at a time: launch latency
        {"name": "norm_token", "op": "norm", "rows": 1, "c": 512, "pad": 0, "dtype": "bf16", "direction": "forward"},
        # a training batch: 64 index maps of 16x16, 512 channels
        {"name": "norm_train", "op": "norm", "rows": 16384, "c": 512, "pad": 0, "dtype": "bf16", "direction": "train"},
        # a 41-channel latent in its padded NHWC rows, 16 maps of 64x64, f32 mode
        {"name": "norm_padded_f32", "op": "norm", "rows": 65536, "c": 41, "pad": 7, "dtype": "f32", "direction": "train"},
        # one position through a wide layer: bound by one read of the weights
        {"name": "linear_token", "op": "linear", "m": 1, "k": 1024, "n": 4096, "act": "gelu", "bias": True, "residual": False,
         "dtype": "bf16", "direction": "forward"},
        # the widening half of a token-wise layer pair, a training batch of 64 maps of 16x16
        {"name": "linear_widen", "op": "linear", "m": 16384, "k": 1024, "n": 4096, "act": "gelu", "bias": True, "residual": False,
         "dtype": "bf16", "direction": "train"},
        # the narrowing half with its residual, 512 channels, a ragged number of positions
        {"name": "linear_narrow", "op": "linear", "m": 16381, "k": 2048, "n": 512, "act": "none", "bias": True, "residual": True,
         "dtype": "bf16", "direction": "train"},
        # the exact-f32 mode at odd sizes
        {"name": "linear_odd_f32", "op": "linear", "m": 1001, "k": 515, "n": 1037, "act": "silu", "bias": True, "residual": True,
         "dtype": "f32", "direction": "train"},
        # the loss of a training batch over a large codebook
        {"name": "logprobs_train", "op": "logprobs", "rows": 16384, "vocab": 8192, "pad": 0, "top": 0, "masked": 0.0, "dtype": "bf16",
         "direction": "train"},
        # the default codebook in f32 with the best alternatives, codes in use only
        {"name": "logprobs_alternatives", "op": "logprobs", "rows": 4096, "vocab": 512, "pad": 0, "top": 4, "masked": 0.3,
         "dtype": "f32", "direction": "train"},
        # a handful of positions over a very large vocabulary, odd, in padded rows: the long axis has to be split
        {"name": "logprobs_few_long", "op": "logprobs", "rows": 3, "vocab": 200003, "pad": 61, "top": 8, "masked": 0.0,
         "dtype": "bf16", "direction": "forward"},
        # the discriminator of the default configuration, 8-bit states
        {"name": "adamw_discriminator_8bit", "op": "adamw", "tensors": "discriminator", "count": 0, "total": 0, "bits": 8, "decay": 0.01,
         "step": 100},
        # the generator of the beta configuration, 169 M parameters, 32-bit states
        {"name": "adamw_beta_generator", "op": "adamw", "tensors": "beta_generator", "count": 0, "total": 0, "bits": 32, "decay": 0.05,
         "step": 1000},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "logprobs", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    direction = rng.choice(["forward", "train", "train"])
    if op == "norm":
        c = _log_int(rng, 16, 8192)
        if rng.random() < 0.5:
            c = (c + 31) // 32 * 32
        rows = _log_int(rng, 1, min(65536, 8388608 // c))
        pad = rng.choice([0, 0, (-c) % 32])
        return {"op": op, "rows": rows, "c": c, "pad": pad, "dtype": dtype, "direction": direction}
    if op == "linear":
        k, n = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        if rng.random() < 0.6:
            k, n = (k + 63) // 64 * 64, (n + 63) // 64 * 64
        most = 16384 * 1024 * 4096 // (1 if dtype == "bf16" else 16)
        m = _log_int(rng, 1, max(1, min(16384, most // (k * n))))
        return {"op": op, "m": m, "k": k, "n": n, "act": rng.choice(["none", "lrelu", "sigmoid", "gelu", "silu"]),
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.5, "dtype": dtype, "direction": direction}
    if op == "logprobs":
        vocab = _log_int(rng, 8, 262144)
        if rng.random() < 0.4:
            vocab = 1 << (vocab.bit_length() - 1)
        rows = _log_int(rng, 1, max(1, min(16384, 67108864 // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 64)]),
                "top": rng.choice([0, 0, 1, 4, 8]), "masked": rng.choice([0.0, 0.0, 0.3]), "dtype": dtype, "direction": direction}
    count = _log_int(rng, 1, 300)
    return {"op": op, "tensors": "mixed", "count": count, "total": _log_int(rng, count, 100_000_000), "bits": rng.choice([8, 32]),
            "decay": rng.choice([0.0, 0.01, 0.1]), "step": _log_int(rng, 1, 100000)}


def work(case):
    c = case
    if c["op"] == "norm":
        e, n, cs = 2 if c["dtype"] == "bf16" else 4, c["rows"] * c["c"], c["rows"] * (c["c"] + c["pad"])
        train = c["direction"] == "train"
        return {"bytes": 2 * cs * e + 8 * c["c"] + train * (2 * cs * e + 12 * c["c"]), "flops": n * (8 + 14 * train)}
    if c["op"] == "linear":
        e, train = 2 if c["dtype"] == "bf16" else 4, c["direction"] == "train"
        xs, ws, ys = c["m"] * c["k"], c["n"] * c["k"], c["m"] * c["n"]
        b = c["n"] if c["bias"] else 0
        res = ys if c["residual"] else 0
        return {"bytes": e * (xs + ws + b + ys + res + train * (ys + xs + ws + b)), "flops": 2.0 * c["m"] * c["n"] * c["k"] * (3 if train else 1)}
    if c["op"] == "logprobs":
        e, n, r = 2 if c["dtype"] == "bf16" else 4, c["rows"] * c["vocab"], c["rows"]
        train = c["direction"] == "train"
        return {"bytes": n * e * (1 + train) + r * (16 + 12 * c["top"] + 8 * train), "flops": n * (6 + 8 * train)}
    n = sum(math.prod(s) for s in _shapes(c))
    return {"bytes": n * 12 + (n * 4 + n / BLOCK * 16 if c["bits"] == 8 else n * 16), "flops": 14 * n}


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _bn(c):
    return [(c,), (c,)]


def _conv(i, o, k):
    return [(o, i, k, k), (o,)]


def _res(c):
    return _conv(c, c, 3) + _conv(c, c, 3) + _bn(c) + _bn(c)


def _shapes(case):
    """The parameter shapes of one optimizer: the layer stacks of the framework's own configurations, or a mixture."""
    ch = [64, 128, 256, 512]
    if case["tensors"] == "discriminator":
        out = _conv(3, 64, 4)
        for a, b in zip(ch, ch[1:]):
            out += _conv(a, b, 4) + _bn(b)
        return out + _conv(512, 1, 4)
    if case["tensors"] == "beta_generator":
        out = _conv(3, 64, 3) + _bn(64)
        for a, b in zip(ch, ch[1:]):
            out += _res(a) + _conv(a, b, 4) + _bn(b)
        out += _res(512) + 2 * [(128, 512 * 32 * 32), (128,)] + [(512 * 16 * 16, 128), (512 * 16 * 16,)] + _bn(512)
        for a, b in zip(ch[:0:-1], ch[-2::-1]):
            out += _res(a) + _conv(b, a, 4)[:1] + [(b,)] + _bn(b)
        return out + _res(64) + _conv(64, 3, 3)
    r = random.Random("%d of %d" % (case["count"], case["total"]))
    share = [math.exp(r.uniform(0.0, 8.0)) for _ in range(case["count"])]
    out = []
    for s in share:
        n = max(1, int(case["total"] * s / sum(share)))
        rows = r.choice([1, 1, 3, 16, 64])
        out.append((rows, n // rows) if 1 < rows <= n else (n,))
    return out


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _layout(shapes):
    """Offsets of tensors in one flat buffer, each begun at a multiple of BLOCK, and the buffer's length."""
    offsets, at = [], 0
    for s in shapes:
        offsets.append(at)
        at += (math.prod(s) + BLOCK - 1) // BLOCK * BLOCK
    return offsets, at


def _round8(blocks):
    """[n, BLOCK] non-negative or signed values as e4m3 with one scale a block (the largest magnitude becomes 448)."""
    scale = (blocks.abs().amax(dim=1) * (1.0 / 448.0)).clamp_min(2.0 ** -126)
    return (blocks * (1.0 / scale)[:, None]).to(torch.float8_e4m3fn), scale


def _root8(v):
    """The root of the second moments in 8 bits; what is not zero stays at least the smallest code, 2^-9 of the scale."""
    root = v.sqrt()
    scale = (root.amax(dim=1) * (1.0 / 448.0)).clamp_min(2.0 ** -126)
    q = root * (1.0 / scale)[:, None]
    return torch.where(root > 0, q.clamp_min(2.0 ** -9), q).to(torch.float8_e4m3fn), scale


def _inputs(case, seed):
    """The tensors of one case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    dt = DTYPES.get(c.get("dtype"))
    if c["op"] == "norm":
        spread = torch.exp(0.5 * _normal(g, c["c"] + c["pad"]))              # channels of different sizes, some far from 0
        x = _normal(g, c["rows"], c["c"] + c["pad"]) * spread + 0.5 * _normal(g, c["c"] + c["pad"])
        x[:, c["c"]:] = 0
        d = {"x": x.to(dt), "w": 1 + 0.2 * _normal(g, c["c"]), "b": 0.1 * _normal(g, c["c"])}
        if c["direction"] == "train":
            dy = _normal(g, c["rows"], c["c"] + c["pad"]) * torch.exp(_normal(g, c["rows"], 1)) * 1e-3
            dy[:, c["c"]:] = 0
            d["dy"] = dy.to(dt)
        return d
    if c["op"] == "linear":
        d = {"x": _normal(g, c["m"], c["k"]).to(dt), "w": (_normal(g, c["n"], c["k"]) / c["k"] ** 0.5).to(dt), "b": None, "res": None}
        if c["bias"]:
            d["b"] = (0.5 * _normal(g, c["n"])).to(dt)
        if c["residual"]:
            d["res"] = _normal(g, c["m"], c["n"]).to(dt)
        if c["direction"] == "train":
            d["dy"] = (1e-2 * _normal(g, c["m"], c["n"])).to(dt)
        return d
    if c["op"] == "logprobs":
        sharp = torch.exp(0.7 * _normal(g, c["rows"], 1))                   # sure positions and unsure ones
        x = _normal(g, c["rows"], c["vocab"]) * (1.5 * sharp)
        tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda")
        if c["masked"] > 0:
            x.masked_fill_(torch.rand(c["rows"], c["vocab"], generator=g, device="cuda") < c["masked"], -math.inf)
            x[torch.arange(c["rows"], device="cuda"), tokens] = _normal(g, c["rows"])   # the code that was taken is allowed
            if c["rows"] > 8:
                x[c["rows"] // 2] = -math.inf                                  # a padded position: nothing is allowed
        tokens[::7] = torch.where(torch.arange(0, c["rows"], 7, device="cuda") > 0, -100, tokens[::7])     # positions without a loss
        store = torch.zeros(c["rows"], c["vocab"] + c["pad"], dtype=dt, device="cuda")
        store[:, :c["vocab"]] = x.to(dt)
        d = {"x": store[:, :c["vocab"]], "tokens": tokens}
        if c["direction"] == "train":
            d["dlogp"] = torch.full((c["rows"],), -1.0 / c["rows"], device="cuda")
            d["dent"] = (0.1 / c["rows"]) * _normal(g, c["rows"])
        return d
    shapes = _shapes(c)
    offsets, n = _layout(shapes)
    valid = torch.zeros(n, device="cuda")
    decay = torch.zeros(n // BLOCK, device="cuda")
    for s, o in zip(shapes, offsets):
        valid[o:o + math.prod(s)] = 1
        decay[o // BLOCK:(o + math.prod(s) + BLOCK - 1) // BLOCK] = float(len(s) > 1)       # biases and norm weights are not decayed
    size = torch.exp(1.5 * _normal(g, n // BLOCK, 1)) * 1e-4
    grad = (_normal(g, n // BLOCK, BLOCK) * size).view(-1) * valid
    m = (0.3 * _normal(g, n // BLOCK, BLOCK) * size).view(-1) * valid
    v = ((torch.exp(0.7 * _normal(g, n // BLOCK, BLOCK)) * size).square()).view(-1) * valid
    d = {"p": 0.05 * _normal(g, n) * valid, "g": grad, "decay": decay}
    if c["bits"] == 8:
        d["m"], d["m_scale"] = _round8(m.view(-1, BLOCK))
        d["r"], d["r_scale"] = _root8(v.view(-1, BLOCK))
        d["m"], d["r"] = d["m"].view(-1), d["r"].view(-1)
    else:
        d["m"], d["v"] = m, v
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if case["op"] == "adamw":
        d["step"] = case["step"]
        if own:
            d["opt"] = _optimizer(case, d)
    return d


def _optimizer(case, d):
    """The framework's optimizer over parameters with these values, in the middle of a training run."""
    from vae_gan_amd.optim import FlatAdamW
    shapes = _shapes(case)
    offsets, _ = _layout(shapes)
    params = [torch.nn.Parameter(d["p"][o:o + math.prod(s)].reshape(s).clone()) for s, o in zip(shapes, offsets)]
    opt = FlatAdamW(params, lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=case["decay"], decay_filter=lambda p: p.dim() > 1,
                    state_bits=case["bits"])
    opt.flat_g.copy_(d["g"])
    opt.exp_avg.copy_(d["m"])
    if case["bits"] == 8:
        opt.exp_avg_scale.copy_(d["m_scale"])
        opt.root_sq.copy_(d["r"])
        opt.root_sq_scale.copy_(d["r_scale"])
    else:
        opt.exp_avg_sq.copy_(d["v"])
    opt.step_count = case["step"] - 1
    for k in ("p", "g", "m", "v", "r", "m_scale", "r_scale", "decay"):
        d.pop(k, None)
    return opt


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(state):
    return {"norm": _norm, "linear": _linear, "logprobs": _logprobs, "adamw": _adamw}[state["case"]["op"]](state)


def _norm(s):
    c = s["case"]
    train = c["direction"] == "train"
    if own:
        from vae_gan_amd import ops
        if not train:
            with torch.no_grad():
                return {"y": ops.layer_norm(s["x"], s["w"], s["b"], EPS, c["c"])}
        x, w, b = (s[k].detach().requires_grad_() for k in ("x", "w", "b"))
        y = ops.layer_norm(x, w, b, EPS, c["c"])
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    n, dt = c["c"], s["x"].dtype
    x = s["x"][:, :n].float()
    mean = x.mean(dim=1, keepdim=True)
    xc = x - mean
    rstd = (xc.square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    xh = xc * rstd
    y = torch.zeros_like(s["x"])
    y[:, :n] = (xh * s["w"] + s["b"]).to(dt)
    if not train:
        return {"y": y}
    dy = s["dy"][:, :n].float()
    g = dy * s["w"]
    dx = torch.zeros_like(s["x"])
    dx[:, :n] = (rstd * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))).to(dt)
    return {"y": y, "dx": dx, "dw": (dy * xh).sum(dim=0), "db": dy.sum(dim=0)}


def _act(z, act):
    if act == "lrelu":
        return torch.where(z > 0, z, 0.2 * z)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "lrelu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, 0.2))
    if act == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 - p)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _linear(s):
    c = s["case"]
    train = c["direction"] == "train"
    names = [k for k in ("x", "w", "b", "res") if s[k] is not None]
    if own:
        from vae_gan_amd import lib, ops
        act = {"none": lib.ACT_NONE, "lrelu": lib.ACT_LRELU, "sigmoid": lib.ACT_SIGMOID, "gelu": lib.ACT_GELU, "silu": lib.ACT_SILU}[c["act"]]
        if not train:
            with torch.no_grad():
                return {"y": ops.linear_act(s["x"], s["w"], s["b"], act, s["res"])}
        t = {k: s[k].detach().requires_grad_() for k in names}
        y = ops.linear_act(t["x"], t["w"], t.get("b"), act, t.get("res"))
        return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, torch.autograd.grad(y, [t[k] for k in names], s["dy"]))}}
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, c["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    out = {"y": y.to(dt)}
    if train:
        dz = s["dy"].float() * _act_slope(z, c["act"])
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if s["b"] is not None:
            out["db"] = dz.sum(dim=0).to(dt)
        if s["res"] is not None:
            out["dres"] = s["dy"]
    return out


def _top(x, k):
    """The k largest of each row and their places, equal values in the order of their places."""
    v = x.shape[1]
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = order * (1 << 32) + (v - 1 - torch.arange(v, device=x.device))
    at = (v - 1) - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    return x.gather(1, at), at


def _logprobs(s):
    c = s["case"]
    train = c["direction"] == "train"
    if own:
        from vae_gan_amd import ops
        x = s["x"].detach().requires_grad_(train)
        logp, entropy, top_logp, top_at = ops.token_logprobs(x, s["tokens"], top=c["top"])
        out = {"logp": logp.detach(), "entropy": entropy.detach()}
        if train:
            out["dx"], = torch.autograd.grad((logp, entropy), (x,), (s["dlogp"], s["dent"]))
    else:
        x, t = s["x"].float(), s["tokens"]
        most = x.amax(dim=1, keepdim=True)
        empty = most == -math.inf
        xs = x - torch.where(empty, torch.zeros_like(most), most)
        e = torch.exp(xs)
        total = e.sum(dim=1, keepdim=True)
        ln_total = torch.log(total)
        weighted = torch.where(e > 0, e * xs, torch.zeros_like(e))
        entropy = torch.where(empty, torch.zeros_like(total), ln_total - weighted.sum(dim=1, keepdim=True) / total)
        used = t >= 0
        logp = torch.where(used, (xs.gather(1, t.clamp_min(0)[:, None]) - ln_total)[:, 0], torch.zeros_like(t, dtype=torch.float32))
        logp = torch.where(used & empty[:, 0], torch.full_like(logp, -math.inf), logp)
        out = {"logp": logp, "entropy": entropy[:, 0]}
        if train:
            p = torch.where(empty, torch.zeros_like(e), e / total)
            ln_p = torch.where(e > 0, xs - ln_total, torch.zeros_like(e))
            a = torch.where(used & ~empty[:, 0], s["dlogp"], torch.zeros_like(s["dlogp"]))
            dx = -p * (a[:, None] + s["dent"][:, None] * (ln_p + entropy))
            dx.scatter_add_(1, t.clamp_min(0)[:, None], a[:, None])
            out["dx"] = dx.to(s["x"].dtype)
        if c["top"]:
            best, top_at = _top(x, c["top"])
            top_logp = torch.where(empty, best, best - torch.where(empty, torch.zeros_like(most), most) - ln_total)
    if c["top"]:
        out["top_logp"], out["top_at"] = top_logp, top_at
    return out


def _adamw(s):
    c = s["case"]
    if own:
        opt = s["opt"]
        opt.step()
        if c["bits"] == 8:
            return {"p": opt.flat_p, "m": opt.exp_avg, "m_scale": opt.exp_avg_scale, "r": opt.root_sq, "r_scale": opt.root_sq_scale}
        return {"p": opt.flat_p, "m": opt.exp_avg, "v": opt.exp_avg_sq}
    t, (b1, b2) = s["step"], BETAS
    s["step"] += 1
    g = s["g"].view(-1, BLOCK)
    if c["bits"] == 8:
        m = s["m"].view(-1, BLOCK).float() * s["m_scale"][:, None]
        v = (s["r"].view(-1, BLOCK).float() * s["r_scale"][:, None]).square()
    else:
        m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = s["p"].view(-1, BLOCK)
    p = p * (1 - LR * c["decay"] * s["decay"])[:, None]
    s["p"] = (p - (LR / (1 - b1 ** t)) * (m / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + ADAM_EPS))).view(-1)
    if c["bits"] == 8:
        s["m"], s["m_scale"] = _round8(m)
        s["r"], s["r_scale"] = _root8(v)
        s["m"], s["r"] = s["m"].view(-1), s["r"].view(-1)
        return {k: s[k] for k in ("p", "m", "m_scale", "r", "r_scale")}
    s["m"], s["v"] = m.view(-1), v.view(-1)
    return {k: s[k] for k in ("p", "m", "v")}


# ----------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    d = _inputs(case, seed)
    c = case
    train = c.get("direction") == "train"
    if c["op"] == "norm":
        n = c["c"]
        x = d["x"].double()[:, :n]
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        r = 1 / torch.sqrt(var + EPS)
        w, wide = d["w"].double(), lambda a: torch.nn.functional.pad(a, (0, c["pad"]))  # noqa: E731
        out = {"y": wide((x - mean) * r * w + d["b"].double())}
        if train:
            dy = d["dy"].double()[:, :n]
            # the Jacobian applied as a product: r (I - 1/n - xh xh^T / n) (w dy)
            u, xh = dy * w, (x - mean) * r
            out["dx"] = wide(r * (u - u.sum(1, True) / n - xh * ((u * xh).sum(1, True) / n)))
            out["dw"], out["db"] = (dy * xh).sum(0), dy.sum(0)
        return out
    if c["op"] == "linear":
        x, w = d["x"].double(), d["w"].double()
        z = torch.mm(x, w.t().contiguous())
        if c["bias"]:
            z += d["b"].double()
        z.requires_grad_(train)
        with torch.enable_grad():
            f = torch.nn.functional
            y = {"none": lambda a: a * 1, "lrelu": lambda a: f.leaky_relu(a, 0.2), "sigmoid": torch.sigmoid, "gelu": f.gelu, "silu": f.silu}[c["act"]](z)
        out = {"y": y.detach() + (d["res"].double() if c["residual"] else 0)}
        if train:
            dz, = torch.autograd.grad(y, z, d["dy"].double())
            out["dx"], out["dw"] = torch.mm(dz, w), torch.mm(dz.t().contiguous(), x)
            if c["bias"]:
                out["db"] = dz.sum(0)
            if c["residual"]:
                out["dres"] = d["dy"].double()
        return out
    if c["op"] == "logprobs":
        out = {k: [] for k in ("logp", "entropy") + (("dx",) if train else ()) + (("top_logp",) if c["top"] else ())}
        step = max(1, (1 << 25) // c["vocab"])
        for r in range(0, c["rows"], step):
            x, t = d["x"][r:r + step].double(), d["tokens"][r:r + step]
            lse = torch.logsumexp(x, 1, keepdim=True)
            empty = torch.isinf(lse)
            ln_p = torch.where(empty, torch.full_like(x, -math.inf), x - lse)
            p = torch.exp(ln_p)
            ent = -torch.special.xlogy(p, p).sum(1, keepdim=True)
            picked = ln_p.gather(1, t.clamp_min(0)[:, None])[:, 0]
            out["logp"].append(torch.where(t < 0, torch.zeros_like(picked), picked))
            out["entropy"].append(ent[:, 0] + 0.0)
            if train:
                a = torch.where((t < 0) | empty[:, 0], 0.0, d["dlogp"][r:r + step].double())
                dx = -a[:, None] * p - d["dent"][r:r + step, None].double() * (torch.special.xlogy(p, p) + p * ent)
                dx[torch.arange(len(t), device=t.device), t.clamp_min(0)] += a
                out["dx"].append(dx)
            if c["top"]:
                out["top_logp"].append(torch.sort(ln_p, dim=1, descending=True).values[:, :c["top"]])
        out = {k: torch.cat(v) for k, v in out.items()}
        return {**out, "top_at": None} if c["top"] else out
    t, (b1, b2) = c["step"], BETAS
    g, p = d["g"].double(), d["p"].double()
    if c["bits"] == 8:
        m = (d["m"].double().view(-1, BLOCK) * d["m_scale"].double()[:, None]).view(-1)
        v = (d["r"].double().view(-1, BLOCK) * d["r_scale"].double()[:, None]).view(-1) ** 2
    else:
        m, v = d["m"].double(), d["v"].double()
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    p = p - p * LR * c["decay"] * d["decay"].double().repeat_interleave(BLOCK)
    p = p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + ADAM_EPS)
    if c["bits"] == 8:
        largest = lambda a: a.abs().view(-1, BLOCK).amax(1) / 448  # noqa: E731
        return {"p": p, "m": None, "m_scale": largest(m), "r": None, "r_scale": largest(torch.sqrt(v))}
    return {"p": p, "m": m, "v": v}
