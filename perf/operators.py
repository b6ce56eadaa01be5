"""Group norm with an activation (channels last) and the AdamW step over many tensors: cases, plain forms, exact forms.

``own`` False: the operators in elementary torch operations, in 32 bits.  ``own`` True: the calls a training program makes
of this package.  A state's tensors lie as such a program has them: activations [N, H, W, C]; the parameters of a model as
views of one flat buffer (every tensor starts on a multiple of 256 elements there), with flat gradients and moments.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-3            # of the normalisation layers of this package
BETA_1, BETA_2, ADAM_EPS, LR = 0.9, 0.999, 1e-7, 1e-3
DECAY, DECAY_STEPS, DECAY_RATE = 0.004, 10, 0.96
BLOCK = 256           # elements of one 8-bit block, and what every tensor of a flat buffer starts on a multiple of
SEED = 1833


# ------------------------------------------------------------------------------------------------ cases
def _autoencoder():
    """The kernels and biases of the 12 035-weight auto-encoder."""
    sizes, cin = [], 3
    for cout in (8, 16, 32, 16, 8, 3):
        sizes += [9 * cin * cout, cout]
        cin = cout
    return sizes


def _gan():
    """The U-Net of 2x2 convolutions and its discriminator of 4x4 ones: kernels, gammas and betas."""
    sizes = []
    for cin in (6, 64, 64, 64):
        sizes += [4 * cin * 64, 64, 64]
    sizes += [4 * 64 * 64, 4 * 128 * 64, 4 * 128 * 64, 4 * 128 * 3, 3]
    sizes += [16 * 9 * 64, 16 * 64 * 128, 128, 128, 16 * 128 * 256, 256, 256, 16 * 256, 1]
    return sizes


def _stack(width, layers, tail):
    """A generic deep stack: square matrices, one four times as wide, vectors, and a ragged last tensor."""
    sizes = []
    for _ in range(layers):
        sizes += [width * width, 4 * width * width, width, 4 * width]
    return sizes + [tail]


def _text(sizes):
    return ",".join(str(n) for n in sizes)


def _norm(name, op, n, h, w, c, groups, dtype, act):
    return {"name": name, "op": op, "n": n, "h": h, "w": w, "c": c, "groups": groups, "dtype": dtype, "act": act}


def _adamw(name, sizes, bits, clip=0.0, copy=False):
    return {"name": name, "op": "adamw", "sizes": _text(sizes), "bits": bits, "clip": clip, "copy": copy}


def listed():
    return [
        # one image of a U-Net's second stage: what a single-sample call costs, latency alone
        _norm("norm_fwd_one_image", "norm_fwd", 1, 8, 8, 64, 8, "float32", "lrelu"),
        # the first stage of a 64-filter stack at the auto-encoder's batch: the largest ordinary call
        _norm("norm_fwd_batch_1024", "norm_fwd", 1024, 32, 32, 64, 8, "float32", "elu"),
        # odd extents and a channel count that leaves 4-byte pieces in bf16
        _norm("norm_fwd_odd", "norm_fwd", 37, 31, 29, 90, 9, "bfloat16", "relu"),
        # few large images: one sample is more than a workgroup can hold
        _norm("norm_fwd_large_image", "norm_fwd", 2, 512, 512, 128, 32, "bfloat16", "elu"),
        # the discriminator's 128-channel stage over [real; generated] at batch 32: an ordinary small backward call
        _norm("norm_bwd_gan", "norm_bwd", 64, 8, 8, 128, 16, "float32", "lrelu"),
        # the bf16 policy at batch 1024
        _norm("norm_bwd_batch_1024", "norm_bwd", 1024, 16, 16, 256, 32, "bfloat16", "lrelu"),
        # odd extents, channels in pieces of two
        _norm("norm_bwd_odd", "norm_bwd", 19, 45, 33, 54, 6, "float32", "elu"),
        # few large images, backward
        _norm("norm_bwd_large_image", "norm_bwd", 4, 256, 256, 64, 8, "float32", "elu"),
        # the step at the end of the auto-encoder's 0.15 ms training step: latency
        _adamw("adamw_autoencoder", _autoencoder(), 32),
        # the GAN models under the bf16 policy, states in 8 bits: parameters, their bf16 copy, moments
        _adamw("adamw_gan_8bit", _gan(), 8, copy=True),
        # a model of 101 M weights, gradients clipped by their global norm
        _adamw("adamw_large_clip", _stack(1024, 19, 1_234_567), 32, clip=1.0),
        # the same model with its states in 8 bits
        _adamw("adamw_large_8bit", _stack(1024, 19, 1_234_567), 8),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "adamw"])
    if op == "adamw":
        bits = rng.choice([32, 8])
        total = _spread(rng, 3_000, 90_000_000)
        count = _spread(rng, 1, 60)
        parts = [_spread(rng, 1, 5_000) for _ in range(count)]
        scale = total / sum(parts)
        sizes = [max(1, int(p * scale)) for p in parts]
        clip = rng.choice([0.0, 1.0]) if bits == 32 else 0.0
        return {"op": op, "sizes": _text(sizes), "bits": bits, "clip": clip, "copy": rng.random() < 0.5}
    while True:
        groups, depth = rng.choice([1, 2, 4, 6, 8, 9, 16, 32]), rng.choice([1, 2, 3, 4, 5, 8, 10, 16, 32])
        n, h, w = _spread(rng, 1, 1024), _spread(rng, 2, 512), _spread(rng, 2, 512)
        total = n * h * w * groups * depth
        # no larger than the largest listed case of the direction, and no kernel is called for a handful of numbers
        if 4_000 <= total <= (16_000_000 if op == "norm_bwd" else 60_000_000):
            break
    return {"op": op, "n": n, "h": h, "w": w, "c": groups * depth, "groups": groups,
            "dtype": rng.choice(["float32", "bfloat16"]), "act": rng.choice(["none", "relu", "elu", "lrelu", "tanh", "sigmoid"])}


def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        # gradient, parameter twice, moments twice; a bf16 copy; moments in 8 bits are also handed out as values
        each = 4 + 8 + (16 if case["bits"] == 32 else 4 + 8) + (2 if case["copy"] else 0)
        return {"bytes": each * n, "flops": 16 * n}
    n = case["n"] * case["h"] * case["w"] * case["c"]
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": (2 if case["op"] == "norm_fwd" else 3) * size * n, "flops": (10 if case["op"] == "norm_fwd" else 20) * n}


def _sizes(case):
    return [int(s) for s in case["sizes"].split(",")]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "adamw":
        return _prepare_adamw(case, normal, dev)
    n, h, w, c, groups = (case[k] for k in ("n", "h", "w", "c", "groups"))
    dtype = getattr(torch, case["dtype"])
    act = None if case["act"] == "none" else case["act"]
    # activations of a convolution: channels of their own level and spread
    x = normal(n, h, w, c).mul_(normal(c).abs_() + 0.3).add_(normal(c)).to(dtype)
    st = {"case": case, "x": x, "gamma": 1 + 0.2 * normal(c), "beta": 0.2 * normal(c), "act": act, "alpha": 0.2}
    if case["op"] == "norm_fwd":
        st["y"] = torch.empty_like(x)
        st["mean"], st["rstd"] = torch.empty(n, groups, device=dev), torch.empty(n, groups, device=dev)
    else:
        v = x.view(n, h * w, groups, c // groups).double()
        mean = v.mean((1, 3))
        var = v.sub_(mean[:, None, :, None]).square_().mean((1, 3))
        st["mean"], st["rstd"] = mean.float(), (var + EPS).rsqrt().float()
        st["dy"] = normal(n, h, w, c).mul_(0.01).to(dtype)
        st["dx"], st["dgamma"], st["dbeta"] = torch.empty_like(x), torch.empty(c, device=dev), torch.empty(c, device=dev)
    if own:  # the scratch that a model keeps
        from spectrum_vae_amd import ops
        nbytes = ops.groupnorm_workspace(n, h * w, c, groups)
        st["ws"] = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
    return st


def _prepare_adamw(case, normal, dev):
    sizes = _sizes(case)
    blocks = [-(-s // BLOCK) for s in sizes]
    starts = [BLOCK * b for b in np.cumsum([0] + blocks[:-1])]
    total = BLOCK * sum(blocks)
    live = torch.zeros(total, dtype=torch.bool, device=dev)
    decay = torch.zeros(total, device=dev)
    for i, (at, s) in enumerate(zip(starts, sizes)):
        live[at:at + s] = True
        if s > 1024:  # vectors (biases, gammas, betas) are not decayed
            decay[at:at + s] = DECAY
    spread = torch.exp(2.0 * normal(total // BLOCK)).repeat_interleave(BLOCK)  # layers differ in their gradients' size
    st = {"case": case, "theta": normal(total).mul_(0.05).mul_(live), "grad": normal(total).mul_(spread).mul_(1e-3).mul_(live)}
    m = normal(total).mul_(spread).mul_(3e-4).mul_(live)
    v = normal(total).mul_(spread).mul_(1e-3).square_().mul_(live).add_(1e-12 * live)
    if case["bits"] == 8:
        half = torch.full((), 1 << 15, dtype=torch.int32, device=dev)
        st["m"], st["m_exp"] = _encode(m, half, 15)
        st["v"], st["v_exp"] = _encode(v, half, 31)
        st["m_out"], st["v_out"] = torch.empty(total, device=dev), torch.empty(total, device=dev)
    else:
        st["m"], st["v"] = m, v
    st["copy"] = st["theta"].bfloat16() if case["copy"] else None
    st["count"] = torch.tensor([25, 0, 0], dtype=torch.int64, device=dev)  # updates so far, and the step's scratch
    if own:  # the plan of a model's tensors
        from spectrum_vae_amd import ops
        cut = lambda t: [t[at:at + s] for at, s in zip(starts, sizes)]  # noqa: E731
        by_block = lambda t: [t[at // BLOCK:at // BLOCK + b] for at, b in zip(starts, blocks)]  # noqa: E731
        st["plan"] = ops.AdamWPlan(cut(st["theta"]), cut(st["grad"]), cut(st["m"]), cut(st["v"]),
                                   [DECAY if s > 1024 else 0.0 for s in sizes],
                                   m_exp=by_block(st["m_exp"]) if case["bits"] == 8 else None,
                                   v_exp=by_block(st["v_exp"]) if case["bits"] == 8 else None,
                                   params_lp=cut(st["copy"]) if case["copy"] else None)
    else:
        st["decay"] = decay
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        return _adamw_own(state) if own else _adamw_plain(state)
    if op == "norm_fwd":
        return _norm_fwd_own(state) if own else _norm_fwd_plain(state)
    return _norm_bwd_own(state) if own else _norm_bwd_plain(state)


def _norm_fwd_own(s):
    from spectrum_vae_amd import ops
    ops.groupnorm_act_fwd(s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"], s["case"]["groups"], EPS, s["act"],
                          s["alpha"], s["ws"])
    return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}


def _norm_bwd_own(s):
    from spectrum_vae_amd import ops
    ops.groupnorm_act_bwd(s["x"], s["dy"], s["gamma"], s["beta"], s["mean"], s["rstd"], s["dx"], s["dgamma"], s["dbeta"],
                          False, s["case"]["groups"], s["act"], s["alpha"], s["ws"])
    return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}


def _adamw_own(s):
    from spectrum_vae_amd import ops
    ops.adamw_step(s["plan"], s["count"], LR, BETA_1, BETA_2, ADAM_EPS, DECAY_STEPS, DECAY_RATE, True,
                   clip_norm=s["case"]["clip"], seed=SEED)
    return _adamw_outputs(s, lambda code, exp, out, second: ops.adamw_decode(code, exp, out, second))


def _adamw_outputs(s, decode):
    out = {"theta": s["theta"]}
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    if s["case"]["bits"] == 8:  # the values that the 8-bit moments stand for
        decode(s["m"], s["m_exp"], s["m_out"], False)
        decode(s["v"], s["v_exp"], s["v_out"], True)
        out["m"], out["v"] = s["m_out"], s["v_out"]
    else:
        out["m"], out["v"] = s["m"], s["v"]
    return out


# ------------------------------------------------------------------------------------------------ plain forms
def _act(z, act, alpha):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "elu":
        return torch.where(z > 0, z, torch.expm1(z))
    if act == "lrelu":
        return torch.where(z >= 0, z, alpha * z)
    if act == "tanh":
        return torch.tanh(z)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_slope(z, act, alpha):
    """d act / d z; at 0 the slope of the negative side."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "elu":
        return torch.where(z > 0, torch.ones_like(z), torch.exp(z))
    if act == "lrelu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, alpha))
    if act == "tanh":
        return 1 - torch.tanh(z).square()
    if act == "sigmoid":
        y = 1 / (1 + torch.exp(-z))
        return y * (1 - y)
    return torch.ones_like(z)


def _norm_fwd_plain(s):
    x, groups = s["x"], s["case"]["groups"]
    n, c = x.shape[0], x.shape[-1]
    v = x.float().view(n, -1, groups, c // groups)
    mean = v.mean((1, 3))
    d = v - mean[:, None, :, None]
    rstd = 1 / torch.sqrt(d.square().mean((1, 3)) + EPS)
    z = (d * rstd[:, None, :, None]).view(n, -1, c) * s["gamma"] + s["beta"]
    return {"y": _act(z, s["act"], s["alpha"]).view(x.shape).to(x.dtype), "mean": mean, "rstd": rstd}


def _norm_bwd_plain(s):
    x, groups = s["x"], s["case"]["groups"]
    n, c = x.shape[0], x.shape[-1]
    split = (n, -1, groups, c // groups)
    rstd = s["rstd"][:, None, :, None]
    xhat = ((x.float().view(split) - s["mean"][:, None, :, None]) * rstd).view(n, -1, c)
    dz = s["dy"].float().view(n, -1, c) * _act_slope(xhat * s["gamma"] + s["beta"], s["act"], s["alpha"])
    dgamma, dbeta = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    gz, xh = (dz * s["gamma"]).view(split), xhat.view(split)
    c1, c2 = gz.mean((1, 3), keepdim=True), (gz * xh).mean((1, 3), keepdim=True)
    return {"dx": (rstd * (gz - c1 - xh * c2)).view(x.shape).to(x.dtype), "dgamma": dgamma, "dbeta": dbeta}


def _adamw_plain(s):
    case, theta = s["case"], s["theta"]
    it = s["count"][0]
    t = (it + 1).double()
    lr = LR * DECAY_RATE ** torch.div(it, DECAY_STEPS, rounding_mode="floor").double()
    alpha = (lr * torch.sqrt(1 - BETA_2 ** t) / (1 - BETA_1 ** t)).float()
    g = s["grad"]
    if case["clip"] > 0:
        norm = torch.sqrt(g.double().square().sum())
        g = g * (case["clip"] / torch.clamp(norm, min=case["clip"])).float()
    if case["bits"] == 8:
        m, v = _decode(s["m"], s["m_exp"], 15), _decode(s["v"], s["v_exp"], 31)
    else:
        m, v = s["m"], s["v"]
    m = m * BETA_1 + g * (1 - BETA_1)
    v = v * BETA_2 + (g * g) * (1 - BETA_2)
    theta.sub_(theta * (lr.float() * s["decay"]))
    theta.sub_(alpha * m / (torch.sqrt(v) + ADAM_EPS))
    if s["copy"] is not None:
        s["copy"].copy_(theta)
    if case["bits"] == 8:
        low, high = _random_16(theta.numel(), it, theta.device)
        code, exp = _encode(m, low, 15)
        s["m"].copy_(code), s["m_exp"].copy_(exp)
        code, exp = _encode(v, high, 31)
        s["v"].copy_(code), s["v_exp"].copy_(exp)
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    s["count"][0] += 1
    return _adamw_outputs(s, lambda code, exp, out, second: out.copy_(_decode(code, exp, 31 if second else 15)))


# 8-bit moments: blocks of 256 elements with one exponent byte e (255: not finite).  A first moment's code is sign, 4 exponent
# bits and 3 mantissa bits, a second moment's 5 and 3 (no sign); a code's value is the float whose bits are code << 20, times
# 2^(e - top), top = 15 or 31.  e is the exponent of the block's largest magnitude once its mantissa is rounded up to 3 bits.
def _power(k):
    """2^k in 64 bits, k an integer tensor."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _decode(code, exp, top):
    code, exp = code.view(-1, BLOCK).to(torch.int32), exp[:, None].to(torch.int32)
    bits = (code & 0x7F) << 20 if top == 15 else code << 20
    value = (bits.view(torch.float32).double() * _power(exp - top)).float()
    if top == 15:
        value = torch.where(code > 127, -value, value)
    return torch.where(exp == 255, torch.full_like(value, float("nan")), value).view(-1)


def _encode(x, random, top):
    """Codes and exponents of x; ``random``: 16 bits an element, what decides whether a value goes up to the next code."""
    x = x.view(-1, BLOCK)
    size = x.view(torch.int32) & 0x7FFFFFFF
    exp = ((size.amax(1, keepdim=True).to(torch.int64) + 0xFFFFF) >> 23).clamp_(max=255)
    scaled = (x.double() * _power(top - exp)).float().view(torch.int32) & 0x7FFFFFFF
    code = (scaled + ((random.view(-1, BLOCK) if random.dim() else random) << 4)) >> 20
    if top == 15:
        code = code | ((x.view(torch.int32) < 0).to(torch.int32) << 7)
    else:  # a positive second moment never becomes 0
        code = torch.where((x > 0) & (code == 0), torch.ones_like(code), code)
    code = torch.where(exp == 255, torch.zeros_like(code), code)
    return code.to(torch.uint8).view(-1), exp.to(torch.uint8).view(-1)


def _signed(k):
    return k - (1 << 64) if k >> 63 else k


def _mix(x):
    """This package's counter hash of 64 bits, on int64 tensors (whose products wrap)."""
    x = x + _signed(0x9E3779B97F4A7C15)
    x = (x ^ ((x >> 30) & ((1 << 34) - 1))) * _signed(0xBF58476D1CE4E5B9)
    x = (x ^ ((x >> 27) & ((1 << 37) - 1))) * _signed(0x94D049BB133111EB)
    return x ^ ((x >> 31) & ((1 << 33) - 1))


def _random_16(total, it, device):
    """The 16 random bits of the first and of the second moment: one hash for two elements, 32 bits each."""
    h = _mix(torch.arange(total // 2, device=device) ^ _mix(_mix(it) ^ SEED))
    r = torch.stack([h & 0xFFFFFFFF, (h >> 32) & 0xFFFFFFFF], 1).view(-1)
    return (r & 0xFFFF).to(torch.int32), (r >> 16).to(torch.int32)


# ------------------------------------------------------------------------------------------------ from the definitions, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    n, c, groups = case["n"], case["c"], case["groups"]
    if n * case["h"] * case["w"] * c > 150_000_000:
        return None
    x = s["x"].double().reshape(n, -1, groups, c // groups)
    gamma, beta = (s[k].double().reshape(groups, c // groups) for k in ("gamma", "beta"))
    act = s["act"]
    if case["op"] == "norm_fwd":
        var, mean = torch.var_mean(x, dim=(1, 3), unbiased=False, keepdim=True)
        rstd = (var + EPS) ** -0.5
    else:
        mean, rstd = (s[k].double()[:, None, :, None] for k in ("mean", "rstd"))
    xhat = (x - mean) * rstd
    z = xhat * gamma + beta
    neg = torch.clamp(z, max=0)
    if case["op"] == "norm_fwd":
        if act is not None:
            z = {"relu": lambda: z.clamp(min=0), "elu": lambda: z.clamp(min=0) + torch.expm1(neg),
                 "lrelu": lambda: z.clamp(min=0) + s["alpha"] * neg, "tanh": lambda: torch.tanh(z),
                 "sigmoid": lambda: torch.sigmoid(z)}[act]()
        return {"y": z.reshape(s["x"].shape), "mean": mean.reshape(n, groups), "rstd": rstd.reshape(n, groups)}
    dz = s["dy"].double().reshape(x.shape)
    if act is not None:
        up = (z > 0).double()
        dz = dz * {"relu": lambda: up, "elu": lambda: torch.exp(neg), "lrelu": lambda: up + (1 - up) * s["alpha"],
                   "tanh": lambda: torch.cosh(z) ** -2, "sigmoid": lambda: torch.sigmoid(z) * torch.sigmoid(-z)}[act]()
    dgamma, dbeta = (dz * xhat).sum((0, 1)).reshape(-1), dz.sum((0, 1)).reshape(-1)
    dxhat = dz * gamma
    dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True) - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
    return {"dx": dx.reshape(s["x"].shape), "dgamma": dgamma, "dbeta": dbeta}


def _exact_adamw(case, s):
    total = s["theta"].numel()
    if total > 8_000_000:
        return None
    sizes = _sizes(case)
    wd = np.concatenate([np.full(-(-k // BLOCK) * BLOCK, DECAY if k > 1024 else 0.0) for k in sizes])
    it = int(s["count"][0])
    lr = LR * DECAY_RATE ** (it // DECAY_STEPS)
    step = lr * math.sqrt(1 - BETA_2 ** (it + 1)) / (1 - BETA_1 ** (it + 1))
    theta, g = (s[k].cpu().numpy().astype(np.float64) for k in ("theta", "grad"))
    if case["clip"] > 0:
        g = g * (case["clip"] / max(case["clip"], math.sqrt(float(np.sum(g * g)))))
    if case["bits"] == 8:
        m = _exact_values(s["m"].cpu().numpy(), s["m_exp"].cpu().numpy(), 4, True)
        v = _exact_values(s["v"].cpu().numpy(), s["v_exp"].cpu().numpy(), 5, False)
    else:
        m, v = (s[k].cpu().numpy().astype(np.float64) for k in ("m", "v"))
    m, v = BETA_1 * m + (1 - BETA_1) * g, BETA_2 * v + (1 - BETA_2) * g * g
    theta = theta * (1 - lr * wd)
    theta = theta - step * m / (np.sqrt(v) + ADAM_EPS)
    out = {"theta": theta}
    if case["copy"]:
        out["copy"] = theta
    if case["bits"] == 8:
        h = _exact_hash(np.arange(total // 2, dtype=np.uint64) ^ _exact_hash(_exact_hash(it) ^ np.uint64(SEED)))
        r = h.view(np.uint32).astype(np.int64)  # little end first: the even element's 32 bits, then the odd one's
        m, v = _exact_round(m, r % 65536, 4), _exact_round(v, r // 65536, 5)
    out["m"], out["v"] = m, v
    return {k: torch.from_numpy(np.ascontiguousarray(a)) for k, a in out.items()}


def _exact_hash(x):
    x = np.atleast_1d(np.asarray(x, dtype=np.uint64)) + np.uint64(0x9E3779B97F4A7C15)
    x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return x ^ (x >> np.uint64(31))


def _exact_values(code, exp, width, signed):
    """What codes of ``width`` exponent bits and 3 mantissa bits stand for."""
    code = code.astype(np.int64).reshape(-1, BLOCK)
    field, low = (code >> 3) & ((1 << width) - 1), code & 7
    size = np.where(field == 0, low * 2.0 ** -129, (8 + low) * 2.0 ** (field - 130.0))
    size = size * 2.0 ** (exp.astype(np.float64)[:, None] - ((1 << width) - 1))
    return np.where((code > 127) & signed, -size, size).reshape(-1)


def _exact_round(x, r, width):
    """x on the grid of its block: down, or up where the distance to the code below and r / 65536 make one step."""
    x = x.reshape(-1, BLOCK)
    big = np.abs(x).max(1, keepdims=True)
    frac, e = np.frexp(big)  # big = frac * 2^e, frac in [0.5, 1)
    e = np.where(np.ceil(frac * 16) == 16, e + 1, e)  # the exponent once the mantissa is rounded up to 3 bits
    lowest = e - (1 << width) + 2  # exponent of the smallest normal code
    own_e = np.maximum(np.frexp(np.abs(x))[1], lowest)
    step = 2.0 ** (own_e - 4)
    k = np.floor(np.abs(x) / step + r.reshape(x.shape) / 65536.0)
    if width == 5:
        k = np.where((x > 0) & (k == 0), 1, k)
    return (np.sign(x) * k * step).reshape(-1)
