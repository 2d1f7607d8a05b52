"""Cases of the position-wise operators (``gwn_amd.layers``): the product with its epilogue, layer
norm, and dropout without a stored mask, forward and backward, over the sizes that the framework's
own workloads and generic wide layers give them.

``listed`` names the cases, ``draw`` gives further ones of the same ranges, ``prepare`` makes a
case's inputs, ``run`` is one pass -- in elementary torch operations, or with ``own`` set through
the framework's operators -- ``work`` is what a pass cannot do without, and ``exact`` is the
definition in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
EPS = 1e-5
SALT = 5  # one operator's place among a step's masks

MOST_PRODUCT = 20800 * 2048 * 8192  # rows * k * n of the largest listed product
MOST_VALUES = 20800 * 4096          # rows * channels of the largest listed norm and dropout
MOST_BYTES = 1100 * 10 ** 6         # read and written by one pass of the largest listed cases


def linear(name, m, k, n, type, act, train, bias=True, residual=False, p=0.0, pad=0):
    """``pad``: the rows of x lie that many values further apart than they are long."""
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "type": type, "act": act, "train": train,
            "bias": bias, "residual": residual, "p": p, "pad": pad}


def norm(name, m, c, type, train, wide_weights=False, pad=0):
    """``wide_weights``: the weights stay in 32 bits beside 16-bit activations."""
    return {"name": name, "op": "norm", "m": m, "c": c, "type": type, "train": train, "wide_weights": wide_weights,
            "pad": pad}


def drop(name, m, c, type, p, residual, train):
    return {"name": name, "op": "dropout", "m": m, "c": c, "type": type, "p": p, "residual": residual, "train": train}


def listed():
    return [
        # one row through a wide layer while serving: all latency and weight reading
        linear("linear_one_row_bf16", 1, 1024, 4096, "bf16", "silu", False),
        # the twelve steps of one forecast, sizes that no tile divides
        linear("linear_few_rows_f16", 12, 1999, 1030, "f16", "gelu", False, residual=True),
        # the output head's first product: 64 samples x 207 sensors, 256 -> 512 channels
        linear("linear_head_f32", 13248, 256, 512, "f32", "relu", True),
        # the graph convolution's product: 64 x 207 sensors x 12 steps, 7 pieces of 32 channels -> 32
        linear("linear_mix_f32", 158976, 224, 32, "f32", "none", True, residual=True, p=0.3),
        # a wide feed-forward layer over 64 samples x 325 sensors
        linear("linear_wide_bf16", 20800, 2048, 8192, "bf16", "gelu", True),
        # odd sizes and rows apart, everything in the epilogue
        linear("linear_ragged_f16", 6501, 1000, 1537, "f16", "gelu_tanh", True, residual=True, p=0.1, pad=24),
        # the norm of one forecast's steps while serving
        norm("norm_few_rows_bf16", 12, 512, "bf16", False),
        # the residual channels of 64 x 207 sensors x 13 steps
        norm("norm_channels_f32", 172224, 32, "f32", True),
        # a wide layer's rows, weights in 32 bits
        norm("norm_wide_bf16", 20800, 4096, "bf16", True, wide_weights=True),
        # an odd width: no row but the first starts on a 16-byte border
        norm("norm_odd_f16", 13247, 1111, "f16", True),
        # the graph convolution's dropout: 64 x 207 sensors x 12 steps x 32 channels
        drop("dropout_channels_f32", 158976, 32, "f32", 0.3, False, True),
        # a wide layer's dropout into its residual
        drop("dropout_wide_bf16", 20800, 4096, "bf16", 0.1, True, True),
    ]


def between(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi; every other one as it falls, else to a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 16:
        v -= v % 8
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("linear", "linear", "norm", "dropout"))
    type = rng.choice(("f32", "f16", "bf16"))
    train = rng.random() < 0.7
    if op == "linear":
        k, n = between(rng, 8, 4096), between(rng, 8, 8192)
        m = between(rng, 1, max(1, min(200000, MOST_PRODUCT // (k * n), 20800 * 8192 // max(k, n))))
        c = linear("", m, k, n, type, rng.choice(ACTS), train, bias=rng.random() < 0.8, residual=rng.random() < 0.4,
                   p=rng.choice((0.0, 0.0, 0.1, 0.3)), pad=rng.choice((0, 0, 3, 8)))
    elif op == "norm":
        width = between(rng, 8, 16384)
        c = norm("", between(rng, 1, max(1, min(200000, MOST_VALUES // width))), width, type, train,
                 wide_weights=rng.random() < 0.3, pad=rng.choice((0, 0, 5, 16)))
    else:
        width = between(rng, 8, 16384)
        c = drop("", between(rng, 1, max(1, min(200000, MOST_VALUES // width))), width, type, rng.choice((0.1, 0.3, 0.5)),
                 rng.random() < 0.5, train)
    del c["name"]
    while c["m"] > 1 and work(c)["bytes"] > MOST_BYTES:
        c["m"] -= c["m"] // 3
    return c


def on_grid(t, step):
    """The values of ``t`` to the next multiple of ``step``, laid out as they were."""
    return t.copy_((t.float() / step).round() * step)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, type=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(type)

    s = {"case": case}
    m, train = case["m"], case["train"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        s["x"] = normal(m, k + case["pad"])[:, :k]
        s["w"] = normal(n, k, scale=k ** -0.5)
        s["b"] = normal(n, scale=0.3) if case["bias"] else None
        if case["act"] == "relu":
            # On grids of whole powers of two every sum of products is exact in 32 bits, in any order:
            # a sum next to zero then lies on the same side of relu's border however it is added up.
            step = 2.0 ** (-6 - math.ceil(math.log2(k) / 2))
            s["x"] = on_grid(s["x"], 2.0 ** -6)
            s["w"] = on_grid(s["w"], step)
            s["b"] = on_grid(s["b"], step * 2.0 ** -6 * 32) if case["bias"] else None
        s["r"] = normal(m, n) if case["residual"] else None
        s["dy"] = normal(m, n) if train else None
    elif case["op"] == "norm":
        c = case["c"]
        wt = torch.float32 if case["wide_weights"] else dt
        # activations with a mean and a spread of their own in every row
        centre = torch.randn(m, 1, generator=gen, device="cuda")
        spread = torch.rand(m, 1, generator=gen, device="cuda") + 0.5
        s["x"] = (torch.randn(m, c + case["pad"], generator=gen, device="cuda") * spread + centre).to(dt)[:, :c]
        s["w"] = normal(c, scale=0.2, shift=1.0, type=wt)
        s["b"] = normal(c, scale=0.2, type=wt)
        s["dy"] = normal(m, c) if train else None
    else:
        c = case["c"]
        s["x"] = normal(m, c)
        s["r"] = normal(m, c) if case["residual"] else None
        s["dy"] = normal(m, c) if train else None
    # the step's counter of random masks, as a training program keeps it on the device
    s["count"] = torch.randint(0, 2 ** 62, (1,), generator=gen, device="cuda", dtype=torch.int64)
    s["leaves"] = [s[q] for q in ("x", "w", "b", "r") if s.get(q) is not None]
    if train:
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


def run(state):
    return run_own(state) if own else run_plain(state)


# ---- the framework's operators -----------------------------------------------------------------

def framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "graph-wavenet_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from gwn_amd import layers
    return layers


def run_own(s):
    layers = framework()
    case = s["case"]
    if case["op"] == "linear":
        y = layers.linear_act(s["x"], s["w"], s["b"], act=case["act"], residual=s["r"], p=case["p"], seed=s["count"],
                              salt=SALT)
    elif case["op"] == "norm":
        y = layers.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
    else:
        y = layers.dropout(s["x"], case["p"], s["count"], salt=SALT, residual=s["r"])
    out = {"y": y.detach()}
    if case["train"]:
        names = [q for q in ("x", "w", "b", "r") if s.get(q) is not None]
        out.update(zip(("d" + q for q in names), torch.autograd.grad(y, s["leaves"], s["dy"])))
    return out


# ---- the plain forms ---------------------------------------------------------------------------

LOW = 0xFFFFFFFF


def signed(v):
    """A 64-bit constant as the signed number torch holds it by."""
    return v - (1 << 64) if v >= 1 << 63 else v


def shift_right(v, by):
    """Logical right shift of 64-bit values held as signed ones."""
    return (v >> by) & ((1 << (64 - by)) - 1)


def mix64(v):
    """The finaliser of the SplitMix64 generator (Steele, Lea and Flood 2014), on int64 tensors."""
    v = (v ^ shift_right(v, 30)) * signed(0xBF58476D1CE4E5B9)
    v = (v ^ shift_right(v, 27)) * signed(0x94D049BB133111EB)
    return v ^ shift_right(v, 31)


def kept(count, total, p, device):
    """Which of ``total`` consecutive elements the mask of (count, SALT) keeps."""
    i = torch.arange(total, device=device, dtype=torch.int64)
    key = mix64(mix64(count + signed(0x9E3779B97F4A7C15 * (SALT + 1) % (1 << 64))) + (i >> 32))
    h = ((i & LOW) * 0x9E3779B1 + key) & LOW
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & LOW
    h = ((h ^ (h >> 15)) + shift_right(key, 32)) & LOW
    h = (h * 0x846CA68B) & LOW
    h = h ^ (h >> 16)
    return (h >> 8) >= math.ceil(p * (1 << 24))


def masked(v, keep, p):
    return torch.where(keep, v * (1.0 / (1.0 - p)), torch.zeros((), device=v.device))


def act_plain(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).float()
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        a = (2 / math.pi) ** 0.5
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    sig = 1 / (1 + torch.exp(-z))
    return z * sig, sig * (1 + z * (1 - sig))


@torch.no_grad()
def run_plain(s):
    case = s["case"]
    dt = TYPES[case["type"]]
    x = s["x"].float()
    out = {}
    if case["op"] == "linear":
        w, p = s["w"].float(), case["p"]
        z = x @ w.t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y, slope = act_plain(z, case["act"])
        keep = kept(s["count"], y.numel(), p, y.device).view(y.shape) if p > 0 else None
        if keep is not None:
            y = masked(y, keep, p)
        if s["r"] is not None:
            y = y + s["r"].float()
        out["y"] = y.to(dt)
        if case["train"]:
            dz = s["dy"].float()
            if keep is not None:
                dz = masked(dz, keep, p)
            dz = dz * slope
            out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
            if s["b"] is not None:
                out["db"] = dz.sum(0).to(dt)
            if s["r"] is not None:
                out["dr"] = s["dy"]
    elif case["op"] == "norm":
        w, b = s["w"].float(), s["b"].float()
        d = x - x.mean(-1, keepdim=True)
        rs = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
        xh = d * rs
        out["y"] = (xh * w + b).to(dt)
        if case["train"]:
            dy = s["dy"].float()
            h = dy * w
            out["dx"] = (rs * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True))).to(dt)
            out["dw"] = (dy * xh).sum(0).to(s["w"].dtype)
            out["db"] = dy.sum(0).to(s["b"].dtype)
    else:
        p = case["p"]
        keep = kept(s["count"], x.numel(), p, x.device).view(x.shape)
        y = masked(x, keep, p)
        if s["r"] is not None:
            y = y + s["r"].float()
        out["y"] = y.to(dt)
        if case["train"]:
            out["dx"] = masked(s["dy"].float(), keep, p).to(dt)
            if s["r"] is not None:
                out["dr"] = s["dy"]
    return out


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    e, m = BYTES[case["type"]], case["m"]
    train = case["train"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        small = n if case["bias"] else 0
        res = m * n if case["residual"] else 0
        values = m * k + n * k + small + res + m * n
        flops = 2 * m * k * n
        if train:  # reads dy, which is the residual's gradient too; writes dx, dw, db
            values += m * n + m * k + n * k + small
            flops *= 3
        return {"bytes": values * e, "flops": flops}
    c = case["c"]
    if case["op"] == "norm":
        we = 4 if case["wide_weights"] else e
        return {"bytes": (m * c * (4 if train else 2)) * e + c * we * (4 if train else 2),
                "flops": m * c * (20 if train else 8)}
    values = m * c * ((3 if case["residual"] else 2) + (2 if train else 0))
    return {"bytes": values * e, "flops": m * c * (24 if train else 12)}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def kept_exact(count, shape, p):
    """The mask from the generator's definition, on whole numbers of the widths it is defined in."""
    total = int(np.prod(shape))
    full = (1 << 64) - 1

    def mix(v):
        v = ((v ^ (v >> 30)) * 0xBF58476D1CE4E5B9) & full
        v = ((v ^ (v >> 27)) * 0x94D049BB133111EB) & full
        return v ^ (v >> 31)

    base = mix((int(count) + 0x9E3779B97F4A7C15 * (SALT + 1)) & full)
    parts = []
    for high in range((total - 1 >> 32) + 1):
        key = mix((base + high) & full)
        h = np.arange(min(total - (high << 32), 1 << 32), dtype=np.uint32)
        h *= np.uint32(0x9E3779B1)
        h += np.uint32(key & 0xFFFFFFFF)
        h ^= h >> np.uint32(16)
        h *= np.uint32(0x7FEB352D)
        h ^= h >> np.uint32(15)
        h += np.uint32(key >> 32)
        h *= np.uint32(0x846CA68B)
        h ^= h >> np.uint32(16)
        parts.append((h >> np.uint32(8)) >= math.ceil(p * 2 ** 24))
    return torch.from_numpy(np.concatenate(parts).reshape(shape)).to("cuda")


def act_exact(z, act):
    """The activation's value; its slope follows from differentiating this in 64 bits."""
    if act == "relu":
        return z * (z.detach() > 0)  # slope 0 on the border itself
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.special.expit(z)
    return z * 1.0


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    leaves = [q for q in ("x", "w", "b", "r") if s.get(q) is not None]
    v = {q: s[q].detach().to(f64).requires_grad_(case["train"]) for q in leaves}
    if case["op"] == "norm":
        var, mean = torch.var_mean(v["x"], dim=-1, correction=0, keepdim=True)
        y = (v["x"] - mean) * torch.rsqrt(var + EPS) * v["w"] + v["b"]
    else:
        y = v["x"]
        if case["op"] == "linear":
            y = act_exact(torch.nn.functional.linear(v["x"], v["w"], v.get("b")), case["act"])
        if case["p"] > 0:
            y = y * (kept_exact(s["count"].item(), tuple(y.shape), case["p"]).to(f64) / (1 - case["p"]))
        if "r" in v:
            y = y + v["r"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [v[q] for q in leaves], s["dy"].to(f64))
        out.update(zip(("d" + q for q in leaves), grads))
    return out
