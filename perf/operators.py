"""The operators of pointwise training blocks on voxel rows, as cases whose speed is measured.

A case is a dict of plain values.  Its "kind" names the operator:

  norm   group norm with an activation over rows [N, C] grouped by cloud (channels last)
  gated  both projections of a gated feed-forward block, the activation and the product
  adamw  an AdamW step over many tensors, moments in 32 bits or in 8

"mode": "forward", or "train" for the forward and the backward pass.
"""
import math
import os
import sys

import torch

sys.path.insert(1, os.path.join(os.getcwd(), "ss-conv_amd"))

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5                                                                # of the norm
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 10  # of the step
BLOCK = 256                       # elements of an 8-bit moment that share a scale


# ---- the cases ----------------------------------------------------------------------------
def _norm(rows, clouds, channels, groups, dtype, act, mode, name=None):
    case = dict(kind="norm", rows=rows, clouds=clouds, channels=channels, groups=groups,
                dtype=dtype, act=act, mode=mode)
    return case if name is None else dict(case, name=name)


def _gated(rows, width, hidden, dtype, act, bias, mode, name=None):
    case = dict(kind="gated", rows=rows, width=width, hidden=hidden, dtype=dtype, act=act,
                bias=bias, mode=mode)
    return case if name is None else dict(case, name=name)


def _adamw(tensors, elements, dtype, bits, name=None):
    case = dict(kind="adamw", tensors=tensors, elements=elements, dtype=dtype, bits=bits)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # two small clouds of a 32-channel layer, inference: launches and the host count
        _norm(2100, 2, 32, 8, "f32", "relu", "forward", "norm small"),
        # the output rows of the 64 -> 128 channel benchmark layer, as a training step has them
        _norm(600153, 32, 128, 16, "f32", "silu", "train", "norm train"),
        # clouds of different sizes, 200 channels in groups of 8, half precision
        _norm(50001, 7, 200, 25, "f16", "relu", "train", "norm ragged half"),
        # wide rows of few clouds, inference in bfloat16
        _norm(100000, 8, 512, 32, "bf16", "silu", "forward", "norm wide bf16"),
        # one row at a time, as a model that answers step by step calls the block
        _gated(1, 4096, 8192, "bf16", "silu", False, "forward", "gated one row"),
        # a few rows, odd widths, with biases
        _gated(24, 1000, 2728, "f16", "gelu", True, "forward", "gated few rows"),
        # a long input, inference
        _gated(4096, 2048, 8192, "bf16", "silu", False, "forward", "gated forward"),
        # a training step on many rows: forward, every gradient
        _gated(16384, 2048, 8192, "bf16", "silu", False, "train", "gated train"),
        # the voxel rows of the benchmark batch through a block of 128 channels, float32
        _gated(57304, 128, 512, "f32", "silu", True, "train", "gated train f32"),
        # the parameters of a small network: many tensors, most of them vectors
        _adamw(120, 3100000, "f32", 32, "adamw many"),
        # a large model's parameters in bfloat16, moments in 32 bits
        _adamw(40, 120000000, "bf16", 32, "adamw large"),
        # the same number of float32 parameters with moments in 8 bits
        _adamw(40, 120000000, "f32", 8, "adamw 8 bit"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "gated", "adamw"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    act = rng.choice(["relu", "silu", "gelu"])
    mode = rng.choice(["forward", "train"])
    if kind == "norm":
        while True:
            per = rng.choice([1, 2, 3, 4, 7, 8, 16, 32])
            groups = _log(rng, 1, 64)
            channels = per * groups
            rows = _log(rng, 100, 600000)
            if 8 <= channels <= 512 and rows * channels <= 600153 * 128:
                return _norm(rows, _log(rng, 1, 64), channels, groups, dtype, act, mode)
    if kind == "gated":
        while True:
            rows = _log(rng, 1, 60000)
            odd = rng.random() < 0.3
            width = _log(rng, 64, 4096) if odd else 8 * _log(rng, 8, 512)
            hidden = _log(rng, 64, 8192) if odd else 8 * _log(rng, 8, 1024)
            # (float32 rows cost several times the matrix work)
            most = 16384 * 2048 * 8192 // (8 if dtype == "f32" else 1)
            if rows * width * hidden <= most:
                return _gated(rows, width, hidden, dtype, act, rng.random() < 0.5, mode)
    return _adamw(_log(rng, 1, 200), _log(rng, 20000, 120000000), dtype, rng.choice([8, 32]))


# ---- sizes that follow from a case --------------------------------------------------------
def _lengths(case):
    """Rows of every cloud: unequal, the third of four or more has none."""
    n, b = case["rows"], case["clouds"]
    weights = [0 if (b >= 4 and i == 2) else 2 + (i * 7) % 5 for i in range(b)]
    total = sum(weights)
    got = [n * w // total for w in weights]
    got[-1] += n - sum(got)
    return got


def _shapes(case):
    """Sizes of the tensors: two in three are vectors of a layer, the rest share the elements."""
    t = case["tensors"]
    small = [16 + (i * 37) % 497 for i in range(t) if i % 3 != 0]
    big = [i for i in range(t) if i % 3 == 0]
    left = max(case["elements"] - sum(small), 64 * len(big))
    weights = [1 + (k * 5) % 7 for k in range(len(big))]
    sizes, at = [], 0
    for i in range(t):
        if i % 3 == 0:
            k = i // 3
            sizes.append(max(1, left * weights[k] // sum(weights)))
        else:
            sizes.append(small[at])
            at += 1
    return sizes


# ---- inputs -------------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return x.mul_(scale).add_(shift).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]] if "dtype" in case else None
    s = {"case": case}
    if case["kind"] == "norm":
        n, c = case["rows"], case["channels"]
        ends = [0]
        for length in _lengths(case):
            ends.append(ends[-1] + length)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["longest"] = max(_lengths(case))
        # what a convolution puts out: every channel with a mean and a spread of its own
        x = _normal(g, n, c)
        x.mul_(_normal(g, c).exp_()).add_(_normal(g, c))
        s["x"] = x.to(dtype)
        s["weight"] = _normal(g, c, scale=0.2, shift=1.0)
        s["bias"] = _normal(g, c, scale=0.2)
        if case["mode"] == "train":
            s["dy"] = _normal(g, n, c, dtype=dtype)
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_()
    elif case["kind"] == "gated":
        m, k, h = case["rows"], case["width"], case["hidden"]
        s["x"] = _normal(g, m, k, dtype=dtype)
        s["w_gate"] = _normal(g, h, k, scale=k ** -0.5, dtype=dtype)
        s["w_up"] = _normal(g, h, k, scale=k ** -0.5, dtype=dtype)
        s["b_gate"] = _normal(g, h, scale=0.1, dtype=dtype) if case["bias"] else None
        s["b_up"] = _normal(g, h, scale=0.1, dtype=dtype) if case["bias"] else None
        if case["mode"] == "train":
            s["dy"] = _normal(g, m, h, dtype=dtype)
            for key in ("x", "w_gate", "w_up", "b_gate", "b_up"):
                if s[key] is not None:
                    s[key].requires_grad_()
    else:
        sizes = _shapes(case)
        starts, at = [], 0
        for n in sizes:  # tensors begin at multiples of 256 elements of one storage
            starts.append(at)
            at += -(-n // BLOCK) * BLOCK
        # what lies between the tensors belongs to none of them
        inside = torch.zeros(at, device="cuda")
        cut = lambda flat: [flat[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731
        for v in cut(inside):
            v.fill_(1.0)
        s["flat"] = _normal(g, at, scale=0.05).mul_(inside).to(dtype)
        # gradients of layers differ by orders of magnitude
        spread = _normal(g, at // BLOCK, 1).exp_().expand(-1, BLOCK).reshape(-1)
        grads = _normal(g, at, scale=1e-2).mul_(spread).mul_(inside)
        m = _normal(g, at, scale=3e-3).mul_(spread).mul_(inside)
        v = _normal(g, at, scale=1e-2).mul_(spread).square_().add_(1e-12).mul_(inside)
        s["grad_flat"] = grads.to(dtype)
        s["params"], s["grads"] = cut(s["flat"]), cut(s["grad_flat"])
        if case["bits"] == 8:
            s["m_flat"], s["m_scale_flat"] = _encode_m(m)
            s["v_flat"], s["v_scale_flat"] = _encode_v(v)
            for key in ("m", "v"):
                s[key] = cut(s[key + "_flat"])
                s[key + "_scale"] = [s[key + "_scale_flat"][a // BLOCK:a // BLOCK + -(-n // BLOCK)]
                                     for a, n in zip(starts, sizes)]
                s[key + "_value_flat"] = torch.zeros(at, device="cuda")
                s[key + "_value"] = cut(s[key + "_value_flat"])
        else:
            s["m_flat"], s["v_flat"] = m, v
            s["m"], s["v"] = cut(m), cut(v)
    return s


# ---- plain forms --------------------------------------------------------------------------
def _act(kind, z):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _slope(kind, z):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + \
        z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _norm_plain(s):
    c = s["case"]
    with torch.no_grad():
        x = s["x"].float()
        n, groups = x.size(0), c["groups"]
        per = x.size(1) // groups
        first = s["offsets"][:-1].long()
        length = s["offsets"].diff().long()
        # clouds side by side, padded to the longest one
        at = torch.arange(s["longest"], device=x.device)
        there = (at < length[:, None])[:, :, None]
        rows = (first[:, None] + at).clamp(max=n - 1)
        cloud = torch.repeat_interleave(length, output_size=n)

        def sums(v):  # [rows, k] -> [clouds, k]
            return (v[rows] * there).sum(1)

        count = (length * per).clamp(min=1)[:, None].float()
        mean = sums(x.view(n, groups, per).sum(2)) / count
        xc = x.view(n, groups, per) - mean[cloud][:, :, None]
        rstd = 1 / torch.sqrt(sums((xc * xc).sum(2)) / count + EPS)
        xhat = (xc * rstd[cloud][:, :, None]).view(n, -1)
        w, b = s["weight"].float(), s["bias"].float()
        z = xhat * w + b
        out = {"y": _act(c["act"], z).to(s["x"].dtype)}
        if c["mode"] == "train":
            dz = s["dy"].float() * _slope(c["act"], z)
            out["dbias"] = dz.sum(0).to(s["bias"].dtype)
            out["dweight"] = (dz * xhat).sum(0).to(s["weight"].dtype)
            gz = (dz * w).view(n, groups, per)
            s1 = sums(gz.sum(2)) / count
            s2 = sums((gz * xhat.view(n, groups, per)).sum(2)) / count
            dx = gz - s1[cloud][:, :, None] - xhat.view(n, groups, per) * s2[cloud][:, :, None]
            out["dx"] = (dx * rstd[cloud][:, :, None]).view(n, -1).to(s["x"].dtype)
        return out


def _gated_plain(s):
    c = s["case"]
    with torch.no_grad():
        x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
        a, b = x @ wg.t(), x @ wu.t()
        if c["bias"]:
            a, b = a + s["b_gate"].float(), b + s["b_up"].float()
        f = _act(c["act"], a)
        dtype = s["x"].dtype
        out = {"y": (f * b).to(dtype)}
        if c["mode"] == "train":
            dy = s["dy"].float()
            da, db = dy * b * _slope(c["act"], a), dy * f
            out["dx"] = (da @ wg + db @ wu).to(dtype)
            out["dw_gate"], out["dw_up"] = (da.t() @ x).to(dtype), (db.t() @ x).to(dtype)
            if c["bias"]:
                out["db_gate"], out["db_up"] = da.sum(0).to(dtype), db.sum(0).to(dtype)
        return out


def _scale(top, steps):
    """Scales of blocks whose largest magnitudes are `top`; NaN where one is no finite number."""
    q = (top * (1.0 / (steps * steps))).clamp(min=2.0 ** -126)
    return torch.where(torch.isfinite(top), q, torch.full_like(q, math.nan))


def _codes(x, q):
    """floor(sqrt(x / q) + 1/2) of non-negative x in blocks with the scales q, 0 where q is NaN."""
    return torch.nan_to_num(torch.floor(torch.sqrt(x / q[:, None]) + 0.5), nan=0.0)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _encode_m(m):
    """Codes and scales of first moments: m = q c |c|, c in -127 .. 127."""
    x = _blocks(m)
    q = _scale(x.abs().amax(1), 127)
    c = torch.copysign(_codes(x.abs(), q).clamp(max=127), x)
    return c.view(-1)[:m.numel()].to(torch.int8), q


def _encode_v(v):
    """Codes and scales of second moments: sqrt(v) = q c^2, c in 0 .. 255, at least 1 where v > 0."""
    x = torch.sqrt(_blocks(v))
    q = _scale(x.amax(1), 255)
    c = torch.maximum(_codes(x, q).clamp(max=255), (x > 0).to(x.dtype))
    c = torch.where(torch.isnan(q)[:, None], torch.zeros_like(c), c)
    return c.view(-1)[:v.numel()].to(torch.uint8), q


def _decode_m(c, q):
    x = c.float()
    return (_blocks(x * x.abs()) * q[:, None]).view(-1)[:c.numel()]


def _decode_v(c, q):
    x = c.float()
    u = (_blocks(x * x) * q[:, None]).view(-1)[:c.numel()]
    return u * u


def _adamw_plain(s):
    with torch.no_grad():
        many = torch._foreach_mul
        p, g = [t.float() for t in s["params"]], [t.float() for t in s["grads"]]
        if s["case"]["bits"] == 8:
            m = [_decode_m(c, q) for c, q in zip(s["m"], s["m_scale"])]
            v = [_decode_v(c, q) for c, q in zip(s["v"], s["v_scale"])]
        else:
            m, v = s["m"], s["v"]
        m = torch._foreach_add(many(m, BETA1), many(g, 1 - BETA1))
        v = torch._foreach_add(many(v, BETA2), many(many(g, g), 1 - BETA2))
        below = torch._foreach_add(many(torch._foreach_sqrt(v), (1 - BETA2 ** STEP) ** -0.5),
                                   ADAM_EPS)
        step = many(torch._foreach_div(m, below), LR / (1 - BETA1 ** STEP))
        p = torch._foreach_sub(many(p, 1 - LR * DECAY), step)
        torch._foreach_copy_(s["params"], p)
        if s["case"]["bits"] == 8:
            em, ev = [_encode_m(t) for t in m], [_encode_v(t) for t in v]
            for key, e in (("m", em), ("v", ev)):
                torch._foreach_copy_(s[key], [c for c, q in e])
                torch._foreach_copy_(s[key + "_scale"], [q for c, q in e])
            torch._foreach_copy_(s["m_value"], [_decode_m(c, q) for c, q in em])
            torch._foreach_copy_(s["v_value"], [_decode_v(c, q) for c, q in ev])
        else:
            torch._foreach_copy_(s["m"], m)
            torch._foreach_copy_(s["v"], v)


# ---- the framework's operators ------------------------------------------------------------
def _norm_own(s):
    from ss_conv.groupnorm import group_norm
    c = s["case"]
    y = group_norm(s["x"], s["offsets"], c["groups"], s["weight"], s["bias"], EPS, c["act"])
    if c["mode"] != "train":
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _gated_own(s):
    from ss_conv.feedforward import gated_linear
    c = s["case"]
    y = gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], c["act"])
    if c["mode"] != "train":
        return {"y": y}
    keys = ["x", "w_gate", "w_up"] + (["b_gate", "b_up"] if c["bias"] else [])
    grads = torch.autograd.grad(y, [s[k] for k in keys], s["dy"])
    return dict({"y": y.detach()}, **{"d" + k: g for k, g in zip(keys, grads)})


def _adamw_own(s):
    from ss_conv.optim import adamw_, state_values
    more = {}
    if s["case"]["bits"] == 8:
        more = dict(exp_avg_scales=s["m_scale"], exp_avg_sq_scales=s["v_scale"])
    adamw_(s["params"], s["grads"], s["m"], s["v"], STEP, lr=LR, betas=(BETA1, BETA2),
           eps=ADAM_EPS, weight_decay=DECAY, **more)
    if s["case"]["bits"] == 8:
        state_values(s["m"], s["v"], s["m_scale"], s["v_scale"], out=(s["m_value"], s["v_value"]))


def run(state):
    kind = state["case"]["kind"]
    if kind == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    if kind == "gated":
        return _gated_own(state) if own else _gated_plain(state)
    _adamw_own(state) if own else _adamw_plain(state)
    if state["case"]["bits"] == 8:
        return {"p": state["flat"], "m": state["m_value_flat"], "v": state["v_value_flat"]}
    return {"p": state["flat"], "m": state["m_flat"], "v": state["v_flat"]}


def work(case):
    if case["kind"] == "norm":
        values = case["rows"] * case["channels"]
        train = case["mode"] == "train"  # the backward pass reads the rows once more
        return {"bytes": values * BYTES[case["dtype"]] * (5 if train else 2),
                "flops": values * (30 if train else 12)}
    if case["kind"] == "gated":
        m, k, h, e = case["rows"], case["width"], case["hidden"], BYTES[case["dtype"]]
        once = (m * k + 2 * h * k + m * h) * e
        train = case["mode"] == "train"
        return {"bytes": once * (2 if train else 1) + (m * h * e if train else 0),
                "flops": 4.0 * m * k * h * (3 if train else 1)}
    n, e = sum(_shapes(case)), BYTES[case["dtype"]]
    # parameter in and out, gradient in, two moments in and out; 8-bit moments are read once
    # more and come back as the numbers they stand for
    return {"bytes": n * (3 * e + (16 if case["bits"] == 32 else 4 + 2 + 8)), "flops": n * 15}


# ---- the definitions in 64 bits -----------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    torch_act = {"relu": torch.relu, "silu": torch.nn.functional.silu,
                 "gelu": torch.nn.functional.gelu}
    if case["kind"] == "norm":
        train = case["mode"] == "train"
        w = s["weight"].detach().double().requires_grad_(train)
        b = s["bias"].detach().double().requires_grad_(train)
        ys, dxs, dw, db, at = [], [], 0, 0, 0
        for length in _lengths(case):  # cloud by cloud
            if length == 0:
                continue
            x = s["x"].detach()[at:at + length].double().requires_grad_(train)
            v = x.view(length, case["groups"], -1).transpose(0, 1).reshape(case["groups"], -1)
            var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
            v = (v - mean) * (var + EPS).rsqrt()
            v = v.view(case["groups"], length, -1).transpose(0, 1).reshape(length, -1)
            y = torch_act[case["act"]](v * w + b)
            if train:
                got = torch.autograd.grad(y, (x, w, b), s["dy"][at:at + length].double())
                dxs.append(got[0])
                dw, db = dw + got[1], db + got[2]
            ys.append(y.detach())
            at += length
        out = {"y": torch.cat(ys)}
        return dict(out, dx=torch.cat(dxs), dweight=dw, dbias=db) if train else out
    if case["kind"] == "gated":
        train = case["mode"] == "train"
        keys = ["x", "w_gate", "w_up"] + (["b_gate", "b_up"] if case["bias"] else [])
        t = {k: s[k].detach().double().requires_grad_(train) for k in keys}
        gate = torch.nn.functional.linear(t["x"], t["w_gate"], t.get("b_gate"))
        up = torch.nn.functional.linear(t["x"], t["w_up"], t.get("b_up"))
        y = torch_act[case["act"]](gate) * up
        if not train:
            return {"y": y}
        got = torch.autograd.grad(y, [t[k] for k in keys], s["dy"].double())
        return dict({"y": y.detach()}, **{"d" + k: v for k, v in zip(keys, got)})
    out = {k: s[v].double() for k, v in (("p", "flat"), ("m", "m_flat"), ("v", "v_flat"))}
    if case["bits"] == 8:
        c = out["m"]
        out["m"] = c.sign() * c.square() * s["m_scale_flat"].double().repeat_interleave(BLOCK)
        out["v"] = (out["v"].square() * s["v_scale_flat"].double().repeat_interleave(BLOCK)).square()
    g = s["grad_flat"].double()
    out["m"].lerp_(g, 1 - BETA1)
    out["v"].mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    mhat, vhat = out["m"] / (1 - BETA1 ** STEP), out["v"] / (1 - BETA2 ** STEP)
    out["p"] -= LR * (mhat / (vhat.sqrt() + ADAM_EPS) + DECAY * out["p"])
    if case["bits"] == 8:
        m = out["m"].view(-1, BLOCK)
        q = m.abs().amax(1, keepdim=True).clamp(min=1e-36) / 127 ** 2
        out["m"] = (m.sign() * (m.abs() / q).sqrt().round().square() * q).view(-1)
        u = out["v"].view(-1, BLOCK).sqrt()
        q = u.amax(1, keepdim=True).clamp(min=1e-36) / 255 ** 2
        c = torch.where(u > 0, (u / q).sqrt().round().clamp(min=1), torch.zeros_like(u))
        out["v"] = (c.square() * q).square().view(-1)
    return out
