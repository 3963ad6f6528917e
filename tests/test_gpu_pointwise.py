"""The operators of pointwise training blocks (group norm with an activation, gated feed-forward,
AdamW) against their definitions in 64 bits.

Bounds, from the arithmetic that the library states (every result rounded once to its type, sums
and statistics in float32 or more):

  u     half a unit in the last place of the result's type, relative
  g(n)  error of a float32 sum of n products relative to the sum of their magnitudes: every
        addition and every product is off by at most 2^-24, and matrix instructions may cut
        instead of rounding, so 2 (n + 8) 2^-24
  an activation and its slope: exponentials of z are off by (|z| + 4) 2^-23, so is what follows

A 16-bit gradient passes through one more rounding of da and db, at most u of the value; the bounds
below add up the errors element by element and leave as much again for what the backward pass
reads.
"""
import math

import numpy as np
import pytest
import torch

from ss_conv import _ext
from ss_conv.feedforward import GatedFeedForward, GatedLinear, gated_linear
from ss_conv.groupnorm import GroupNorm, group_norm
from ss_conv.optim import BLOCK, AdamW, adamw_, state_values
from ss_conv.sp_ops.tensor import SparseTensor

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "sigmoid", "tanh", "silu", "gelu"]


def act64(kind, z):
    return {None: lambda v: v, "relu": torch.relu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
            "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[kind](z)


def slope64(kind, z):
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(kind, z).sum(), z)[0]


def gamma(n):
    return 2.0 * (n + 8) * 2.0 ** -24


def act_error(z):
    return (z.abs() + 4) * 2.0 ** -22


def within(got, exact, bound, what):
    got = got.double()
    bad = ~((got - exact).abs() <= bound)
    assert not bad.any(), "%s: %d of %d elements off, worst by %.3g of its bound" % (
        what, int(bad.sum()), bad.numel(), float(((got - exact).abs() / bound).max()))


def normal(shape, seed, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).cuda()


# ---- group norm ---------------------------------------------------------------------------
def norm64(x, offsets, groups, w, b, eps, act, dy=None):
    """y, the spread 1 / sqrt(var + eps) of every element's group and, with dy, the gradients."""
    x = x.double().requires_grad_(dy is not None)
    w, b = [None if t is None else t.detach().double().requires_grad_(dy is not None)
            for t in (w, b)]
    ends = offsets.tolist()
    parts, rstds = [], []
    for s, e in zip(ends[:-1], ends[1:]):
        if s == e:
            continue
        v = x[s:e].view(e - s, groups, -1)
        mean = v.mean((0, 2), keepdim=True)
        var = ((v - mean) ** 2).mean((0, 2), keepdim=True)
        rstd = 1 / torch.sqrt(var + eps)
        parts.append(((v - mean) * rstd).reshape(e - s, -1))
        rstds.append((rstd + 0 * v).reshape(e - s, -1).detach())
    h = torch.cat(parts) if parts else x * 0
    z = h * (1 if w is None else w) + (0 if b is None else b)
    y = act64(act, z)
    rstd = torch.cat(rstds) if rstds else h.detach()
    if dy is None:
        return y, z, h, rstd
    leaves = [t for t in (x, w, b) if t is not None]
    return (y, z, h, rstd) + torch.autograd.grad(y, leaves, dy.double())


NORM_CASES = [
    # rows of the clouds, channels, groups, activation
    ([1], 1, 1, None),
    ([1], 8, 2, "silu"),                         # variance 0 over one row of 4 channels
    ([0, 5, 0, 0, 3, 0], 12, 3, "relu"),         # empty clouds, at both ends too
    ([31, 1, 33], 7, 7, "gelu"),                 # a group for each channel, odd channels
    ([100, 29, 64, 200], 32, 8, "relu"),
    ([257], 200, 25, "tanh"),
    ([5] * 70, 16, 4, "silu"),                   # more clouds than a wave has lanes
    ([3] * 300, 6, 2, "sigmoid"),
    ([1000, 4000], 24, 1, "silu"),               # one group of all channels
    ([9], 1200, 4, "silu"),                      # more channels than a workgroup has threads
    ([40, 2], 2056, 2, "relu"),                  # over 1024 channels in a group
    ([70001], 20, 5, "gelu"),                    # chunks of more than the least rows
]


def norm_inputs(rows, c, dtype, seed):
    n = sum(rows)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32).cuda()
    x = normal((n, c), seed).mul_(normal((c,), seed + 1).exp_()).add_(normal((c,), seed + 2, scale=3))
    return x.to(dtype), offsets, normal((n, c), seed + 5, dtype)


def norm_bounds(x, offsets, groups, w, b, eps, act, dy, dtype, wdtype):
    """Exact results with bounds: [(name, exact, bound)]."""
    y, z, h, rstd, dx, dw, db = norm64(x, offsets, groups, w, b, eps, act, dy)
    u, c = U[dtype], x.size(1)
    wd, bd = w.double().abs(), b.double().abs()
    # a channel's partial sums run over a chunk's rows of a thread and a tree; mean and spread are
    # then right to a few units of float32 relative to the largest value of the group
    n = x.size(0)
    terms = n / 64 + 64
    big = x.double().abs().max() * rstd  # |x| in units of the spread
    e_h = (4 + big) * 2.0 ** -23 + h.abs() * gamma(min(terms, 600)) * 8
    e_z = e_h * wd + (z.abs() + bd) * 2.0 ** -23
    d1 = 1.2 if act != "none" else 1.0
    e_y = u * y.abs() + TINY[dtype] + d1 * e_z + act_error(z) * (y.abs() + e_z)
    # |second derivative| <= 1.2 for every activation; relu's slope jumps where z is 0
    dyd = dy.double().abs()
    slope = slope64(act, z)
    jump = (z.abs() <= e_z).double() if act == "relu" else 0
    e_dz = dyd * (1.2 * e_z + act_error(z) * (1 + z.abs()) + jump)
    dz = dy.double() * slope
    e_dw = (e_dz * h.abs() + dz.abs() * e_h).sum(0) + gamma(min(terms * 4, 4000)) * (dz * h).abs().sum(0)
    e_db = e_dz.sum(0) + gamma(min(terms * 4, 4000)) * dz.abs().sum(0)
    # means over the group of |gradient|, per element of the group
    def mean_of(v):
        out = torch.zeros_like(v)
        ends = offsets.tolist()
        for s, e in zip(ends[:-1], ends[1:]):
            if e > s:
                t = v[s:e].view(e - s, groups, -1)
                out[s:e] = t.mean((0, 2), keepdim=True).expand_as(t).reshape(e - s, -1)
        return out
    g = dz.abs() * wd
    e_g = e_dz * wd + g * gamma(min(terms * 4, 4000))
    e_dx = rstd * (e_dz * wd + mean_of(e_g) + h.abs() * mean_of(e_g * h.abs() + g * e_h) +
                   e_h * mean_of(g * h.abs()) + 2.0 ** -22 * (g + mean_of(g) +
                                                             h.abs() * mean_of(g * h.abs())))
    e_dx = e_dx + (4 + big) * 2.0 ** -22 * dx.abs() + u * dx.abs() + TINY[dtype]
    uw = U[wdtype]
    return [("y", y.detach(), e_y.detach()), ("dx", dx, e_dx.detach()),
            ("dweight", dw, (e_dw + uw * dw.abs()).detach() + TINY[wdtype]),
            ("dbias", db, (e_db + uw * db.abs()).detach() + TINY[wdtype])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(NORM_CASES)))
def test_norm_forward_and_gradients(case, dtype):
    rows, c, groups, act = NORM_CASES[case]
    x, offsets, dy = norm_inputs(rows, c, dtype, 10 * case)
    wdtype = dtype if case % 2 else torch.float32
    w = normal((c,), 3, wdtype, 0.3, 1.0).requires_grad_()
    b = normal((c,), 4, wdtype, 0.3).requires_grad_()
    x.requires_grad_()
    y = group_norm(x, offsets, groups, w, b, 1e-5, act)
    assert y.dtype == dtype and y.shape == x.shape
    got = (y,) + torch.autograd.grad(y, (x, w, b), dy)
    for t, (name, exact, bound) in zip(got, norm_bounds(x.detach(), offsets, groups, w.detach(),
                                                        b.detach(), 1e-5, act, dy, dtype, wdtype)):
        within(t, exact, bound, name)


def test_norm_without_parameters_and_of_some_gradients():
    x, offsets, dy = norm_inputs([50, 0, 70], 16, torch.float32, 3)
    one, zero = torch.ones(16).cuda(), torch.zeros(16).cuda()
    assert torch.equal(group_norm(x, offsets, 4, activation="silu"),
                       group_norm(x, offsets, 4, one, zero, activation="silu"))
    w = normal((16,), 1).requires_grad_()
    for args in ((x, w, zero), (x.clone().requires_grad_(), w, zero),
                 (x.clone().requires_grad_(), one, zero)):
        full = [t.detach().clone().requires_grad_() for t in args]
        want = torch.autograd.grad(group_norm(full[0], offsets, 4, full[1], full[2]), full, dy)
        leaves = [t for t in args if t.requires_grad]
        got = torch.autograd.grad(group_norm(args[0], offsets, 4, args[1], args[2]), leaves, dy)
        want = [g for g, t in zip(want, args) if t.requires_grad]
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    w2 = normal((16,), 1)
    assert torch.equal(group_norm(x, offsets, 4, w2, None), group_norm(x, offsets, 4, w2, zero))


def test_norm_of_rows_far_from_zero():
    """A spread of 1 around 10^4: deviations, not differences of squares, give the variance."""
    x = normal((3000, 8), 1, scale=1.0, shift=1e4)
    offsets = torch.tensor([0, 1000, 3000], dtype=torch.int32).cuda()
    y = group_norm(x, offsets, 2)
    exact, _, _, _ = norm64(x, offsets, 2, None, None, 1e-5, None)
    # the mean is right to a unit of float32 at 10^4 (2^-10), so are the deviations
    assert float((y.double() - exact).abs().max()) < 4e-3


def test_norm_gradient_against_differences():
    x, offsets, dy = norm_inputs([40, 25], 12, torch.float32, 8)
    w, b = normal((12,), 3, scale=0.3, shift=1), normal((12,), 4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = group_norm(leaves[0], offsets, 3, leaves[1], leaves[2], activation="gelu")
    grads = torch.autograd.grad(y, leaves, dy)
    for i, (t, g) in enumerate(zip((x, w, b), grads)):
        d = normal(t.shape, 20 + i)
        step = 1e-2
        f = []
        for s in (step, -step):
            args = [x, w, b]
            args[i] = t + s * d
            v = group_norm(args[0], offsets, 3, args[1], args[2], activation="gelu")
            f.append(float((v.double() * dy.double()).sum()))
        slope, want = (f[0] - f[1]) / (2 * step), float((g.double() * d.double()).sum())
        # third derivatives of the composition times step^2 / 6, over some hundred elements
        assert abs(slope - want) <= 2e-2 * (1 + float((g.double() * d.double()).abs().sum()) ** 0.5 * 2)


def test_norm_strides_streams_and_empty():
    x, offsets, dy = norm_inputs([33, 12], 24, torch.bfloat16, 5)
    wide = torch.zeros(45, 40, dtype=torch.bfloat16).cuda()
    wide[:, 3:27] = x
    w = normal((48,), 1)[::2]
    assert torch.equal(group_norm(wide[:, 3:27], offsets, 4, w),
                       group_norm(x, offsets, 4, w.contiguous()))
    flat = torch.empty(45 * 24 + 1, dtype=torch.bfloat16).cuda()
    odd = flat[1:].view(45, 24).copy_(x)  # rows that do not begin at 16 bytes
    ours, theirs = group_norm(odd, offsets, 4, w), group_norm(x, offsets, 4, w)
    # (another split of the sums: a unit in the last place at most)
    assert float((ours.float() - theirs.float()).abs().max()) <= 2.0 ** -7 * float(theirs.abs().max())
    assert torch.equal(group_norm(x, offsets.long(), 4), group_norm(x, offsets, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = group_norm(x, offsets, 4, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, group_norm(x, offsets, 4, w))
    none = torch.zeros(0, 24, dtype=torch.bfloat16).cuda().requires_grad_()
    w = w.contiguous().requires_grad_()
    y = group_norm(none, torch.zeros(3, dtype=torch.int32).cuda(), 4, w)
    dx, dw = torch.autograd.grad(y, (none, w), torch.zeros_like(y))
    assert y.shape == (0, 24) and dx.shape == (0, 24) and not dw.any()


def test_norm_nan_stays_in_its_group():
    x, offsets, _ = norm_inputs([20, 20], 8, torch.float32, 6)
    want = group_norm(x, offsets, 2)
    x[3, 1] = float("nan")
    x[30, 7] = float("inf")
    got = group_norm(x, offsets, 2, activation="relu")
    assert got[:20, :4].isnan().all() and got[20:, 4:].isnan().all()
    assert torch.equal(got[:20, 4:], want[:20, 4:].relu())
    assert torch.equal(got[20:, :4], want[20:, :4].relu())


def test_norm_module_and_repetition():
    torch.manual_seed(0)
    idx = torch.tensor([[b, i, 0, 0] for b in range(3) for i in range(10 + b)],
                       dtype=torch.int32).cuda()
    x = normal((33, 16), 1)
    m = GroupNorm(4, 16, activation=torch.nn.SiLU()).cuda()
    out = m(SparseTensor(x, idx, [16, 1, 1], 3))
    offsets = torch.tensor([0, 10, 21, 33], dtype=torch.int32).cuda()
    assert torch.equal(out.features, group_norm(x, offsets, 4, m.weight, m.bias, 1e-5, "silu"))
    m.load_state_dict(GroupNorm(4, 16).state_dict())
    # a result does not depend on the other clouds of the batch
    alone = group_norm(x[10:21].contiguous(), torch.tensor([0, 11], dtype=torch.int32).cuda(), 4,
                       activation="silu")
    assert float((alone - out.features[10:21]).detach().abs().max()) < 1e-5
    big, offsets, dy = norm_inputs([20000, 7000], 64, torch.float32, 2)
    big.requires_grad_()
    runs = []
    for _ in range(3):
        y = group_norm(big, offsets, 8, activation="gelu")
        runs.append((y.detach(), torch.autograd.grad(y, big, dy)[0]))
    assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(r, runs[0]))


def test_norm_refusals():
    x, offsets, _ = norm_inputs([4, 4], 8, torch.float32, 1)
    w = torch.ones(8).cuda()
    for error, call in (
            (RuntimeError, lambda: group_norm(x.cpu(), offsets, 2)),
            (RuntimeError, lambda: group_norm(x, offsets.cpu(), 2)),
            (RuntimeError, lambda: group_norm(x, offsets, 2, w.cpu())),
            (ValueError, lambda: group_norm(x, offsets, 3)),
            (ValueError, lambda: group_norm(x, offsets, 0)),
            (ValueError, lambda: group_norm(x, offsets[:1], 2)),
            (ValueError, lambda: group_norm(x, offsets, 2, eps=-1.0)),
            (ValueError, lambda: group_norm(x, offsets, 2, eps=float("nan"))),
            (ValueError, lambda: group_norm(x, offsets, 2, w[:4])),
            (ValueError, lambda: group_norm(x[0], offsets, 2)),
            (ValueError, lambda: group_norm(x, offsets, 2, activation="swish")),
            (ValueError, lambda: group_norm(x, offsets, 2, activation=torch.nn.GELU("tanh"))),
            (TypeError, lambda: group_norm(x.double(), offsets, 2)),
            (TypeError, lambda: group_norm(x, offsets.float(), 2)),
            (TypeError, lambda: group_norm(x, offsets, 2, w.double())),
            (TypeError, lambda: group_norm(x.half(), offsets, 2, w, w.half())),
            (TypeError, lambda: group_norm(x.half(), offsets, 2, w.bfloat16())),
            (ValueError, lambda: GroupNorm(3, 8)),
            (ValueError, lambda: GroupNorm(2, 16).cuda()(
                SparseTensor(x, torch.zeros(8, 4, dtype=torch.int32).cuda(), [4, 4, 4], 2)))):
        with pytest.raises(error):
            call()


# ---- gated feed-forward -------------------------------------------------------------------
GATED_CASES = [
    # rows, width, hidden, activation, bias
    (1, 1, 1, "silu", True),
    (1, 64, 16, "silu", False),
    (1, 520, 100, "gelu", True),
    (3, 7, 5, "relu", True),            # odd widths: no row begins at 16 bytes
    (16, 40, 17, "silu", True),
    (17, 128, 48, None, False),
    (32, 1000, 30, "tanh", True),       # the last rows of the kernel for few
    (33, 96, 64, "sigmoid", True),      # the first of the tiles
    (64, 72, 130, "silu", True),
    (65, 33, 66, "gelu", True),
    (257, 136, 300, "silu", False),
    (300, 8, 8, "relu", True),
    (1000, 64, 24, "silu", True),
    (2049, 200, 523, "gelu", True),
    (700, 1032, 264, "silu", False),    # many steps along k
    (4100, 256, 4096, "silu", True),    # large tiles, the last ones ragged
]


def gated_inputs(m, k, h, dtype, bias, seed):
    x = normal((m, k), seed, dtype)
    wg, wu = [normal((h, k), seed + i, dtype, k ** -0.5) for i in (1, 2)]
    bg, bu = [normal((h,), seed + i, dtype, 0.3) if bias else None for i in (3, 4)]
    return x, wg, wu, bg, bu, normal((m, h), seed + 5, dtype)


def gated_bounds(x, wg, wu, bg, bu, act, dy, dtype):
    m, k = x.shape
    xd, gd, ud, yd = x.double(), wg.double(), wu.double(), dy.double()
    zero = torch.zeros(wg.size(0), dtype=torch.float64, device=x.device)
    bgd, bud = [zero if t is None else t.double() for t in (bg, bu)]
    a, b = xd @ gd.t() + bgd, xd @ ud.t() + bud
    u = U[dtype]
    # float operands in parts leave out 2^-24 of every product
    gk = gamma(k) + 2.0 ** -22
    ea = gk * (xd.abs() @ gd.abs().t() + bgd.abs())
    eb = gk * (xd.abs() @ ud.abs().t() + bud.abs())
    f, s = act64(act, a), slope64(act, a)
    y = f * b
    ef = 1.2 * ea + act_error(a) * (f.abs() + ea)
    ey = u * y.abs() + TINY[dtype] + (f.abs() + ef) * eb + ef * b.abs() + 2.0 ** -23 * y.abs()
    # the backward pass reads a and b rounded to the type (u), and rounds da and db
    ea2, eb2 = ea + u * a.abs() + TINY[dtype], eb + u * b.abs() + TINY[dtype]
    jump = (a.abs() <= ea2).double() if act == "relu" else 0
    es = 1.2 * ea2 + act_error(a) * (1 + a.abs()) + jump
    da, db = yd * b * s, yd * f
    eda = yd.abs() * (eb2 * (s.abs() + es) + b.abs() * es) + 2 * u * da.abs() + TINY[dtype]
    edb = yd.abs() * (1.2 * ea2 + act_error(a) * (f.abs() + ea2)) + 2 * u * db.abs() + TINY[dtype]
    gh, gm = gamma(2 * wg.size(0)) + 2.0 ** -22, gamma(m) + 2.0 ** -22
    dx = da @ gd + db @ ud
    edx = eda @ gd.abs() + edb @ ud.abs() + gh * (da.abs() @ gd.abs() + db.abs() @ ud.abs()) + \
        u * dx.abs() + TINY[dtype]
    out = [("y", y, ey), ("dx", dx, edx)]
    for name, d, e in (("dw_gate", da, eda), ("dw_up", db, edb)):
        dw = d.t() @ xd
        out.append((name, dw, e.t() @ xd.abs() + gm * (d.abs().t() @ xd.abs()) + u * dw.abs() + TINY[dtype]))
    if bg is not None:
        for name, d, e in (("db_gate", da, eda), ("db_up", db, edb)):
            out.append((name, d.sum(0), e.sum(0) + gm * d.abs().sum(0) + u * d.sum(0).abs() + TINY[dtype]))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(GATED_CASES)))
def test_gated_forward_and_gradients(case, dtype):
    m, k, h, act, bias = GATED_CASES[case]
    x, wg, wu, bg, bu, dy = gated_inputs(m, k, h, dtype, bias, 10 * case)
    with torch.no_grad():
        plain = gated_linear(x, wg, wu, bg, bu, act)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    y = gated_linear(x, wg, wu, bg, bu, act)
    assert y.dtype == dtype and y.shape == (m, h) and torch.equal(y, plain)
    got = (y,) + torch.autograd.grad(y, leaves, dy)
    args = [None if t is None else t.detach() for t in (x, wg, wu, bg, bu)]
    for t, (name, exact, bound) in zip(got, gated_bounds(*args, act, dy, dtype)):
        assert t.dtype == dtype
        within(t, exact, bound, name)


def test_gated_some_gradients_strides_streams():
    x, wg, wu, bg, bu, dy = gated_inputs(90, 48, 40, torch.bfloat16, True, 1)
    all_of = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    want = torch.autograd.grad(gated_linear(*all_of), all_of, dy)
    for i in range(5):
        args = [t.clone() for t in (x, wg, wu, bg, bu)]
        args[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(gated_linear(*args), args[i], dy)[0], want[i])
    y = gated_linear(x, wg, wu, bg, bu)
    turned = x.t().contiguous().t()
    assert torch.equal(gated_linear(turned, wg, wu, bg, bu), y)
    assert torch.equal(gated_linear(x.view(2, 3, 15, 48), wg, wu, bg, bu), y.view(2, 3, 15, 40))
    assert torch.equal(gated_linear(x[0], wg, wu, bg, bu), gated_linear(x[:1], wg, wu, bg, bu)[0])
    flat = torch.empty(90 * 48 + 1, dtype=torch.bfloat16).cuda()
    odd = flat[1:].view(90, 48).copy_(x)  # not at 16 bytes: laid out anew first
    assert torch.equal(gated_linear(odd, wg, wu, bg, bu), y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = gated_linear(x, wg, wu, bg, bu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, y)
    none = x[:0].requires_grad_()
    y = gated_linear(none, all_of[1], wu)
    dx, dw = torch.autograd.grad(y, (none, all_of[1]), torch.zeros_like(y))
    assert y.shape == (0, 40) and dx.shape == (0, 48) and not dw.any()


def test_gated_gradient_against_differences():
    x, wg, wu, bg, bu, dy = gated_inputs(50, 20, 12, torch.float32, True, 2)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(gated_linear(*leaves), leaves, dy)
    for i, g in enumerate(grads):
        d, step, f = normal(leaves[i].shape, 30 + i), 1e-2, []
        for s in (step, -step):
            args = [t.detach() for t in leaves]
            args[i] = args[i] + s * d
            f.append(float((gated_linear(*args).double() * dy.double()).sum()))
        slope, want = (f[0] - f[1]) / (2 * step), float((g.double() * d.double()).sum())
        # third derivatives times step^2 / 6 over some hundred elements
        assert abs(slope - want) <= 2e-2 * (1 + float((g.double() * d.double()).abs().sum()) ** 0.5 * 2)


def test_gated_floats_far_apart():
    """Every product counts with its 24 bits whatever stands beside it, the largest floats too."""
    m, k, h = 70, 64, 40
    x, wg, wu, _, _, _ = gated_inputs(m, k, h, torch.float32, False, 3)
    x = x * torch.exp2(normal((m, 1), 9, scale=20).round())
    wg[:, ::2] *= 1e-12
    y = gated_linear(x, wg, wu, activation=None)
    a, b = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    ea = (gamma(k) + 2.0 ** -22) * (x.double().abs() @ wg.double().abs().t())
    eb = (gamma(k) + 2.0 ** -22) * (x.double().abs() @ wu.double().abs().t())
    within(y, a * b, ea * b.abs() + eb * a.abs() + ea * eb + 2.0 ** -22 * (a * b).abs() + 1e-37, "y")
    big = torch.zeros(40, 8).cuda()
    big[:, 0] = torch.finfo(torch.float32).max
    one = torch.zeros(8, 8).cuda()
    one[:, 0] = 0.5
    got = gated_linear(big, one, one * 2.0 ** -127, activation=None)
    want = (big.double() @ one.double().t()) * (big.double() @ (one * 2.0 ** -127).double().t())
    assert float(((got.double() - want) / want).abs().max()) < 2.0 ** -20


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_nan_stays_in_its_row(dtype):
    for m in (20, 100):
        x, wg, wu, _, _, _ = gated_inputs(m, 24, 40, dtype, False, 4)
        want = gated_linear(x, wg, wu)
        x[7, 5] = float("nan")
        got = gated_linear(x, wg, wu)
        rest = [i for i in range(m) if i != 7]
        assert got[7].isnan().all() and torch.equal(got[rest], want[rest])


def test_gated_modules_train():
    """A small network of blocks of the kind learns: norm, gated block, AdamW with 8-bit moments."""
    torch.manual_seed(0)
    idx = torch.tensor([[b, i, 0, 0] for b in range(4) for i in range(64)], dtype=torch.int32).cuda()
    x = normal((256, 24), 1)
    target = torch.sin(x @ normal((24, 24), 2, scale=0.3))
    net = torch.nn.Sequential(GatedFeedForward(24, 48, GroupNorm(4, 24), bias=True),
                              GatedFeedForward(24, 48, GroupNorm(4, 24), activation="gelu")).cuda()
    for bits in (32, 8):
        opt = AdamW(net.parameters(), lr=1e-2, state_bits=bits)
        losses = []
        for _ in range(30):
            opt.zero_grad()
            out = net(SparseTensor(x, idx, [64, 1, 1], 4))
            loss = (out.features - target).square().mean()
            loss.backward()
            opt.step()
            losses.append(float(loss))
        assert losses[-1] < 0.7 * losses[0], losses
    m = GatedLinear(24, 48, bias=True)
    assert sorted(m.state_dict()) == ["b_gate", "b_up", "w_gate", "w_up"]


def test_gated_and_norm_replay_in_a_graph():
    x, wg, wu, bg, bu, _ = gated_inputs(200, 64, 96, torch.bfloat16, True, 6)
    offsets = torch.tensor([0, 120, 200], dtype=torch.int32).cuda()
    w = torch.ones(96, dtype=torch.bfloat16).cuda()
    few = x[:5].clone()

    def both():
        y = gated_linear(x, wg, wu, bg, bu)
        return group_norm(y, offsets, 8, w, activation="relu"), gated_linear(few, wg, wu, bg, bu)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    for i in range(4):
        x.copy_(normal((200, 64), 50 + i, torch.bfloat16))
        few.copy_(x[:5])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, both()))


def test_gated_refusals():
    x, wg, wu, bg, bu, _ = gated_inputs(4, 8, 6, torch.float32, True, 1)
    for error, call in (
            (RuntimeError, lambda: gated_linear(x.cpu(), wg, wu)),
            (RuntimeError, lambda: gated_linear(x, wg.cpu(), wu)),
            (RuntimeError, lambda: gated_linear(x, wg, wu, bg.cpu())),
            (ValueError, lambda: gated_linear(x[:, :7], wg, wu)),
            (ValueError, lambda: gated_linear(x, wg, wu[:5])),
            (ValueError, lambda: gated_linear(x, wg[0], wu)),
            (ValueError, lambda: gated_linear(x, wg, wu, bg[:5])),
            (ValueError, lambda: gated_linear(x, wg, wu, activation="swish")),
            (TypeError, lambda: gated_linear(x, wg, None)),
            (TypeError, lambda: gated_linear(x.double(), wg.double(), wu.double())),
            (TypeError, lambda: gated_linear(x.half(), wg, wu))):
        with pytest.raises(error):
            call()
    with pytest.raises(RuntimeError):  # no second derivative
        leaf = x.clone().requires_grad_()
        g, = torch.autograd.grad(gated_linear(leaf, wg, wu).square().sum(), leaf, create_graph=True)
        g.sum().backward()


# ---- AdamW --------------------------------------------------------------------------------
CONFIG = dict(lr=3e-3, betas=(0.8, 0.95), eps=1e-7, weight_decay=0.1)


def adamw64(p, g, m, v, step, lr, betas, eps, weight_decay):
    p, g, m, v = [t.double() for t in (p, g, m, v)]
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    below = (v / (1 - betas[1] ** step)).sqrt() + eps
    return p * (1 - lr * weight_decay) - lr * (m / (1 - betas[0] ** step)) / below, m, v


def decode(mc, vc, mq, vq):
    """The definition, in numpy and 64 bits."""
    mc, vc, mq, vq = [t.cpu().numpy() for t in (mc, vc, mq, vq)]
    shape = mc.shape
    c, e = mc.reshape(-1).astype(np.float64), vc.reshape(-1).astype(np.float64)
    block = np.arange(c.size) // BLOCK
    return ((c * np.abs(c) * mq[block]).reshape(shape),
            ((e * e * vq[block]) ** 2).reshape(shape))


SIZES = [(1,), (3,), (255,), (256,), (257,), (64, 48), (3, 5, 7), (0,), (5000,), (2049, 3)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_adamw_32_bit(dtype):
    params = [normal(s, i, dtype) for i, s in enumerate(SIZES)]
    grads = [normal(s, 20 + i, dtype) for i, s in enumerate(SIZES)]
    ms = [normal(s, 40 + i) for i, s in enumerate(SIZES)]
    vs = [normal(s, 60 + i).square() for i, s in enumerate(SIZES)]
    for step in (1, 7, 100000):
        want = [adamw64(p, g, m, v, step, **CONFIG) for p, g, m, v in zip(params, grads, ms, vs)]
        versions = [p._version for p in params]
        adamw_(params, grads, ms, vs, step, **CONFIG)
        assert all(p._version > n for p, n in zip(params, versions))
        for p, m, v, (wp, wm, wv), g in zip(params, ms, vs, want, grads):
            # three roundings of each term
            within(m, wm, 2.0 ** -22 * (wm.abs() + g.double().abs() + 1), "m")
            within(v, wv, 2.0 ** -22 * (wv.abs() + 1e-30), "v")
            within(p, wp, U[dtype] * wp.abs() + 2.0 ** -21 * (wp.abs() + 0.1) + TINY[dtype], "p")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("skew", [0, 1])
def test_adamw_8_bit_follows_its_definition(dtype, skew):
    """Codes are the nearest in the root of the magnitude: decoded, encoded values lie within half
    a code of the exact moments, and a v that is not zero is never 0.  skew: tensors that do not
    begin at 4 or 16 bytes."""
    cut = lambda t: torch.cat([t.reshape(-1)[:1].expand(skew), t.reshape(-1)])[skew:].view(t.shape) \
        if t.numel() else t  # noqa: E731
    sizes = SIZES
    params = [cut(normal(s, i, dtype)) for i, s in enumerate(sizes)]
    grads = [cut(normal(s, 20 + i, dtype, 1e-2) * normal(s, 30 + i, scale=2).exp().to(dtype))
             for i, s in enumerate(sizes)]
    ms = [cut(torch.zeros(s, dtype=torch.int8).cuda()) for s in sizes]
    vs = [cut(torch.zeros(s, dtype=torch.uint8).cuda()) for s in sizes]
    mq = [torch.zeros(-(-p.numel() // BLOCK)).cuda() for p in params]
    vq = [torch.zeros(-(-p.numel() // BLOCK)).cuda() for p in params]
    for step in (1, 2, 3):
        before = [[torch.from_numpy(a).cuda() for a in decode(*t)] for t in zip(ms, vs, mq, vq)]
        want = [adamw64(p, g, m, v, step, **CONFIG)
                for p, g, (m, v) in zip(params, grads, before)]
        adamw_(params, grads, ms, vs, step, exp_avg_scales=mq, exp_avg_sq_scales=vq, **CONFIG)
        values = state_values(ms, vs, mq, vq)
        for i, (wp, wm, wv) in enumerate(want):
            n = wp.numel()
            if n == 0:
                continue
            # (m / sqrt(v) is at most sqrt of 1 / (1 - beta2) and more in the first steps)
            within(params[i], wp, U[dtype] * wp.abs() + 2.0 ** -20 * (wp.abs() + 0.1) + TINY[dtype], "p")
            dm, dv = decode(ms[i], vs[i], mq[i], vq[i])
            np.testing.assert_allclose(values[0][i].cpu().numpy(), dm, rtol=2.0 ** -23, atol=0)
            np.testing.assert_allclose(values[1][i].cpu().numpy(), dv, rtol=2.0 ** -22, atol=0)
            for got, exact, steps in ((dm, wm, 127), (np.sqrt(dv), wv.sqrt(), 255)):
                got, exact = got.reshape(-1), exact.cpu().numpy().reshape(-1)
                for s in range(0, n, BLOCK):
                    x, e = got[s:s + BLOCK], exact[s:s + BLOCK]
                    top = np.abs(e).max()
                    if top == 0:
                        assert not x.any()
                        continue
                    code = steps * np.sqrt(np.abs(x) / top)
                    true = steps * np.sqrt(np.abs(e) / top)
                    ok = np.abs(code - true) <= 0.5 + 1e-3
                    if steps == 255:
                        ok |= (np.abs(code - 1) < 1e-3) & (true < 0.5)
                        assert (x[e > 0] > 0).all()
                    assert ok.all() and (np.sign(x[x != 0]) == np.sign(e[x != 0])).all()


def test_adamw_more_tensors_than_a_launch_holds():
    sizes = [(1 + (7 * i) % 600,) for i in range(300)]
    for bits in (32, 8):
        ps = [normal(s, i) for i, s in enumerate(sizes)]
        ref = [p.clone() for p in ps]
        opt, each = AdamW([p.requires_grad_() for p in ps], state_bits=bits), []
        for p, r in zip(ps, ref):
            p.grad = normal(p.shape, 3)
            r.requires_grad_()
            r.grad = p.grad.clone()
            each.append(AdamW([r], state_bits=bits))
        for _ in range(2):
            opt.step()
            for o in each:
                o.step()
        assert all(torch.equal(p, r) for p, r in zip(ps, ref))


def test_adamw_nan_and_infinity():
    for bits in (32, 8):
        p = normal((600,), 1).requires_grad_()
        opt = AdamW([p], state_bits=bits)
        for step in range(2):
            p.grad = normal((600,), 2 + step)
            if step == 0:
                p.grad[5] = float("nan")
                p.grad[590] = float("inf")
            opt.step()
        bad = p.detach().isnan()
        if bits == 32:
            assert bad.nonzero().view(-1).tolist() == [5, 590]
        else:
            assert bad[:256].all() and not bad[256:512].any() and bad[512:].all()


def test_adamw_optimizer_state():
    def make(bits):
        torch.manual_seed(3)
        net = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 4)).cuda()
        net[0].weight.data = net[0].weight.data.t().contiguous().t()  # dense, in another order
        half = torch.nn.Parameter(normal((300,), 5, torch.bfloat16))
        return net, half, AdamW([dict(params=net.parameters(), lr=1e-2),
                                 dict(params=[half], weight_decay=0.0)], state_bits=bits)

    def run(net, half, opt, first, last):
        for i in range(first, last):
            opt.zero_grad()
            (net(normal((8, 20), i)).square().sum() + (half.float() * (i + 1)).sin().sum()).backward()
            opt.step()

    for bits in (32, 8):
        net, half, opt = make(bits)
        run(net, half, opt, 0, 6)
        net2, half2, opt2 = make(bits)
        run(net2, half2, opt2, 0, 3)
        saved = opt2.state_dict()
        net3, half3, opt3 = make(bits)
        net3.load_state_dict(net2.state_dict())
        half3.data.copy_(half2.data)
        opt3.load_state_dict(saved)
        for s in opt3.state.values():
            assert s["step"] == 3
            assert all(s[k].dtype == torch.float32 for k in s if k.endswith("scale"))
            assert s["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.int8)
        run(net3, half3, opt3, 3, 6)
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), net3.parameters()))
        assert torch.equal(half, half3)
    # one that has no gradient keeps its place, and its count of steps
    p, q = [torch.nn.Parameter(normal((4,), i)) for i in range(2)]
    opt = AdamW([p, q])
    p.grad = torch.ones_like(p)
    opt.step()
    assert opt.state[p]["step"] == 1 and len(opt.state[q]) == 0
    q.grad = torch.ones_like(q)
    opt.step()
    assert opt.state[p]["step"] == 2 and opt.state[q]["step"] == 1
    assert opt.step(lambda: torch.ones(1)) == 1


def test_adamw_strides_and_streams():
    p = normal((40, 30), 1).t()
    g = normal((30, 40), 2)          # another order than the parameter's
    m, v = torch.zeros(40, 30).cuda().t(), torch.zeros(40, 30).cuda().t()
    want = adamw64(p, g, m, v, 1, **CONFIG)
    adamw_([p], [g], [m], [v], 1, **CONFIG)
    within(p, want[0], 2.0 ** -20 * (want[0].abs() + 0.1), "p")
    within(m, want[1], 2.0 ** -22 * (want[1].abs() + 1), "m")
    side = torch.cuda.Stream()
    p2 = normal((40, 30), 1).t()
    m2, v2 = torch.zeros(40, 30).cuda().t(), torch.zeros(40, 30).cuda().t()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adamw_([p2], [g], [m2], [v2], 1, **CONFIG)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, p2) and torch.equal(v, v2)


def test_adamw_refusals():
    p, g, m, v = [normal((8, 4), i) for i in range(4)]
    v = v.square()
    c, q = torch.zeros(8, 4, dtype=torch.int8).cuda(), torch.zeros(1).cuda()
    for error, call in (
            (ValueError, lambda: adamw_([p], [g, g], [m], [v], 1)),
            (ValueError, lambda: adamw_([p], [g[:4]], [m], [v], 1)),
            (ValueError, lambda: adamw_([p], [g.half()], [m], [v], 1)),
            (ValueError, lambda: adamw_([p], [g], [m.half()], [v], 1)),
            (ValueError, lambda: adamw_([p], [g], [m[:4]], [v], 1)),
            (ValueError, lambda: adamw_([p], [g], [c], [c.byte()], 1)),
            (ValueError, lambda: adamw_([p], [g], [c], [c.byte()], 1, exp_avg_scales=[q])),
            (ValueError, lambda: adamw_([p], [g], [c], [c.byte()], 1, exp_avg_scales=[q],
                                        exp_avg_sq_scales=[torch.zeros(2).cuda()])),
            (ValueError, lambda: adamw_([p[:, :2]], [g[:, :2]], [m[:, :2].clone()],
                                        [v[:, :2].clone()], 1)),
            (ValueError, lambda: adamw_([p], [g], [m], [v], 0)),
            (ValueError, lambda: adamw_([p], [g], [m], [v], 1, lr=-1.0)),
            (ValueError, lambda: adamw_([p], [g], [m], [v], 1, lr=float("nan"))),
            (ValueError, lambda: adamw_([p], [g], [m], [v], 1, betas=(1.0, 0.9))),
            (TypeError, lambda: adamw_([p.double()], [g.double()], [m], [v], 1)),
            (RuntimeError, lambda: adamw_([p.cpu()], [g.cpu()], [m], [v], 1)),
            (RuntimeError, lambda: adamw_([p], [g], [m.cpu()], [v], 1)),
            (RuntimeError, lambda: adamw_([p], [g.to_sparse()], [m], [v], 1)),
            (ValueError, lambda: AdamW([p], lr=-1.0)),
            (ValueError, lambda: AdamW([p], betas=(0.9, 1.0))),
            (ValueError, lambda: AdamW([p], state_bits=16))):
        before = p.clone()
        with pytest.raises(error):
            call()
        assert torch.equal(p, before)


def test_pointwise_c_abi_refusals():
    """Arguments that the library itself turns away, without a launch."""
    lib = _ext._lib
    x = torch.zeros(4, 8).cuda()
    ws = torch.zeros(1 << 16, dtype=torch.uint8).cuda()
    off = torch.tensor([0, 4], dtype=torch.int32).cuda()
    norm = lambda **k: lib.ssc_groupnorm_fwd(*dict(  # noqa: E731
        dict(dtype=0, x=x.data_ptr(), n=4, c=8, off=off.data_ptr(), clouds=1, groups=2, wtype=0,
             w=None, b=None, eps=1e-5, act=0, y=x.data_ptr(), mean=ws.data_ptr(),
             rstd=ws.data_ptr(), ws=ws.data_ptr(), bytes=ws.numel(), stream=None), **k).values())
    assert norm(dtype=3) == norm(groups=3) == norm(act=9) == norm(clouds=0) == norm(off=None) == \
        norm(eps=-1.0) == norm(wtype=7) == norm(n=-1) == norm(x=None) == _ext.SSC_EINVAL
    assert norm(bytes=16) == norm(ws=None) == _ext.SSC_EWORKSPACE
    assert norm(n=0, x=None) == 0
    gated = lambda **k: lib.ssc_gated_fwd(*dict(  # noqa: E731
        dict(dtype=0, x=x.data_ptr(), m=4, k=8, wg=x.data_ptr(), wu=x.data_ptr(), h=4, bg=None,
             bu=None, act=0, y=ws.data_ptr(), kept=None, ws=ws.data_ptr(), bytes=ws.numel(),
             stream=None), **k).values())
    assert gated(dtype=5) == gated(k=0) == gated(h=0) == gated(act=6) == gated(m=-1) == \
        gated(m=2 ** 40) == gated(wg=None) == gated(kept=ws.data_ptr() + 8) == _ext.SSC_EINVAL
    assert gated(bytes=0) == _ext.SSC_EWORKSPACE
    assert gated(m=0, x=None) == 0
    table = _ext.adamw_table([[x.data_ptr()]] + [None] * 5 + [[32], [0]], 1)
    bad = table.buffer_info()[0]
    assert lib.ssc_adamw_step(bad, 1, 32, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None) == _ext.SSC_EINVAL
    assert lib.ssc_adamw_step(None, 1, 32, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None) == _ext.SSC_EINVAL
    assert lib.ssc_adamw_step(None, 0, 16, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None) == _ext.SSC_EINVAL
    assert lib.ssc_adamw_step(None, 0, 8, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None) == 0
    assert math.isfinite(float(x.sum()))


@pytest.mark.parametrize("rows", [60, 6000])  # one launch, and passes over chunks
def test_norm_of_squares_beyond_float(rows):
    """Deviations whose squares pass float have an infinite variance: the bias is left."""
    x, offsets, dy = norm_inputs([rows, rows], 16, torch.float32, 4)
    want = group_norm(x, offsets, 2)
    big = x.clone()
    big[:rows, :8] *= 1e25
    bias = normal((16,), 3)
    got = group_norm(big.requires_grad_(), offsets, 2, None, bias)
    assert torch.equal(got[:rows, :8], bias[:8].expand(rows, 8))
    assert torch.equal(got[rows:] - bias, group_norm(x, offsets, 2, None, bias)[rows:] - bias)
    assert want.isfinite().all()
    dx, = torch.autograd.grad(got, big, dy)
    assert not dx[:rows, :8].any() and dx.isfinite().all()


@pytest.mark.parametrize("most", [1, 3])  # rows of a cloud: one launch, and passes over chunks
def test_norm_of_more_groups_than_a_launch_has(most):
    """40000 clouds of 64 groups are more workgroups than go into one grid."""
    clouds, c, groups = 40000, 128, 64
    size = torch.randint(0, most + 1, (clouds,), generator=torch.Generator().manual_seed(1))
    if most == 1:
        size[16000:39000] = 0  # (few rows)
    ends = size.cumsum(0)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).cuda()
    n = int(ends[-1])
    x, dy = normal((n, c), 2), normal((n, c), 3)
    cloud = torch.repeat_interleave(torch.arange(clouds), size).cuda()

    def mean_of(v):  # over the group of every element
        s = torch.zeros(clouds, groups, dtype=torch.float64, device="cuda")
        s.index_add_(0, cloud, v.view(n, groups, -1).sum(2))
        return (s / (size.clamp(min=1).cuda()[:, None] * (c // groups)))[cloud].repeat_interleave(
            c // groups, 1)

    x64, g64 = x.double(), dy.double()
    d = x64 - mean_of(x64)
    rstd = 1 / torch.sqrt(mean_of(d * d) + 1e-2)
    h = d * rstd
    dx64 = rstd * (g64 - mean_of(g64) - h * mean_of(g64 * h))
    x.requires_grad_()
    y = group_norm(x, offsets, groups, eps=1e-2)
    dx, = torch.autograd.grad(y, x, dy)
    # sums of at most 6 values; |x|, |dy| below 6, rstd at most 10 and |h| below 3: a few units of
    # float32 of the values at hand
    within(y, h, rstd * 2.0 ** -19 + h.abs() * rstd * 2.0 ** -19, "y")
    within(dx, dx64, (1 + rstd) ** 3 * 2.0 ** -16, "dx")


def pointwise_calls(dtype=torch.float32):
    """(function, its differentiable arguments) of both layers, on a few rows."""
    x, offsets, _ = norm_inputs([9, 4], 16, dtype, 2)
    w, b = normal((16,), 3, dtype, 0.3, 1.0), normal((16,), 4, dtype)
    wg, wu, bg = [normal(s, 5 + i, dtype, 0.3) for i, s in enumerate(((24, 16), (24, 16), (24,)))]
    return [(lambda p, q, r: group_norm(p, offsets, 4, q, r, activation="silu"), (x, w, b)),
            (lambda p, q, r, s: gated_linear(p, q, r, s), (x, wg, wu, bg))]


@pytest.mark.parametrize("which", [0, 1])
def test_pointwise_autograd_rules(which):
    call, args = pointwise_calls()[which]
    leaves = [t.clone().requires_grad_() for t in args]
    y = call(*leaves)
    want = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    # the same again, and for any of the inputs alone
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y.sum(), leaves), want))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y.sum(), leaves)
    for i, t in enumerate(leaves):
        assert torch.equal(torch.autograd.grad(call(*leaves).sum(), t)[0], want[i])
    # once differentiable: what a gradient is made from is no constant
    first = torch.autograd.grad(call(*leaves).sum(), leaves, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, want))
    with pytest.raises(RuntimeError, match="differentiate"):
        torch.autograd.grad(first[0].sum(), leaves)
    # changed in place between forward and backward
    z = [t.clone() for t in leaves]
    y = call(*z)
    with torch.no_grad():
        z[0].add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    # no forward mode, which would lose its tangents without a word
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(RuntimeError):
            call(dual, *args[1:])
    with torch.inference_mode():
        assert torch.equal(call(*args), call(*leaves))
    with torch.no_grad():
        assert not call(*leaves).requires_grad
    assert not call(*args).requires_grad


@pytest.mark.parametrize("which", [0, 1])
def test_pointwise_checkpoint_hooks_and_accumulation(which):
    from torch.utils.checkpoint import checkpoint
    call, args = pointwise_calls()[which]
    leaves = [t.clone().requires_grad_() for t in args]
    want = torch.autograd.grad(call(*leaves).sum(), leaves)
    y = checkpoint(call, *leaves, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y.sum(), leaves), want))
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.cpu()) or len(kept) - 1,
                                                  lambda i: kept[i].cuda()):
        y = call(*leaves)
    assert len(kept) >= 4  # all that the backward pass reads goes through the hooks
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y.sum(), leaves), want))
    for _ in range(2):
        call(*leaves).sum().backward()
    assert all(torch.equal(t.grad, 2 * g) for t, g in zip(leaves, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,h", [(33, 200, 40), (48, 1000, 24), (70, 264, 130), (96, 77, 33),
                                   (97, 136, 64), (130, 320, 48), (17, 640, 16), (20, 1100, 50)])
def test_gated_few_rows_in_blocks(m, k, h, dtype):
    """Blocks of 16, 32, 48 and 64 rows, steps along k that some waves have and others do not."""
    x, dy = normal((m, k), 1, dtype), normal((m, h), 2, dtype)
    wg, wu = normal((h, k), 3, dtype, k ** -0.5), normal((h, k), 4, dtype, k ** -0.5)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    y = gated_linear(*leaves, activation="silu")
    a, b = [x.detach().double() @ w.detach().double().t() for w in (wg, wu)]
    f = act64("silu", a)
    mag_a, mag_b = [x.detach().double().abs() @ w.detach().double().abs().t() for w in (wg, wu)]
    e_a, e_b = gamma(k) * mag_a, gamma(k) * mag_b
    e_f = 1.2 * e_a + act_error(a) * (f.abs() + e_a)
    within(y, f * b, U[dtype] * (f * b).abs() + TINY[dtype] + 2 * (e_f * (b.abs() + e_b) + f.abs() * e_b),
           "y")
    assert torch.equal(y.detach(), gated_linear(*[t.detach() for t in leaves]))
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(g.shape == t.shape and g.isfinite().all() for g, t in zip(grads, leaves))
