"""Gated feed-forward blocks on voxel rows.

    y = act(x w_gate^T + b_gate) * (x w_up^T + b_up)

Both projections, the activation and the product are one kernel (`ssc_gated_fwd`), the gradients
come from hand-written kernels too (`ssc_gated_bwd`): float32, float16 and bfloat16, sums in
float32, one rounding of the result.  A training step keeps both projections for the backward
pass, in 24 bits for 16-bit types and in 32 for floats.

A block mixes the channels of a row: use it on scalar (order 0) fields, where that keeps the
network equivariant.
"""
import math

import torch
import torch.nn as nn

from ss_conv import pointwise


def _at_16_bytes(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """activation(x w_gate^T + b_gate) * (x w_up^T + b_up) for x [..., K] and weights [H, K].

    All tensors have one type (float32, float16 or bfloat16); biases [H] or None.
    activation: a name (None, "relu", "sigmoid", "tanh", "silu", "gelu"), the torch function or the
    torch.nn module of one.  Differentiable once in everything."""
    act = pointwise.activation_code(activation)
    y = pointwise.binding.gated_linear(x, w_gate, w_up, b_gate, b_up, act)
    if y is None:  # something needs a look
        y = pointwise.binding.gated_linear(*_laid_out(x, w_gate, w_up, b_gate, b_up), act)
        pointwise.check_taken(y)
        if x.dim() != 2:
            y = y.view(x.shape[:-1] + y.shape[-1:])
    return y


def _laid_out(x, w_gate, w_up, b_gate, b_up):
    """Checks gated_linear's arguments and lays them out as the kernels want them."""
    pointwise.check_rows("x", x)
    if x.dim() < 1:
        raise ValueError("x has no dimension")
    if not torch.is_tensor(w_gate) or w_gate.dim() != 2 or w_gate.size(0) < 1 or \
            w_gate.size(1) < 1:
        raise ValueError("w_gate is a matrix [hidden, width]")
    h, k = w_gate.shape
    if x.size(-1) != k:
        raise ValueError("x has {} columns, w_gate {}".format(x.size(-1), k))
    for what, t, shape in (("w_gate", w_gate, (h, k)), ("w_up", w_up, (h, k)),
                           ("b_gate", b_gate, (h,)), ("b_up", b_up, (h,))):
        pointwise.check_like(what, t, shape, (x.dtype,), x.device)
    if w_up is None:
        raise TypeError("w_up is missing")
    b_gate, b_up = [None if t is None else t.contiguous() for t in (b_gate, b_up)]
    return [_at_16_bytes(t) for t in (x.reshape(-1, k), w_gate, w_up)] + [b_gate, b_up]


class GatedLinear(nn.Module):
    """gated_linear with its parameters: width columns in, hidden columns out."""

    def __init__(self, width, hidden, bias=False, activation="silu"):
        super().__init__()
        self.width, self.hidden = width, hidden
        self.activation = pointwise.activation_name(activation)
        self.w_gate = nn.Parameter(torch.empty(hidden, width))
        self.w_up = nn.Parameter(torch.empty(hidden, width))
        for name in ("b_gate", "b_up"):
            self.register_parameter(name, nn.Parameter(torch.empty(hidden)) if bias else None)
        self.reset_parameters()

    def reset_parameters(self):
        bound = 1 / math.sqrt(self.width)
        for p in self.parameters():
            nn.init.uniform_(p, -bound, bound)

    def extra_repr(self):
        return "{} -> {}, bias={}, activation={}".format(self.width, self.hidden,
                                                         self.b_gate is not None, self.activation)

    def forward(self, x):
        return gated_linear(x, self.w_gate, self.w_up, self.b_gate, self.b_up, self.activation)


class GatedFeedForward(nn.Module):
    """x + w_down gated(norm(x)) on the features of a SparseTensor: the residual block of a
    pointwise network.  norm: a module on SparseTensors (groupnorm.GroupNorm, batchnorm.BatchNorm)
    or None; the projection back is a plain torch.nn.Linear."""

    def __init__(self, width, hidden, norm=None, bias=False, activation="silu"):
        super().__init__()
        self.norm = norm
        self.gated = GatedLinear(width, hidden, bias, activation)
        self.down = nn.Linear(hidden, width, bias=bias)

    def forward(self, input):  # pylint: disable=W
        x = input.features
        rows = input if self.norm is None else self.norm(input)
        input.features = x + self.down(self.gated(rows.features))
        return input
