"""Group norm with an activation on sparse tensors, channels last.

The channels of a voxel row are cut into groups of neighbours; every cloud of the batch (rows
offsets[b] to offsets[b + 1]) and group is normalised by its own mean and variance, so the
result depends neither on the other clouds nor on running statistics, in training as in
evaluation.  Forward and backward run on the library's kernels (`ssc_groupnorm_fwd`,
`ssc_groupnorm_bwd`): float32, float16 and bfloat16 rows, statistics in float32 or more, one
rounding of every result.  Only the rows and the statistics are kept for the backward pass.

The mean of a group mixes its channels: use it on scalar (order 0) fields, where that keeps the
network equivariant; `ss_conv.batchnorm.BatchNorm` is the norm of fields of higher order.
"""
import torch
import torch.nn as nn

from ss_conv import pointwise


def group_norm(x, offsets, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """activation(weight * (x - mean) / sqrt(var + eps) + bias) for rows x [N, C].

    offsets: [clouds + 1] whole numbers on the device of x, ascending from 0 to N (what
    SparseTensor.get_offsets returns; int32 is used as it is).  Clouds may be empty.
    weight, bias: [C], of the type of x or float32 (both the same), or None.
    activation: a name (None, "relu", "sigmoid", "tanh", "silu", "gelu"), the torch function or
    the torch.nn module of one.
    Differentiable once in x, weight and bias."""
    act = pointwise.activation_code(activation)
    y = pointwise.binding.group_norm(x, offsets, num_groups, weight, bias, eps, act)
    if y is None:  # something needs a look
        x, offsets, weight, bias = _laid_out(x, offsets, num_groups, weight, bias, eps)
        y = pointwise.binding.group_norm(x, offsets, num_groups, weight, bias, eps, act)
        pointwise.check_taken(y)
    return y


def _laid_out(x, offsets, num_groups, weight, bias, eps):
    """Checks group_norm's arguments and lays them out as the kernels want them."""
    pointwise.check_rows("x", x)
    if x.dim() != 2:
        raise ValueError("x has {} dimensions, not 2".format(x.dim()))
    n, c = x.shape
    if num_groups < 1 or c < 1 or c % num_groups != 0:
        raise ValueError("{} channels cannot be cut into {} groups".format(c, num_groups))
    if not eps >= 0:
        raise ValueError("eps = {} is negative".format(eps))
    if not torch.is_tensor(offsets) or offsets.dim() != 1 or offsets.is_floating_point() or \
            offsets.is_complex() or offsets.dtype == torch.bool:
        raise TypeError("offsets is a vector of whole numbers")
    if offsets.numel() < (2 if n > 0 else 1):
        raise ValueError("offsets has {} elements for {} rows".format(offsets.numel(), n))
    if offsets.device != x.device:
        raise RuntimeError("offsets is on {}, the rows are on {}".format(offsets.device, x.device))
    kinds = (x.dtype, torch.float32)
    pointwise.check_like("weight", weight, (c,), kinds, x.device)
    pointwise.check_like("bias", bias, (c,), kinds, x.device)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight has type {}, bias {}".format(weight.dtype, bias.dtype))
    weight, bias = [None if t is None else t.contiguous() for t in (weight, bias)]
    return x.contiguous(), offsets.to(torch.int32).contiguous(), weight, bias


class GroupNorm(nn.Module):
    """group_norm on the features of a SparseTensor whose rows are grouped by batch index in
    ascending order (as Point2Voxel and Convolution return them).

    num_groups groups of num_channels channels; weight and bias [num_channels] with affine."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None):
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups != 0:
            raise ValueError("{} channels cannot be cut into {} groups".format(num_channels,
                                                                               num_groups))
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.eps = eps
        self.affine = affine
        self.activation = pointwise.activation_name(activation)
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels))
            self.bias = nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter('weight', None)
            self.register_parameter('bias', None)

    def __repr__(self):
        return "{} ({} groups of {} channels, eps={}, affine={}, activation={})".format(
            self.__class__.__name__, self.num_groups, self.num_channels, self.eps, self.affine,
            self.activation)

    def forward(self, input):  # pylint: disable=W
        x = input.features
        if x.size(1) != self.num_channels:
            raise ValueError("features have {} channels, the norm {}".format(
                x.size(1), self.num_channels))
        input.features = group_norm(x, input.get_offsets(), self.num_groups, self.weight,
                                    self.bias, self.eps, self.activation)
        return input
