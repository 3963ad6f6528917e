"""AdamW over all parameters of a model in one launch, moments in 32 bits or in 8.

    m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

in float32 whatever the parameters' type (float32, float16, bfloat16; those of 16 bits are
rounded once, to nearest).  Moments in 8 bits take 1/4 of the memory: 256 neighbouring elements
of a tensor share a float32 scale q, m = q c |c| with an int8 c, sqrt(v) = q c^2 with a uint8 c
that is at least 1 where v > 0.  A gradient that is no finite number makes its element NaN, and
with 8-bit moments the block it lies in from the next step on.

Sparse gradients, gradients of another type than their parameter and tensors whose elements do not
fill their memory one after another are refused.  The number of the step is an argument of the
launch: a step cannot be captured into a graph and replayed.
"""
import torch

from ss_conv import _ext
from ss_conv import pointwise

BLOCK = 256  # elements that share a scale


def _dense(t):
    """Whether the elements of `t` fill a stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    dims = sorted((s, n) for n, s in zip(t.shape, t.stride()) if n != 1)
    at = 1
    for s, n in dims:
        if s != at:
            return False
        at *= n
    return True


def _like(t, p):
    """`t` with its elements in the order in which those of p lie in memory."""
    if t.stride() == p.stride():
        return t
    return torch.empty_like(p).copy_(t)


def _check_param(i, p, g):
    if p.layout is not torch.strided or g.layout is not torch.strided:
        raise RuntimeError("parameter {}: sparse tensors are not supported".format(i))
    if p.dtype not in _ext.ELEM:
        raise TypeError("parameter {} has type {}: float32, float16 and bfloat16 are "
                        "supported".format(i, p.dtype))
    if g.dtype is not p.dtype or g.shape != p.shape:
        raise ValueError("parameter {}: gradient of {} {}, parameter of {} {}".format(
            i, g.dtype, tuple(g.shape), p.dtype, tuple(p.shape)))
    _ext._need_gpu(p, g)
    if not _dense(p):
        raise ValueError("parameter {}: its elements do not fill their memory".format(i))


def _check_moments(i, n, dev, items, dtypes, sizes):
    for t, dtype, size in zip(items, dtypes, sizes):
        if t.dtype is not dtype or t.numel() != size:
            raise ValueError("moments of tensor {}: {} elements of {}, not {} of {}".format(
                i, t.numel(), t.dtype, size, dtype))
        if t.device != dev:
            raise RuntimeError("moments of tensor {} are on {}, not on {}".format(i, t.device, dev))
        if not _dense(t):
            raise ValueError("moments of tensor {}: their elements do not fill their "
                             "memory".format(i))


def _check_order(i, p, items):
    for t in items:
        if t.shape != p.shape or (t.stride() != p.stride() and
                                  not (t.is_contiguous() and p.is_contiguous())):
            raise ValueError("moments of tensor {} are laid out as {} {}, their parameter as "
                             "{} {}".format(i, tuple(t.shape), t.stride(), tuple(p.shape),
                                            p.stride()))


_BITS8 = (torch.int8, torch.uint8, torch.float32, torch.float32)
_BITS32 = (torch.float32, torch.float32)


def _scales(n):
    return -(-n // BLOCK)


def adamw_(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
           weight_decay=1e-2, exp_avg_scales=None, exp_avg_sq_scales=None):
    """One AdamW step over lists of tensors, all on one device, in place.

    exp_avgs, exp_avg_sqs: the moments, float32 and of the shape and strides of their parameter;
    or, with exp_avg_scales and exp_avg_sq_scales (float32, one for each 256 elements in the order
    in which they lie in memory), int8 and uint8 codes.  step: the number of this step, from 1.
    Tensors must not share memory."""
    eight = exp_avg_scales is not None
    if eight != (exp_avg_sq_scales is not None):
        raise ValueError("8-bit moments have scales for both, 32-bit ones have none")
    count = len(params)
    lists = [grads, exp_avgs, exp_avg_sqs] + ([exp_avg_scales, exp_avg_sq_scales] if eight else [])
    if any(len(x) != count for x in lists):
        raise ValueError("{} parameters with lists of {} tensors".format(
            count, [len(x) for x in lists]))
    if count == 0:
        return
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("an AdamW step cannot be captured into a graph: the number of the step "
                           "is an argument of its launch")
    if pointwise.binding.adamw(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales,
                               exp_avg_sq_scales, step, lr, betas[0], betas[1], eps,
                               weight_decay):
        return
    # something needs a look
    dtypes = _BITS8 if eight else _BITS32
    dev = params[0].device
    lists[0] = grads = list(grads)
    for i, p in enumerate(params):
        _check_param(i, p, grads[i])
        if p.device != dev or grads[i].device != dev:
            raise RuntimeError("parameter {} is on {}, its gradient on {}, the first on "
                               "{}".format(i, p.device, grads[i].device, dev))
        n = p.numel()
        _check_moments(i, n, dev, [x[i] for x in lists[1:]], dtypes,
                       (n, n, _scales(n), _scales(n)))
        _check_order(i, p, [x[i] for x in lists[1:3]])
        grads[i] = _like(grads[i], p)
    columns = [map(torch.Tensor.data_ptr, x) for x in [params] + lists]
    if not eight:
        columns += [None, None]
    columns += [map(torch.Tensor.numel, params), [_ext.ELEM[p.dtype] for p in params]]
    _ext.call_on(params[0], _ext.adamw_step, columns, count, 8 if eight else 32, lr, betas[0],
                 betas[1], eps, weight_decay, step, _ext._raw_stream(dev.index))
    torch.autograd.graph.increment_version(params)


def state_values(exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, out=None):
    """The float32 moments that lists of 8-bit ones stand for: (exp_avgs, exp_avg_sqs).
    out: the two lists of float32 tensors, laid out as the moments, to write them to."""
    count = len(exp_avgs)
    lists = [exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales] + (list(out) if out is not None else [])
    if any(len(x) != count for x in lists):
        raise ValueError("{} moments with lists of {} tensors".format(count,
                                                                      [len(x) for x in lists]))
    if count == 0:
        return [], []
    dev = exp_avgs[0].device
    _ext._need_gpu(exp_avgs[0])
    if out is None:
        out = tuple([torch.empty_like(t, dtype=torch.float32) for t in x]
                    for x in (exp_avgs, exp_avg_sqs))
    moments = [exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales]
    if pointwise.binding.adamw_values(*out, *moments):
        return tuple(out)
    # something needs a look
    sizes = [t.numel() for t in exp_avgs]
    for i, n in enumerate(sizes):
        _check_moments(i, n, dev, [x[i] for x in moments], _BITS8,
                       (n, n, _scales(n), _scales(n)))
        _check_moments(i, n, dev, (out[0][i], out[1][i]), _BITS32, (n, n))
        # (a new tensor has the layout of the codes, a given one has to have it)
        _check_order(i, exp_avgs[i], (exp_avg_sqs[i], out[0][i], out[1][i]))
    columns = [map(torch.Tensor.data_ptr, x) for x in list(out) + moments]
    columns += [sizes, None]
    _ext.call_on(exp_avgs[0], _ext.adamw_values, columns, count, _ext._raw_stream(dev.index))
    return tuple(out)


class AdamW(torch.optim.Optimizer):
    """torch.optim.Optimizer with adamw_ as its step; state_bits: 32 or 8, for each group.

    state[p] holds step, exp_avg and exp_avg_sq, with 8 bits also exp_avg_scale and
    exp_avg_sq_scale."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 state_bits=32):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                        state_bits=state_bits)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        group = dict(self.defaults, **param_group)
        for key in ("lr", "eps", "weight_decay"):
            if not float(group[key]) >= 0:
                raise ValueError("{} = {} is negative".format(key, group[key]))
        if len(group["betas"]) != 2 or not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError("betas = {} are not in [0, 1)".format(group["betas"]))
        if group["state_bits"] not in (32, 8):
            raise ValueError("state_bits = {}: 32 and 8 are supported".format(group["state_bits"]))
        super().add_param_group(param_group)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # torch casts the state to the parameter's type; moments, codes and scales keep theirs and
        # the parameter's order in memory
        given = [i for g in state_dict["param_groups"] for i in g["params"]]
        held = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(given, held):
            for key, t in state_dict["state"].get(i, {}).items():
                if not torch.is_tensor(t):
                    continue
                if t.shape != p.shape or t.dim() < 2:
                    self.state[p][key] = t.to(device=p.device, copy=True)
                    continue
                if t.dtype is not torch.float32 and t.stride() != p.stride():
                    raise ValueError("8-bit moments of a parameter with the strides {} do not fit "
                                     "one with {}".format(t.stride(), p.stride()))
                self.state[p][key] = torch.empty_like(p, dtype=t.dtype).copy_(t)

    def _init(self, p, bits):
        s = self.state[p]
        s["step"] = 0
        if bits == 32:
            s["exp_avg"] = torch.zeros_like(p, dtype=torch.float32,
                                            memory_format=torch.preserve_format)
            s["exp_avg_sq"] = torch.zeros_like(s["exp_avg"])
        else:
            s["exp_avg"] = torch.zeros_like(p, dtype=torch.int8,
                                            memory_format=torch.preserve_format)
            s["exp_avg_sq"] = torch.zeros_like(s["exp_avg"], dtype=torch.uint8)
            for key in ("exp_avg_scale", "exp_avg_sq_scale"):
                s[key] = torch.zeros(_scales(p.numel()), dtype=torch.float32, device=p.device)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            bits = group["state_bits"]
            together = {}  # by device and number of steps
            for i, p in enumerate(group["params"]):
                if p.grad is None:
                    continue
                if len(self.state[p]) == 0:
                    _check_param(i, p, p.grad)
                    self._init(p, bits)
                s = self.state[p]
                if ("exp_avg_scale" in s) != (bits == 8):
                    raise ValueError("parameter {} has moments of {} bits, its group asks for "
                                     "{}".format(i, 8 if bits == 32 else 32, bits))
                together.setdefault((p.device, s["step"]), []).append(p)
            for (_, done), ps in together.items():
                states = [self.state[p] for p in ps]
                more = {}
                if bits == 8:
                    more = dict(exp_avg_scales=[s["exp_avg_scale"] for s in states],
                                exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states])
                adamw_(ps, [p.grad for p in ps], [s["exp_avg"] for s in states],
                       [s["exp_avg_sq"] for s in states], done + 1, float(group["lr"]),
                       group["betas"], group["eps"], group["weight_decay"], **more)
                for s in states:
                    s["step"] = done + 1
        return loss
