"""What the pointwise operators (groupnorm.py, feedforward.py) check in common."""
import torch

from ss_conv import _ext

try:
    from ss_conv import _pointwise as binding  # (csrc/pointwise_torch.cpp)
except ImportError as e:
    raise ImportError("ss_conv/_pointwise.so is not built, or not for this torch: run `python "
                      "ss-conv_amd/build.py --force`") from e

_NAMES = {None: _ext.ACT_NONE, "none": _ext.ACT_NONE, "relu": _ext.ACT_RELU,
          "sigmoid": _ext.ACT_SIGMOID, "tanh": _ext.ACT_TANH, "silu": _ext.ACT_SILU,
          "gelu": _ext.ACT_GELU}
_CALLABLES = {torch.relu: "relu", torch.nn.functional.relu: "relu", torch.sigmoid: "sigmoid",
              torch.nn.functional.sigmoid: "sigmoid", torch.tanh: "tanh",
              torch.nn.functional.tanh: "tanh", torch.nn.functional.silu: "silu",
              torch.nn.functional.gelu: "gelu"}


def activation_name(fn):
    """Name of an activation given by its name (None, "none", "relu", "sigmoid", "tanh", "silu",
    "gelu": the one with the error function), as a torch function or as a torch.nn module."""
    if fn is None or isinstance(fn, str):
        if fn in _NAMES:
            return fn or "none"
    elif isinstance(fn, torch.nn.Module):
        for cls, name in ((torch.nn.Identity, "none"), (torch.nn.ReLU, "relu"),
                          (torch.nn.Sigmoid, "sigmoid"), (torch.nn.Tanh, "tanh"),
                          (torch.nn.SiLU, "silu"), (torch.nn.GELU, "gelu")):
            if type(fn) is cls and getattr(fn, "approximate", "none") == "none":
                return name
    else:
        for known, name in _CALLABLES.items():
            if fn is known:
                return name
    raise ValueError("activation {!r} is none of {}".format(
        fn, ", ".join(str(k) for k in _NAMES)))


def activation_code(fn):
    """The kernels' code of an activation (see activation_name)."""
    code = _NAMES.get(fn) if fn is None or isinstance(fn, str) else None
    return _NAMES[activation_name(fn)] if code is None else code


def check_rows(what, x):
    """Floating-point rows on the GPU, of a type the kernels know."""
    if not torch.is_tensor(x):
        raise TypeError("{} is a {}, not a tensor".format(what, type(x).__name__))
    _ext._need_gpu(x)
    if x.dtype not in _ext.ELEM:
        raise TypeError("{} has type {}: float32, float16 and bfloat16 are supported".format(
            what, x.dtype))


def check_like(what, t, shape, dtypes, device):
    """An optional tensor of a given shape, type and device."""
    if t is None or (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype in dtypes and
                     t.device == device):
        return
    if not torch.is_tensor(t):
        raise TypeError("{} is a {}, not a tensor".format(what, type(t).__name__))
    if tuple(t.shape) != tuple(shape):
        raise ValueError("{} has shape {}, not {}".format(what, tuple(t.shape), tuple(shape)))
    if t.dtype not in dtypes:
        raise TypeError("{} has type {}, not {}".format(
            what, t.dtype, " or ".join(str(d) for d in dict.fromkeys(dtypes))))
    if t.device != device:
        raise RuntimeError("{} is on {}, the rows are on {}".format(what, t.device, device))


def check_taken(y):
    """What the binding makes of arguments that have been checked and laid out."""
    if y is None:
        raise RuntimeError("tensors of this kind or size are not supported")
