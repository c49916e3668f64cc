"""Dense layers over the rows that the tables hold: heads that decode features, trained with them and served.

    fused_linear   y = act(x W^T + b) + r          one launch; gradients of x, W, b and r
    rms_norm       s = x + r,  y = s / sqrt(mean(s^2) + eps) * w          one launch, y in 8 bits if wanted; gradients

and the modules built from them (the reference keeps its MLP helpers in a file of this name, ash/mlp.py):
``Linear``, ``MLP``, ``SirenLayer``, ``SirenNet`` and ``ResidualMLP``, which can be served in 8 bits.

Types are float32, float16 and bfloat16, the same for all tensors of a call; sums and statistics are float32 and a result
is rounded once.  float32 layers are as exact as float32 sums (their factors are multiplied as exact sums of three
bfloat16 parts), except that an infinity among x or W makes NaN of what it touches.  Both functions are differentiable
any number of times: a backward pass that is itself recorded (``create_graph=True``) is composed of the same functions and
elementwise ones.

A training step may be captured in a CUDA graph under the conditions that torch puts on any: run it a few times on a side
stream first, and let the outputs of those runs go before the capture, since autograd otherwise meets the leaves'
accumulation on the stream that they were made for and the capture fails.
"""
import math
from typing import List, Optional, Tuple, Union

import torch
import torch.nn as nn

from .common import _get_c_extension
from .quant import QuantizedRows, VALUE_TYPES, quantize_rows

backend = _get_c_extension()

ACTIVATIONS = ("none", "relu", "silu", "gelu", "sin")


# ------------------------------------------------------------------------------------------------ checks
def _check_like(t: Optional[torch.Tensor], name: str, shape, like: torch.Tensor, dtype: torch.dtype) -> None:
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype} as the other tensors of the call, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, x on {like.device}")


def _check_value(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in VALUE_TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")


def _check_activation(activation: str, omega: float) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, got {activation!r}")
    if not math.isfinite(omega):
        raise ValueError(f"omega must be finite, got {omega}")


def _recorded(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


_transforms_open = getattr(backend, "transforms_open", lambda: False)


def _refuse_tangents(*tensors) -> None:
    """Forward-mode derivatives are not computed: rather than dropped without a word they are refused."""
    if _transforms_open():
        for t in tensors:
            if t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("forward-mode derivatives of dense layers and norms are not implemented")


# ------------------------------------------------------------------------------------------------ dense layer
def _slope(z: torch.Tensor, activation: str, omega: float) -> torch.Tensor:
    """act'(z) of the activations that have a second derivative, by elementwise operations that autograd records."""
    if activation == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    if activation == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return omega * torch.cos(omega * z)


class _FusedLinear(torch.autograd.Function):
    """2-D x and residual."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, omega):
        # relu without a residual: the output's sign is its slope
        sign = activation == "relu" and residual is None
        with_slope = activation != "none" and not sign
        y, slope = backend.linear_forward(x, weight, bias, activation, residual, omega, with_slope)
        ctx.activation, ctx.omega = activation, omega
        ctx.kind = 0 if activation == "none" else 2 if activation == "relu" else 1      # relu: by sign
        ctx.has_bias = bias is not None
        ctx.save_for_backward(x, weight, bias, y if sign else slope)
        return y

    @staticmethod
    def backward(ctx, grad):
        x, weight, bias, slope = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dr = grad if want_r else None
        if torch.is_grad_enabled():
            dz = grad
            if ctx.activation == "relu":      # the saved sign: its slope has no derivative
                dz = torch.where(slope.detach() > 0, grad, 0)
            elif ctx.kind == 1:
                # The formula in float32, and of the float32 sum, as the slope is without recording: a sum rounded to 16 bits
                # first is off by up to 2^-8 of itself, times omega in a sine's phase (omega 30, bf16: 9 % of the slope, against 0.2 %).
                # The casts keep 16-bit factors what they are; the product of float32 rows is the price.
                z = fused_linear(x.float(), weight.float(), None if bias is None else bias.float())
                dz = (grad.float() * _slope(z, ctx.activation, ctx.omega)).to(grad.dtype)
            dx = fused_linear(dz, weight.t()) if want_x else None
            # without rows there is no product to take
            dw = (fused_linear(dz.t(), x.t()) if x.shape[0] else torch.zeros_like(weight)) if want_w else None
            db = dz.float().sum(0).to(dz.dtype) if want_b else None
        elif want_x or want_w or want_b:
            dx, dw, db = backend.linear_backward(grad, slope, ctx.kind, x, weight, want_x, want_w, want_b)
        else:
            dx = dw = db = None
        return dx, dw, db, dr, None, None


def fused_linear(x: Union[torch.Tensor, QuantizedRows], weight: Union[torch.Tensor, QuantizedRows],
                 bias: Optional[torch.Tensor] = None, activation: str = "none", residual: Optional[torch.Tensor] = None,
                 omega: float = 1.0, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one launch.

    x (..., inputs), weight (outputs, inputs), bias (outputs), residual (..., outputs); ``activation`` is ``"none"``,
    ``"relu"``, ``"silu"``, ``"gelu"`` (with erf) or ``"sin"`` (sin(omega z)).

    With x and weight both ``QuantizedRows`` in e4m3 (a scale a row each) the product is taken of the codes and the
    result, bias and residual are of ``dtype`` (bfloat16 if not given); that form is for serving and has no gradient.
    """
    _check_activation(activation, omega)
    if isinstance(x, QuantizedRows) or isinstance(weight, QuantizedRows):
        if not (isinstance(x, QuantizedRows) and isinstance(weight, QuantizedRows)):
            raise ValueError("x and weight must both be QuantizedRows or both be tensors")
        return _quantized_linear(x, weight, bias, activation, residual, omega, dtype or torch.bfloat16)
    _check_value(x, "x")
    kept = x.dtype
    if dtype is not None and dtype != kept:
        raise ValueError(f"dtype is for QuantizedRows: the result of {kept} rows is {kept}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[-1] or weight.numel() == 0:
        raise ValueError(f"x (..., inputs) and weight (outputs, inputs) are wanted, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    outputs, flat = weight.shape[0], x.dim() == 2
    shape = (*x.shape[:-1], outputs)
    if weight.dtype is not kept or weight.device != x.device:
        _check_like(weight, "weight", weight.shape, x, kept)
    if bias is not None:
        _check_like(bias, "bias", (outputs,), x, kept)
    if residual is not None:
        _check_like(residual, "residual", shape, x, kept)
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    r2 = residual if residual is None or flat else residual.reshape(-1, outputs)
    if _recorded(x, weight, bias, residual):
        y = _FusedLinear.apply(x2, weight, bias, r2, activation, float(omega))
    else:
        _refuse_tangents(x, weight, bias, residual)
        y = backend.linear_forward(x2, weight, bias, activation, r2, float(omega), False)[0]
    return y if flat else y.reshape(shape)


def check_waits(device: Union[None, int, str, torch.device] = None) -> None:
    """Wait for ``device`` (the current one) and raise ``RuntimeError`` if a layer's kernel gave up on a wait there since this was
    last asked: what that layer returned is incomplete.  The waits inside the kernels are bounded, by seconds where they
    take microseconds, so that a launch always ends.  Layers called later raise the same without waiting; for work
    that no call follows, or that a replayed CUDA graph does, ask here."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device("cuda", device) \
        if isinstance(device, int) else torch.device(device)
    count = backend.layer_timeouts(device)
    if count:
        raise RuntimeError(f"waits inside the kernels of dense layers ran out in {count} thread blocks on {device}: what those layers "
                           "returned is incomplete")


def _quantized_linear(x, weight, bias, activation, residual, omega, dtype):
    x.check("x")
    weight.check("weight")
    if x.format != "e4m3" or weight.format != "e4m3":
        raise ValueError(f"x and weight must be e4m3 rows, got {x.format} and {weight.format}")
    if dtype not in VALUE_TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    if weight.codes.dim() != 2 or x.codes.shape[-1] != weight.codes.shape[1] or weight.codes.numel() == 0:
        raise ValueError(f"x (..., inputs) and weight (outputs, inputs) are wanted, got {tuple(x.codes.shape)} and "
                         f"{tuple(weight.codes.shape)}")
    if weight.codes.device != x.codes.device:
        raise ValueError(f"weight is on {weight.codes.device}, x on {x.codes.device}")
    shape = (*x.codes.shape[:-1], weight.codes.shape[0])
    _check_like(bias, "bias", shape[-1:], x.codes, dtype)
    _check_like(residual, "residual", shape, x.codes, dtype)
    if _recorded(bias, residual):
        raise RuntimeError("a product of QuantizedRows has no gradient: call it under torch.no_grad()")
    r2 = None if residual is None else residual.reshape(-1, shape[-1])
    y, _ = backend.linear_forward(x.codes.reshape(-1, x.codes.shape[-1]), weight.codes, bias, activation, r2, float(omega),
                                  False, scales=(x.scales.reshape(-1), weight.scales), out_dtype=dtype)
    return y.reshape(shape)


# ------------------------------------------------------------------------------------------------ norm
class _RMSNorm(torch.autograd.Function):
    """2-D x and residual; (y, s), s an output of its own only with a residual."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, _, total, rstd = backend.rms_norm_forward(x, weight, residual, eps, False, True)
        ctx.eps, ctx.has_residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, residual, total, rstd)
        return (y, total) if residual is not None else y

    @staticmethod
    def backward(ctx, dy, ds=None):
        x, weight, residual, total, rstd = ctx.saved_tensors
        if dy is None and ds is None:
            return None, None, None, None
        if dy is None:
            return ds, None, ds if ctx.has_residual else None, None
        if torch.is_grad_enabled():
            dx, dw = _composed_norm_gradients(x, weight, residual, ctx.eps, dy, ds)
            return dx, dw, dx if ctx.has_residual else None, None
        dx, dw = backend.rms_norm_backward(dy, ds, x if total is None else total, weight, rstd)
        return dx, dw, dx if ctx.has_residual else None, None


def _composed_norm_gradients(x, weight, residual, eps, dy, ds):
    """The gradients of x (and the residual) and of the weight, by elementwise operations that autograd records.  Written out:
    asking autograd for those of a composed norm would count what reaches x by way of a residual made from it twice."""
    s, g = x.float() if residual is None else x.float() + residual.float(), dy.float()
    # by the row's largest value, or the root of eps if that is larger: squares stay in range, and it cancels
    size = s.detach().abs().amax(1, keepdim=True).clamp_min(max(math.sqrt(eps), 2.0**-126))
    t = s / size
    r = torch.rsqrt((t * t).mean(1, keepdim=True) + eps / size / size)
    n, gw = t * r, g * weight.float()
    dx = (gw - n * (gw * n).mean(1, keepdim=True)) * (r / size)
    if ds is not None:
        dx = dx + ds.float()
    return dx.to(x.dtype), (g * n).sum(0).to(weight.dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
             quantize: bool = False):
    """Root-mean-square norm of the rows of x (..., width), or of ``s = x + residual``: ``s / sqrt(mean(s^2) + eps) *
    weight``.  Returns y, with a residual ``(y, s)``.

    ``quantize``: y comes as ``QuantizedRows`` in e4m3, the operand of ``fused_linear``; that form is for serving and has no
    gradient.  A row of zeros gives zeros (with an eps of 0 NaN, 0/0); a row that holds an infinity or a NaN gives NaN
    throughout; one of finite values has its norm, whether their squares are in float32's range or not.
    """
    _check_value(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one value, got {tuple(x.shape)}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    _check_like(weight, "weight", x.shape[-1:], x, x.dtype)
    _check_like(residual, "residual", x.shape, x, x.dtype)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    r2 = residual if residual is None or residual.dim() == 2 else residual.reshape(-1, x.shape[-1])
    if quantize:
        if _recorded(x, weight, residual):
            raise RuntimeError("a quantised norm has no gradient: call it under torch.no_grad()")
        _refuse_tangents(x, weight, residual)
        _, codes, scales, s, _ = backend.rms_norm_forward(x2, weight, r2, float(eps), True, False)
        y = QuantizedRows(codes.reshape(x.shape), scales.reshape(x.shape[:-1]))
        return y if residual is None else (y, s.reshape(x.shape))
    if _recorded(x, weight, residual):
        got = _RMSNorm.apply(x2, weight, r2, float(eps))
    else:
        _refuse_tangents(x, weight, residual)
        y, _, _, s, _ = backend.rms_norm_forward(x2, weight, r2, float(eps), False, False)
        got = y if residual is None else (y, s)
    if x.dim() == 2:
        return got
    if residual is None:
        return got.reshape(x.shape)
    return got[0].reshape(x.shape), got[1].reshape(x.shape)


# ------------------------------------------------------------------------------------------------ modules
class Linear(nn.Module):
    """``fused_linear`` with its parameters: ``weight`` (outputs, inputs) and ``bias``, uniform in +-1/sqrt(inputs), or
    for ``"sin"`` within the bound that keeps the variance of its phases (sqrt(6/inputs)/omega; 1/inputs for the first
    layer of a network)."""

    def __init__(self, inputs: int, outputs: int, bias: bool = True, activation: str = "none", omega: float = 1.0,
                 first: bool = False, device=None, dtype: torch.dtype = torch.float32):
        super().__init__()
        _check_activation(activation, omega)
        if inputs < 1 or outputs < 1:
            raise ValueError(f"a layer of {inputs} inputs and {outputs} outputs")
        self.activation, self.omega = activation, float(omega)
        bound = 1 / math.sqrt(inputs)
        if activation == "sin":
            bound = 1 / inputs if first else math.sqrt(6 / inputs) / omega
        self.weight = nn.Parameter(torch.empty(outputs, inputs, device=device, dtype=dtype).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(outputs, device=device, dtype=dtype).uniform_(-bound, bound)) if bias else None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return fused_linear(x, self.weight, self.bias, self.activation, residual, self.omega)

    def extra_repr(self) -> str:
        outputs, inputs = self.weight.shape
        return f"{inputs}, {outputs}, bias={self.bias is not None}, activation={self.activation!r}, omega={self.omega}"


class MLP(nn.Module):
    """``num_layers`` hidden layers and a last one.  ``residual``: hidden layers between equal widths add their input."""

    def __init__(self, dim_in: int, dim_hidden: int, dim_out: int, num_layers: int, use_bias: bool = True,
                 activation: str = "relu", final_activation: str = "none", residual: bool = False, device=None,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        if num_layers < 1:
            raise ValueError("at least one hidden layer is wanted")
        self.residual = residual
        widths = [dim_in] + [dim_hidden] * num_layers
        self.layers = nn.ModuleList(Linear(i, o, use_bias, activation, device=device, dtype=dtype)
                                    for i, o in zip(widths, widths[1:]))
        self.last_layer = Linear(dim_hidden, dim_out, use_bias, final_activation, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for layer in self.layers:
            same = self.residual and layer.weight.shape[0] == layer.weight.shape[1]
            x = layer(x, x if same else None)
        return self.last_layer(x)


class SirenLayer(Linear):
    """A sine layer: sin(w0 (x W^T + b))."""

    def __init__(self, dim_in: int, dim_out: int, w0: float = 30.0, is_first: bool = False, use_bias: bool = True,
                 activation: str = "sin", device=None, dtype: torch.dtype = torch.float32):
        super().__init__(dim_in, dim_out, use_bias, activation, w0, is_first, device, dtype)


class SirenNet(nn.Module):
    """``num_layers`` sine layers (frequency ``w0_initial`` in the first, ``w0`` after it) and a last layer.  Smooth, with
    gradients of any order, so positions can be supervised through them (an eikonal term)."""

    def __init__(self, dim_in: int, dim_hidden: int, dim_out: int, num_layers: int, w0: float = 1.0,
                 w0_initial: float = 30.0, use_bias: bool = True, final_activation: str = "none", device=None,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        if num_layers < 1:
            raise ValueError("at least one sine layer is wanted")
        self.layers = nn.ModuleList(
            SirenLayer(dim_in if i == 0 else dim_hidden, dim_hidden, w0_initial if i == 0 else w0, i == 0, use_bias,
                       device=device, dtype=dtype) for i in range(num_layers))
        self.last_layer = Linear(dim_hidden, dim_out, use_bias, final_activation, w0, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for layer in self.layers:
            x = layer(x)
        return self.last_layer(x)


class ResidualMLP(nn.Module):
    """A first layer, ``num_blocks`` blocks ``h <- h + W2 act(W1 norm(h))``, and a last layer on the normed sum.  The
    addition happens in the norm that follows it.  ``quantize_()`` keeps a copy of the blocks' weights in e4m3 and serves
    from it, the norms writing the 8-bit operands; calls that record gradients go on using the parameters."""

    def __init__(self, dim_in: int, dim_hidden: int, dim_out: int, num_blocks: int, expansion: int = 4,
                 activation: str = "silu", eps: float = 1e-6, device=None, dtype: torch.dtype = torch.float32):
        super().__init__()
        if num_blocks < 1 or expansion < 1:
            raise ValueError("at least one block and an expansion of one are wanted")
        make = lambda i, o, act="none": Linear(i, o, True, act, device=device, dtype=dtype)
        self.eps = eps
        self.first_layer = make(dim_in, dim_hidden)
        self.up = nn.ModuleList(make(dim_hidden, expansion * dim_hidden, activation) for _ in range(num_blocks))
        self.down = nn.ModuleList(make(expansion * dim_hidden, dim_hidden) for _ in range(num_blocks))
        self.norms = nn.ParameterList(nn.Parameter(torch.ones(dim_hidden, device=device, dtype=dtype))
                                      for _ in range(num_blocks + 1))
        self.last_layer = make(dim_hidden, dim_out)
        self._rows: Optional[List[Tuple[QuantizedRows, QuantizedRows]]] = None

    def quantize_(self, enable: bool = True) -> "ResidualMLP":
        """Serve the blocks in 8 bits from the weights as they are now (call it again after they change), or stop to."""
        self._rows = [(quantize_rows(u.weight), quantize_rows(d.weight)) for u, d in zip(self.up, self.down)] if enable else None
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        eight = self._rows is not None and not _recorded(x, *self.parameters())
        h, f = self.first_layer(x), None
        for i, (up, down) in enumerate(zip(self.up, self.down)):
            n = rms_norm(h, self.norms[i], f, self.eps, quantize=eight)
            if f is not None:
                n, h = n
            if eight:
                w1, w2 = self._rows[i]
                u = fused_linear(n, w1, up.bias, up.activation, omega=up.omega, dtype=h.dtype)
                f = fused_linear(quantize_rows(u), w2, down.bias, dtype=h.dtype)
            else:
                f = down(up(n))
        n, _ = rms_norm(h, self.norms[len(self.up)], f, self.eps)
        return self.last_layer(n)
