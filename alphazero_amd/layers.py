"""Network layers as single operators: `dense` and `layer_norm`, with their gradients.

The reference's networks are stacks of flax Dense layers and activations
(networks/networks.py:25-48, kernel [in, out], bias [out]); these are such layers, and the ones a
residual network puts around them, as HIP kernels of libaz_mcts.so (include/az_layers.h).  Float32,
bfloat16 and float16; sums are held in float32 and an output is rounded once.  There is no CPU path.
"""
import torch
from torch.autograd import forward_ad
from torch.fx.experimental import proxy_tensor

from . import _native as nat

DTYPES = {torch.float32: nat.TYPE_F32, torch.bfloat16: nat.TYPE_BF16, torch.float16: nat.TYPE_F16}
MAX_ROWS = 0x7fff0000   # rows and widths are 32-bit numbers in the C ABI
ACTIVATIONS = {None: nat.ACT_NONE, "relu": nat.ACT_RELU, "swish": nat.ACT_SWISH, "gelu": nat.ACT_GELU}


# the current stream's handle without the Stream object (a dozen microseconds in the autograd engine's thread)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _native(device, fn, *args):
    """Calls a native entry point on `device`, which it makes the current one (launches go to the current device's
    stream).  Tensor arguments are contiguous; they are passed as pointers."""
    args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index) if _raw_stream is not None else nat.stream_ptr())
    else:
        with torch.cuda.device(device):
            rc = fn(*args, nat.stream_ptr())
    if rc != 0:
        nat.check(rc)


# Whether torch.jit.trace or, by a dispatch mode, make_fx records the calls: they would see the outputs' allocation alone, and
# the recorded program would return memory that nothing has written.  (The quick forms of the public questions where there are
# such: a call costs ten microseconds.)
_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 1)


def _no_tangents(op, *tensors):
    """Refuses the dual tensors of forward-mode differentiation, whose tangents a native call would drop."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{op}: no forward-mode derivatives")


def _checked(op, x, others, same_type=False):
    """Refuses tensors of other types or devices than the kernels take, and calls that are being recorded."""
    if _tracing() or (_modes() and proxy_tensor.get_proxy_mode() is not None):
        raise NotImplementedError(f"{op}: a native call cannot be traced")
    if x.dtype not in DTYPES:
        raise TypeError(f"{op}: float32, bfloat16 or float16 tensors, got {x.dtype}")
    at = x.get_device()
    for name, t in others:
        if t is None:
            continue
        if same_type and t.dtype != x.dtype:
            raise TypeError(f"{op}: {name} is {t.dtype}, x {x.dtype}")
        if t.get_device() != at or (at < 0 and t.device != x.device):
            raise ValueError(f"{op}: {name} is on {t.device}, x on {x.device}")
    if not x.is_cuda:
        raise NotImplementedError(f"{op}: tensors must be on the GPU (there is no CPU path)")


def _rows(x):
    """x as contiguous [rows, width] (x itself where it is: a view would be a node of the autograd graph)."""
    if x.numel() > MAX_ROWS and (x.shape[-1] > MAX_ROWS or x.numel() // x.shape[-1] > MAX_ROWS):
        raise NotImplementedError(f"{tuple(x.shape)} holds more than {MAX_ROWS} rows or columns")
    return (x if x.dim() == 2 else x.reshape(-1, x.shape[-1])).contiguous()


# ---------------------------------------------------------------- dense
def _dense_forward(x, kernel, bias, residual, act, keep_z):
    """(y, z): x [M, K] and residual [M, N] contiguous."""
    M, K = x.shape
    N = kernel.shape[1]
    code = DTYPES[x.dtype]
    lib = nat.lib()
    y = x.new_empty((M, N))
    z = None
    if keep_z and act != nat.ACT_NONE:
        z = torch.empty((M, N), dtype=torch.float32 if x.dtype == torch.float32 else torch.float16, device=x.device)
    n = lib.az_dense_workspace_bytes(code, M, K, N, 0)
    if n < 0:
        nat.check(-2)
    ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
    _native(x.device, lib.az_dense_forward, code, act, M, K, N, x, kernel, bias, residual, y, z, ws, n)
    return y, z


def _dense_backward(ctx, dy):
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents("dense", dy)
    x, kernel, z = ctx.saved_tensors
    M, K = x.shape
    N = kernel.shape[1]
    need = ctx.needs_input_grad
    dx = torch.empty_like(x) if need[0] else None
    dkernel = torch.empty_like(kernel) if need[1] else None
    dbias = x.new_empty(N) if need[2] else None
    if need[0] or need[1] or need[2]:
        g = dy.contiguous()
        code = DTYPES[x.dtype]
        lib = nat.lib()
        n = lib.az_dense_workspace_bytes(code, M, K, N, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
        _native(x.device, lib.az_dense_backward, code, ctx.act, M, K, N, x, kernel, z, g, dx, dkernel, dbias, ws, n)
    return dx, dkernel, dbias, dy if need[3] else None, None


# (the wrapper makes a second differentiation an error; it is only needed where one is being recorded)
_dense_backward_once = torch.autograd.function.once_differentiable(_dense_backward)


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, residual, act):
        y, z = _dense_forward(x, kernel, bias, residual, act, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, kernel, z)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_dense_backward_once if torch.is_grad_enabled() else _dense_backward)(ctx, dy)


def dense(x, kernel, bias=None, activation=None, residual=None):
    """act(x @ kernel + bias) + residual, differentiable (backwards, once) in every tensor.

    x [..., fan_in], kernel [fan_in, fan_out], bias [fan_out], residual [..., fan_out] of one type
    (float32, bfloat16 or float16) on one GPU; strided tensors are copied first.
    activation: None, "relu", "swish" (z * sigmoid(z), networks/networks.py:25-48) or "gelu" (erf form).
    """
    act = ACTIVATIONS.get(activation, -1)
    N = kernel.shape[1] if kernel.dim() == 2 else 0
    if act < 0 or N < 1 or x.dim() < 1 or x.shape[-1] != kernel.shape[0] or not x.shape[-1] or \
            (bias is not None and bias.shape != (N,)) or \
            (residual is not None and (residual.shape[-1:] != (N,) or residual.shape[:-1] != x.shape[:-1])):
        _refuse_dense(x, kernel, bias, activation, residual)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents("dense", x, kernel, bias, residual)
    _checked("dense", x, (("kernel", kernel), ("bias", bias), ("residual", residual)), True)
    x2, r2 = _rows(x), None if residual is None else _rows(residual)
    kernel = kernel.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x2.requires_grad or kernel.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (r2 is not None and r2.requires_grad)):
        y = _Dense.apply(x2, kernel, bias, r2, act)
    else:
        y, _ = _dense_forward(x2, kernel, bias, r2, act, False)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (N,))


def _refuse_dense(x, kernel, bias, activation, residual):
    if activation not in ACTIVATIONS:
        raise ValueError(f"dense: activation {activation!r} is not one of {list(ACTIVATIONS)}")
    if kernel.dim() != 2 or x.dim() < 1 or x.shape[-1] != kernel.shape[0]:
        raise ValueError(f"dense: x {tuple(x.shape)} and kernel {tuple(kernel.shape)} do not match")
    if 0 in kernel.shape:
        raise ValueError(f"dense: empty kernel {tuple(kernel.shape)}")
    shape = tuple(x.shape[:-1]) + (kernel.shape[1],)
    if bias is not None and tuple(bias.shape) != shape[-1:]:
        raise ValueError(f"dense: bias {tuple(bias.shape)} does not match kernel {tuple(kernel.shape)}")
    raise ValueError(f"dense: residual {tuple(residual.shape)} is not of the output's shape {shape}")


# ---------------------------------------------------------------- layer norm
def _norm_forward(x, scale, bias, eps, keep):
    M, D = x.shape
    code = DTYPES[x.dtype]
    p = scale if scale is not None else bias
    pcode = code if p is None else DTYPES[p.dtype]
    y = torch.empty_like(x)
    mean = rstd = None
    if keep:
        mean, rstd = torch.empty((2, M), dtype=torch.float32, device=x.device)
    _native(x.device, nat.lib().az_layer_norm_forward, code, pcode, M, D, x, scale, bias,
            eps, y, mean, rstd)
    return y, mean, rstd


def _norm_backward(ctx, dy):
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents("layer_norm", dy)
    x, scale, mean, rstd = ctx.saved_tensors
    M, D = x.shape
    need = ctx.needs_input_grad
    code = DTYPES[x.dtype]
    ptype = scale.dtype if scale is not None else ctx.bias_dtype or x.dtype
    dx = torch.empty_like(x) if need[0] else None
    dscale = torch.empty(D, dtype=ptype, device=x.device) if need[1] else None
    dbias = torch.empty(D, dtype=ptype, device=x.device) if need[2] else None
    lib = nat.lib()
    n = lib.az_layer_norm_workspace_bytes(M, D) if need[1] or need[2] else 0
    ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
    _native(x.device, lib.az_layer_norm_backward, code, DTYPES[ptype], M, D, x, scale, mean, rstd, dy.contiguous(), dx,
            dscale, dbias, ws, n)
    return dx, dscale, dbias, None


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, eps):
        y, mean, rstd = _norm_forward(x, scale, bias, eps, True)
        ctx.save_for_backward(x, scale, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, dy)


def layer_norm(x, scale=None, bias=None, eps=1e-6):
    """(x - mean) / sqrt(variance + eps) * scale + bias over the last axis, differentiable (backwards, once) in
    every tensor.

    x [..., width] in float32, bfloat16 or float16; scale and bias [width], both of x's type or
    both float32; strided tensors are copied first.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x {tuple(x.shape)} has no last axis to normalise")
    D = x.shape[-1]
    ptype = None
    for name, t in (("scale", scale), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (D,):
            raise ValueError(f"layer_norm: {name} {tuple(t.shape)} does not match x {tuple(x.shape)}")
        if t.dtype not in (x.dtype, torch.float32) or (ptype is not None and t.dtype != ptype):
            raise TypeError(f"layer_norm: scale and bias must share a type, x's ({x.dtype}) or float32")
        ptype = t.dtype
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"layer_norm: eps {eps}")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents("layer_norm", x, scale, bias)
    _checked("layer_norm", x, (("scale", scale), ("bias", bias)))
    x2 = _rows(x)
    scale = None if scale is None else scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x2.requires_grad or (scale is not None and scale.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(x2, scale, bias, eps)
    else:
        y = _norm_forward(x2, scale, bias, eps, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)
