"""The pointwise product with its epilogue (include/psfm_linear.h, csrc/psfm_linear*.hip).

  linear_act(x, weight, bias, act, residual, drop)   y = residual + drop(act(x weight^T + bias)) over the last
                                                     dimension, one pass; drop is a dropout.Drop
  conv1x1_act(x, weight, bias, act, ...)             the same as a 1x1 convolution on [B, C, H, W] images, whose
                                                     channels_last storage is the product's rows

The residual blocks' shortcut (packnet_sfm/networks/layers/packnet/layers01.py:40-61: 1x1 convolution, channel
dropout, sum) and the pose decoder's squeeze (packnet_sfm/networks/layers/resnet/pose_decoder.py:14-49) are of this
form.  fp32, fp16 and bf16 tensors on a ROCm device run the HIP kernels, forward and backward; under autocast the
tensors are cast to its type first, as torch's linear does.  Anything else (CPU tensors, fp64) runs the same
arithmetic as plain torch ops.
"""
import ctypes

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ... import _hip
from .dropout import as_rows, check_drop, check_like, mask_rows, on_device, plain_drop
from .fused import ACT_ELU, ACT_NONE, ACT_RELU, ACT_SIGMOID

ACT_SILU, ACT_GELU = 4, 5   # PSFM_ACT_SILU, PSFM_ACT_GELU
_PLAIN = {ACT_NONE: lambda z: z, ACT_RELU: torch.relu, ACT_SIGMOID: torch.sigmoid, ACT_ELU: F.elu, ACT_SILU: F.silu,
          ACT_GELU: F.gelu}


# what the values before the activation are kept in (psfm_linear_fwd's z; ReLU's: the tensors' own type)
_Z = {torch.float32: torch.float32, torch.float16: torch.float32, torch.bfloat16: torch.float16}


def _at(t):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, residual, act, p, rng, share, want_z):
    """(x as the kernel took it, its row stride, weight, y, z)"""
    x, ldx = as_rows(x)
    weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    ldr = 0
    if residual is not None:
        residual, ldr = as_rows(residual)
    N, K = weight.shape
    device, dtype, lead = x.device, x.dtype, x.shape[:-1]
    y = torch.empty(lead + (N,), device=device, dtype=dtype)
    z = torch.empty(lead + (N,), device=device, dtype=dtype if act == ACT_RELU else _Z[dtype]) if want_z else None
    d = ctypes.byref(_hip.Linear(lead.numel(), N, K, ldx, ldr, _hip.DTYPES[dtype], act, p, share, _at(rng)))
    L = _hip.lib()
    n = L.psfm_linear_fwd_ws_bytes(d)
    if n < 0:
        _hip.check(-1, "psfm_linear_fwd_ws_bytes")
    ws = torch.empty(n, device=device, dtype=torch.uint8) if n else None
    with on_device(device):
        _hip.check(L.psfm_linear_fwd(d, x.data_ptr(), weight.data_ptr(), _at(bias), _at(residual), y.data_ptr(), _at(z),
                                     _at(ws), _hip.stream(device)), "psfm_linear_fwd")
    return x, ldx, weight, y, z


class _LinearAct(torch.autograd.Function):
    """Saves x, the weight and the values before the activation (_Z).  ReLU's slope is the sign of its output
    where nothing follows it."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, p, rng, share):
        _hip.note_forward(ctx)
        from_y = act == ACT_RELU and residual is None and rng is None
        want_z = act != ACT_NONE and not from_y and any(ctx.needs_input_grad[:3])
        need = ctx.needs_input_grad
        xk, ldx, wk, y, z = _forward(x, weight, bias, residual, act, p, rng, share, want_z)
        ctx.save_for_backward(xk if need[1] else None, wk if need[0] else None, y if from_y else z, rng)
        ctx.meta = (x.shape, ldx, wk.shape, act, p, share)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _hip.capture_guard(ctx, leaves=True)
        x, weight, z, rng = ctx.saved_tensors
        xshape, ldx, (N, K), act, p, share = ctx.meta
        want_dx, want_dw, want_db, want_dres = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_dx or want_dw or want_db:
            g = dy.contiguous()
            device, dtype = g.device, g.dtype
            if want_dx:
                dx = torch.empty(xshape, device=device, dtype=dtype)
            if want_dw:
                dw = torch.empty((N, K), device=device, dtype=dtype)
            if want_db:
                db = torch.empty((N,), device=device, dtype=dtype)
            d = ctypes.byref(_hip.Linear(xshape[:-1].numel(), N, K, ldx, 0, _hip.DTYPES[dtype], act, p, share, _at(rng)))
            L = _hip.lib()
            n = L.psfm_linear_bwd_ws_bytes(d, want_dx, want_dw, want_db)
            if n < 0:
                _hip.check(-1, "psfm_linear_bwd_ws_bytes")
            ws = torch.empty(n, device=device, dtype=torch.uint8) if n else None
            with on_device(device):
                _hip.check(L.psfm_linear_bwd(d, g.data_ptr(), _at(x), _at(weight), _at(z), _at(dx), _at(dw), _at(db),
                                             _at(ws), _hip.stream(device)), "psfm_linear_bwd")
        return dx, dw, db, dy if want_dres else None, None, None, None, None


def linear_act(x, weight, bias=None, act=ACT_NONE, residual=None, drop=None):
    """residual + drop(act(x weight^T + bias)): x [..., K], weight [N, K], bias [N], residual [..., N].  Sums and the
    epilogue in fp32, y rounded once.  x and residual may be slices of wider buffers (rows at one
    stride); other layouts are copied."""
    if act not in _PLAIN:
        raise ValueError(f"linear_act: unknown activation {act}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"linear_act: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias, residual = (t if t is None or t.dtype not in _hip.DTYPES else t.to(dt)
                                     for t in (x, weight, bias, residual))
    N = weight.shape[0]
    check_like(weight, "weight", weight.shape, x)
    if bias is not None:
        check_like(bias, "bias", (N,), x)
    if residual is not None:
        check_like(residual, "residual", x.shape[:-1] + (N,), x)
    if drop is not None:
        drop = check_drop(drop, x.device)
    if not x.is_cuda or x.dtype not in _hip.DTYPES:
        wide = torch.promote_types(x.dtype, torch.float32)
        y = _PLAIN[act](F.linear(x.to(wide), weight.to(wide), None if bias is None else bias.to(wide)))
        if drop is not None:
            y = plain_drop(y, drop)
        return (y if residual is None else y + residual.to(wide)).to(x.dtype)
    p, rng, share = (0.0, None, 1) if drop is None else (drop.p, drop.rng, mask_rows(x.shape, drop.channels))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias is not None and bias.requires_grad
                                    or residual is not None and residual.requires_grad):
        return _LinearAct.apply(x, weight, bias, residual, act, p, rng, share)
    return _forward(x, weight, bias, residual, act, p, rng, share, False)[3]


def conv1x1_act(x, weight, bias=None, act=ACT_NONE, residual=None, drop=None):
    """linear_act as a 1x1 convolution: x [B, C, H, W], weight [N, C, 1, 1], residual [B, N, H, W]; the result is
    channels_last.  A drop with `channels` drops whole channels of a sample, as nn.Dropout2d does."""
    if x.dim() != 4 or weight.dim() != 4 or weight.shape[2:] != (1, 1):
        raise RuntimeError(f"conv1x1_act: x {tuple(x.shape)} and weight {tuple(weight.shape)} are no 1x1 convolution")
    res = None if residual is None else residual.permute(0, 2, 3, 1)
    return linear_act(x.permute(0, 2, 3, 1), weight.flatten(1), bias, act, res, drop).permute(0, 3, 1, 2)
