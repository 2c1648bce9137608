"""The pointwise product with its epilogue (include/psfm_linear.h, csrc/psfm_linear*.hip).

  linear_act(x, weight, bias, act, residual, drop)   y = residual + drop(act(x weight^T + bias)) over the last
                                                     dimension, one pass; drop is a dropout.Drop
  conv1x1_act(x, weight, bias, act, ...)             the same as a 1x1 convolution on [B, C, H, W] images, whose
                                                     channels_last storage is the product's rows

The residual blocks' shortcut (packnet_sfm/networks/layers/packnet/layers01.py:40-61: 1x1 convolution, channel
dropout, sum) is of this form and runs on it with dropout_seed (layers01.ResidualConv).  fp32, fp16 and bf16 tensors on
a ROCm device run the HIP kernels, forward and backward; under autocast the tensors are cast to its type first, as
torch's linear does.  Anything else (CPU tensors, fp64) runs the same arithmetic as plain torch ops.  Gradients: z is
kept in fp16 for bf16 layers and in fp32 for the others, and large 16-bit layers round dz to their type before its
products (include/psfm_linear.h).  The autograd node is in C++ (csrc/psfm_autograd.cpp); under torch.jit.trace a call
is recorded as a Python operator.
"""
import torch
import torch.nn.functional as F

from ... import _hip
from .dropout import check_drop, check_like, plain_drop, run
from .fused import ACT_ELU, ACT_NONE, ACT_RELU, ACT_SIGMOID

ACT_SILU, ACT_GELU = 4, 5   # PSFM_ACT_SILU, PSFM_ACT_GELU
_PLAIN = {ACT_NONE: lambda z: z, ACT_RELU: torch.relu, ACT_SIGMOID: torch.sigmoid, ACT_ELU: F.elu, ACT_SILU: F.silu,
          ACT_GELU: F.gelu}


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
        z = F.linear(x.to(wide), weight.to(wide), None if bias is None else bias.to(wide))
        y = _PLAIN[act](z) if drop is None else plain_drop(z, drop, _PLAIN[act])
        return (y if residual is None else y + residual.to(wide)).to(x.dtype)
    p, rng, channels = (0.0, None, False) if drop is None else drop
    return run(_hip.ext().linear_act, x, weight, bias, act, residual, p, rng, channels)


def conv1x1_act(x, weight, bias=None, act=ACT_NONE, residual=None, drop=None):
    """linear_act as a 1x1 convolution: x [B, C, H, W], weight [N, C, 1, 1], residual [B, N, H, W]; the result is
    channels_last.  A drop with `channels` drops whole channels of a sample, as nn.Dropout2d does."""
    if x.dim() != 4 or weight.dim() != 4 or weight.shape[2:] != (1, 1):
        raise RuntimeError(f"conv1x1_act: x {tuple(x.shape)} and weight {tuple(weight.shape)} are no 1x1 convolution")
    res = None if residual is None else residual.permute(0, 2, 3, 1)
    return linear_act(x.permute(0, 2, 3, 1), weight.flatten(1), bias, act, res, drop).permute(0, 3, 1, 2)
