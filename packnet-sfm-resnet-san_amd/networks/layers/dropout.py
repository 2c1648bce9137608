"""Dropout from a counter-based generator (include/psfm_dropout.h, csrc/psfm_dropout.hip).

The reference's ResidualConv drops whole channels of its shortcut (nn.Dropout2d,
packnet_sfm/networks/layers/packnet/layers01.py:40-61).  Here a mask is a function of (seed, offset, position)
(Philox4x32-10; the header says which word is whose), so the forward and the backward pass each make it
again and neither stores it, and a run can be repeated from its seed whatever else drew random numbers:

  dropout(x, drop, residual)     y = [residual +] x with dropped values 0 and kept ones times 1 / (1 - p),
                                 columns along the last dimension
  dropout2d(x, drop, residual)   the same on [B, C, H, W] images, columns along C
  Drop(p, rng, channels)         one mask: probability, int64 pair (seed, offset) on x's device, and whether all
                                 positions of a sample (the first dimension) share one row of it
  CounterDropout(p, seed)        the module: draws a new offset on the device at every training forward

linear.linear_act takes the same Drop into its epilogue: the mask is the one that `dropout` would
give its output.  fp32, fp16 and bf16 tensors on a ROCm device run the HIP kernel; anything else
(CPU tensors, fp64) runs the same arithmetic as plain torch ops.  The autograd nodes are in C++ (csrc/psfm_autograd.cpp).
"""
from contextlib import nullcontext
from typing import NamedTuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ... import _hip
from ...utils.horovod import rank


class Drop(NamedTuple):
    p: float
    rng: torch.Tensor
    channels: bool = False


def check_drop(drop, device):
    """Drop's arguments; returns it, or None where it drops nothing."""
    p, rng, _ = drop
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is not in 0 .. 1")
    if p == 0.0:
        return None
    if rng.dtype != torch.int64 or rng.numel() != 2 or rng.device != device or not rng.is_contiguous():
        raise RuntimeError(f"rng must be a contiguous int64 pair (seed, offset) on {device}; got {rng.dtype} "
                           f"{tuple(rng.shape)} on {rng.device}")
    return drop


def mask_rows(shape, channels):
    """How many consecutive rows of a [..., columns] tensor share a row of the mask."""
    if not channels:
        return 1
    n = 1
    for s in shape[1:-1]:
        n *= s
    return max(n, 1)


_HERE = nullcontext()


def on_device(device):
    """Launches go to the current device: make it this one."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


_tracing = torch._C._get_tracing_state


class _Recorded(torch.autograd.Function):
    """fn(*args) as a Python operator, which torch.jit.trace records as a call of it."""

    @staticmethod
    def forward(ctx, fn, *args):
        with torch.enable_grad():
            inner = [a.detach().requires_grad_(a.requires_grad) if torch.is_tensor(a) else a for a in args]
            y = fn(*inner)
        ctx.inner = inner, y
        return y.detach()

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        inner, y = ctx.inner
        leaves = [k for k, a in enumerate(inner) if torch.is_tensor(a) and a.requires_grad]
        grads = dict(zip(leaves, torch.autograd.grad(y, [inner[k] for k in leaves], dy, retain_graph=True)))
        return (None, *(grads.get(k) for k in range(len(inner))))


def run(fn, *args):
    """fn(*args), for an fn that allocates its result and fills it by address: a trace would hold the allocation alone."""
    return fn(*args) if _tracing() is None else _Recorded.apply(fn, *args)


def rng_next(state, add):
    used = torch.empty_like(state)
    with on_device(state.device):
        _hip.check(_hip.lib().psfm_rng_next(state.data_ptr(), add, used.data_ptr(), _hip.stream(state.device)),
                   "psfm_rng_next")
    return used


def keep_mask(rows, cols, p, rng):
    """The kept values of a [rows, cols] mask, in plain torch integer operations on rng's device."""
    blocks, low = (cols + 3) // 4, 0xFFFFFFFF
    at = torch.arange(rows * blocks, device=rng.device)
    c0, c1 = at & low, at >> 32
    c2, c3 = (rng[1] & low).expand_as(at), (rng[1] >> 32 & low).expand_as(at)
    k0, k1 = rng[0] & low, rng[0] >> 32 & low
    for _ in range(10):
        # 32 x 32 bits: the product wraps into int64's sign and keeps its bits
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack((c0, c1, c2, c3), 1).view(rows, 4 * blocks)[:, :cols]
    return words >= int(p * 2.0 ** 32 + 0.5)


def plain_drop(t, drop, act=None):
    """dropout of act(t) in plain torch operations."""
    shape = t.shape
    if t.numel() == 0:
        return t
    share = mask_rows(shape, drop.channels)
    keep = keep_mask(t.numel() // shape[-1] // share, shape[-1], drop.p, drop.rng).unsqueeze(1)
    scale = 1.0 / (1.0 - drop.p) if drop.p < 1.0 else 0.0
    t = t.reshape(-1, share, shape[-1])
    if act is not None:   # of a finite value where it is dropped, so that the slope there is finite too
        t = act(torch.where(keep, t, 0.0))
    return torch.where(keep, t * scale, 0.0).view(shape)


def check_like(t, name, shape, x):
    if t.shape != shape or t.dtype != x.dtype or t.device != x.device:
        raise RuntimeError(f"{name} must be {tuple(shape)} {x.dtype} on {x.device}; got {tuple(t.shape)} {t.dtype} on "
                           f"{t.device}")


def dropout(x, drop, residual=None):
    """[residual +] drop(x) over the last dimension's columns; drop None: nothing is dropped.  A dropped value is
    0 whatever it was, infinities and NaN included.  The sum is taken in fp32 and rounded once."""
    if x.dim() == 0:
        raise RuntimeError("dropout needs at least one dimension")
    if residual is not None:
        check_like(residual, "residual", x.shape, x)
    if drop is not None:
        drop = check_drop(drop, x.device)
    if drop is None:
        return x if residual is None else x + residual
    if not x.is_cuda or x.dtype not in _hip.DTYPES:
        wide = torch.promote_types(x.dtype, torch.float32)
        y = plain_drop(x.to(wide), drop)
        return (y if residual is None else y + residual.to(wide)).to(x.dtype)
    return run(_hip.ext().dropout, x, residual, drop.p, drop.rng, drop.channels)


def dropout2d(x, drop, residual=None):
    """dropout of [B, C, H, W] images with C as the mask's columns (channels_last storage is taken as it is); with
    drop.channels whole channels of a sample are dropped, as nn.Dropout2d does."""
    if x.dim() != 4:
        raise RuntimeError(f"dropout2d takes [B, C, H, W] images, got {tuple(x.shape)}")
    res = None if residual is None else residual.permute(0, 2, 3, 1)
    return dropout(x.permute(0, 2, 3, 1), drop, res).permute(0, 3, 1, 2)


class CounterDropout(nn.Module):
    """Dropout whose masks are (seed, offset), the offset counted on the device: in training every forward draws
    the next one, also in a captured graph's replays.  The ranks of a data-parallel job, which hold the same
    buffers, take seed + rank (jobs whose masks must differ take seeds further apart than their ranks); the layers of
    one network take different first offsets.  The state is no part of the state_dict: checkpoints of networks with
    nn.Dropout load as they are.  dropout_states(network) saves the layers' states beside it, and
    load_dropout_states goes on from them; DDPTrainer.checkpoint() holds them under 'dropout'.

    A forward that is run again for its backward (activation checkpointing) would draw another mask: draw() before
    it, and give the Drop to dropout or linear_act inside."""

    def __init__(self, p, seed, offset=0, channels=False):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability {p} is not in 0 .. 1")
        self.p, self.channels = float(p), channels
        self.register_buffer("state", torch.tensor([_int64(seed), _int64(offset)]), persistent=False)

    def extra_repr(self):
        return f"p={self.p}, channels={self.channels}"

    def draw(self):
        """The Drop of this forward (None where nothing is dropped)."""
        if not self.training or self.p == 0.0:
            return None
        state = self.state
        if not state.is_cuda:
            used = torch.stack((state[0] + rank(), state[1]))
            state[1] += 1
        else:
            used = run(rng_next, state, rank())
        return Drop(self.p, used, self.channels)

    def forward(self, x, residual=None):
        return (dropout2d if x.dim() == 4 else dropout)(x, self.draw(), residual)


def dropout_states(network):
    """{module name: [seed, offset]} of the network's CounterDropout layers."""
    return {n: m.state.tolist() for n, m in network.named_modules() if isinstance(m, CounterDropout)}


@torch.no_grad()
def load_dropout_states(network, states):
    """Goes on from dropout_states' masks, in place: captured graphs hold the states' addresses."""
    layers = {n: m for n, m in network.named_modules() if isinstance(m, CounterDropout)}
    if set(layers) != set(states):
        raise RuntimeError(f"dropout states of other layers: {sorted(set(layers) ^ set(states))}")
    for n, m in layers.items():
        m.state.copy_(torch.tensor(states[n], dtype=torch.int64))


def _int64(v):
    """v of 64 bits as the signed number of the same bits."""
    return (int(v) + 2 ** 63) % 2 ** 64 - 2 ** 63
