"""linear_act where its arithmetic can lose a value: gradients that are not finite, tails of the activations, launches at
their limits.  test_linear.formulas gives values and tolerances in float64."""
import ctypes
import math

import pytest
import torch

import packnet_sfm_amd  # noqa: F401
from packnet_sfm_amd import _hip
from packnet_sfm_amd.networks.layers import linear as LI
from packnet_sfm_amd.networks.layers.dropout import Drop, dropout
from packnet_sfm_amd.networks.layers.linear import conv1x1_act, linear_act
from test_dropout import oracle_mask, pair
from test_linear import ACTS, TYPES, U, check, drop_and_keep, formulas, make

gpu = pytest.mark.gpu
# rows x columns x reduction: gradients that make dz as they stage it, the same with odd rows, dz as a pass of its own
SIZES = [(20, 16, 24), (67, 45, 37), (130, 72, 200), (3000, 264, 1200), (2049, 515, 777)]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda", 0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_relu_selects_its_gradient(dev, dtype, M, N, K):
    """An infinite or NaN gradient of a value below 0 is no gradient, and a NaN passes its own, as in torch.relu.  The slope's
    tensor is z or y."""
    for res, p in ((False, 0), (True, 0), (True, 0.4)):
        t = make(M, N, K, dtype, dev, M + N, True, res)
        drop, keep = drop_and_keep(M, N, p, dev)
        leaves = [t["x"], t["w"], t["bias"]]
        y = linear_act(*leaves, LI.ACT_RELU, t["res"], drop)
        z = t["x"].double() @ t["w"].double().t() + t["bias"].double()
        off = z < -0.01
        zero = t["dy"].masked_fill(off, 0)
        want = torch.autograd.grad(y, leaves, zero, retain_graph=True)
        for bad in (float("inf"), -float("inf"), float("nan")):
            got = torch.autograd.grad(y, leaves, zero.masked_fill(off, bad), retain_graph=True)
            assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(got, want))
        x = t["x"].detach().clone()
        x[3] = float("nan")
        x.requires_grad_(True)
        y = linear_act(x, t["w"], t["bias"], LI.ACT_RELU, t["res"], drop)
        dx, db = torch.autograd.grad(y, [x, t["bias"]], zero)
        passed = zero[3:4].double() * (1 if keep is None else keep[3:4].double() / (1 - p))
        ref = formulas(torch.zeros(1, K, device=dev, dtype=dtype), t["w"], None, None, "none", None, 0, passed)
        check(dx[3:4], (ref["dx"][0], ref["dx"][1] + 4 * U * (passed.abs() @ t["w"].detach().double().abs())), "row of a NaN")
        assert bool(db.isfinite().all()) and bool(dx.isfinite().all())
