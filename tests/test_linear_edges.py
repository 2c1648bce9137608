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
from test_linear import ACTS, CURVE, TYPES, U, check, drop_and_keep, formulas, make

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


def tails(act, z):
    """act(z), act'(z) in float64 and the sums of magnitudes that their fp32 errors count from, with steps of 2^-24 each.
    exp(a) of an fp32 a: a's own rounding and log2(e)'s are 2 |a| steps, the function, sums, reciprocals and products
    after it 12 at most.  The normal distribution's z^2 / 2, or z / sqrt(2) in erfc, whose logarithm has the slope
    z^2 + 1 in it: 2 z^2 + 2, and 38 for erfc itself (16 units) and the rest."""
    steps = 2 * z * z + 40 if act == "gelu" else 2 * z.abs() + 12
    if act == "gelu":
        c = torch.erfc(-z / math.sqrt(2)) / 2
        d = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * c, c + d, steps * U * (z * c).abs(), steps * U * (c + d.abs())
    s = torch.sigmoid(z)
    t = torch.sigmoid(-z)
    if act == "sigmoid":
        return s, s * t, steps * U * s, steps * U * s * t
    if act == "silu":
        return z * s, s * (1 + z * t), steps * U * (z * s).abs(), steps * U * s * (1 + z.abs())
    a, slope = torch.where(z > 0, z, torch.expm1(z)), torch.where(z > 0, 1.0, torch.exp(z))
    return a, slope, steps * U * a.abs(), steps * U * slope


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["sigmoid", "elu", "silu", "gelu"])
def test_tails_keep_their_scale(dev, dtype, act):
    """Relative bounds where the activations and their slopes are small: one rounding of the type, the steps of `tails`, and the
    smallest values of the type (the hardware's exponential gives 0 below the normal ones)."""
    f = torch.finfo(dtype)
    v = torch.linspace(-13, 25, 4001, device=dev, dtype=torch.float64).to(dtype)
    small = max(f.tiny * f.eps, 2.0 ** -125)

    def near(got, value, err, what):
        got, tol = got.detach().double().flatten(), f.eps / 2 * 1.02 * value.abs() + err + small
        bad = (got - value).abs() / tol
        assert bool((bad <= 1).all()), f"{what}: {float(bad.max())} of the bound at z = {float(v[int(bad.argmax())])}"

    a, slope, ea, es = tails(act, v.double())
    # z = x, one column; z = bias, few rows (no tiles) and more
    x, w = v[:, None].clone().requires_grad_(True), torch.ones(1, 1, device=dev, dtype=dtype)
    y = linear_act(x, w, None, ACTS[act])
    near(y, a, ea, "y of x")
    near(torch.autograd.grad(y, x, torch.ones_like(y))[0], slope, es, "dx")
    for M, K in ((1, 8), (8, 8), (40, 8), (300, 64)):
        x, w = torch.zeros(M, K, device=dev, dtype=dtype), torch.zeros(4001, K, device=dev, dtype=dtype, requires_grad=True)
        b = v.clone().requires_grad_(True)
        y = linear_act(x, w, b, ACTS[act])
        dy = torch.zeros_like(y)
        dy[M // 2] = 1
        near(y[M - 1], a, ea, f"y of the bias, {M} rows")
        near(torch.autograd.grad(y, b, dy, retain_graph=True)[0], slope, es, "dbias alone")
        near(torch.autograd.grad(y, [b, w], dy)[0], slope, es, "dbias beside dw")


@gpu
@pytest.mark.parametrize("act", ["sigmoid", "elu", "silu", "gelu"])
@pytest.mark.parametrize("dtype,kept", [(torch.float32, 0.0), (torch.float16, 0.0), (torch.bfloat16, 2.0 ** -11)])
def test_what_z_is_kept_in(dev, dtype, kept, act):
    """Slopes at values of z between those of the layer's type: fp32 and fp16 layers keep z in fp32, bf16 ones in fp16, off by 2^-11 of
    it, which moves the slope by at most |act''| times that.  Beside it the bounds of test_tails_keep_their_scale, and
    two steps for z's own sum."""
    f = torch.finfo(dtype)
    b = torch.linspace(-6, 6, 4001, device=dev, dtype=torch.float64).to(dtype).requires_grad_(True)
    x = torch.full((1, 1), 1.25 * 2.0 ** -9, device=dev, dtype=dtype)
    w = torch.ones(4001, 1, device=dev, dtype=dtype, requires_grad=True)
    z = b.detach().double() + float(x)
    _, slope, _, es = tails(act, z)
    tol = f.eps / 2 * 1.02 * slope.abs() + es + CURVE[act] * (kept + 2 * U) * z.abs() + f.tiny * f.eps
    for some in ([b], [b, w]):
        y = linear_act(x, w, b, ACTS[act])
        got = torch.autograd.grad(y, some, torch.ones_like(y))[0].double()
        assert bool(((got - slope).abs() <= tol).all()), float(((got - slope).abs() / tol).max())


def test_more_than_a_launch_holds_is_refused():
    """A launch's threads are counted in 32 bits; the check comes before anything is launched."""
    L, a = _hip.lib(), ctypes.c_void_p(4096)
    good = dict(M=4, N=8, K=8, ldx=8, ldr=8, dtype=2, act=0, p=0.0, mask_rows=1, rng=None)
    for dtype in (0, 1, 2):
        for sizes in (dict(M=2 ** 31), dict(N=2 ** 31, ldr=2 ** 31), dict(M=2 ** 33, N=1), dict(M=2 ** 17, N=2 ** 32, ldr=2 ** 32)):
            d = _hip.Linear(**{**good, **sizes, "dtype": dtype})
            assert L.psfm_linear_fwd(ctypes.byref(d), a, a, None, None, a, None, a, None) == -8, sizes
            assert b"launch" in L.psfm_linear_last_error()
            for act in (LI.ACT_NONE, LI.ACT_SILU):
                d.act = act
                assert L.psfm_linear_bwd(ctypes.byref(d), a, a, a, a, a, a, None, a, None) == -8, sizes
        d = _hip.Linear(**{**good, "N": 2 ** 28, "ldr": 2 ** 28, "dtype": dtype})
        assert L.psfm_linear_bwd(ctypes.byref(d), a, a, a, None, a, a, a, a, None) == -8
        assert L.psfm_dropout(a, 1, None, 0, dtype, 2 ** 34, 1, 1, 0.5, a, a, None) == -1


@gpu
def test_rows_and_columns_past_the_smaller_launches(dev):
    """More columns than the few-row kernel's launch holds (2^27), more rows than the smallest tiles' (2^30)."""
    N, K = 2 ** 27 + 5, 8
    t = make(1, 300, K, torch.bfloat16, dev, 2, True)
    w = torch.zeros(N, K, device=dev, dtype=torch.bfloat16)
    b = torch.zeros(N, device=dev, dtype=torch.bfloat16)
    w[-300:], b[-300:] = t["w"].detach(), t["bias"].detach()
    with torch.no_grad():
        y = linear_act(t["x"], w, b, LI.ACT_GELU)
    ref = formulas(t["x"], t["w"], t["bias"], None, "gelu", None, 0, t["dy"])
    check(y[:, -300:], ref["y"], "columns")
    assert bool((y[:, :-300] == 0).all())
    del w, b, y
    M, N = 2 ** 30 + 77, 1
    t = make(300, N, K, torch.bfloat16, dev, 4, True, grad=False)
    x = torch.zeros(M, K, device=dev, dtype=torch.bfloat16)
    x[-300:] = t["x"]
    dy = torch.zeros(M, N, device=dev, dtype=torch.bfloat16)
    dy[-300:] = t["dy"]
    leaves = [x.requires_grad_(True), t["w"].requires_grad_(True)]
    y = linear_act(*leaves, t["bias"], LI.ACT_SILU)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    ref = formulas(t["x"], t["w"], t["bias"], None, "silu", None, 0, t["dy"])
    check(y[-300:], ref["y"], "rows")
    check(dx[-300:], ref["dx"], "dx")
    assert bool((dx[:-300] == 0).all())
    check(dw, ref["dw"], "dw")


@pytest.mark.parametrize("where", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_dropped_value_has_no_gradient_whatever_it_was(where):
    """z infinite or NaN, dy infinite or NaN, at dropped places only: y and every gradient are those of zeros there."""
    if where == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    M, N, K = 12, 20, 9
    drop, keep = drop_and_keep(M, N, 0.5, where)
    t = make(M, N, K, torch.float32, torch.device(where), 3, False, False, grad=False)
    # z is not finite in the columns that row 2 drops; rows 0 and 1, which keep some of them, are not looked at
    off = (~keep[2]).nonzero().flatten()
    for act in ACTS.values():
        for bad in (float("inf"), -float("inf"), float("nan")):
            bias = torch.zeros(N, device=where)
            bias[off] = bad
            x = t["x"][2:3]
            grads = []
            for b, dyv in ((bias, bad), (torch.zeros_like(bias), 0.0)):
                b = b.requires_grad_(True)
                xs = torch.cat((t["x"][:2], x)).requires_grad_(True)
                y = linear_act(xs, t["w"], b, act, None, drop)
                dy = torch.zeros_like(y)
                dy[2] = torch.where(keep[2], t["dy"][2], torch.full((), dyv, device=where))
                dx, = torch.autograd.grad(y, xs, dy)
                grads.append((y[2], dx[2]))
            for a, b in zip(*grads):
                assert torch.equal(a, b) and bool(a.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_gradients_that_are_dropped_reach_nothing(dev, dtype, M, N, K):
    """dy infinite or NaN at dropped places: dx, dw and db, asked for together and each alone, are those of zeros there, whether
    the products make dz as they stage it (dw's with the column sums) or a pass does."""
    for act in ACTS.values():
        t = make(M, N, K, dtype, dev, N, True, False)
        drop, keep = drop_and_keep(M, N, 0.4, dev)
        leaves = [t["x"], t["w"], t["bias"]]
        y = linear_act(*leaves, act, None, drop)
        zero = t["dy"].masked_fill(~keep, 0)
        for bad in (float("inf"), float("nan")):
            for some in (leaves, leaves[1:], leaves[:1], leaves[1:2], leaves[2:]):
                a, b = (torch.autograd.grad(y, some, d, retain_graph=True) for d in (zero.masked_fill(~keep, bad), zero))
                for u, v in zip(a, b):
                    assert bool(u.isfinite().all()) and torch.equal(u, v)


@gpu
def test_counter_blocks_past_32_bits(dev):
    """Masks of more than 2^34 values: the last rows' counters have a high word, in the dropout pass, in the product's epilogue
    and in its gradients."""
    rows = 2 ** 32 + 300
    y = dropout(torch.ones(rows, 1, device=dev, dtype=torch.float16), Drop(0.25, pair(1, 2, dev)))
    keep = torch.from_numpy(oracle_mask(600, 1, 0.25, 1, 2, rows - 600)).to(dev)
    assert torch.equal(y[-600:] != 0, keep)
    del y
    M, N, K = 2 ** 20 + 64, 2 ** 14 + 8, 8
    assert (M - 40) * (N // 4) > 2 ** 32
    t = make(40, N, K, torch.bfloat16, dev, 4, True, grad=False)
    x = torch.zeros(M, K, device=dev, dtype=torch.bfloat16)
    x[-40:] = t["x"]
    leaves = [x.requires_grad_(True), t["w"].requires_grad_(True)]
    y = linear_act(*leaves, t["bias"], drop=Drop(0.25, pair(3, 2 ** 35, dev)))
    keep = torch.from_numpy(oracle_mask(40, N, 0.25, 3, 2 ** 35, M - 40)).to(dev)
    dy = torch.zeros(M, N, device=dev, dtype=torch.bfloat16)
    dy[-40:] = t["dy"]
    ref = formulas(t["x"], t["w"], t["bias"], None, "none", keep, 0.25, t["dy"])
    check(y[-40:], ref["y"], "y")
    dx, dw = torch.autograd.grad(y, leaves, dy)
    check(dx[-40:], ref["dx"], "dx")
    check(dw, ref["dw"], "dw")
