"""The pointwise product with its epilogue (networks/layers/linear.py, include/psfm_linear.h) against its formulas in
float64.  Tolerances count, element by element:
  * one rounding of each result, eps / 2 of its type;
  * fp32 sums of R terms, at most R 2^-24 of the sum of the terms' magnitudes (any order), and as much for the few
    operations of the epilogue, whose functions are good to 2^-20;
  * backward: dz rounded to the type before the products, its slope taken at a z rounded to the type:
    eps / 2 |dz| + |dy| max|act''| (eps / 2 |z| + the error of z's sum); ReLU's slope may flip where |z| is below
    that error."""
import ctypes
import gc
import math

import numpy as np
import pytest
import torch

import packnet_sfm_amd  # noqa: F401
from packnet_sfm_amd import _hip
from packnet_sfm_amd.networks.layers import linear as LI
from packnet_sfm_amd.networks.layers.dropout import Drop, dropout
from packnet_sfm_amd.networks.layers.linear import conv1x1_act, linear_act
from test_dropout import oracle_mask, pair

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = {"none": LI.ACT_NONE, "relu": LI.ACT_RELU, "sigmoid": LI.ACT_SIGMOID, "elu": LI.ACT_ELU, "silu": LI.ACT_SILU,
        "gelu": LI.ACT_GELU}
CURVE = {"none": 0.0, "relu": 0.0, "sigmoid": 0.1, "elu": 1.0, "silu": 0.5, "gelu": 0.8}   # max |act''|
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda", 0)


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    if act == "elu":
        e = torch.exp(z.clamp(max=0))
        return torch.where(z > 0, z, torch.expm1(z.clamp(max=0))), torch.where(z > 0, torch.ones_like(z), e)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def formulas(x, w, bias, res, act, keep, p, dy):
    """{name: (value, tolerance)} in float64 on x's device, over [M, ...] matrices."""
    f, half = torch.finfo(x.dtype), torch.finfo(x.dtype).eps / 2
    x, w, dy = x.detach().double(), w.detach().double(), dy.detach().double()
    (M, K), N = x.shape, w.shape[0]
    b = torch.zeros(N, dtype=torch.float64, device=x.device) if bias is None else bias.detach().double()
    z = x @ w.t() + b
    ze = (K + 2) * U * (x.abs() @ w.abs().t() + b.abs())
    a, slope = act64(z, act)
    d = torch.ones_like(z) if keep is None else keep.double() / (1 - p if p < 1 else 1)
    y = a * d + (0 if res is None else res.detach().double())
    # act' is at most 1.13
    tiny = f.tiny * f.eps
    out = {"y": (y, half * y.abs() + 1.2 * d * (ze + 2 ** -20 * a.abs()) + 4 * U * y.abs() + tiny)}
    dz = dy * d * slope
    near = CURVE[act] * (half * z.abs() + ze) + 2 ** -20 * 1.2
    if act == "relu":
        near = (z.abs() <= ze + tiny).double()
    if act == "none":
        near = torch.zeros_like(z)
    es = dy.abs() * d * near
    # dz is rounded unscaled: its subnormal step counts with the scale
    e = es + (half * dz.abs() if act != "none" else 0) + (tiny * d if act != "none" else 0) + 4 * U * dz.abs()
    for name, value, err in (("dx", dz @ w, e @ w.abs() + (N + 2) * U * (dz.abs() @ w.abs())),
                             ("dw", dz.t() @ x, e.t() @ x.abs() + (M + 2) * U * (dz.abs().t() @ x.abs())),
                             ("dbias", dz.sum(0), (es + 4 * U * dz.abs()).sum(0) + (M + 2) * U * dz.abs().sum(0))):
        out[name] = value, half * value.abs() + 1.1 * err + tiny
    return out


def check(got, ref, what):
    value, tol = ref
    got = got.detach().double().reshape(value.shape)
    d = (got - value).abs()
    assert bool((d <= tol).all()), f"{what}: {float((d - tol).max()):.3e} over a tolerance of about {float(tol.mean()):.1e}"


def make(M, N, K, dtype, dev, seed, bias=True, res=False, grad=True):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, a=1.0: (torch.randn(*s, generator=g) * a).to(dtype).to(dev)  # noqa: E731
    t = {"x": n(M, K), "w": n(N, K, a=max(K, 1) ** -0.5), "bias": n(N, a=0.2) if bias else None,
         "res": n(M, N) if res else None, "dy": n(M, N)}
    return {k: v.requires_grad_(True) if grad and k != "dy" and v is not None else v for k, v in t.items()}


def drop_and_keep(M, N, p, dev, share=1, seed=77):
    if p == 0:
        return None, None
    keep = torch.from_numpy(oracle_mask(-(-M // share), N, p, seed, 5)).to(dev).repeat_interleave(share, 0)[:M]
    return Drop(p, pair(seed, 5, dev), share > 1), keep


# sizes around the tiles (64, 128), the LDS stages (32, 64) and the 16-byte chunks; single rows and columns; long
# reductions that are split; every direction has its long one
SIZES = [(1, 1, 1), (1, 512, 512), (2, 33, 1031), (5, 17, 33), (16, 64, 4096), (17, 1030, 64), (64, 64, 64),
         (65, 63, 66), (130, 257, 129), (128, 128, 32), (127, 256, 40), (1000, 64, 32), (300, 2056, 72), (4099, 24, 48),
         (9001, 13, 7), (2500, 320, 264), (70001, 3, 5), (6000, 1, 70)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward_and_gradients(dev, dtype, M, N, K):
    for i, (act, bias, res, p) in enumerate((("none", True, False, 0), ("gelu", True, True, 0.2), ("relu", False, False, 0),
                                             ("elu", True, False, 0), ("silu", False, True, 0), ("none", False, True, 0.5),
                                             ("sigmoid", True, False, 0.9), ("relu", True, True, 0.3))):
        t = make(M, N, K, dtype, dev, 100 * i + M + N + K, bias, res)
        drop, keep = drop_and_keep(M, N, p, dev)
        y = linear_act(t["x"], t["w"], t["bias"], ACTS[act], t["res"], drop)
        ref = formulas(t["x"], t["w"], t["bias"], t["res"], act, keep, p, t["dy"])
        check(y, ref["y"], f"{act} y")
        names = [k for k in ("x", "w", "bias", "res") if t[k] is not None]
        grads = dict(zip(names, torch.autograd.grad(y, [t[k] for k in names], t["dy"])))
        for k in names:
            if k == "res":
                assert torch.equal(grads[k], t["dy"])
            else:
                assert grads[k].dtype == dtype
                check(grads[k], ref["d" + k], f"{act} d{k}")
        with torch.no_grad():
            assert torch.equal(linear_act(t["x"], t["w"], t["bias"], ACTS[act], t["res"], drop), y)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_every_subset_of_gradients(dev, dtype):
    """Only what is asked for is made, and it does not depend on what else is: bit for bit, but for the bias
    gradient, whose rows are summed in another order where no product runs beside it.  Two orders of 70 fp32 terms
    differ by at most 2 x 72 x 2^-24 of the sum of their magnitudes, and each result is rounded once, eps / 2."""
    t = make(70, 48, 90, dtype, dev, 4, True, True, grad=False)
    drop, _ = drop_and_keep(70, 48, 0.3, dev)
    names, full = ("x", "w", "bias", "res"), None
    for bits in (15, 1, 2, 4, 8, 3, 5, 6, 12):
        for act in (LI.ACT_NONE, LI.ACT_GELU):
            leaf = {k: t[k].clone().requires_grad_(bool(bits >> i & 1)) for i, k in enumerate(names)}
            y = linear_act(leaf["x"], leaf["w"], leaf["bias"], act, leaf["res"], drop)
            y.backward(t["dy"])
            got = {k: v.grad for k, v in leaf.items()}
            if bits == 15:
                full = {**(full or {}), act: got}
            for i, k in enumerate(names):
                assert (got[k] is None) == (not bits >> i & 1)
                if k == "bias" and got[k] is not None:
                    most = 1.13 / 0.7 * t["dy"].double().abs().sum(0)
                    step = torch.finfo(dtype).eps * full[act][k].double().abs()
                    assert bool(((got[k].double() - full[act][k].double()).abs() <= 144 * U * most + 1.01 * step).all())
                else:
                    assert got[k] is None or torch.equal(got[k], full[act][k])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("share,M", [(5, 35), (64, 192), (333, 999), (1000, 3000)])
def test_channel_masks(dev, dtype, share, M):
    """A mask row of each sample, forward and backward; a narrow layer and a wide one."""
    for N, K in ((64, 32), (37, 50)):
        t = make(M, N, K, dtype, dev, share, True, True)
        drop, keep = drop_and_keep(M, N, 0.5, dev, share)
        x = t["x"].view(M // share, share, K)
        y = linear_act(x, t["w"], t["bias"], LI.ACT_SILU, t["res"].view(M // share, share, N), drop)
        ref = formulas(t["x"], t["w"], t["bias"], t["res"], "silu", keep, 0.5, t["dy"])
        check(y, ref["y"], "y")
        for k, gr in zip(("x", "w", "bias"), torch.autograd.grad(y, [t["x"], t["w"], t["bias"]], t["dy"].view_as(y))):
            check(gr, ref["d" + k], "d" + k)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_the_mask_is_dropouts(dev, dtype):
    """In the epilogue or afterwards, the same values are dropped."""
    for shape, N, channels in (((3, 41, 64), 70, True), ((130, 64), 129, False), ((1, 8), 5, False)):
        t = make(int(np.prod(shape[:-1])), N, shape[-1], dtype, dev, N, False)
        drop = Drop(0.4, pair(1 << 63, 3, dev), channels)
        x, ones = t["x"].view(shape), torch.ones(N, device=dev, dtype=dtype)
        with torch.no_grad():
            fused = linear_act(torch.zeros_like(x), t["w"], ones, drop=drop)
            assert torch.equal(fused, dropout(ones.expand(*shape[:-1], N), drop))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_and_alignment(dev, dtype):
    """Slices of wider buffers, odd bases, turned, expanded tensors and gradients: the dense copies' values, to
    the order of the fp32 sums."""
    g = torch.Generator().manual_seed(6)
    base = torch.randn(4, 60, 49, generator=g).to(dtype).to(dev)
    wide = torch.randn(40, 60, generator=g).to(dtype).to(dev) * 0.15
    for v in (base[..., :40], base[..., 1:41], base[..., 3:40], base[:, :55, 8:], base[:, ::2, :16], base[..., ::3],
              base.transpose(0, 1), base[:, :1].expand(4, 60, 49), base[2:3, :, 5:9], base[0, 0]):
        K = v.shape[-1]
        for w in (wide[:, :K], wide[:, 3:3 + K], wide.t()[:K].t()):
            w = w.detach()
            x = v.detach().requires_grad_(True)
            wl = w.requires_grad_(True)
            r = base[..., 1:41].expand(4, 60, 40)[:v.shape[0] if v.dim() == 3 else 1, :v.shape[1] if v.dim() == 3 else 1]
            r = r[0, 0] if v.dim() == 1 else r if r.shape[:-1] == v.shape[:-1] else None
            y = linear_act(x, wl, None, LI.ACT_GELU, r)
            for dy in (torch.ones_like(y), torch.ones((), device=dev, dtype=dtype).expand(y.shape),
                       torch.randn(y.shape[::-1], generator=g).to(dtype).to(dev).permute(*reversed(range(y.dim())))):
                ref = formulas(v.reshape(-1, K), w, None, None if r is None else r.reshape(-1, 40), "gelu", None, 0,
                               dy.reshape(-1, 40))
                check(y, ref["y"], "y")
                dx, dw = torch.autograd.grad(y, [x, wl], dy, retain_graph=True)
                assert dx.shape == x.shape
                check(dx, ref["dx"], "dx")
                check(dw, ref["dw"], "dw")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_large_products_at_odd_addresses(dev, dtype):
    """Whole chunks of rows from bases that are no multiple of 16 bytes, at a size whose gradients take the largest
    tiles; and the same from odd rows."""
    for M, N, K in ((4096, 8192, 2048), (2050, 4097, 1023)):
        t = make(M, N, K, dtype, dev, 9, False, grad=False)
        buf = torch.empty(M * K + 1, device=dev, dtype=dtype)
        x = buf[1:].view(M, K).copy_(t["x"]).requires_grad_(True)
        w = t["w"].requires_grad_(True)
        y = linear_act(x, w, None, LI.ACT_SILU)
        ref = formulas(x, w, None, None, "silu", None, 0, t["dy"])
        check(y, ref["y"], "y")
        for k, got in zip(("dx", "dw"), torch.autograd.grad(y, [x, w], t["dy"])):
            check(got, ref[k], k)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_images(dev, dtype):
    """conv1x1_act on NCHW and channels_last images against F.conv2d's formula."""
    g = torch.Generator().manual_seed(2)
    img = torch.randn(2, 24, 6, 10, generator=g).to(dtype).to(dev)
    w = (torch.randn(40, 24, 1, 1, generator=g) * 0.2).to(dtype).to(dev)
    b = torch.randn(40, generator=g).to(dtype).to(dev)
    drop, keep = drop_and_keep(120, 40, 0.5, dev, 60)
    rows = lambda t: t.permute(0, 2, 3, 1).reshape(120, -1)  # noqa: E731
    for fmt in (torch.contiguous_format, torch.channels_last):
        x = img.contiguous(memory_format=fmt).requires_grad_(True)
        for wf in (w, w.contiguous(memory_format=torch.channels_last)):
            wl = wf.detach().requires_grad_(True)
            res = torch.randn(2, 40, 6, 10, generator=g).to(dtype).to(dev).contiguous(memory_format=fmt)
            y = conv1x1_act(x, wl, b, LI.ACT_ELU, res, drop)
            assert y.shape == (2, 40, 6, 10) and y.is_contiguous(memory_format=torch.channels_last)
            dy = torch.randn(2, 40, 6, 10, generator=g).to(dtype).to(dev)
            ref = formulas(rows(x), w[:, :, 0, 0], b, rows(res), "elu", keep, 0.5, rows(dy))
            check(rows(y), ref["y"], "y")
            dx, dw = torch.autograd.grad(y, [x, wl], dy)
            assert dw.shape == w.shape
            check(rows(dx), ref["dx"], "dx")
            check(dw, ref["dw"], "dw")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dev, dtype):
    """A row's infinities and NaN stay in its row (tails of tiles and chunks take none in), ReLU keeps NaN, and a
    dropped place is 0 in y, dx, dw and dbias whatever z and dy hold there."""
    for M, N, K in ((67, 45, 37), (64, 64, 64), (9, 24, 136)):
        t = make(M, N, K, dtype, dev, M, True, False, grad=False)
        clean = linear_act(t["x"], t["w"], t["bias"], LI.ACT_RELU)
        x = t["x"].clone()
        x[3] = float("nan")
        x[5, K - 1] = float("inf")
        y = linear_act(x, t["w"], t["bias"], LI.ACT_RELU)
        rest = [i for i in range(M) if i not in (3, 5)]
        assert bool(y[3].isnan().all()) and torch.equal(y[rest], clean[rest]) and not bool(y[5].isfinite().all())
        drop, keep = drop_and_keep(M, N, 0.5, dev)
        for act in ACTS.values():
            x = t["x"].clone().requires_grad_(True)
            w, b = t["w"].clone().requires_grad_(True), t["bias"].clone().requires_grad_(True)
            with torch.no_grad():
                x[3] = float("nan")
            y = linear_act(x, w, b, act, None, drop)
            assert bool((y[3][~keep[3]] == 0).all()) and bool(y[3][keep[3]].isnan().all())
            dy = t["dy"].clone()
            dy[~keep] = float("inf")
            dy[3] = float("nan")
            dy[3, keep[3]] = 0
            dx, db = torch.autograd.grad(y, [x, b], dy)
            assert bool(dx[rest].isfinite().all())
            if act == LI.ACT_NONE:      # no slope at the NaN: its row's gradients are zero
                assert bool((dx[3] == 0).all()) and bool(db.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_gradient_gives_infinities(dev, dtype):
    """Of the weights' signs, in its row of dx alone; small layers and one whose dz is a pass of its own."""
    for M, N, K in ((20, 16, 24), (130, 72, 200), (3000, 264, 1200)):
        t = make(M, N, K, dtype, dev, 5, True)
        dy = t["dy"].clone()
        dy[7, 3] = float("inf")
        for act in (LI.ACT_NONE, LI.ACT_SIGMOID):
            y = linear_act(t["x"], t["w"], t["bias"], act)
            dx, db = torch.autograd.grad(y, [t["x"], t["bias"]], dy)
            assert torch.equal(dx[7], t["w"][3].detach().sign() * float("inf"))
            assert bool(dx[8:].isfinite().all()) and bool(dx[:7].isfinite().all())
            assert float(db[3]) == float("inf") and int(db.isfinite().sum()) == N - 1


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_everything_dropped(dev, dtype):
    t = make(40, 24, 16, dtype, dev, 1, True, True)
    drop, _ = drop_and_keep(40, 24, 1.0, dev)
    y = linear_act(t["x"], t["w"], t["bias"], LI.ACT_GELU, t["res"], drop)
    assert torch.equal(y, t["res"])
    for gr in torch.autograd.grad(y, [t["x"], t["w"], t["bias"]], t["dy"]):
        assert bool((gr == 0).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_empty_sizes(dev, dtype):
    for M, N, K in ((0, 8, 16), (8, 0, 16), (8, 16, 0), (0, 0, 0), (100, 16, 0), (0, 100, 200), (200, 0, 64)):
        t = make(M, N, K, dtype, dev, 1, True, True)
        y = linear_act(t["x"], t["w"], t["bias"], LI.ACT_SILU, t["res"], Drop(0.5, pair(1, 1, dev)))
        dx, dw, db = torch.autograd.grad(y, [t["x"], t["w"], t["bias"]], t["dy"])
        assert y.shape == (M, N) and dx.shape == (M, K) and dw.shape == (N, K) and db.shape == (N,)
        assert bool((dx == 0).all()) and bool((dw == 0).all())
        if K == 0:
            keep = torch.from_numpy(oracle_mask(M, N, 0.5, 1, 1)).to(dev) if M and N else None
            ref = formulas(t["x"], t["w"], t["bias"], t["res"], "silu", keep, 0.5, t["dy"])
            check(y, ref["y"], "y")
            check(db, ref["dbias"], "dbias")
        else:
            assert bool((db == 0).all())


@gpu
def test_offsets_past_32_bits(dev):
    """More than 2^31 values in x, then in y: the last rows are right, forward and backward."""
    rows, K, N = (2 ** 31) // 2048 + 201, 2048, 8
    x = torch.zeros(rows, K, device=dev, dtype=torch.bfloat16)
    t = make(300, N, K, torch.bfloat16, dev, 3, True, True, grad=False)
    x[-300:] = t["x"]
    x.requires_grad_(True)
    w = t["w"].requires_grad_(True)
    y = linear_act(x, w, t["bias"])
    dy = torch.zeros(rows, N, device=dev, dtype=torch.bfloat16)
    dy[-300:] = t["dy"]
    ref = formulas(t["x"], w, t["bias"], None, "none", None, 0, t["dy"])
    check(y[-300:], ref["y"], "y")
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    check(dx[-300:], ref["dx"], "dx")
    value, tol = ref["dw"]
    check(dw, (value, tol + (rows * U) * value.abs()), "dw")
    del x, y, dx, dy
    t = make(rows, 8, 8, torch.bfloat16, dev, 3, True, False, grad=False)
    w = torch.randn(2048, 8, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    y = linear_act(t["x"], w, None, LI.ACT_RELU, None, Drop(0.25, pair(4, 4, dev)))
    keep = torch.from_numpy(oracle_mask(300, 2048, 0.25, 4, 4, rows - 300)).to(dev)
    ref = formulas(t["x"][-300:], w, None, None, "relu", keep, 0.25, y[-300:])
    check(y[-300:], ref["y"], "y")


@gpu
def test_autocast_and_module_weights(dev):
    """Under autocast fp32 leaves are cast as torch's linear casts them; their gradients come back in fp32."""
    t = make(50, 40, 30, torch.float32, dev, 9)
    for dt in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype=dt):
            y = linear_act(t["x"], t["w"], t["bias"], LI.ACT_ELU)
        assert y.dtype == dt
        c = lambda k: t[k].detach().to(dt)  # noqa: E731
        ref = formulas(c("x"), c("w"), c("bias"), None, "elu", None, 0, c("dy"))
        check(y, ref["y"], "y")
        for k, gr in zip(("x", "w", "bias"), torch.autograd.grad(y, [t[k] for k in ("x", "w", "bias")], c("dy"))):
            assert gr.dtype == torch.float32
            check(gr, ref["d" + k], "d" + k)


@gpu
@pytest.mark.parametrize("M,N,K", [(8, 512, 2048), (700, 64, 48), (96, 80, 33)])
def test_captured_and_replayed_with_new_inputs(dev, M, N, K):
    """A step captured on its own stream replays bit for bit what the eager call gives, with eager calls of the same
    operator (whose workspaces are others) between the replays; two graphs do not share theirs."""
    t = make(M, N, K, torch.bfloat16, dev, 5, True, True)
    leaves = [t["x"], t["w"], t["bias"]]
    rng = pair(3, 1, dev)

    def step():
        y = linear_act(t["x"], t["w"], t["bias"], LI.ACT_SILU, t["res"], Drop(0.3, rng))
        return (y.detach(),) + torch.autograd.grad(y, leaves, t["dy"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gc.collect()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(step())
    g = torch.Generator().manual_seed(8)
    for n in range(4):
        with torch.no_grad():
            t["x"].copy_(torch.randn(M, K, generator=g).to(torch.bfloat16))
            rng[1] = n
        graphs[n % 2].replay()
        graphs[1 - n % 2].replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@gpu
def test_second_derivatives_are_refused(dev):
    """A gradient with a graph of its own has the right values and raises when that graph is differentiated; the residual's,
    which is dy itself, goes on being differentiable."""
    t = make(40, 24, 16, torch.float32, dev, 1, True, True)
    names = ("x", "w", "bias", "res")
    for drop in (None, Drop(0.5, pair(1, 1, dev))):
        for f in (lambda: linear_act(t["x"], t["w"], t["bias"], LI.ACT_SILU, t["res"], drop),
                  lambda: dropout(t["res"], drop or Drop(0.1, pair(2, 2, dev)), t["res"])):
            leaves = [t[k] for k in names]
            dy = t["dy"].clone().requires_grad_(True)
            once = torch.autograd.grad(f(), leaves, dy, allow_unused=True)
            graph = torch.autograd.grad(f(), leaves, dy, create_graph=True, allow_unused=True)
            assert all(a is None or torch.equal(a, b) for a, b in zip(once, graph))
            for g in graph:
                if g is not None and g is not graph[3]:
                    with pytest.raises(RuntimeError, match="differentiated twice"):
                        g.sum().backward(retain_graph=True)
    dy = t["dy"].clone().requires_grad_(True)
    g, = torch.autograd.grad(linear_act(t["x"], t["w"], residual=t["res"]), t["res"], dy, create_graph=True)
    assert torch.equal(torch.autograd.grad((g * g).sum(), dy)[0], 2 * dy)


@gpu
def test_forward_mode_derivatives_are_refused(dev):
    import torch.autograd.forward_ad as fwd
    t = make(4, 8, 6, torch.float32, dev, 3, True, True, grad=False)
    drop = Drop(0.5, pair(1, 2, dev))
    with fwd.dual_level():
        for k in ("x", "w", "bias", "res"):
            a = {**t, k: fwd.make_dual(t[k], torch.ones_like(t[k]))}
            with pytest.raises(RuntimeError, match="forward-mode"):
                linear_act(a["x"], a["w"], a["bias"], LI.ACT_SILU, a["res"])
        dual = fwd.make_dual(t["res"], torch.ones_like(t["res"]))
        for args in ((dual, drop), (t["res"], drop, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                dropout(*args)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_checkpointed_and_offloaded(dev, dtype):
    """A forward that is run again for its backward makes the same mask; saved tensors may rest on the host."""
    from torch.utils.checkpoint import checkpoint
    t = make(300, 72, 136, dtype, dev, 8, True, True)
    leaves = [t[k] for k in ("x", "w", "bias", "res")]
    drop = Drop(0.4, pair(6, 7, dev))

    def block(x, w, b, r):
        return dropout(linear_act(x, w, b, LI.ACT_RELU, r, drop), drop, r)

    want = torch.autograd.grad(block(*leaves), leaves, t["dy"])
    again = torch.autograd.grad(checkpoint(block, *leaves, use_reentrant=False), leaves, t["dy"])
    with torch.autograd.graph.save_on_cpu():
        y = block(*leaves)
    away = torch.autograd.grad(y, leaves, t["dy"])
    for w, a, b in zip(want, again, away):
        assert torch.equal(w, a) and torch.equal(w, b)


@gpu
def test_saved_tensors_changed_in_place_are_refused(dev):
    for change, act in (("x", LI.ACT_NONE), ("w", LI.ACT_NONE), ("y", LI.ACT_RELU)):
        t = make(40, 24, 16, torch.bfloat16, dev, 1, False)
        y = linear_act(t["x"], t["w"], None, act)
        with torch.no_grad():
            (y if change == "y" else t[change]).mul_(2)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(y, [t["x"], t["w"]], t["dy"])


@gpu
def test_capture_with_a_leaf_that_an_eager_graph_holds_is_refused(dev):
    """Whichever operator made that graph: the leaf's accumulator is bound to the default stream.  Freed, the same
    capture goes ahead."""
    t = make(40, 24, 16, torch.float32, dev, 1)
    held = torch.nn.functional.linear(t["x"], t["w"], t["bias"])
    torch.autograd.grad(held, t["w"], t["dy"], retain_graph=True)
    drop, buf = Drop(0.5, pair(1, 1, dev)), torch.zeros(8, device=dev)
    for call in (lambda: linear_act(t["x"], t["w"]), lambda: dropout(t["x"], drop)):
        with pytest.raises(RuntimeError, match="still holds one of this call's leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                buf.add_(1)
                call()
        torch.cuda.synchronize()
    del held
    gc.collect()
    want = torch.autograd.grad(linear_act(t["x"], t["w"], t["bias"]), [t["x"], t["w"]], t["dy"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(linear_act(t["x"], t["w"], t["bias"]), [t["x"], t["w"]], t["dy"])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_streams_side_by_side(dev):
    """Calls on two streams at once have workspaces of their own."""
    ts = [make(300 + s, 96, 4096, torch.float16, dev, s, True, True) for s in range(2)]
    refs = [formulas(t["x"], t["w"], t["bias"], t["res"], "gelu", None, 0, t["dy"]) for t in ts]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for t, st, out in zip(ts, streams, got):
            with torch.cuda.stream(st):
                y = linear_act(t["x"], t["w"], t["bias"], LI.ACT_GELU, t["res"])
                out.append((y.detach(),) + torch.autograd.grad(y, [t["x"], t["w"], t["bias"]], t["dy"]))
    torch.cuda.synchronize()
    for ref, out in zip(refs, got):
        for tensors in out:
            for k, v in zip(("y", "dx", "dw", "dbias"), tensors):
                check(v, ref[k], k)
            assert all(torch.equal(a, b) for a, b in zip(tensors, out[0]))   # sums in a fixed order


@gpu
def test_gradients_against_differences(dev):
    """fp32 central differences along random directions: step h has an error of h^2 and of 2^-24 of the sums / h."""
    for act in ("sigmoid", "elu", "silu", "gelu"):
        t = make(33, 20, 41, torch.float32, dev, 3, True, True)
        drop, _ = drop_and_keep(33, 20, 0.25, dev)
        names = ("x", "w", "bias", "res")

        def loss(v):
            y = linear_act(v["x"], v["w"], v["bias"], ACTS[act], v["res"], drop)
            return (y.double() * t["dy"].double()).sum()

        grads = dict(zip(names, torch.autograd.grad(loss(t), [t[k] for k in names])))
        g, h = torch.Generator().manual_seed(1), 2.0 ** -7
        for k in names:
            u = torch.randn(t[k].shape, generator=g).to(dev)
            u = u / u.norm()
            with torch.no_grad():
                hi, lo = (loss({**t, k: t[k] + s * h * u}) for s in (1, -1))
            want = float((grads[k].double() * u.double()).sum())
            # third derivatives along u are below 10 of what the loss sums; 660 values of magnitude 2 off by 2^-23 each
            assert abs(float(hi - lo) / (2 * h) - want) < 10 * h * h + 660 * 2 * 2 ** -23 / h, (act, k)


def test_plain_path_on_the_cpu():
    for dtype in TYPES + [torch.float64]:
        t = make(21, 10, 12, dtype, torch.device("cpu"), 2, True, True)
        drop, keep = drop_and_keep(21, 10, 0.5, "cpu", 7)
        x = t["x"].view(3, 7, 12)
        y = linear_act(x, t["w"], t["bias"], LI.ACT_GELU, t["res"].view(3, 7, 10), drop)
        ref = formulas(t["x"], t["w"], t["bias"], t["res"], "gelu", keep, 0.5, t["dy"])
        assert y.dtype == dtype and y.shape == (3, 7, 10)
        if dtype == torch.float64:
            assert torch.allclose(y.view(21, 10), ref["y"][0], rtol=1e-12, atol=1e-12)
        else:
            check(y, ref["y"], "y")
        img = torch.randn(2, 12, 3, 4).to(dtype)
        got = conv1x1_act(img, t["w"].detach()[:, :, None, None], t["bias"].detach(), LI.ACT_RELU)
        want = torch.relu(torch.nn.functional.conv2d(img.double(), t["w"].detach().double()[:, :, None, None],
                                                     t["bias"].detach().double()))
        assert torch.allclose(got.double(), want, rtol=torch.finfo(dtype).eps, atol=1e-3 if dtype != torch.float64 else 1e-12)


def test_refusals():
    x, w, b = torch.ones(2, 4), torch.ones(3, 4), torch.ones(3)
    for args in ((torch.ones(()), w), (x, torch.ones(3, 5)), (x, torch.ones(4)), (x, w.double()), (x, w, torch.ones(4)),
                 (x, w, b.half()), (x, w, b, LI.ACT_RELU, torch.ones(2, 4)), (x, w, b, LI.ACT_RELU, torch.ones(3)),
                 (x, w, None, LI.ACT_NONE, None, Drop(0.5, torch.zeros(2)))):
        with pytest.raises(RuntimeError):
            linear_act(*args)
    with pytest.raises(ValueError, match="activation"):
        linear_act(x, w, b, 6)
    with pytest.raises(ValueError, match="probability"):
        linear_act(x, w, b, drop=Drop(-1.0, pair(0, 0)))
    for args in ((x, w), (torch.ones(1, 4, 2, 2), w), (torch.ones(1, 4, 2, 2), torch.ones(3, 4, 3, 3)),
                 (torch.ones(1, 5, 2, 2), torch.ones(3, 4, 1, 1))):
        with pytest.raises(RuntimeError):
            conv1x1_act(*args)
    L, a = _hip.lib(), ctypes.c_void_p(4096)
    good = dict(M=4, N=8, K=8, ldx=8, ldr=8, dtype=0, act=0, p=0.0, mask_rows=1, rng=None)
    for bad, code in ((dict(M=-1), -2), (dict(K=2 ** 41), -2), (dict(ldx=7), -3), (dict(ldr=-1), -3), (dict(dtype=3), -4),
                      (dict(act=6), -5), (dict(act=-1), -5), (dict(p=-0.5), -6), (dict(p=float("nan")), -6),
                      (dict(p=0.5), -7), (dict(p=0.5, rng=4096, mask_rows=0), -7),
                      (dict(M=2 ** 39, N=2 ** 39, K=0), -3)):
        d = _hip.Linear(**{**good, **bad})
        assert L.psfm_linear_fwd(ctypes.byref(d), a, a, None, None, a, None, None, None) == code, bad
        assert L.psfm_linear_bwd(ctypes.byref(d), a, a, a, a, a, a, a, a, None) == code, bad
        assert L.psfm_linear_fwd_ws_bytes(ctypes.byref(d)) == -1 and L.psfm_linear_last_error()
        assert L.psfm_linear_bwd_ws_bytes(ctypes.byref(d), 1, 1, 1) == -1
    d = _hip.Linear(**good)
    assert L.psfm_linear_fwd(ctypes.byref(d), None, a, None, None, a, None, None, None) == -9
    assert L.psfm_linear_fwd(ctypes.byref(d), a, a, None, None, None, None, None, None) == -9
    d.ldr = 7
    assert L.psfm_linear_fwd(ctypes.byref(d), a, a, None, a, a, None, None, None) == -3
    d = _hip.Linear(**{**good, "act": LI.ACT_SILU})
    assert L.psfm_linear_bwd(ctypes.byref(d), a, a, a, None, a, None, None, a, None) == -9     # no z
    d = _hip.Linear(**{**good, "act": LI.ACT_SILU, "M": 100000})   # a long reduction is split: no workspace
    assert L.psfm_linear_bwd_ws_bytes(ctypes.byref(d), 0, 1, 0) > 0
    assert L.psfm_linear_bwd(ctypes.byref(d), a, a, a, a, None, a, None, None, None) == -10
    d = _hip.Linear(**{**good, "M": 64, "K": 65536, "ldx": 65536})
    assert L.psfm_linear_fwd_ws_bytes(ctypes.byref(d)) > 0
    assert L.psfm_linear_fwd(ctypes.byref(d), a, a, None, None, a, None, None, None) == -10
    assert L.psfm_linear_fwd(None, a, a, None, None, a, None, a, None) == -1
    d = _hip.Linear(**{**good, "M": 0})
    assert L.psfm_linear_fwd(ctypes.byref(d), None, a, None, None, None, None, None, None) == 0
