"""Counter-based dropout (networks/layers/dropout.py, include/psfm_dropout.h) against Philox4x32-10 written in numpy
and float64 arithmetic.  A mask has to be equal; a value is off by its one rounding, eps / 2 of the type,
and by two fp32 operations (scale, sum) of 2^-24 of their results each."""
import ctypes
import gc

import numpy as np
import pytest
import torch

import packnet_sfm_amd  # noqa: F401
from packnet_sfm_amd import _hip
from packnet_sfm_amd.networks.layers.dropout import CounterDropout, Drop, dropout, dropout2d, keep_mask

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def philox(counter, key):
    """Ten rounds on one counter of four words (numpy uint64 arithmetic)."""
    c, k = [np.uint64(v) for v in counter], [int(v) for v in key]
    m, h = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> h) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> h) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def oracle_mask(rows, cols, p, seed, offset, first_row=0):
    """keep [rows, cols] of mask rows first_row ..., rows vectorised."""
    blocks = -(-cols // 4)
    at = np.arange(rows * blocks, dtype=np.uint64) + np.uint64(first_row * blocks)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    words = philox([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.full_like(at, offset % 2 ** 32),
                    np.full_like(at, offset >> 32)], [seed % 2 ** 32, seed >> 32])
    return np.stack(words, -1).reshape(rows, 4 * blocks)[:, :cols] >= np.uint64(round(p * 2 ** 32))


def pair(seed, offset, dev="cpu"):
    return torch.tensor([(v + 2 ** 63) % 2 ** 64 - 2 ** 63 for v in (seed, offset)], device=dev)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda", 0)


def test_oracle_gives_the_published_answers():
    """Random123's known answers of philox4x32-10."""
    for ctr, key, out in (([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
                          ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
                          ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0],
                           [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])):
        assert [int(v) for v in philox(ctr, key)] == out


@pytest.mark.parametrize("seed,offset", [(0, 0), (7, 2 ** 32 + 5), (2 ** 64 - 1, 2 ** 63), (2 ** 63 + 11, 2 ** 64 - 2)])
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.5), (3, 7, 0.1), (5, 64, 0.9), (2, 130, 1.0), (4, 8, 1e-12)])
def test_plain_mask_equals_the_oracle(rows, cols, p, seed, offset):
    assert np.array_equal(keep_mask(rows, cols, p, pair(seed, offset)).numpy(), oracle_mask(rows, cols, p, seed, offset))


def reference(x, res, drop, share):
    """float64 values, and how far a result of x's type may be."""
    cols = x.shape[-1]
    seed, off = (int(v) for v in drop.rng.tolist())
    keep = torch.from_numpy(oracle_mask(x.numel() // cols // share, cols, drop.p, seed, off))
    keep = keep.unsqueeze(1).expand(-1, share, -1).reshape(x.shape)
    a = torch.where(keep, x.detach().cpu().double() / (1 - drop.p if drop.p < 1 else 1), 0.0)
    r = torch.zeros_like(a) if res is None else res.detach().cpu().double()
    f = torch.finfo(x.dtype)
    tol = f.eps / 2 * (a + r).abs() + 2 ** -24 * (2 * a.abs() + (a + r).abs()) * 1.01 + f.tiny * f.eps
    return a + r, tol, keep


def check(y, ref, tol):
    d = (y.detach().cpu().double() - ref).abs()
    assert bool((d <= tol).all()), f"{float((d - tol).max()):.3e} over, at {int((d - tol).argmax())}"


SHAPES = [((1,), False), ((7,), False), ((1, 1), False), ((4, 4), False), ((3, 5, 8), True), ((2, 33, 130), True),
          ((2, 9, 11, 64), True), ((5, 4097), False), ((513, 3), False), ((6, 17, 1), True), ((3, 2050, 40), False)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,channels", SHAPES)
def test_forward_and_gradients(dev, dtype, shape, channels):
    g = torch.Generator().manual_seed(sum(shape))
    for p, with_res in ((0.1, False), (0.5, True), (1.0, True)):
        x = torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_(True)
        res = torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_(True) if with_res else None
        drop = Drop(p, pair(2 ** 63 + sum(shape), 2 ** 40 + 3, dev), channels)
        share = int(np.prod(shape[1:-1])) if channels else 1
        y = dropout(x, drop, res)
        assert y.dtype == dtype and y.is_contiguous()
        ref, tol, _ = reference(x, res, drop, share)
        check(y, ref, tol)
        dy = torch.randn(shape, generator=g).to(dtype).to(dev)
        grads = torch.autograd.grad(y, [x] + ([res] if with_res else []), dy)
        ref, tol, keep = reference(dy, None, drop, share)
        check(grads[0], ref, tol)
        assert bool((grads[0].cpu()[~keep] == 0).all())
        if with_res:
            assert torch.equal(grads[1], dy)
        with torch.no_grad():
            assert torch.equal(dropout(x, drop, res), y)   # the same bits without a graph


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_and_alignment(dev, dtype):
    """Slices of wider buffers, odd bases, turned and expanded tensors: the values of the dense copy."""
    g = torch.Generator().manual_seed(5)
    drop = Drop(0.3, pair(11, 12, dev), True)
    base = torch.randn(4, 6, 49, generator=g).to(dtype).to(dev)
    views = [base[..., :40], base[..., 1:41], base[..., 3:40], base[:, :5, 8:], base[:, ::2, :16], base[..., ::3],
             base.transpose(0, 1), base[:, :1].expand(4, 6, 49), base[..., :1].expand(4, 6, 9), base[2:3, :, 5:9]]
    for v in views:
        for r in (None, v, v.contiguous()):
            assert torch.equal(dropout(v, drop, r), dropout(v.contiguous(), drop, None if r is None else r.contiguous()))
    img = torch.randn(2, 24, 5, 7, generator=g).to(dtype).to(dev)
    cl = img.contiguous(memory_format=torch.channels_last)
    want = dropout(img.permute(0, 2, 3, 1).contiguous(), drop).permute(0, 3, 1, 2)
    assert torch.equal(dropout2d(img, drop), want) and torch.equal(dropout2d(cl, drop), want)
    assert dropout2d(cl, drop).is_contiguous(memory_format=torch.channels_last)
    whole = (want == 0).flatten(2)   # by channel: all of it or nothing
    assert bool((whole.all(-1) == whole.any(-1)).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dropped_values_are_zero_whatever_they_were(dev, dtype):
    drop = Drop(0.5, pair(3, 4, dev))
    keep = torch.from_numpy(oracle_mask(64, 96, 0.5, 3, 4)).to(dev)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        x = torch.full((64, 96), bad, device=dev, dtype=dtype).masked_fill(keep, 1.0)
        assert torch.equal(dropout(x, drop), keep.to(dtype) * 2)
        y = dropout(torch.full((64, 96), bad, device=dev, dtype=dtype), drop)
        assert bool((y[~keep] == 0).all()) and not bool((y[keep] == 0).any())


@gpu
def test_offsets_past_32_bits(dev):
    """2^31 values and more in one tensor: the last rows have the mask and the values of their place."""
    rows, cols = (2 ** 31) // 4096 + 77, 4096
    x = torch.ones(rows, cols, device=dev, dtype=torch.float16)
    y = dropout(x, Drop(0.25, pair(1, 2, dev)))
    keep = torch.from_numpy(oracle_mask(50, cols, 0.25, 1, 2, rows - 50)).to(dev)
    assert torch.equal(y[-50:] != 0, keep)
    del x, y
    # counter blocks past 32 bits: many rows of few columns, by a mask row of each
    got = dropout(torch.ones(3, 1, device=dev, dtype=torch.float32), Drop(0.5, pair(9, 9, dev)))
    assert torch.equal(got[:, 0] != 0, torch.from_numpy(oracle_mask(3, 1, 0.5, 9, 9)[:, 0]).to(dev))


@gpu
def test_empty_tensors_and_no_dropout(dev):
    drop = Drop(0.5, pair(0, 0, dev))
    for shape in ((0,), (0, 4), (4, 0), (2, 0, 3)):
        x = torch.ones(shape, device=dev, requires_grad=True)
        y = dropout(x, drop, x)
        y.sum().backward()
        assert y.shape == shape and x.grad.shape == shape
    x = torch.randn(3, 4, device=dev)
    assert dropout(x, None) is x and dropout(x, Drop(0.0, None)) is x
    assert torch.equal(dropout(x, None, x), x + x)


@gpu
def test_module_draws_new_masks_also_in_replays(dev):
    m = CounterDropout(0.5, seed=5, offset=2 ** 32 - 1).to(dev)
    x = torch.ones(64, 64, device=dev)

    def mask(n):
        return torch.from_numpy(oracle_mask(64, 64, 0.5, 5, 2 ** 32 - 1 + n)).to(dev).float() * 2

    assert torch.equal(m(x), mask(0)) and torch.equal(m(x), mask(1))
    m.eval()
    assert m(x) is x
    m.train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(m(x), mask(2))
    torch.cuda.current_stream().wait_stream(side)
    xs = torch.ones(64, 64, device=dev, requires_grad=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(xs)
        dx, = torch.autograd.grad(y, xs, torch.ones_like(y))
    for n in range(3, 7):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, mask(n)) and torch.equal(dx, mask(n))
        assert float((x + x).sum()) == 2 * 64 * 64   # eager work between the replays
    assert m.state.tolist()[1] == 2 ** 32 - 1 + 7
    assert "state" not in m.state_dict()


@gpu
def test_changed_rng_is_refused_by_the_backward(dev):
    rng = pair(1, 1, dev)
    x = torch.ones(4, 4, device=dev, requires_grad=True)
    y = dropout(x, Drop(0.5, rng))
    rng += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@gpu
def test_capture_is_refused_while_an_eager_graph_lives(dev):
    """Its leaves' accumulators are bound to the default stream; freed, the capture goes ahead."""
    rng = pair(1, 1, dev)
    w = torch.ones(8, 8, device=dev, requires_grad=True)
    y = dropout(w, Drop(0.5, rng))
    y.sum().backward()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="refusing to begin"):
        graph.capture_begin()
    del y
    gc.collect()
    w.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dropout(w, Drop(0.5, rng)).sum().backward()
    want = torch.from_numpy(oracle_mask(8, 8, 0.5, 1, 1)).to(dev).float() * 2
    for _ in range(3):
        w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w.grad, want)


def test_plain_path_on_the_cpu():
    """CPU tensors: the same masks, differentiable; float64 stays float64."""
    g = torch.Generator().manual_seed(1)
    for dtype in TYPES + [torch.float64]:
        x = torch.randn(2, 3, 5, generator=g).to(dtype).requires_grad_(True)
        drop = Drop(0.4, pair(8, 9), True)
        y = dropout(x, drop, x)
        ref, tol, keep = reference(x, x, drop, 3)
        assert y.dtype == dtype
        check(y, ref, tol)
        gx, = torch.autograd.grad(y.sum(), x)
        check(gx, 1.0 + keep.double() / 0.6, torch.finfo(dtype).eps * 4)
    m = CounterDropout(0.4, 8, 9, channels=True)
    a, b = m(torch.ones(2, 3, 5)), m(torch.ones(2, 3, 5))
    assert np.array_equal((a[:, 0] != 0).numpy(), oracle_mask(2, 5, 0.4, 8, 9))
    assert np.array_equal((b[:, 0] != 0).numpy(), oracle_mask(2, 5, 0.4, 8, 10))


def test_refusals():
    x, rng = torch.ones(2, 4), pair(0, 0)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            dropout(x, Drop(p, rng))
    with pytest.raises(ValueError, match="probability"):
        CounterDropout(2.0, 0)
    for bad in (rng.int(), torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(RuntimeError, match="rng"):
            dropout(x, Drop(0.5, bad))
    for res in (torch.ones(2, 5), torch.ones(2, 4, dtype=torch.float64), torch.ones(4)):
        with pytest.raises(RuntimeError, match="residual"):
            dropout(x, Drop(0.5, rng), res)
    with pytest.raises(RuntimeError, match="dimension"):
        dropout(torch.ones(()), Drop(0.5, rng))
    with pytest.raises(RuntimeError, match="images"):
        dropout2d(x, Drop(0.5, rng))
    L, a = _hip.lib(), ctypes.c_void_p(4096)
    for args, code in (((a, 4, None, 0, 0, -1, 4, 1, 0.5, a, a), -1), ((a, 4, None, 0, 0, 2 ** 41, 4, 1, 0.5, a, a), -1),
                       ((a, 4, None, 0, 3, 2, 4, 1, 0.5, a, a), -2), ((a, 4, None, 0, 0, 2, 4, 1, 1.5, a, a), -3),
                       ((a, 4, None, 0, 0, 2, 4, 1, float("nan"), a, a), -3),
                       ((a, 4, None, 0, 0, 2, 4, 1, 0.5, None, a), -4), ((a, 4, None, 0, 0, 2, 4, 0, 0.5, a, a), -4),
                       ((None, 4, None, 0, 0, 2, 4, 1, 0.5, a, a), -5), ((a, 3, None, 0, 0, 2, 4, 1, 0.5, a, a), -6),
                       ((a, 4, a, 3, 0, 2, 4, 1, 0.5, a, a), -6)):
        assert L.psfm_dropout(*args, None) == code, args
        assert L.psfm_dropout_last_error()
    assert L.psfm_dropout(a, 4, None, 0, 0, 0, 4, 1, 0.5, a, a, None) == 0      # nothing to do
    assert L.psfm_rng_next(None, 0, a, None) == -1 and L.psfm_rng_next(a, 0, None, None) == -1
