"""The residual block with counter-based channel dropout (layers01.ResidualConv, dropout_seed): the 1x1 product, its mask
and the sum of linear.conv1x1_act, then gn_act, together and inside the networks and the trainer that call them."""
import copy

import pytest
import torch
import torch.nn.functional as F

import packnet_sfm_amd  # noqa: F401
from packnet_sfm_amd.networks.layers import dropout as DR
from packnet_sfm_amd.networks.layers.packnet.layers01 import ResidualBlock, ResidualConv
from test_dropout import oracle_mask

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda", 0)


def tail(block, x, r, keep, p):
    """ELU(GN(r + drop(shortcut(x)))) in float64, keep [B, C]."""
    c, n = block.conv3[0], block.normalize
    h = F.conv2d(x, c.weight.double(), c.bias.double(), c.stride) * keep[:, :, None, None] / (1 - p)
    return F.elu(F.group_norm(r + h, n.num_groups, n.weight.double(), n.bias.double(), n.eps))


@pytest.mark.parametrize("stride", [1, 2])
def test_block_on_the_cpu(stride):
    """fp32: the formula's output and gradients with the oracle's mask, a new mask each forward, the plain module in
    eval, and the plain module's parameter names.  fp32 sums of up to 9 x 32 terms through two GroupNorms: 1e-4."""
    torch.manual_seed(0)
    m = ResidualConv(16, 32, stride, dropout=0.4, dropout_seed=9, dropout_offset=5)
    plain = ResidualConv(16, 32, stride, dropout=0.4)
    assert list(m.state_dict()) == list(plain.state_dict())
    plain.load_state_dict(m.state_dict())
    x = torch.randn(3, 16, 6, 8, requires_grad=True)
    for n in range(2):
        keep = torch.from_numpy(oracle_mask(3, 32, 0.4, 9, 5 + n)).double()
        y = m(x)
        want = tail(m, x.double(), m.conv2(m.conv1(x)).double(), keep, 0.4)
        assert torch.allclose(y.double(), want, rtol=1e-4, atol=1e-4)
        dy = torch.randn_like(y)
        leaves = [x] + list(m.parameters())
        for a, b in zip(torch.autograd.grad(y, leaves, dy, retain_graph=True),
                        torch.autograd.grad(want, leaves, dy.double())):
            assert torch.allclose(a, b.float(), rtol=1e-3, atol=1e-3 * float(b.abs().max()))
    m.eval(), plain.eval()
    assert torch.allclose(m(x), plain(x), rtol=1e-5, atol=1e-5)


def test_masks_of_blocks_ranks_and_networks_differ(monkeypatch):
    b = ResidualBlock(16, 16, 3, 1, dropout=0.5, dropout_seed=1, dropout_offset=7 << 40)
    drops = [m.conv3[1] for m in b]
    assert [d.state.tolist() for d in drops] == [[1, (7 << 40) + (i << 32)] for i in range(3)]
    monkeypatch.setattr(DR, "rank", lambda: 3)
    assert drops[0].draw().rng.tolist() == [4, 7 << 40] and drops[0].draw().rng.tolist() == [4, (7 << 40) + 1]
    from packnet_sfm_amd.networks import load_depth_net
    for name in ("PackNet01", "PackNetSAN01"):
        net = load_depth_net(name, version="1A", dropout=0.5, dropout_seed=3)
        states = [tuple(m.state.tolist()) for m in net.modules() if isinstance(m, DR.CounterDropout)]
        assert len(states) == 10 and len(set(states)) == 10 and {s[0] for s in states} == {3}
        plain = load_depth_net(name, version="1A", dropout=0.5)
        assert list(net.state_dict()) == list(plain.state_dict())
        assert not any(isinstance(m, DR.CounterDropout) for m in plain.modules())


@gpu
@pytest.mark.parametrize("cin,cout,stride,size", [(32, 64, 1, (24, 40)), (64, 64, 1, (7, 9)), (32, 32, 2, (12, 16))])
def test_block_in_bf16(dev, cin, cout, stride, size):
    """Under bf16 autocast, from the block's own conv branch r (bf16): the sum is rounded once (2^-9 of up to 5 deviations:
    1e-2 of y's deviation), y once more; its gradients pass two to three such roundings: 2e-2 of the largest."""
    torch.manual_seed(1)
    m = ResidualConv(cin, cout, stride, dropout=0.5, dropout_seed=4).to(dev).to(memory_format=torch.channels_last)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, cin, *size, generator=g).to(dev, torch.bfloat16).contiguous(memory_format=torch.channels_last)
    x.requires_grad_(True)
    real, kept = m.conv2.forward, []

    def conv2(t):
        kept.append(real(t).detach().requires_grad_(True))
        return kept[0]

    m.conv2.forward = conv2
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
    assert y.dtype == torch.bfloat16 and y.is_contiguous(memory_format=torch.channels_last)
    keep = torch.from_numpy(oracle_mask(3, cout, 0.5, 4, 0)).to(dev).double()
    c = m.conv3[0]
    ref = copy.deepcopy(m)
    with torch.no_grad():      # autocast's weights are the bf16 ones
        for p in (ref.conv3[0].weight, ref.conv3[0].bias):
            p.copy_(p.to(torch.bfloat16).float())
    x64, r64 = x.detach().double().requires_grad_(True), kept[0].detach().double().requires_grad_(True)
    want = tail(ref, x64, r64, keep, 0.5)
    dy = torch.randn(y.shape, generator=g).to(dev, torch.bfloat16)
    got = torch.autograd.grad(y, [kept[0], c.weight, c.bias, m.normalize.weight], dy)
    exp = torch.autograd.grad(want, [r64, ref.conv3[0].weight, ref.conv3[0].bias, ref.normalize.weight], dy.double())
    for a, b in zip((y,) + got, (want,) + exp):
        assert a.shape == b.shape
        assert float((a.double() - b.double()).abs().max()) < 2e-2 * float(b.abs().max())


@gpu
def test_captured_block_draws_a_mask_each_replay(dev):
    torch.manual_seed(3)
    m = ResidualBlock(32, 32, 2, 1, dropout=0.5, dropout_seed=8).to(dev).to(memory_format=torch.channels_last)
    x = torch.randn(2, 32, 16, 24, device=dev).contiguous(memory_format=torch.channels_last)
    drops = [b.conv3[1] for b in m]

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            y = m(x)
        grads = torch.autograd.grad(y, list(m.parameters()), torch.ones_like(y))
        return y.detach(), grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grads = step()
    seen = []
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert [d.state.tolist()[1] for d in drops] == [3 + n, (1 << 32) + 3 + n]
        assert bool(y.isfinite().all()) and all(bool(t.isfinite().all()) for t in grads)
        seen.append(y.clone())
        assert float((x * 0).sum()) == 0.0
    assert all(not torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])
    # a replayed mask is the seed's: the states before the first replay (they were 3 after it) give its block again
    for d, s in zip(drops, (2, (1 << 32) + 2)):
        d.state[1] = s
    graph.replay()
    torch.cuda.synchronize()
    off, most = float((y - seen[0]).float().abs().max()), float(seen[0].float().abs().max())
    assert off < 2e-2 * most


@gpu
def test_trainer_step_of_a_network_with_seeded_dropout(dev):
    """DDPTrainer's captured bf16 step of PackNetSAN01: the warm-up's draws are taken back with the rest of the training
    state, every step draws once per block, weights and loss stay finite."""
    import bench
    from packnet_sfm_amd.models.SelfSupModel import SelfSupModel
    from packnet_sfm_amd.networks import load_depth_net, load_pose_net
    from packnet_sfm_amd.trainers.ddp_trainer import DDPTrainer, make_optimizer
    torch.manual_seed(5)
    model = SelfSupModel(**bench.loss_kw(0.5, 80.0), upsample_depth_maps=True, rotation_mode="euler")
    model.add_depth_net(load_depth_net("PackNetSAN01", version="1A", dropout=0.5, dropout_seed=6))
    model.add_pose_net(load_pose_net("PoseNet", nb_ref_imgs=2))
    model = bench.to_channels_last(model.to(dev).train())
    trainer = DDPTrainer(model, make_optimizer(model, 1e-4, 1e-4, capturable=True), dev, amp_dtype=torch.bfloat16, graph=True)
    batch = bench.synthetic_batch(1, 64, 128, dev, seed=1, channels_last=True)
    states = [m.state for m in model.modules() if isinstance(m, DR.CounterDropout)]
    first = [s.tolist() for s in states]
    w = model.depth_net.encoder.conv2[0].conv3[0].weight
    before = w.detach().clone()
    for n in range(3):
        out = trainer.train_step(batch)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(out["loss"]).all())
        assert [s.tolist() for s in states] == [[a, b + n + 1] for a, b in first]
    assert not torch.equal(w, before) and bool(w.isfinite().all())
