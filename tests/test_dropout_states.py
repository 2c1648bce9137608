"""The states of counter-based dropout in a trainer's checkpoint: a resumed run draws the masks that the run would have drawn."""
import pytest
import torch

import packnet_sfm_amd  # noqa: F401
from packnet_sfm_amd.networks.layers.dropout import CounterDropout, dropout_states, load_dropout_states
from packnet_sfm_amd.trainers.ddp_trainer import DDPTrainer, make_optimizer


class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.depth_net = torch.nn.Sequential(torch.nn.Linear(8, 16), CounterDropout(0.5, 7, 2 ** 40), torch.nn.Linear(16, 4),
                                             CounterDropout(0.25, -3, 2 ** 63 + 5))
        self.pose_net = torch.nn.Linear(8, 4)

    def forward(self, batch, progress=0.0):
        return {"loss": (self.depth_net(batch["x"]) - self.pose_net(batch["x"])).square().mean()}


def trainer(seed):
    torch.manual_seed(seed)
    m = Model()
    return m, DDPTrainer(m, make_optimizer(m, 1e-2, 1e-2), torch.device("cpu"), amp_dtype=None, graph=False, flat=True)


def test_a_resumed_run_goes_on(tmp_path):
    batches = [{"x": torch.randn(6, 8, generator=torch.Generator().manual_seed(n))} for n in range(5)]
    m, tr = trainer(0)
    for b in batches[:3]:
        tr.train_step(b)
    torch.save(tr.checkpoint(epoch=1), tmp_path / "c.ckpt")
    for b in batches[3:]:
        tr.train_step(b)
    ck = torch.load(tmp_path / "c.ckpt", weights_only=True)
    assert ck["dropout"] == {"depth_net.1": [7, 2 ** 40 + 3], "depth_net.3": [-3, 5 - 2 ** 63 + 3]}
    again, tr2 = trainer(1)
    again.load_state_dict({k[len("model."):]: v for k, v in ck["state_dict"].items()})
    tr2.optimizer.load_state_dict(ck["optimizer"])
    addresses = [b.data_ptr() for b in again.buffers()]
    load_dropout_states(again, ck["dropout"])
    assert addresses == [b.data_ptr() for b in again.buffers()]
    for b in batches[3:]:
        tr2.train_step(b)
    assert dropout_states(again) == dropout_states(m)
    for (k, a), b in zip(m.state_dict().items(), again.state_dict().values()):
        assert torch.equal(a, b), k


def test_states_of_other_layers_are_refused():
    m = Model()
    for states in ({}, {"depth_net.1": [1, 2]}, {**dropout_states(m), "depth_net.0": [1, 2]}):
        with pytest.raises(RuntimeError, match="other layers"):
            load_dropout_states(m, states)
    assert dropout_states(torch.nn.Linear(2, 2)) == {}
    load_dropout_states(torch.nn.Linear(2, 2), {})
