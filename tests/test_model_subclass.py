"""A Model subclass with a setup_optimizer of its own: the train iteration it inherits must run as it did before optim.clip_norm existed."""
import torch

from neural_invertible_warp_amd.model import barf_inn_dtu, nerf
from neural_invertible_warp_amd.util import edict


class Graph(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(3))

    def forward(self, opt, var, mode=None, iter=None):
        return edict(var, out=(self.weight * var.x).sum())

    def compute_loss(self, opt, var, mode=None):
        return edict(render=var.out ** 2)


def own(base):
    class Model(base):
        def __init__(self):
            self.it, self.trainer, self.graph = 0, None, Graph()

        def setup_optimizer(self, opt):
            self.optim = torch.optim.SGD(self.graph.parameters(), lr=0.01)
            self.optim_pose = torch.optim.SGD([torch.nn.Parameter(torch.zeros(1))], lr=0.01)
            self.sched_pose = torch.optim.lr_scheduler.ExponentialLR(self.optim_pose, gamma=1.0)

        def summarize_loss(self, opt, var, loss):
            return edict(loss, all=loss.render)
    return Model()


def test_a_subclass_that_sets_up_its_own_optimizer_trains():
    for base in (nerf.Model, barf_inn_dtu.Model):
        model = own(base)
        if base is barf_inn_dtu.Model:
            model.graph.nerf = torch.nn.Module()
            model.graph.nerf.set_progress = lambda progress: None
        model.setup_optimizer(None)
        loss = model.train_iteration(edict(max_iter=10), edict(x=torch.tensor([1.0, 2.0, 3.0])))
        assert float(loss.all.detach()) == 36.0 and model.it == 1
        assert torch.allclose(model.graph.weight.detach(), 1 - 0.01 * 12 * torch.tensor([1.0, 2.0, 3.0]))
