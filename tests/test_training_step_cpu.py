"""The mixed-precision step's bookkeeping (masters, skipped steps) on the CPU, with the clipping operator replaced by
its formula; any module whose call gives a loss will do."""

import copy

import pytest
import torch
from torch import nn

from morphottention_b200 import language
from morphottention_b200.language import MixedPrecisionStep

OPTIMIZERS = {
    "adamw": lambda ps: torch.optim.AdamW(ps, lr=1e-2),
    "adam": lambda ps: torch.optim.Adam(ps, lr=1e-2),
    "momentum": lambda ps: torch.optim.SGD(ps, lr=1e-2, momentum=0.9, dampening=0.5),
    "decay": lambda ps: torch.optim.SGD(ps, lr=1e-2, weight_decay=0.1),
}


def clip(grads, max_norm, *, out, loss_scale):
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt() / loss_scale
    by = torch.clamp(max_norm / (norm + 1e-6), max=1.0) / loss_scale
    for g, o in zip(grads, out):
        o.copy_(g.double() * by)
    return norm.float()


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.a, self.b = nn.Linear(6, 4), nn.Linear(6, 4)

    def forward(self, x, both=True):
        y = self.a(x) + self.b(x) if both else self.a(x)
        return y.square().mean()


@pytest.fixture(params=sorted(OPTIMIZERS))
def step(request, monkeypatch):
    monkeypatch.setattr(language, "clip_grad_norm", clip)
    torch.manual_seed(0)
    return MixedPrecisionStep(Model(), OPTIMIZERS[request.param], loss_scale=8.0)


def everything(step):
    return copy.deepcopy(([p.detach() for p in step.params], [m.detach() for m in step.masters],
                          step.optimizer.state_dict()))


def same(a, b):
    if isinstance(a, torch.Tensor):
        return isinstance(b, torch.Tensor) and torch.equal(a, b)
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(same(a[k], b[k]) for k in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(same(x, y) for x, y in zip(a, b))
    return a == b


@pytest.mark.parametrize("good", [0, 1, 3])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_step_that_is_not_finite_changes_nothing(step, good, bad):
    for _ in range(good):
        step(torch.randn(5, 6))
    before = everything(step)
    _, norm = step(torch.full((5, 6), bad))
    assert not torch.isfinite(norm)
    assert same(before, everything(step))
    _, norm = step(torch.randn(5, 6))  # and the next one works again
    assert torch.isfinite(norm) and not same(before, everything(step))
    assert all(torch.isfinite(m).all() for m in step.masters)


def test_a_parameter_without_a_gradient_is_left_alone(step):
    step(torch.randn(5, 6))
    alone = {id(p) for p in step.model.b.parameters()}
    before = copy.deepcopy([(p.detach(), m.detach(), step.optimizer.state[m]) for p, m in zip(step.params, step.masters)])
    x = torch.randn(5, 6)
    _, norm = step(x, False)  # `b` takes no part
    after = [(p.detach(), m.detach(), step.optimizer.state[m]) for p, m in zip(step.params, step.masters)]
    for p, old, new in zip(step.params, before, after):
        assert same(old, new) == (id(p) in alone)
    _, norm = step(x)  # takes part again
    assert all(m.grad is not None for m in step.masters)
