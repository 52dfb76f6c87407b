"""The causal language model: the operators together, against the same model with torch's operators, and
trained for a while."""

import pytest
import torch
from torch.nn import functional as F

import morphottention_b200 as M
from morphottention_b200 import capi
from morphottention_b200.language import CausalLanguageModel, MixedPrecisionStep, main, synthetic_batch

pytestmark = pytest.mark.gpu


def torch_loss(model, tokens, targets):
    """The model's loss with torch's residual adds, layer norms and cross entropy in fp32 around the same
    attention and MLP."""
    def norm(m, x):
        return F.layer_norm(x.float(), (m.dim,), m.weight.float(), m.bias.float(), m.eps).to(x.dtype)
    h = model.embed(tokens)
    for b in model.blocks:
        h = h + b.attn(norm(b.norm1, h))
        h = h + b.mlp(norm(b.norm2, h))
    z = norm(model.norm, h).float() @ model.head.float().t()
    return F.cross_entropy(z.view(-1, z.shape[-1]), targets.view(-1), ignore_index=-100)


def test_loss_and_gradients_match_torch(cuda):
    torch.manual_seed(1)
    model = CausalLanguageModel(1003, 128, 2, 16, 2, device="cuda")
    tokens, targets = synthetic_batch(3, 100, 1003, 5, cuda)
    scale = 256.0
    loss = model(tokens, targets)
    (loss * scale).backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    want = torch_loss(model, tokens, targets)
    (want * scale).backward()
    assert capi.device_status(reset=True) == 0
    assert abs(loss.item() - want.item()) <= 1e-3 * want.item()  # fp16 activations on both sides
    for n, p in model.named_parameters():
        # two fp16 backward passes whose roundings differ: the encoder's tolerance for gradients, gate
        # gradients (sums of cancelling terms) as in the attention tests
        tol = 1.5e-2 if "gate" in n else 5e-3
        err = (got[n].double() - p.grad.double()).norm() / p.grad.double().norm()
        assert err <= 2 * tol, (n, err.item())


def test_scores_are_log_probabilities(cuda):
    torch.manual_seed(2)
    model = CausalLanguageModel(500, 128, 2, 16, 1, device="cuda")
    tokens, targets = synthetic_batch(1, 1, 500, 0, cuda)
    targets[:] = 3
    s = model.score(tokens, targets)
    z = model.hidden(tokens).float() @ model.head.float().t()
    assert s.shape == (1, 1)
    assert abs(s.item() - torch.log_softmax(z, -1)[0, 0, 3].item()) <= 1e-5 * 10
    every = torch.arange(500, device=cuda).view(1, -1)
    total = model.score(tokens.expand(1, 500).contiguous()[:, :1].expand(500, 1).contiguous(), every.view(500, 1)).exp().sum()
    assert abs(total.item() - 1.0) <= 1e-3


def test_training_learns_the_sequence(cuda):
    losses = main(["--steps", "60"])
    assert losses[0] > 6.0 and losses[-1] < 0.5 * losses[0], (losses[0], losses[-1])


def test_step_with_overflow_changes_nothing(cuda):
    torch.manual_seed(3)
    model = CausalLanguageModel(300, 64, 1, 16, 1, device="cuda")
    step = MixedPrecisionStep(model, lambda ps: torch.optim.SGD(ps, lr=0.1), loss_scale=2.0 ** 40)
    before = [p.detach().clone() for p in model.parameters()]
    _, norm = step(*synthetic_batch(2, 20, 300, 0, cuda))
    assert not torch.isfinite(norm)
    assert all(torch.equal(a, b) for a, b in zip(before, model.parameters()))


def test_step_clips(cuda):
    torch.manual_seed(4)
    model = CausalLanguageModel(300, 64, 1, 16, 1, device="cuda")
    step = MixedPrecisionStep(model, lambda ps: torch.optim.SGD(ps, lr=0.0), max_norm=0.01, loss_scale=512.0)
    _, norm = step(*synthetic_batch(2, 20, 300, 0, cuda))
    total = torch.stack([m.grad.double().square().sum() for m in step.masters]).sum().sqrt()
    assert norm.item() > 0.01 and abs(total.item() - 0.01) <= 1e-5


def test_captured_forward_and_backward(cuda):
    torch.manual_seed(5)
    model = CausalLanguageModel(300, 64, 1, 16, 1, device="cuda")
    tokens, targets = synthetic_batch(2, 50, 300, 0, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            model.zero_grad()
            (model(tokens, targets) * 64).backward()
    torch.cuda.current_stream().wait_stream(side)
    want = [p.grad.clone() for p in model.parameters()]
    model.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (model(tokens, targets) * 64).backward()
    graph.replay()
    torch.cuda.synchronize()
    for (n, p), w in zip(model.named_parameters(), want):
        if "embed" in n:  # torch's embedding backward adds in any order
            assert (p.grad.double() - w.double()).norm() <= 1e-2 * w.double().norm()
        else:
            assert (p.grad.double() - w.double()).norm() <= 5e-3 * w.double().norm(), n


def test_overflow_after_a_good_step_changes_nothing(cuda):
    """With an optimizer that has momentum and weight decay, which zero gradients would still move."""
    torch.manual_seed(3)
    model = CausalLanguageModel(300, 64, 1, 16, 1, device="cuda")
    step = MixedPrecisionStep(model, lambda ps: torch.optim.AdamW(ps, lr=1e-2), loss_scale=512.0)
    step(*synthetic_batch(2, 20, 300, 0, cuda))

    def everything():
        state = [v for s in step.optimizer.state.values() for v in s.values()]
        return [t.detach().clone() for t in (*model.parameters(), *step.masters, *state)]
    before = everything()
    step.loss_scale = 2.0 ** 40
    _, norm = step(*synthetic_batch(2, 20, 300, 1, cuda))
    assert not torch.isfinite(norm)
    assert all(torch.equal(a, b) for a, b in zip(before, everything()))
