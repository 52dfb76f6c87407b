"""A small causal language model on MorphoAttention, trained with this package's operators: the residual
adds and norms of its pre-norm blocks run as one kernel each (:class:`~.training.LayerNorm` with a
residual), the loss over the vocabulary never stores the logits, and :class:`MixedPrecisionStep` keeps
float32 masters of the float16 weights, with the loss scale removed and the gradients clipped on the way.

``python -m morphottention_b200.language`` trains one for a few steps on a synthetic sequence and prints
the losses.
"""

from __future__ import annotations

import argparse
import math

import torch
from torch import nn

from .autograd import MorphoAttention
from .encoder import MLP
from .training import LayerNorm, clip_grad_norm, linear_cross_entropy, linear_cross_entropy_forward


class CausalBlock(nn.Module):
    """One pre-norm block on a residual stream ``h`` and the last branch's output ``out``, which is still
    to be added to it: both adds happen inside the norms."""

    def __init__(self, dim: int, num_heads: int, cube_m: int, *, mlp_ratio: float = 4.0, scale: float = 1.0,
                 dtype=torch.float16, device=None) -> None:
        super().__init__()
        self.norm1 = LayerNorm(dim, dtype=dtype, device=device)
        self.attn = MorphoAttention(dim, num_heads, cube_m, scale=scale, causal=True, dtype=dtype, device=device)
        self.norm2 = LayerNorm(dim, dtype=dtype, device=device)
        self.mlp = MLP(dim, int(dim * mlp_ratio), dtype=dtype, device=device)

    def forward(self, out: torch.Tensor, h: torch.Tensor):
        y, h = self.norm1(out, h)
        y, h = self.norm2(self.attn(y), h)
        return self.mlp(y), h


class CausalLanguageModel(nn.Module):
    """Token embedding, ``depth`` causal blocks, a last norm, and an output embedding.

    ``forward(tokens, targets)`` is the mean cross entropy over the targets that are not
    ``ignore_index``; ``hidden(tokens)`` the states before the output embedding; ``score(tokens,
    targets)`` each target's log probability, without gradients.

    :param vocab: vocabulary size (any).
    :param dim: model width, a multiple of 8 and of ``num_heads`` with a head width of 32, 64 or 128."""

    def __init__(self, vocab: int, dim: int, num_heads: int, cube_m: int, depth: int, *, mlp_ratio: float = 4.0,
                 scale: float = 1.0, ignore_index: int = -100, dtype=torch.float16, device=None) -> None:
        super().__init__()
        self.ignore_index = ignore_index
        self.embed = nn.Embedding(vocab, dim, dtype=dtype, device=device)
        self.blocks = nn.ModuleList(CausalBlock(dim, num_heads, cube_m, mlp_ratio=mlp_ratio, scale=scale, dtype=dtype,
                                                device=device) for _ in range(depth))
        self.norm = LayerNorm(dim, dtype=dtype, device=device)
        self.head = nn.Parameter(torch.empty(vocab, dim, dtype=dtype, device=device))
        with torch.no_grad():
            for w in (self.embed.weight, self.head):
                w.copy_(torch.empty(w.shape, dtype=torch.float32, device=w.device).normal_(0.0, dim ** -0.5))

    def hidden(self, tokens: torch.Tensor) -> torch.Tensor:
        out = self.embed(tokens)
        h = torch.zeros_like(out)
        for block in self.blocks:
            out, h = block(out, h)
        return self.norm(out, h)[0]

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(self.hidden(tokens), self.head, targets, ignore_index=self.ignore_index)

    @torch.no_grad()
    def score(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        loss, _ = linear_cross_entropy_forward(self.hidden(tokens), self.head, targets, self.ignore_index, "none")
        return -loss


class MixedPrecisionStep:
    """Training steps of a float16 model with float32 master weights: the loss is multiplied by
    ``loss_scale``, the gradients are brought to float32 and clipped to ``max_norm`` in one operator, an
    optimizer updates the masters, and the model's weights are copied from them.  A step whose gradient
    norm is not finite changes nothing: masters, weights and the optimizer's state keep their values.
    (The optimizer is not called then, since zero gradients would still move what has momentum or weight
    decay; so the host reads the norm, and waits for the backward pass, once a step.)

    :param make_optimizer: builds the optimizer from the list of masters.
    :returns: ``step(tokens, targets)`` gives ``(loss, gradient norm)``, tensors on the device."""

    def __init__(self, model: nn.Module, make_optimizer, *, max_norm: float = 1.0, loss_scale: float = 1024.0) -> None:
        self.model, self.max_norm, self.loss_scale = model, max_norm, loss_scale
        self.params = [p for p in model.parameters() if p.requires_grad]
        self.masters = [p.detach().float().requires_grad_() for p in self.params]
        self.grads = [torch.zeros_like(m) for m in self.masters]  # what the masters' gradients are written to
        self.optimizer = make_optimizer(self.masters)

    def __call__(self, *batch):
        loss = self.model(*batch)
        for p in self.params:
            p.grad = None
        (loss * self.loss_scale).backward()
        for p, m, g in zip(self.params, self.masters, self.grads):  # a parameter that took no part has no gradient
            m.grad = None if p.grad is None else g
        norm = clip_grad_norm([p.grad for p in self.params if p.grad is not None], self.max_norm,
                              out=[m.grad for m in self.masters if m.grad is not None], loss_scale=self.loss_scale)
        if math.isfinite(norm.item()):
            self.optimizer.step()
            with torch.no_grad():
                torch._foreach_copy_(self.params, self.masters)
        return loss.detach(), norm


def synthetic_batch(batch: int, length: int, vocab: int, seed: int, device):
    """Sequences in which each token follows from the one before it by a fixed affine map of the
    vocabulary, from random first tokens, with a tenth of the targets ignored."""
    g = torch.Generator().manual_seed(seed)
    rows = [torch.randint(0, vocab, (batch,), generator=g)]
    for _ in range(length):
        rows.append((rows[-1] * 5 + 7) % vocab)
    seq = torch.stack(rows, 1)
    targets = seq[:, 1:].clone()
    targets[torch.rand(targets.shape, generator=g) < 0.1] = -100
    return seq[:, :-1].contiguous().to(device), targets.to(device)


def main(argv=None) -> list:
    ap = argparse.ArgumentParser(description="train a small causal language model on a synthetic sequence")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=128)
    ap.add_argument("--vocab", type=int, default=1000)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--depth", type=int, default=2)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = CausalLanguageModel(a.vocab, a.dim, a.dim // 64, 16, a.depth, device="cuda")
    step = MixedPrecisionStep(model, lambda ps: torch.optim.AdamW(ps, lr=2e-3))
    losses = []
    for i in range(a.steps):
        loss, norm = step(*synthetic_batch(a.batch, a.length, a.vocab, i, "cuda"))
        losses.append(loss)
        if i % 10 == 0 or i == a.steps - 1:
            print(f"step {i:4d}  loss {loss.item():.4f}  gradient norm {norm.item():.3f}")
    return [v.item() for v in losses]


if __name__ == "__main__":
    main()
