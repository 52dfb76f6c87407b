"""The training-step operators as registered: torch's checks of schema and fake implementation against the real
ones, and a step through them traced by torch.compile (graphs run eagerly) with the eager step's bits."""

import pytest
import torch
from torch.library import opcheck

import morphottention_b200 as M

pytestmark = pytest.mark.gpu
UTILS = ("test_schema", "test_faketensor")


def randn(*size, seed=0, kind=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(size))
    return torch.randn(*size, generator=g, device="cuda").to(kind)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("wkind", [torch.float16, torch.float32, None])
def test_layer_norm(cuda, residual, wkind):
    o = torch.ops.morphottention
    x, r = randn(3, 6, 64), randn(3, 6, 64, seed=1) if residual else None
    w, b = (None, None) if wkind is None else (randn(64, kind=wkind), randn(64, seed=2, kind=wkind))
    opcheck(o.layer_norm_forward.default, (x, w, b, 1e-5, r), test_utils=UTILS)
    _, mean, rstd, *h = M.layer_norm_forward(x, w, b, 1e-5, r)
    opcheck(o.layer_norm_backward.default, (randn(3, 6, 64, seed=3), h[0] if h else x, w, mean, rstd, r), test_utils=UTILS)


@pytest.mark.parametrize("reduction", [0, 1, 2])
def test_linear_cross_entropy(cuda, reduction):
    o = torch.ops.morphottention
    h, w, t = randn(2, 9, 64), randn(50, 64), torch.arange(18, device="cuda").view(2, 9)
    opcheck(o.linear_cross_entropy_forward.default, (h, w, t, -100, reduction), test_utils=UTILS)
    loss, lse = o.linear_cross_entropy_forward(h, w, t, -100, reduction)
    opcheck(o.linear_cross_entropy_backward.default, (torch.ones_like(loss), h, w, t, lse, -100, reduction), test_utils=UTILS)


def test_clip_grad_norm(cuda):
    g = [randn(9), randn(3, 4, kind=torch.float32)]
    out = [torch.zeros(x.shape, device="cuda") for x in g]
    opcheck(torch.ops.morphottention.clip_grad_norm.default, (g, out, 0.1, 8.0), test_utils=UTILS)


def test_compiled(cuda):
    ln = M.LayerNorm(64, device="cuda")
    head, x = randn(100, 64).requires_grad_(), randn(6, 64).requires_grad_()
    t = torch.arange(6, device="cuda") * 7

    def f(x):
        y, h = ln(x, x * 2)
        return M.linear_cross_entropy(y + h, head, t)
    want = torch.autograd.grad(f(x), (x, head, ln.weight))
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x), (x, head, ln.weight))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
