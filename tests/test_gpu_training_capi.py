"""The training-step operators through the C ABI binding: the same bits as the torch ops, workspaces that are
too small refused, launches counted and timed like the other kernels'."""

import ctypes

import pytest
import torch

import morphottention_b200 as M
from morphottention_b200 import capi

pytestmark = pytest.mark.gpu


def test_layer_norm(cuda):
    g = torch.Generator(device="cuda").manual_seed(0)
    x, r, gy, gh = (torch.randn(700, 328, generator=g, device=cuda, dtype=torch.float16) for _ in range(4))
    w, b = torch.randn(328, generator=g, device=cuda), torch.randn(328, generator=g, device=cuda)
    want = M.layer_norm_forward(x, w, b, 1e-5, r)
    p = capi.layer_norm_problem(x, w)
    y, h, mean, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(700, device=cuda), torch.empty(700, device=cuda)
    capi.layer_norm_forward(p, x, r, w, b, y, h, mean, rstd)
    assert capi.last_launch_count() == 1
    assert all(torch.equal(a, c) for a, c in zip((y, mean, rstd, h), want))
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    capi.layer_norm_backward(p, gy, gh, h, w, mean, rstd, dx, dw, db)
    assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), M.layer_norm_backward(gy, h, w, mean, rstd, gh)))
    dx2 = torch.empty_like(x)  # dx alone
    capi.layer_norm_backward(p, gy, gh, h, w, mean, rstd, dx2, None, None)
    assert torch.equal(dx, dx2)
    L = capi.lib()
    rc = L.morpho_sm100_layer_norm_backward(ctypes.byref(p), *(t.data_ptr() for t in (gy, gh, h, w, mean, rstd, dx, dw, db)),
                                            dx2.data_ptr(), 16, None)
    assert rc == capi.MORPHO_ERR_WORKSPACE


def test_linear_cross_entropy(cuda):
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(150, 64, generator=g, device=cuda, dtype=torch.bfloat16)
    w = torch.randn(777, 64, generator=g, device=cuda, dtype=torch.bfloat16) / 8
    t = torch.randint(0, 777, (150,), generator=g, device=cuda)
    want = M.linear_cross_entropy_forward(h, w, t)
    p = capi.vocab_loss_problem(h, w)
    loss, lse = torch.empty((), device=cuda), torch.empty(150, device=cuda)
    capi.profile_enable(True)
    capi.linear_cross_entropy_forward(p, h, w, t, loss, lse)
    capi.profile_enable(False)
    assert set(capi.profile_collect()) == {"vocab_stats", "vocab_join"}
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    one, dh, dw = torch.ones((), device=cuda), torch.empty_like(h), torch.empty_like(w)
    capi.linear_cross_entropy_backward(p, one, h, w, t, lse, dh, dw)
    a, b = M.linear_cross_entropy_backward(one, h, w, t, lse)
    assert torch.equal(dh, a) and torch.equal(dw, b)
    L = capi.lib()
    rc = L.morpho_sm100_linear_cross_entropy_forward(ctypes.byref(p), h.data_ptr(), w.data_ptr(), t.data_ptr(), loss.data_ptr(),
                                                     lse.data_ptr(), dh.data_ptr(), 64, None)
    assert rc == capi.MORPHO_ERR_WORKSPACE
    assert capi.device_status(reset=True) == 0


def test_clip_grad_norm(cuda):
    g = [torch.randn(n, device=cuda).half() for n in (5, 3000, 70001)]
    out, want = [torch.empty(n.shape, device=cuda) for n in g], [torch.empty(n.shape, device=cuda) for n in g]
    norm = torch.empty((), device=cuda)
    capi.clip_grad_norm(g, out, 0.5, norm, 2.0)
    assert capi.last_launch_count() == 2
    assert torch.equal(norm, M.clip_grad_norm(g, 0.5, out=want, loss_scale=2.0))
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    pair = capi.MorphoTensorPair(g[0].data_ptr(), out[0].data_ptr(), 5, 0, 2)
    rc = capi.lib().morpho_sm100_clip_grad_norm(ctypes.byref(pair), 1, 1.0, 1.0, norm.data_ptr(), out[2].data_ptr(), 8, None)
    assert rc == capi.MORPHO_ERR_WORKSPACE


@pytest.mark.parametrize("rows,dim", [(700, 328), (3, 64), (5000, 777), (40, 33), (300, 9000)])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_layer_norm_sum_in_place(cuda, rows, dim, over):
    g = torch.Generator(device="cuda").manual_seed(dim)
    x, r = (torch.randn(rows, dim, generator=g, device=cuda, dtype=torch.float16) for _ in range(2))
    w, b = torch.randn(dim, generator=g, device=cuda), torch.randn(dim, generator=g, device=cuda)
    want = M.layer_norm_forward(x, w, b, 1e-5, r)
    p = capi.layer_norm_problem(x, w)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    h = x if over == "x" else r
    capi.layer_norm_forward(p, x, r, w, b, y, h, mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip((y, mean, rstd, h), want))
