"""The training-step operators without a GPU: exports, schemas, shapes under fake tensors, refusals of the
Python forms and of the C ABI (nothing here launches a kernel)."""

import ctypes

import pytest
import torch

import morphottention_b200 as M
from morphottention_b200 import capi


def test_exports_and_schemas():
    for name in ("LayerNorm", "layer_norm", "layer_norm_forward", "layer_norm_backward", "linear_cross_entropy",
                 "linear_cross_entropy_forward", "linear_cross_entropy_backward", "clip_grad_norm", "clip_grad_norm_"):
        assert name in M.__all__ and callable(getattr(M, name))
    ops = torch.ops.morphottention
    assert str(ops.layer_norm_forward.default._schema).endswith(
        "(Tensor x, Tensor? weight, Tensor? bias, float eps, Tensor? residual=None) -> Tensor[]")
    assert str(ops.linear_cross_entropy_backward.default._schema).endswith("int reduction=1) -> Tensor[]")


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 5, 64, device="cuda", dtype=torch.float16)
        w = torch.empty(64, device="cuda", dtype=torch.float16)
        y, mean, rstd = M.layer_norm_forward(x, w, w)
        assert y.shape == x.shape and mean.shape == (2, 5) and rstd.dtype == torch.float32
        assert len(M.layer_norm_forward(x, w, w, 1e-5, x)) == 4
        dx, dw, db = M.layer_norm_backward(x, x, w, mean, rstd)
        assert dx.shape == x.shape and dw.shape == db.shape == (64,)
        v = torch.empty(100, 64, device="cuda", dtype=torch.float16)
        t = torch.empty(2, 5, device="cuda", dtype=torch.int64)
        loss, lse = M.linear_cross_entropy_forward(x, v, t)
        assert loss.shape == () and lse.shape == (2, 5) and loss.dtype == torch.float32
        assert M.linear_cross_entropy_forward(x, v, t, -100, "none")[0].shape == (2, 5)
        dh, dv = M.linear_cross_entropy_backward(loss, x, v, t, lse)
        assert dh.shape == x.shape and dv.shape == v.shape
        assert M.clip_grad_norm([x, w], 1.0).shape == ()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="expects a CUDA tensor"):
        M.layer_norm(x)
    with pytest.raises(ValueError, match="expects a CUDA tensor"):
        M.LayerNorm(64)(x)
    with pytest.raises(ValueError, match="expects CUDA tensors"):
        M.linear_cross_entropy(x, x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="reduction must be one of"):
        M.linear_cross_entropy(x, x, torch.zeros(2, dtype=torch.int64), reduction="total")
    with pytest.raises(NotImplementedError):
        M.clip_grad_norm([x], 1.0)
    with pytest.raises(ValueError, match="dim must be positive"):
        M.LayerNorm(0)


def test_layer_norm_module_state():
    m, ref = M.LayerNorm(32), torch.nn.LayerNorm(32, dtype=torch.float16)
    assert m.state_dict().keys() == ref.state_dict().keys()
    m.load_state_dict(ref.state_dict())
    assert torch.all(m.weight == 1) and torch.all(m.bias == 0)
    assert [n for n, _ in M.LayerNorm(32, bias=False).named_parameters()] == ["weight"]


def norm_problem(**kw):
    d = dict(rows=4, dim=64, type=0, weight_type=0, eps=1e-5, stride_x=0, stride_residual=0, stride_grad_y=0, stride_grad_h=0)
    return capi.MorphoLayerNorm(*{**d, **kw}.values())


def loss_problem(**kw):
    d = dict(tokens=4, vocab=100, dim=64, type=0, reduction=1, ignore_index=-100, stride_hidden=0, stride_weight=0)
    return capi.MorphoVocabLoss(*{**d, **kw}.values())


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(dim=0), dict(type=3), dict(type=0, weight_type=1), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(stride_x=63), dict(rows=1 << 40)], ids=str)
def test_layer_norm_problems_refused(bad):
    L, p = capi.lib(), norm_problem(**bad)
    assert L.morpho_sm100_layer_norm_forward(ctypes.byref(p), *[None] * 9) == capi.MORPHO_ERR_INVALID
    assert "layer norm" in capi.last_error()
    assert L.morpho_sm100_layer_norm_backward_workspace_size(ctypes.byref(p)) == 0


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(vocab=0), dict(dim=60), dict(dim=16392), dict(type=2), dict(reduction=3),
                                 dict(stride_hidden=65), dict(stride_weight=56)], ids=str)
def test_cross_entropy_problems_refused(bad):
    L, p = capi.lib(), loss_problem(**bad)
    for name in ("forward", "backward"):
        assert getattr(L, f"morpho_sm100_linear_cross_entropy_{name}_workspace_size")(ctypes.byref(p)) == 0
        assert "cross entropy" in capi.last_error()
    assert L.morpho_sm100_linear_cross_entropy_forward(ctypes.byref(p), *[None] * 6, 0, None) == capi.MORPHO_ERR_INVALID


def test_null_and_misaligned_pointers_refused():
    L = capi.lib()
    assert L.morpho_sm100_layer_norm_forward(ctypes.byref(norm_problem()), *[None] * 9) == capi.MORPHO_ERR_INVALID
    assert "x is NULL" in capi.last_error()
    p = loss_problem()
    at = [0x1000, 0x2008, 0x3000, 0x4000, 0x5000, 0x6000]  # weight at 8 bytes
    rc = L.morpho_sm100_linear_cross_entropy_forward(ctypes.byref(p), *at, 1 << 30, None)
    assert rc == capi.MORPHO_ERR_INVALID and "weight is not 16-byte aligned" in capi.last_error()
    assert L.morpho_sm100_layer_norm_forward(None, *[None] * 9) == capi.MORPHO_ERR_INVALID


def test_clip_arguments_refused():
    L = capi.lib()
    pair = capi.MorphoTensorPair(0x1000, 0x1000, 8, 0, 0)
    ws = 0x10000
    call = lambda p, n, m, s, norm=0x8000, w=ws: L.morpho_sm100_clip_grad_norm(ctypes.byref(p), n, m, s, norm, w, 1 << 20, None)  # noqa: E731
    for args in ((pair, 1, -1.0, 1.0), (pair, 1, float("nan"), 1.0), (pair, 1, 1.0, 0.0), (pair, -1, 1.0, 1.0),
                 (pair, 1, 1.0, 1.0, None), (pair, 1, 1.0, 1.0, 0x8000, None),
                 (capi.MorphoTensorPair(0x1000, 0x1000, 8, 0, 2), 1, 1.0, 1.0), (capi.MorphoTensorPair(0x1001, 0x1001, 8, 0, 0), 1, 1.0, 1.0),
                 (capi.MorphoTensorPair(0x1000, None, 8, 0, 0), 1, 1.0, 1.0), (capi.MorphoTensorPair(0x1000, 0x1000, 8, 7, 7), 1, 1.0, 1.0)):
        assert call(*args) == capi.MORPHO_ERR_INVALID
        assert "clip" in capi.last_error()


def test_backward_workspace_is_bounded():
    """One piece of dz at a time: the workspace of a large problem stays far below the logits."""
    L = capi.lib()
    p = loss_problem(tokens=1 << 16, vocab=131072, dim=2048)
    n = L.morpho_sm100_linear_cross_entropy_backward_workspace_size(ctypes.byref(p))
    assert 0 < n < 2 * (1 << 16) * 131072 // 8


def test_misaligned_parameters_refused():
    """Pointers off their element's size, which a kernel would fault on, in every place that takes one."""
    L, p = capi.lib(), norm_problem(weight_type=2)
    at = [0x1000 * (i + 1) for i in range(9)]
    names = ["x", "residual", "weight", "bias", "y", "h", "mean", "rstd"]
    for i, name in enumerate(names):
        bad = [a + (i == k) for k, a in enumerate(at[:8])]
        assert L.morpho_sm100_layer_norm_forward(ctypes.byref(p), *bad, None) == capi.MORPHO_ERR_INVALID, name
        assert f"{name} is not aligned" in capi.last_error()
    assert L.morpho_sm100_layer_norm_forward(ctypes.byref(p), *at[:2], at[2] + 2, *at[3:8], None) == capi.MORPHO_ERR_INVALID
    names = ["grad_y", "grad_h", "h", "weight", "mean", "rstd", "dx", "dweight", "dbias"]
    for rows in (4, 0):
        p = norm_problem(weight_type=2, rows=rows)
        for i, name in enumerate(names):
            if rows == 0 and not name.startswith(("dw", "db")):
                continue
            bad = [a + (i == k) for k, a in enumerate(at)]
            rc = L.morpho_sm100_layer_norm_backward(ctypes.byref(p), *bad, 0xA0000, 1 << 30, None)
            assert rc == capi.MORPHO_ERR_INVALID, name
            assert f"{name} is not aligned" in capi.last_error()
    pair = capi.MorphoTensorPair(0x1000, 0x1000, 8, 0, 0)
    rc = L.morpho_sm100_clip_grad_norm(ctypes.byref(pair), 1, 1.0, 1.0, 0x8002, 0x10000, 1 << 20, None)
    assert rc == capi.MORPHO_ERR_INVALID and "norm" in capi.last_error()


def test_sum_in_place_of_strided_rows_refused():
    """h is contiguous: written over rows with gaps it would overtake rows that are not read yet."""
    L, at = capi.lib(), [0x1000 * (i + 1) for i in range(8)]
    for strides, over in ((dict(stride_x=80), 0), (dict(stride_residual=72), 1)):
        p = norm_problem(**strides)
        args = [*at[:5], at[over], *at[6:]]
        assert L.morpho_sm100_layer_norm_forward(ctypes.byref(p), *args, None) == capi.MORPHO_ERR_INVALID
        assert "in place" in capi.last_error()
