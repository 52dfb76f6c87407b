"""Layer norm with its residual add against a plain 64-bit form.

Tolerances, per element: an output rounded to a type of unit roundoff u is off by at most u of its
value; everything before that rounding is fp32, whose error is a few 2^-24 of the terms that are added
(ARITH bounds the count: sums over dim run as trees and short chains)."""

import ctypes

import pytest
import torch

import morphottention_b200 as M
from morphottention_b200 import capi

pytestmark = pytest.mark.gpu

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half the smallest fp16 step
ARITH = 64 * 2.0 ** -24
EPS = 1e-5


def make(rows, dim, kind, wkind, residual, seed=0, offset=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    d = {"x": (n(rows, dim) + offset).to(kind), "w": (1 + 0.2 * n(dim)).to(wkind), "b": (0.2 * n(dim)).to(wkind),
         "gy": n(rows, dim).to(kind), "res": n(rows, dim).to(kind) if residual else None,
         "gh": n(rows, dim).to(kind) if residual else None}
    return d


def plain(d, eps=EPS):
    """The formulas in 64 bits, and for each gradient the magnitudes its terms are summed at."""
    x = d["x"].double()
    h = x if d["res"] is None else (x + d["res"].double()).to(d["x"].dtype).double()
    mu = h.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((h - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (h - mu) * rstd
    w = torch.ones_like(h[0]) if d["w"] is None else d["w"].double()
    b = torch.zeros_like(w) if d["b"] is None else d["b"].double()
    gy = d["gy"].double()
    g = gy * w
    mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - mg - xh * mgx)
    if d["gh"] is not None:
        dx = dx + d["gh"].double()
    size_x = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)
                     * 2) * (1 + h.abs().amax(-1, keepdim=True) * rstd)
    # an error of the mean (a few 2^-24 of |h|) moves xh by rstd as much
    slack = h.abs().amax(-1, keepdim=True) * rstd
    return {"h": h, "y": xh * w + b, "size_y": (xh.abs() + slack) * w.abs() + b.abs(), "dx": dx, "size_x": size_x,
            "dw": (gy * xh).sum(0), "size_w": (gy.abs() * (xh.abs() + slack)).sum(0), "db": gy.sum(0),
            "size_b": gy.abs().sum(0), "mean": mu[:, 0], "rstd": rstd[:, 0]}


def near(got, want, size, what):
    u, tiny = ROUND[got.dtype], TINY[got.dtype]
    bound = u * want.abs() + (1 + u) * ARITH * size + tiny
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound).all(), f"{what}: {(off / bound).max().item():.2f} of its bound"


def check(d, eps=EPS):
    y, mean, rstd, *h = M.layer_norm_forward(d["x"], d["w"], d["b"], eps, d["res"])
    e = plain(d, eps)
    if d["res"] is not None:
        assert torch.equal(h[0].double(), e["h"])
    near(y, e["y"], e["size_y"], "y")
    near(mean, e["mean"], e["h"].abs().amax(-1), "mean")
    hh = h[0] if h else d["x"]
    dx, dw, db = M.layer_norm_backward(d["gy"], hh, d["w"], mean, rstd, d["gh"])
    near(dx, e["dx"], e["size_x"], "dx")
    near(dw, e["dw"], e["size_w"], "dweight")
    near(db, e["db"], e["size_b"], "dbias")
    again = M.layer_norm_backward(d["gy"], hh, d["w"], mean, rstd, d["gh"])
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))


# widths on both sides of every change of kernel: one vector, a warp's 1024, a CTA's 8192, beyond; odd ones
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 64, 197, 256, 264, 768, 1001, 1024, 1032, 2048, 2056, 4100, 8192, 8200])
def test_widths(cuda, dim, kind):
    check(make(5, dim, kind, kind, residual=True, seed=dim))


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 197, 1500, 5000])
@pytest.mark.parametrize("residual", [False, True])
def test_rows(cuda, rows, residual):
    check(make(rows, 264, torch.float16, torch.float16, residual, seed=rows))


# enough rows for the streaming kernels: every number of warps to a row, full and part-filled lanes
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,dim", [(4736, 8), (5001, 200), (4999, 256), (6000, 264), (4800, 512), (5003, 776), (4740, 1024),
                                      (2400, 1032), (2501, 2048), (1300, 2056), (1201, 4096), (600, 4104), (700, 8192)])
def test_many_rows(cuda, rows, dim, kind):
    check(make(rows, dim, kind, kind, residual=True, seed=dim))
    check(make(rows, dim, kind, torch.float32, residual=False, seed=dim))


# rows whose length is no multiple of 16 bytes: every group width, and widths where the widest offset just
# fits or needs the next group
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,dim", [(5000, 3), (4999, 57), (5001, 63), (5003, 121), (4801, 249), (4805, 250), (4799, 507),
                                      (5007, 777), (4741, 1001), (2500, 1017), (2501, 1019), (2399, 2045), (1301, 4091),
                                      (1300, 6001), (1201, 8185), (1203, 8187)])
def test_many_shifted_rows(cuda, rows, dim, kind):
    check(make(rows, dim, kind, kind, residual=True, seed=dim))
    check(make(rows, dim, kind, torch.float32, residual=False, seed=dim))


@pytest.mark.parametrize("at", [1, 3])
@pytest.mark.parametrize("dim", [256, 777])
def test_contiguous_rows_off_a_boundary(cuda, at, dim):
    """Contiguous inputs that begin inside a 16-byte pack: the backward's alike, the forward's unlike its outputs."""
    d = make(5000, dim, torch.float16, torch.float16, residual=True)
    for k in ("x", "res", "gy", "gh"):
        flat = torch.full((5000 * dim + 8,), float("nan"), device="cuda", dtype=torch.float16)
        flat[at:at + 5000 * dim] = d[k].flatten()
        d[k] = flat[at:at + 5000 * dim].view(5000, dim)
    check(d)


def test_shifted_rows_do_not_see_their_neighbours(cuda):
    d = make(5000, 777, torch.float16, torch.float16, residual=True)
    y0, mean, rstd, h0 = M.layer_norm_forward(d["x"], d["w"], d["b"], EPS, d["res"])
    dx0 = M.layer_norm_backward(d["gy"], h0, d["w"], mean, rstd, d["gh"])[0]
    d["x"][1::2] = float("nan")
    y, mean, rstd, h = M.layer_norm_forward(d["x"], d["w"], d["b"], EPS, d["res"])
    assert torch.equal(y[::2], y0[::2]) and torch.equal(h[::2], h0[::2]) and y[1::2].isnan().all()
    dx = M.layer_norm_backward(d["gy"], h, d["w"], mean, rstd, d["gh"])[0]
    assert torch.equal(dx[::2], dx0[::2]) and dx[1::2].isnan().all()


def test_many_strided_rows(cuda):
    d = make(5000, 256, torch.float16, torch.float16, residual=True)
    for k in ("x", "res", "gy", "gh"):
        wide = torch.zeros(5000, 280, device="cuda", dtype=torch.float16)
        wide[:, 8:264] = d[k]
        d[k] = wide[:, 8:264]
    check(d)
    d["gy"] = d["gy"][:1].expand(5000, 256)
    check(d)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_fp32_weights(cuda, kind):
    check(make(77, 512, kind, torch.float32, residual=True))
    check(make(77, 2500, kind, torch.float32, residual=True))


def test_without_weight_or_bias(cuda):
    d = make(9, 320, torch.float16, torch.float16, residual=False)
    d["b"] = None
    check(d)
    d["w"] = None
    check(d)


@pytest.mark.parametrize("dim", [256, 200, 33])
def test_strided_rows_and_odd_bases(cuda, dim):
    """Rows that are views of wider ones, at offsets of one element (no 16-byte alignment)."""
    for at in (0, 1, 8):
        d = make(24, dim, torch.float16, torch.float16, residual=True)
        for k in ("x", "res", "gy", "gh"):
            wide = torch.zeros(24, dim + 24, device="cuda", dtype=torch.float16)
            wide[:, at:at + dim] = d[k]
            d[k] = wide[:, at:at + dim]
        check(d)


def test_leading_dimensions_and_transposes(cuda):
    d = make(24, 64, torch.float16, torch.float16, residual=True)
    y, mean, rstd, h = M.layer_norm_forward(d["x"], d["w"], d["b"], EPS, d["res"])
    x3 = d["x"].view(4, 6, 64).transpose(0, 1).contiguous().transpose(0, 1)  # rows without one stride
    y3, mean3, _, h3 = M.layer_norm_forward(x3, d["w"], d["b"], EPS, d["res"].view(4, 6, 64))
    assert y3.shape == (4, 6, 64) and mean3.shape == (4, 6)
    assert torch.equal(y3.reshape(24, 64), y) and torch.equal(h3.reshape(24, 64), h)
    xt = d["x"].t().contiguous().t()  # last dimension not contiguous
    assert torch.equal(M.layer_norm_forward(xt, d["w"], d["b"], EPS, d["res"])[0], y)
    ge = d["gy"][:1].expand(24, 64)  # a broadcast gradient
    a = M.layer_norm_backward(ge, h, d["w"], mean, rstd)
    b = M.layer_norm_backward(ge.contiguous(), h, d["w"], mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_large_offset_keeps_the_variance(cuda):
    """|mean| a thousand times the deviation: a one-pass variance would lose it."""
    check(make(16, 1024, torch.float32, torch.float32, residual=False, offset=1000.0))


def test_constant_rows(cuda):
    d = make(4, 128, torch.float16, torch.float16, residual=False)
    d["x"] = torch.full_like(d["x"], 3.0)
    check(d)  # variance 0: rstd = eps^-1/2


def test_no_rows(cuda):
    x = torch.empty(0, 64, device="cuda", dtype=torch.float16)
    w = torch.ones(64, device="cuda", dtype=torch.float16)
    y, mean, rstd = M.layer_norm_forward(x, w, w)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = M.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_non_finite_rows_stay_in_their_rows(cuda):
    d = make(8, 256, torch.float16, torch.float16, residual=False)
    clean = M.layer_norm_forward(d["x"], d["w"], d["b"])[0]
    d["x"][3, 7] = float("inf")
    d["x"][5, 9] = float("nan")
    y = M.layer_norm_forward(d["x"], d["w"], d["b"])[0]
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[keep], clean[keep]) and y[3].isnan().any() and y[5].isnan().all()


def test_more_than_2_31_elements(cuda):
    rows, dim = 1 << 21, 1032
    x = torch.empty(rows, dim, device="cuda", dtype=torch.float16)
    g = torch.Generator(device="cuda").manual_seed(3)
    for c in x.split(1 << 18):
        c.normal_(generator=g)
    w = torch.ones(dim, device="cuda", dtype=torch.float16)
    y, mean, rstd = M.layer_norm_forward(x, w, None)
    dx, dw, db = M.layer_norm_backward(x, x, w, mean, rstd)
    d = {"x": x[-7:], "w": w, "b": None, "gy": x[-7:], "res": None, "gh": None}
    e = plain(d)
    near(y[-7:], e["y"], e["size_y"], "y")
    near(dx[-7:], e["dx"], e["size_x"], "dx")
    db64 = sum(c.double().sum(0) for c in x.split(1 << 18))
    # 2^21 terms through partial sums of up to 2^11 (a CTA's rows) and 2^9 (the CTAs)
    assert ((db.double() - db64).abs() <= ROUND[db.dtype] * db64.abs() + 2.0 ** -24 * 2600 * 0.8 * 2100).all()


def test_gradients_against_differences(cuda):
    """The kernel's gradients along random directions against central differences of the 64-bit form."""
    d = make(6, 72, torch.float32, torch.float32, residual=True)
    y, mean, rstd, h = M.layer_norm_forward(d["x"], d["w"], d["b"], EPS, d["res"])
    dx, dw, db = M.layer_norm_backward(d["gy"], h, d["w"], mean, rstd, d["gh"])
    g = torch.Generator(device="cuda").manual_seed(5)

    def loss(x, w, b):
        h = x + d["res"].double()
        c = h - h.mean(-1, keepdim=True)
        y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS) * w + b
        return (y * d["gy"].double()).sum() + (h * d["gh"].double()).sum()

    at = [d[k].double() for k in ("x", "w", "b")]
    for i, grad in enumerate((dx, dw, db)):
        v = torch.randn(at[i].shape, generator=g, device="cuda", dtype=torch.float64)
        step = 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step * v, at[i] - step * v
        want = (loss(*up) - loss(*down)) / (2 * step)
        got = (grad.double() * v).sum()
        size = (grad.double().abs() * v.abs()).sum()
        # differences are good to step^2 and 1e-16 / step; h = x + residual is rounded once, to 2^-24
        assert abs(got - want) <= 1e-5 * size, (i, got.item(), want.item())


def test_autograd_module_and_residual(cuda):
    torch.manual_seed(0)
    ln = M.LayerNorm(96, device="cuda")
    ref = torch.nn.LayerNorm(96, device="cuda", dtype=torch.float64)
    with torch.no_grad():
        ln.weight.add_(0.1 * torch.randn_like(ln.weight))
    ref.load_state_dict({k: v.double() for k, v in ln.state_dict().items()})
    x = torch.randn(3, 5, 96, device="cuda", dtype=torch.float16, requires_grad=True)
    r = torch.randn(3, 5, 96, device="cuda", dtype=torch.float16, requires_grad=True)
    y, h = ln(x, r)
    (y.float().square().sum() + h.float().sum()).backward()
    h64 = h.detach().double().requires_grad_()
    y64 = ref(h64)
    (y64.square().sum() + h64.sum()).backward()
    # dy itself is rounded (2 y, with y rounded): two roundings of each term, and the result's
    for got, want in ((x.grad, h64.grad), (r.grad, h64.grad), (ln.weight.grad, ref.weight.grad), (ln.bias.grad, ref.bias.grad)):
        assert (got.double() - want).norm() <= 3 * 2.0 ** -11 * want.norm()
    assert torch.equal(x.grad, r.grad)
    # only h used: the gradient passes straight through
    y, h = ln(x, r)
    x.grad = None
    h.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))
    # without a residual
    x.grad = None
    ln(x).sum().backward()
    assert x.grad is not None


def test_no_second_derivative(cuda):
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    one = torch.ones(64, device="cuda")
    (dx,) = torch.autograd.grad(M.layer_norm(x, one, one).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_on_another_stream(cuda):
    d = make(64, 512, torch.float16, torch.float16, residual=True)
    want = M.layer_norm_forward(d["x"], d["w"], d["b"], EPS, d["res"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = M.layer_norm_forward(d["x"], d["w"], d["b"], EPS, d["res"])
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda):
    d = make(4, 64, torch.float16, torch.float16, residual=True)
    f = M.layer_norm_forward
    with pytest.raises(RuntimeError, match="weight must be"):
        f(d["x"], d["w"][:63], d["b"])
    with pytest.raises(RuntimeError, match="same type"):
        f(d["x"], d["w"], d["b"].float())
    with pytest.raises(RuntimeError, match="x's type or be float32|x's type or float32"):
        f(d["x"], d["w"].bfloat16(), d["b"].bfloat16())
    with pytest.raises(RuntimeError, match="residual must have x's shape"):
        f(d["x"], d["w"], d["b"], EPS, d["res"][:2])
    with pytest.raises(RuntimeError, match="residual must have x's type"):
        f(d["x"], d["w"], d["b"], EPS, d["res"].float())
    with pytest.raises(RuntimeError, match="must be float16, bfloat16 or float32"):
        f(d["x"].double(), None, None)
    with pytest.raises(RuntimeError, match="bias needs a weight"):
        f(d["x"], None, d["b"])
    with pytest.raises(RuntimeError, match="empty last dimension"):
        f(d["x"][:, :0], None, None)
    with pytest.raises(RuntimeError, match="eps must be non-negative"):
        f(d["x"], d["w"], d["b"], -1.0)
    y, mean, rstd, h = f(d["x"], d["w"], d["b"], EPS, d["res"])
    with pytest.raises(RuntimeError, match="grad_y must match"):
        M.layer_norm_backward(d["gy"].float(), h, d["w"], mean, rstd)
    with pytest.raises(RuntimeError, match="mean must be"):
        M.layer_norm_backward(d["gy"], h, d["w"], mean[:2], rstd)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        f(d["x"], d["w"].cpu(), None)


def test_last_dimension_past_32_bits_is_refused(cuda):
    x = torch.zeros(1, device="cuda", dtype=torch.float16).expand((1 << 32) + 64)
    one = torch.ones((), device="cuda")
    with pytest.raises(RuntimeError, match="last dimension"):
        M.layer_norm_forward(x)
    with pytest.raises(RuntimeError, match="last dimension"):
        M.layer_norm_backward(x, x, None, one, one)


def test_a_group_gives_up_as_one(cuda):
    """One warp of a group waits for a row that never comes: the wait is bounded, both warps of the group
    leave together (neither is left at the group's barrier) and the others go on."""
    assert capi.device_status(reset=True) == 0
    seen = torch.full((8,), -1, device="cuda", dtype=torch.int32)
    capi.selftest_row_wait(seen)
    assert seen.tolist() == [1, 1, 0, 0, 1, 1, 1, 1]
    with pytest.raises(capi.MorphoError) as e:
        capi.device_status(reset=False)
    assert e.value.code == capi.MORPHO_ERR_TIMEOUT
    word = ctypes.c_uint32(0)
    capi.lib().morpho_sm100_device_status(torch.cuda.current_stream().cuda_stream, 1, ctypes.byref(word))
    assert word.value == (0x80000000 | (2 << 8) | 7)
    check(make(2400, 1032, torch.float16, torch.float16, residual=True))
    assert capi.device_status(reset=True) == 0
