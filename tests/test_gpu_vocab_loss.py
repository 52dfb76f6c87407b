"""The vocabulary loss (linear layer, softmax cross entropy, no logits kept) against a plain 64-bit form.

Tolerances, per element.  A logit is an fp32 sum of exact products, added up in at most dim / 16 steps
each good to 2^-23 of the magnitudes S = |hidden| . |weight|: dz = dim 2^-27 S.  lse, loss and the
probabilities inherit it (plus a few 2^-22 of their own).  dz is rounded once to the inputs' type (u of
itself; 2^-40 below fp16's range), the products' fp32 sums add (terms / 16) 2^-23 of their magnitudes,
and the result is rounded once."""

import threading

import pytest
import torch

import morphottention_b200 as M
from morphottention_b200 import capi

pytestmark = pytest.mark.gpu

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
IGNORE = -100


def make(T, V, D, kind, seed=0, ignored=0.2, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * T + V + D)
    w = (spread * D ** -0.5 * torch.randn(V, D, generator=g, device="cuda")).to(kind)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    h = (torch.randn(T, D, generator=g, device="cuda") + w[y].float()).to(kind)
    y[torch.rand(T, generator=g, device="cuda") < ignored] = IGNORE
    return h, w, y


def plain(h, w, y, reduction, grad, ignore=IGNORE):
    h, w = h.double(), w.double()
    T = y.numel()
    keep = y != ignore
    label = torch.where(keep, y, 0)
    z = h @ w.t()
    size_z = (h.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(z, 1)
    rows = torch.arange(T, device=y.device)
    each = torch.where(keep, lse - z[rows, label], 0.0)
    count = max(1, int(keep.sum()))
    loss = each if reduction == "none" else each.sum() / (count if reduction == "mean" else 1)
    g = torch.where(keep, grad.double() / (count if reduction == "mean" else 1), 0.0).expand(T)
    p = torch.exp(z - lse[:, None])
    dz = p.clone()
    dz[rows, label] -= 1.0
    dz, p = dz * g[:, None], p * g.abs()[:, None]
    return {"loss": loss, "lse": lse, "size_z": size_z, "dh": dz @ w, "dw": dz.t() @ h, "dz": dz, "p": p, "g": g,
            "keep": keep}


def check(h, w, y, reduction="mean", grad=None, ignore=IGNORE):
    T, D = h.shape
    V = w.shape[0]
    kind = h.dtype
    u = ROUND[kind]
    if grad is None:
        grad = torch.rand(T, device="cuda") + 0.5 if reduction == "none" else torch.tensor(64.0, device="cuda")
    loss, lse = M.linear_cross_entropy_forward(h, w, y, ignore, reduction)
    dh, dw = M.linear_cross_entropy_backward(grad, h, w, y, lse, ignore, reduction)
    again = M.linear_cross_entropy_backward(grad, h, w, y, lse, ignore, reduction)
    assert capi.device_status(reset=True) == 0
    assert torch.equal(dh, again[0]) and torch.equal(dw, again[1])
    e = plain(h, w, y, reduction, grad, ignore)
    off_z = D * 2.0 ** -27 * e["size_z"] + 2.0 ** -20  # of a logit, per row
    assert (torch.abs(lse.double() - e["lse"]) <= off_z + 2.0 ** -22 * e["lse"].abs()).all()
    each = 2 * off_z + 2.0 ** -21 * (e["lse"].abs() + e["size_z"])
    bound = torch.where(e["keep"], each, 0.0)
    if reduction != "none":
        bound = (bound.sum() / (max(1, int(e["keep"].sum())) if reduction == "mean" else 1)) + 2.0 ** -22 * e["loss"].abs()
    assert (torch.abs(loss.double() - e["loss"]) <= bound).all()
    # dz: probabilities off by 2 off_z + 2^-20 of themselves, rounded once
    gmax = e["g"].abs().max()
    off_dz = e["p"] * (2 * off_z + 2.0 ** -20)[:, None] + u * e["dz"].abs() + 2.0 ** -39 * gmax
    a_h, a_w = h.double().abs(), w.double().abs()
    tiny = 2.0 ** -25 if kind == torch.float16 else 0.0
    for got, want, size in ((dh, e["dh"], off_dz @ a_w + V / 16 * 2.0 ** -23 * (e["dz"].abs() @ a_w)),
                            (dw, e["dw"], off_dz.t() @ a_h + T / 16 * 2.0 ** -23 * (e["dz"].abs().t() @ a_h))):
        assert torch.isfinite(got).all()
        off = (got.double() - want).abs()
        limit = u * want.abs() + (1 + u) * (size + 2.0 ** -22 * want.abs()) + tiny
        assert (off <= limit).all(), f"{(off / limit).max().item():.2f} of the bound"
        # errors of many roundings do not line up: the whole is within two roundings
        if want.norm() > 0:
            assert off.norm() <= 2 * u * want.norm() + (tiny * off.numel() ** 0.5)
    assert not dh[~e["keep"]].any()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (1, 1000, 64), (2, 255, 72), (3, 256, 128), (127, 257, 256), (128, 128, 64),
                                   (129, 1001, 136), (197, 511, 200), (256, 513, 512), (300, 4099, 1024), (1000, 777, 264)])
def test_sizes(cuda, T, V, D, kind):
    check(*make(T, V, D, kind))


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("V,D", [(5, 8), (33, 264), (20011, 72), (1000, 5128), (300, 16384)])
def test_few_tokens(cuda, T, V, D):
    """On both sides of the change to the kernel for a few tokens, in tokens and in width."""
    check(*make(T, V, D, torch.float16, ignored=0.0), reduction="none")
    check(*make(T, V, D, torch.bfloat16, ignored=0.4), reduction="mean")


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_reductions(cuda, reduction, kind):
    grad = torch.tensor(0.5, device="cuda") if reduction == "sum" else None
    check(*make(200, 700, 128, kind), reduction=reduction, grad=grad)


@pytest.mark.parametrize("T,V,D", [(4096, 1000, 256), (5000, 3001, 128), (70, 30011, 64)])
def test_many_tiles(cuda, T, V, D):
    check(*make(T, V, D, torch.float16))
    check(*make(T, V, D, torch.bfloat16), reduction="none")


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [256, 1024, 2048])
def test_logits_are_not_biased(cuda, D, kind):
    """The tensor core loses up to 2.1e-8 of a sum at each of its D / 16 steps, always towards zero; what is
    put back leaves at most a third of that on average, beside the random part of an fp32 sum (2^-24 of the
    result for the root of the steps, averaged over the tokens)."""
    h, w, y = make(400, 3000, D, kind, ignored=0.0)
    h = (h.float() + w[y].float()).to(kind)
    loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "none")
    zt = (h.double() * w.double()[y]).sum(1)
    short = (zt - (lse.double() - loss.double())) / zt
    steps = D / 16
    assert abs(short.mean().item()) <= steps * 2.1e-8 / 3 + 3 * steps ** 0.5 * 2.0 ** -24 / 400 ** 0.5 + 2.0 ** -23


def test_gradients_of_very_different_rows(cuda):
    """Row gradients over eight orders of magnitude, zeros and negative ones among them."""
    h, w, y = make(64, 300, 64, torch.bfloat16, ignored=0.0)
    grad = 10.0 ** torch.linspace(-8, 0, 64, device="cuda")
    grad[::5] *= -1
    grad[7] = 0.0
    check(h, w, y, "none", grad)
    check(h, w, y, "none", torch.zeros(64, device="cuda"))


@pytest.mark.parametrize("kind,tokens", [(torch.bfloat16, 40), (torch.float16, 40), (torch.float16, (1 << 20) + 77)])
def test_gradients_below_the_normal_range(cuda, kind, tokens):
    """2^-140 a row: below fp32's normal numbers, so the gradients stay within sum |dz| max |operand| of
    zero (sum over v of |dz| is at most 2 g, each |dz| at most g).  The many tokens make two pieces of dz."""
    g = torch.Generator(device="cuda").manual_seed(3)
    h = torch.randn(tokens, 8, generator=g, device="cuda").to(kind)
    w = torch.randn(300, 8, generator=g, device="cuda").to(kind)
    y = torch.randint(0, 300, (tokens,), generator=g, device="cuda")
    grad = torch.full((tokens,), 2.0 ** -140, device="cuda")
    _, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "none")
    dh, dw = M.linear_cross_entropy_backward(grad, h, w, y, lse, IGNORE, "none")
    assert dh.double().abs().max() <= 2 * w.double().abs().max() * 2.0 ** -140
    assert dw.double().abs().max() <= tokens * h.double().abs().max() * 2.0 ** -140


def test_no_second_derivative(cuda):
    h, w, y = make(16, 40, 64, torch.float16)
    h.requires_grad_()
    (dh,) = torch.autograd.grad(M.linear_cross_entropy(h, w, y).square(), h, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dh.float().sum().backward()


def test_all_ignored(cuda):
    for reduction, grad in (("none", torch.ones(40, device="cuda")), ("mean", torch.ones((), device="cuda")),
                            ("sum", torch.ones((), device="cuda"))):
        h, w, y = make(40, 300, 64, torch.float16)
        y[:] = IGNORE
        loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, reduction)
        dh, dw = M.linear_cross_entropy_backward(grad, h, w, y, lse, IGNORE, reduction)
        assert not loss.any() and not dh.any() and not dw.any()


def test_ignore_index_within_the_vocabulary(cuda):
    h, w, y = make(100, 300, 64, torch.float16, ignored=0.0)
    y[::3] = 0
    check(h, w, y, ignore=0)


def test_target_outside_the_vocabulary_is_nan(cuda):
    h, w, y = make(20, 300, 64, torch.float16, ignored=0.0)
    y[4], y[9] = 300, -7
    loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "none")
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[[4, 9]] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(lse.isnan(), bad)
    dh, _ = M.linear_cross_entropy_backward(torch.ones(20, device="cuda"), h, w, y, lse, IGNORE, "none")
    assert dh[bad].isnan().all() and torch.isfinite(dh[~bad]).all()
    assert M.linear_cross_entropy_forward(h, w, y, IGNORE, "mean")[0].isnan()


def test_non_finite_hidden_stays_in_its_row(cuda):
    h, w, y = make(20, 300, 64, torch.float16, ignored=0.0)
    h[3, 5] = float("nan")
    h[6, 1] = float("inf")
    loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "none")
    assert loss[3].isnan() and not torch.isfinite(loss[6])
    rest = [i for i in range(20) if i not in (3, 6)]
    assert torch.isfinite(loss[rest]).all()
    y[3] = y[6] = IGNORE  # padding may hold anything
    loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "mean")
    assert torch.isfinite(loss)
    dh, _ = M.linear_cross_entropy_backward(torch.ones((), device="cuda"), h, w, y, lse, IGNORE, "mean")
    assert torch.isfinite(dh).all() and not dh[[3, 6]].any()


def test_large_logits(cuda):
    """Logits of several hundred: exponentials relative to a row's maximum only."""
    h, w, y = make(64, 500, 128, torch.bfloat16, spread=60.0)
    check(h, w, y)


@pytest.mark.parametrize("at,extra", [(0, 8), (8, 16), (1, 7), (4, 4)])
def test_strides_and_offsets(cuda, at, extra):
    """Rows inside wider ones; bases and strides that tensor maps refuse are copied."""
    h, w, y = make(90, 333, 64, torch.float16)
    hs = torch.zeros(90, 64 + at + extra, device="cuda", dtype=torch.float16)
    ws = torch.zeros(333, 64 + at + extra, device="cuda", dtype=torch.float16)
    hs[:, at:at + 64], ws[:, at:at + 64] = h, w
    grad = torch.ones((), device="cuda")
    a = M.linear_cross_entropy_forward(h, w, y)
    b = M.linear_cross_entropy_forward(hs[:, at:at + 64], ws[:, at:at + 64], y)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a = M.linear_cross_entropy_backward(grad, h, w, y, a[1])
    b = M.linear_cross_entropy_backward(grad, hs[:, at:at + 64], ws[:, at:at + 64], y, b[1])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_leading_dimensions(cuda):
    h, w, y = make(60, 333, 64, torch.float16)
    loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "none")
    l3, e3 = M.linear_cross_entropy_forward(h.view(4, 15, 64), w, y.view(4, 15), IGNORE, "none")
    assert l3.shape == (4, 15) and torch.equal(l3.reshape(-1), loss) and torch.equal(e3.reshape(-1), lse)
    one, _ = M.linear_cross_entropy_forward(h[5], w, y[5], IGNORE, "none")
    assert one.shape == () and torch.equal(one, M.linear_cross_entropy_forward(h[5:6], w, y[5:6], IGNORE, "none")[0][0])


def test_no_tokens(cuda):
    h, w, y = make(4, 50, 64, torch.float16)
    for reduction in ("none", "mean", "sum"):
        loss, lse = M.linear_cross_entropy_forward(h[:0], w, y[:0], IGNORE, reduction)
        assert lse.shape == (0,) and not loss.any()
        grad = torch.ones(0 if reduction == "none" else (), device="cuda")
        dh, dw = M.linear_cross_entropy_backward(grad, h[:0], w, y[:0], lse, IGNORE, reduction)
        assert dh.shape == (0, 64) and not dw.any()


def test_pieces_of_the_vocabulary_and_offsets_past_32_bits(cuda):
    """So many tokens that a 256-column piece of dz has over 2^31 elements and the vocabulary takes two."""
    T, V, D = (1 << 23) + 77, 300, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(T, D, generator=g, device="cuda", dtype=torch.float16)
    w = torch.randn(V, D, generator=g, device="cuda", dtype=torch.float16)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    grad = torch.ones(T, device="cuda")
    loss, lse = M.linear_cross_entropy_forward(h, w, y, IGNORE, "none")
    dh, dw = M.linear_cross_entropy_backward(grad, h, w, y, lse, IGNORE, "none")
    assert capi.device_status(reset=True) == 0
    dw64 = torch.zeros(V, D, device="cuda", dtype=torch.float64)
    for i in range(0, T, 1 << 19):
        e = plain(h[i:i + (1 << 19)], w, y[i:i + (1 << 19)], "none", grad[i:i + (1 << 19)])
        dw64 += e["dw"]
        last = e
    n = last["loss"].numel()
    assert (loss[-n:].double() - last["loss"]).norm() <= 1e-5 * last["loss"].norm()
    assert (dh[-n:].double() - last["dh"]).norm() <= 2 * 2.0 ** -11 * last["dh"].norm()
    # 2^23 terms per element, rounded to 2^-11 each with no common sign, and summed in fp32 (2^-23 of
    # a running sum of at most sum |dz h|, 2^19 steps that do not line up either)
    fits = dw64.abs() < 65504
    assert torch.equal(dw[~fits].double(), dw64[~fits].to(torch.float16).double()) and fits.sum() > fits.numel() // 2
    assert (dw.double() - dw64)[fits].norm() <= 4 * 2.0 ** -11 * dw64[fits].norm()


def test_gradients_against_differences(cuda):
    """The kernel's gradients along random directions against central differences of the 64-bit loss."""
    h, w, y = make(30, 200, 64, torch.bfloat16)
    loss, lse = M.linear_cross_entropy_forward(h, w, y)
    dh, dw = M.linear_cross_entropy_backward(torch.ones((), device="cuda"), h, w, y, lse)
    g = torch.Generator(device="cuda").manual_seed(2)
    one = torch.ones((), device="cuda")
    for i, (at, grad) in enumerate(((h, dh), (w, dw))):
        v = torch.randn(at.shape, generator=g, device="cuda", dtype=torch.float64)
        step = 1e-5
        moved = [(at.double() + s * step * v) for s in (1, -1)]
        ls = [plain(m if i == 0 else h, w if i == 0 else m, y, "mean", one)["loss"] for m in moved]
        want = (ls[0] - ls[1]) / (2 * step)
        got = (grad.double() * v).sum()
        # independent roundings of 2^-8 (dz and the result) weighted by v: five deviations
        dev = (grad.double() * v).norm() * 2 * 2.0 ** -8
        assert abs(got - want) <= 5 * dev, (i, got.item(), want.item())


def test_autograd(cuda):
    h, w, y = make(64, 300, 128, torch.float16)
    h, w = h.view(4, 16, 128).requires_grad_(), w.requires_grad_()
    y = y.view(4, 16)
    loss = M.linear_cross_entropy(h, w, y)
    (loss * 16.0).backward()
    _, lse = M.linear_cross_entropy_forward(h.detach(), w.detach(), y)
    dh, dw = M.linear_cross_entropy_backward(torch.tensor(16.0, device="cuda"), h.detach(), w.detach(), y, lse)
    assert torch.equal(h.grad, dh) and torch.equal(w.grad, dw)
    h.grad = None  # per-token losses with an expanded gradient
    M.linear_cross_entropy(h, w, y, reduction="none").sum().backward()
    a = h.grad.clone()
    h.grad = None
    M.linear_cross_entropy(h, w, y, reduction="sum").backward()
    assert torch.equal(a, h.grad)


def test_first_call_of_a_thread(cuda):
    """A thread that has not used the device yet, as autograd's worker when the loss is what backward starts from."""
    h, w, y = make(64, 300, 128, torch.float16)
    one = torch.ones((), device="cuda")
    _, lse = M.linear_cross_entropy_forward(h, w, y)
    want = [t.clone() for t in M.linear_cross_entropy_backward(one, h, w, y, lse)]
    got = []
    t = threading.Thread(target=lambda: got.extend(M.linear_cross_entropy_backward(one, h, w, y, lse)))
    t.start()
    t.join()
    assert len(got) == 2 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_another_stream_and_captured(cuda):
    h, w, y = make(64, 300, 128, torch.float16)
    one = torch.ones((), device="cuda")
    want = M.linear_cross_entropy_forward(h, w, y)
    want_b = M.linear_cross_entropy_backward(one, h, w, y, want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = M.linear_cross_entropy_forward(h, w, y)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse = M.linear_cross_entropy_forward(h, w, y)
        dh, dw = M.linear_cross_entropy_backward(one, h, w, y, lse)
    dh.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(dh, want_b[0]) and torch.equal(dw, want_b[1])


def test_refusals(cuda):
    h, w, y = make(8, 50, 64, torch.float16)
    f = M.linear_cross_entropy_forward
    for args, words in (((h.float(), w.float(), y), "float16 or bfloat16"), ((h, w.bfloat16(), y), "hidden's type"),
                        ((h[:, :60], w[:, :60], y), "multiple of 8"), ((h, w[:, :32], y), "weight must be"),
                        ((torch.zeros(2, 16392, device="cuda", dtype=torch.float16),
                          torch.zeros(3, 16392, device="cuda", dtype=torch.float16), y[:2]), "at most 16384"),
                        ((h, w, y.int()), "int64"), ((h, w, y[:4]), "leading shape"), ((h, w[:0], y), "weight must be"),
                        ((h, w.cpu(), y), "CUDA")):
        with pytest.raises(RuntimeError, match=words):
            f(*args)
    with pytest.raises(ValueError, match="reduction"):
        f(h, w, y, IGNORE, "average")
    loss, lse = f(h, w, y)
    one = torch.ones((), device="cuda")
    with pytest.raises(RuntimeError, match="grad_loss must be float32"):
        M.linear_cross_entropy_backward(one.half(), h, w, y, lse)
    with pytest.raises(RuntimeError, match="one element"):
        M.linear_cross_entropy_backward(torch.ones(8, device="cuda"), h, w, y, lse)
    with pytest.raises(RuntimeError, match="target's shape"):
        M.linear_cross_entropy_backward(one, h, w, y, lse, IGNORE, "none")
    with pytest.raises(RuntimeError, match="lse must be"):
        M.linear_cross_entropy_backward(one, h, w, y, lse[:3])


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,V,D", [(1, 50, 64), (2, 300, 72), (20, 300, 64), (129, 777, 136), (1000, 300, 512), (5000, 3001, 128),
                                   (300, 20000, 64), ((1 << 20) + 77, 300, 8)])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_rows_that_count_for_nothing_may_hold_anything(cuda, T, V, D, kind, reduction):
    """Ignored rows with NaN and infinities give the same bits as zeros in their place, in dweight too (whose
    product meets them): few and many tokens, one block of rows and many, split sums, two pieces of dz."""
    g = torch.Generator(device="cuda").manual_seed(T + V + D)
    h = torch.randn(T, D, generator=g, device="cuda").to(kind)
    w = (torch.randn(V, D, generator=g, device="cuda") * D ** -0.5).to(kind)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    grad = torch.rand(T, generator=g, device="cuda") + 0.5 if reduction == "none" else torch.ones((), device="cuda")
    off = torch.rand(T, generator=g, device="cuda") < 0.2
    off[256:640] = False  # blocks of rows without any
    off[-1] = True
    y[off] = IGNORE
    if reduction == "none" and T > 2:  # a gradient of zero is as good
        y[-1], grad[-1] = 0, 0.0
    bad = torch.nonzero(off)[:, 0]
    dirty, clean = h.clone(), h.clone()
    for i, x in enumerate((float("nan"), float("inf"), -float("inf"))):
        dirty[bad[i::3], (3 * i) % D] = x
    dirty[-1] = float("nan")
    clean[bad] = 0.0
    got, want = [], []
    for x, res in ((dirty, got), (clean, want)):
        loss, lse = M.linear_cross_entropy_forward(x, w, y, IGNORE, reduction)
        res += [loss[y != IGNORE][:-1] if reduction == "none" else loss,
                *M.linear_cross_entropy_backward(grad, x, w, y, lse, IGNORE, reduction)]
    assert capi.device_status(reset=True) == 0
    for name, a, b in zip(("loss", "dhidden", "dweight"), got, want):
        assert torch.isfinite(b).all() and torch.equal(a, b), name


def test_non_finite_rows_that_count_are_seen(cuda):
    h, w, y = make(300, 500, 64, torch.float16, ignored=0.2)
    at = torch.nonzero(y != IGNORE)[7, 0]
    h[at, 3] = float("nan")
    _, lse = M.linear_cross_entropy_forward(h, w, y)
    dh, dw = M.linear_cross_entropy_backward(torch.ones((), device="cuda"), h, w, y, lse)
    assert dh[at].isnan().all() and dw.isnan().all()
