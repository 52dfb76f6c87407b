"""The global gradient norm and clipping against a plain 64-bit form.

Tolerances: the squares of one thread are summed in fp32 (at most 32 of a chunk, 2^-24 each and all
positive, so the norm is off by at most 16 2^-24 of itself), the rest in fp64; an output is one more
fp32 product and one rounding."""

import pytest
import torch

import morphottention_b200 as M

pytestmark = pytest.mark.gpu

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
NORM = 20 * 2.0 ** -24
KINDS = [torch.float16, torch.bfloat16, torch.float32]


def make(sizes, kinds, seed=0, at=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        store = torch.randn(n + at, generator=g, device="cuda") * 10.0 ** (-(i % 3))
        out.append(store.to(kinds[i % len(kinds)])[at:])
    return out


def plain(grads, max_norm, scale):
    norm = torch.stack([(g.double() ** 2).sum() for g in grads]).sum().sqrt() / scale
    c = torch.clamp(max_norm / (norm + 1e-6), max=1.0) / scale
    return norm, [g.double() * c for g in grads]


def check(grads, max_norm, scale=1.0, out_kind=None, at=0):
    want_norm, want = plain(grads, max_norm, scale)
    outs = None
    if out_kind is not None:
        outs = [torch.full((g.numel() + at,), float("nan"), device="cuda", dtype=out_kind)[at:].view(g.shape) for g in grads]
    norm = M.clip_grad_norm(grads, max_norm, out=outs, loss_scale=scale)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(norm.double() - want_norm) <= NORM * want_norm
    for got, w in zip(grads if outs is None else outs, want):
        u = ROUND[got.dtype]
        tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
        assert ((got.double() - w).abs() <= (u + NORM + 4 * 2.0 ** -24) * w.abs() + tiny).all()


@pytest.mark.parametrize("sizes", [[1], [7, 1, 8193], [256, 4096, 8192, 8191, 65536 + 5], [3_000_001]], ids=str)
@pytest.mark.parametrize("kinds", [[k] for k in KINDS] + [KINDS], ids=["fp16", "bf16", "fp32", "mixed"])
def test_in_place(cuda, sizes, kinds):
    grads = make(sizes, kinds, seed=len(sizes))
    check(grads, 0.5)


@pytest.mark.parametrize("at", [0, 1, 3, 8])
@pytest.mark.parametrize("out_kind", KINDS, ids=["fp16", "bf16", "fp32"])
def test_into_other_tensors_at_odd_offsets(cuda, at, out_kind):
    for kinds in ([torch.float16], KINDS):
        check(make([5, 8192 + 13, 100, 20000], kinds, at=at), 0.25, 8.0, out_kind, at=at)
        check(make([5, 8192 + 13, 100, 20000], kinds, at=at), 0.25, 8.0, out_kind, at=(at * 5) % 7)


def test_nothing_to_clip_keeps_every_bit(cuda):
    grads = make([100, 9000], KINDS)
    before = [g.clone() for g in grads]
    M.clip_grad_norm(grads, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    M.clip_grad_norm(grads, 1e6, out=outs, loss_scale=4.0)
    assert all(torch.equal(o, g.float() / 4) for o, g in zip(outs, grads))


def test_many_tensors(cuda):
    """More tensors than one launch's table holds, empty ones among them."""
    sizes = [(i * 37) % 300 for i in range(2000)]
    check(make(sizes, KINDS), 0.1)
    check(make(sizes, KINDS), 0.1, 2.0, torch.float32)


def test_zero_and_empty(cuda):
    z = [torch.zeros(10, device="cuda"), torch.empty(0, device="cuda")]
    assert M.clip_grad_norm(z, 1.0).item() == 0.0 and not z[0].any()
    assert M.clip_grad_norm([torch.empty(0, device="cuda")], 1.0).item() == 0.0
    g = make([50], [torch.float32])
    M.clip_grad_norm(g, 0.0)
    assert not g[0].any()


def test_non_finite(cuda):
    g = make([1000, 20], [torch.float32])
    g[0][17] = float("inf")
    assert M.clip_grad_norm(g, 1.0).item() == float("inf")
    assert g[0][17].isnan() and not g[0][:17].any() and not g[1].any()
    g = make([1000, 20], [torch.float32])
    g[1][3] = float("nan")
    assert M.clip_grad_norm(g, 1.0).isnan()
    assert g[0].isnan().all() and g[1].isnan().all()


def test_fp16_squares_do_not_overflow(cuda):
    check([torch.full((5000,), 60000.0, device="cuda", dtype=torch.float16)], 1.0)


def test_dense_but_permuted(cuda):
    g = make([64 * 48], [torch.float16])[0].view(64, 48).t()
    check([g], 0.1)
    wide = torch.randn(8, 16, device="cuda")
    with pytest.raises(RuntimeError, match="dense"):
        M.clip_grad_norm([wide[:, :8]], 1.0)
    with pytest.raises(RuntimeError, match="same strides"):
        M.clip_grad_norm([wide.t()], 1.0, out=[torch.empty(16, 8, device="cuda")])


def test_same_bits_every_run(cuda):
    grads = make([70001, 9, 300000], KINDS)
    outs = [[torch.empty_like(g) for g in grads] for _ in range(2)]
    norms = [M.clip_grad_norm(grads, 0.3, out=o) for o in outs]
    assert torch.equal(*norms) and all(torch.equal(a, b) for a, b in zip(*outs))


def test_more_than_2_31_elements(cuda):
    n = (1 << 31) + 4099
    g = torch.full((n,), 0.5, device="cuda", dtype=torch.float16)
    g[-1] = 100.0
    want = (0.25 * (n - 1) + 1e4) ** 0.5
    norm = M.clip_grad_norm([g], want / 4)
    assert abs(norm.item() - want) <= NORM * want
    assert g[-1].item() == 25.0 and g[-2].item() == 0.125 and g[0].item() == 0.125


def test_parameters_form_and_another_stream(cuda):
    lin = torch.nn.Linear(64, 64, device="cuda")
    free = torch.nn.Parameter(torch.zeros(3, device="cuda"))  # no gradient
    x = torch.randn(8, 64, device="cuda")
    lin(x).square().sum().backward()
    want_norm, want = plain([p.grad for p in lin.parameters()], 0.1, 1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = M.clip_grad_norm_([*lin.parameters(), free], 0.1)
    torch.cuda.current_stream().wait_stream(s)
    assert abs(norm.double() - want_norm) <= NORM * want_norm
    for p, w in zip(lin.parameters(), want):
        assert ((p.grad.double() - w).abs() <= (NORM + 5 * 2.0 ** -24) * w.abs()).all()
    assert M.clip_grad_norm_([free], 1.0).item() == 0.0


def test_refusals(cuda):
    g = make([10], [torch.float32])
    for bad, words in ((dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"),
                       (dict(max_norm=1.0, loss_scale=0.0), "loss_scale"),
                       (dict(max_norm=1.0, loss_scale=float("inf")), "loss_scale")):
        with pytest.raises(RuntimeError, match=words):
            M.clip_grad_norm(g, **bad)
    with pytest.raises(RuntimeError, match="as many tensors"):
        M.clip_grad_norm(g, 1.0, out=[])
    with pytest.raises(RuntimeError, match="shape"):
        M.clip_grad_norm(g, 1.0, out=[torch.empty(9, device="cuda")])
    with pytest.raises(RuntimeError, match="float16, bfloat16 or float32"):
        M.clip_grad_norm([g[0].double()], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        M.clip_grad_norm(g, 1.0, out=[torch.empty(10)])


def test_a_graph_that_saved_what_is_written_notices(cuda):
    p = torch.nn.Parameter(torch.randn(100, device="cuda"))
    p.grad = torch.randn(100, device="cuda")
    x = torch.randn(100, device="cuda", requires_grad=True)
    y = (x * p.grad).sum()
    M.clip_grad_norm_([p], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out = torch.empty(100, device="cuda")
    saved, read = out._version, p.grad._version
    M.clip_grad_norm([p.grad], 0.1, out=[out])
    assert out._version > saved and p.grad._version == read
    with torch.inference_mode():
        M.clip_grad_norm([torch.randn(100, device="cuda")], 0.1)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("size", [1e20, 3e30, 1e-25, 1e-30])
def test_squares_past_the_range_of_fp32(cuda, kind, size):
    """Elements whose squares overflow or vanish in fp32 (the scale brings the results back to the size of one)."""
    grads = [(g.float() * size).to(kind) for g in make([5, 8192 + 3, 40000, 33], [torch.float32])]
    scale = min(size, 1e30)
    check(grads, 0.5, float(torch.tensor(scale)), torch.float32)
    # beside zeros, and as a few among smaller ones
    for g in grads:
        g[::3] = 0.0
        g[1::7] *= 1e-6
    check([*grads, torch.zeros(3000, device="cuda", dtype=kind)], 0.5, float(torch.tensor(scale)), torch.float32)
