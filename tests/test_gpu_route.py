"""Routing from logits on the GPU (rwkvmoe_route, rwkvmoe_route_backward)
against the 64-bit oracle: experts equal; gates and gradients, computed in 64
bits and rounded once, within half a step of their type (and the 64-bit sums'
own error, taken as 2^-40)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import ops_oracle as O
from rwkv_mlx_amd import GroupRouter, route_topk

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# (rows, E, k, groups, top_groups, group_score)
SHAPES = [
    (1, 1, 1, 1, 1, "max"),
    (1, 256, 8, 8, 4, "top2"),
    (5, 8, 8, 1, 1, "max"),
    (33, 60, 6, 5, 3, "top2"),       # groups that lie on no whole lanes
    (33, 60, 6, 5, 3, "max"),
    (70, 64, 32, 2, 2, "max"),
    (7, 512, 32, 64, 5, "top2"),
    (9, 320, 20, 1, 1, "max"),
    (4099, 160, 6, 8, 3, "top2"),    # 16 lanes a row
    (4099, 64, 32, 1, 1, "max"),
    (4097, 512, 9, 16, 2, "max"),
    (4097, 33, 3, 3, 2, "top2"),
    (4096, 96, 5, 12, 7, "top2"),
]


def make(rows, E, dtype, masked, seed):
    rng = np.random.default_rng(seed)
    l = torch.from_numpy(rng.normal(size=(rows, E)) * 2).to(DT[dtype])
    if masked:
        gone = torch.from_numpy(rng.random((rows, E)) < masked)
        l = l.masked_fill(gone, float("-inf"))
        l[0] = float("-inf")  # a row with nothing left
        l[-1, ::2] = float("nan")
    return l, torch.from_numpy(rng.normal(size=E) * 0.1).float()


def check(l, inds, gates, want_i, want_g):
    assert inds.dtype == torch.int32 and gates.dtype == torch.float32
    assert (inds.cpu().numpy() == want_i).all()
    g = gates.cpu().numpy().astype(np.float64)
    assert (np.abs(g - want_g) <= np.abs(want_g) * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -150).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype,bias,masked,renorm", [("f32", True, 0.0, True), ("bf16", False, 0.4, True),
                                                      ("f16", True, 0.9, False), ("f32", False, 0.0, False)])
def test_route(device, shape, score, dtype, bias, masked, renorm):
    R, E, k, G, tg, gs = shape
    l, b = make(R, E, dtype, masked, seed=R * 7 + E)
    kw = dict(score=score, n_groups=G, top_groups=tg, group_score=gs, renormalize=renorm, scale=1.5)
    ld = l.to(device).requires_grad_(True)
    bd = b.to(device) if bias else None
    inds, gates = route_topk(ld, k, bias=bd, **kw)
    want_i, want_g = O.route(l.double().numpy(), k, bias=b.numpy() if bias else None, **kw)
    check(l, inds, gates.detach(), want_i, want_g)
    with torch.no_grad():
        again = route_topk(ld, k, bias=bd, **kw)
    assert torch.equal(again[0], inds) and torch.equal(again[1], gates)

    dg = torch.from_numpy(np.random.default_rng(3).normal(size=(R, k))).float()
    (got,) = torch.autograd.grad(gates, ld, dg.to(device))
    want = O.route_backward(l.double().numpy(), want_i, want_g, dg.double().numpy(), score=score,
                            renormalize=renorm, scale=1.5)
    assert got.dtype == ld.dtype and got.shape == ld.shape
    eps = torch.finfo(DT[dtype]).eps / 2
    # 64-bit sums of up to 32 terms of size |d| / U · s, whose difference is the result
    s, _ = O.route_scores(l.double().numpy(), score)
    size = np.abs(dg.numpy()).max(1, keepdims=True) * 1.5 * (1.0 / np.maximum(
        np.where(renorm, np.abs(np.take_along_axis(s, want_i, 1)).sum(1, keepdims=True), 1.0), 1e-30)) * s
    tiny = torch.finfo(DT[dtype]).smallest_normal * eps * 2
    err = np.abs(got.cpu().double().numpy() - want)
    assert (err <= np.abs(want) * eps + size * 2.0 ** -40 + tiny).all()


def test_route_ties_take_the_lower_index(device):
    l = torch.zeros(5, 64, device=device)
    l[1, 40:] = 1.0
    l[2, ::2] = 1.0
    inds, gates = route_topk(l, 4)
    assert inds.tolist() == [[0, 1, 2, 3], [40, 41, 42, 43], [0, 2, 4, 6], [0, 1, 2, 3], [0, 1, 2, 3]]
    assert torch.equal(gates, torch.full_like(gates, 0.25))
    inds, _ = route_topk(l, 4, score="sigmoid", n_groups=8, top_groups=2, group_score="top2")
    assert inds.tolist() == [[0, 1, 2, 3], [40, 41, 42, 43], [0, 2, 4, 6], [0, 1, 2, 3], [0, 1, 2, 3]]


def test_route_resolves_scores_that_fp32_does_not(device):
    # sigmoid(17) and sigmoid(18) are both 1 in fp32 with a bias beside them
    l = torch.tensor([[17.0, 18.0, 3.0, 17.5]], device=device)
    inds, _ = route_topk(l, 3, bias=torch.full((4,), 0.25, device=device), score="sigmoid")
    assert inds.tolist() == [[1, 3, 0]]


def test_route_of_masks_and_extremes(device):
    low = torch.finfo(torch.float32).min
    l = torch.tensor([[low, low, low, low], [low, 0.0, low, 1.0], [float("-inf")] * 4,
                      [float("nan"), 2.0, float("-inf"), 1.0], [float("inf"), 0.0, float("inf"), 1.0]], device=device)
    inds, gates = route_topk(l, 2)
    assert inds.tolist() == [[0, 1], [3, 1], [0, 1], [1, 3], [0, 2]]
    e = float(torch.sigmoid(torch.tensor(1.0, dtype=torch.float64)))
    want = torch.tensor([[0.5, 0.5], [e, 1 - e], [0, 0], [e, 1 - e], [0.5, 0.5]])
    assert torch.allclose(gates.cpu(), want, rtol=2.0 ** -23, atol=0)
    b = torch.tensor([0.0, float("-inf"), float("nan"), 0.0], device=device)
    inds, gates = route_topk(torch.zeros(1, 4, device=device), 3, bias=b, score="sigmoid")
    assert inds.tolist() == [[0, 3, 1]] and gates.tolist() == [[0.5, 0.5, 0.0]]


def test_route_strides_shapes_and_empty(device):
    base = torch.randn(10, 40, device=device)
    want = route_topk(base[:, 8:24].contiguous(), 3)
    for l in (base[:, 8:24], base[:, 8:24].t().contiguous().t()):
        got = route_topk(l, 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    strided = base[::2, 1:17].detach().requires_grad_(True)
    i, g = route_topk(strided, 2)
    (d,) = torch.autograd.grad(g, strided, torch.ones_like(g) * torch.arange(2., device=device))
    dense = strided.detach().contiguous().requires_grad_(True)
    i2, g2 = route_topk(dense, 2)
    (d2,) = torch.autograd.grad(g2, dense, torch.ones_like(g) * torch.arange(2., device=device))
    assert torch.equal(i, i2) and torch.equal(d, d2)
    i3, g3 = route_topk(base.view(2, 5, 40), 3)
    assert i3.shape == (2, 5, 3) and torch.equal(i3.view(10, 3), route_topk(base, 3)[0])
    z = torch.zeros(0, 16, device=device, requires_grad=True)
    i, g = route_topk(z, 2)
    assert i.shape == g.shape == (0, 2)
    (d,) = torch.autograd.grad(g.sum(), z)
    assert d.shape == (0, 16)
    leaf = torch.randn(2, 5, 16, device=device, requires_grad=True)
    (d,) = torch.autograd.grad(route_topk(leaf, 2)[1][..., 0].sum(), leaf)
    assert d.shape == leaf.shape


def test_route_refuses(device):
    l = torch.zeros(4, 16, device=device)
    for call, err in ((lambda: route_topk(l, 0), RuntimeError), (lambda: route_topk(l, 17), RuntimeError),
                      (lambda: route_topk(l, 2, n_groups=3), RuntimeError),
                      (lambda: route_topk(l, 5, n_groups=4, top_groups=1), RuntimeError),
                      (lambda: route_topk(l, 2, score="tanh"), ValueError),
                      (lambda: route_topk(l, 2, group_score="sum"), ValueError),
                      (lambda: route_topk(l, 2, bias=torch.zeros(15, device=device)), ValueError),
                      (lambda: route_topk(l, 2, bias=torch.zeros(16)), ValueError),
                      (lambda: route_topk(l.double(), 2), TypeError)):
        with pytest.raises(err):
            call()


def test_route_on_a_side_stream_and_in_a_graph(device):
    l = torch.randn(300, 64, device=device)
    want = route_topk(l, 4, score="sigmoid", n_groups=4, top_groups=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = route_topk(l, 4, score="sigmoid", n_groups=4, top_groups=2)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = route_topk(l, 4, score="sigmoid", n_groups=4, top_groups=2)
    for seed in range(3):
        l.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        want = route_topk(l, 4, score="sigmoid", n_groups=4, top_groups=2)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_group_router(device):
    torch.manual_seed(0)
    r = GroupRouter(64, 16, 3, n_groups=4, top_groups=2, scale=2.0).to(device)
    x = torch.randn(2, 7, 64, device=device, requires_grad=True)
    inds, w, aux, z = r(x)
    assert inds.shape == (2, 7, 3) and w.dtype == x.dtype and float(aux) == float(z) == 0
    want_i, want_g = O.route((x.detach() @ r.gate.weight.detach().t()).double().cpu().numpy().reshape(14, 16), 3,
                             bias=np.zeros(16), score="sigmoid", n_groups=4, top_groups=2, group_score="top2", scale=2.0)
    assert (inds.cpu().numpy().reshape(14, 3) == want_i).all()
    (w * torch.arange(3.0, device=device)).sum().backward()
    assert x.grad.abs().sum() > 0 and r.gate.weight.grad.abs().sum() > 0
    r.update_balance(inds, 0.5)
    load = np.bincount(inds.cpu().numpy().ravel(), minlength=16)
    assert (np.sign(load.mean() - load) * 0.5 == r.balance_bias.cpu().numpy()).all()


def test_route_past_32_bits(device):
    R, E = 4_300_000, 256
    l = torch.empty(R, E, device=device).normal_()
    tail = l[-300:].clone().requires_grad_(True)
    assert l.numel() * 4 > 1 << 32
    b = torch.randn(E, device=device) * 0.1
    kw = dict(bias=b, score="sigmoid", n_groups=8, top_groups=4, group_score="top2")
    l.requires_grad_(True)
    inds, gates = route_topk(l, 8, **kw)
    i1, g1 = route_topk(tail, 8, **kw)
    assert torch.equal(inds[-300:], i1) and torch.equal(gates[-300:], g1)
    dg = torch.empty(R, 8, device=device).normal_()
    (d,) = torch.autograd.grad(gates, l, dg)
    (d1,) = torch.autograd.grad(g1, tail, dg[-300:])
    assert torch.equal(d[-300:], d1)


def test_route_rows_of_near_ties(device):
    """Scores closer than fp32 resolves, many of them in a row: 16 and 64 lanes
    a row, a few and more than a wave settles, and at the border of groups."""
    rng = np.random.default_rng(0)
    for R in (70, 4100):
        base = rng.normal(size=(R, 1))
        l = (base + rng.integers(0, 4, (R, 64)) * 2.0 ** -22).astype(np.float32)
        l[::3] = rng.normal(size=l[::3].shape)
        l[1::3, ::5] += rng.normal(size=l[1::3, ::5].shape).astype(np.float32)
        b = (rng.integers(0, 3, 64) * 2.0 ** -25).astype(np.float32)
        for score in ("sigmoid", "softmax"):
            for k, G, tg, bias in ((3, 1, 1, True), (6, 8, 2, True), (12, 4, 2, True), (5, 8, 3, False), (14, 2, 2, True)):
                kw = dict(score=score, n_groups=G, top_groups=tg, group_score="top2")
                inds, gates = route_topk(torch.from_numpy(l).to(device), k,
                                         bias=torch.from_numpy(b).to(device) if bias else None, **kw)
                wi, wg = O.route(l.astype(np.float64), k, bias=b if bias else None, **kw)
                # (softmax's scores are sums' quotients: the last bit of 64 may fall either way, so their values
                # are compared, and the experts where no two scores lie within 2^-48)
                s, _ = O.route_scores(l.astype(np.float64), score)
                val = s + (b if bias else 0)
                got = np.take_along_axis(val, inds.cpu().numpy().astype(np.int64), 1)
                want = np.take_along_axis(val, wi, 1)
                assert (np.abs(got - want) <= 2.0 ** -48 * np.abs(want)).all()
                if score == "sigmoid" and G == 1:
                    assert (inds.cpu().numpy() == wi).all()


def test_route_gradient_in_a_graph(device):
    l = torch.randn(500, 64, device=device, requires_grad=True)
    dg = torch.randn(500, 4, device=device)
    step = lambda: torch.autograd.grad(route_topk(l, 4, score="sigmoid", n_groups=4, top_groups=2)[1], l, dg)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in range(3):
        with torch.no_grad():
            l.copy_(torch.randn(500, 64, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


@pytest.mark.parametrize("score,want", [("sigmoid", 2), ("softmax", 5)])
def test_group_router_keeps_fp32_logits_under_autocast(device, score, want):
    """Two experts with logits of 64 and 64 (1 + 2^-12): bf16 logits tie and
    leave expert 2 in front.  So do their sigmoids, 1 - e^-64 = 1 - 2^-92 in 64
    bits, but not their softmax."""
    r = GroupRouter(64, 8, 1, score=score).to(device)
    with torch.no_grad():
        r.gate.weight.zero_()
        r.gate.weight[5], r.gate.weight[2] = 1.0 + 2.0 ** -12, 1.0
    x = torch.ones(1, 3, 64, device=device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        inds, w, _, _ = r(x)
    assert (inds == want).all() and w.dtype == x.dtype and torch.equal(inds, r(x)[0])
