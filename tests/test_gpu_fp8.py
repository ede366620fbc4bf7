"""8-bit block operands and their products on the GPU against the 64-bit
oracle.  Rounding to blocks is exact (the same e4m3 values and scales).  A
product of K terms is summed in fp32: each result is within half a step of its
type, plus 2^-23 · (128 + Kb) of Σ |a| |b|, a bound on the sums' roundings
(2^-23 a term within a block of 128, whatever its order, then one fma and one
product of scales a block).

fp16 and bf16 results of more than 64 rows come from the e4m3 matrix
instruction.  It aligns every 8 consecutive k to their largest product and
drops what lies below 2^-13 of it (measured on the card: 2^16 + 127 · 2^2 comes
out 7 · 2^2 too small, 2^16 + 127 · 2^3 exact).  The largest product keeps all
its bits (two 4-bit significands), so at most 7 products of a group lose less
than 2^-13 of the largest each: ``ops_oracle.dropped`` adds that up."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import ops_oracle as O
from rwkv_mlx_amd import (Fp8MoE_CMix, Fp8Weight, GroupRouter, MoE_CMix, RWKVConfig, channel_mixing_rnn, fp8_experts,
                          fp8_grouped_linear, fp8_linear, fp8_quantize)

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rand(shape, dtype, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    v = rng.normal(size=shape) * np.exp(rng.normal(size=(*shape[:-1], 1)) * spread)
    return torch.from_numpy(v).to(DT[dtype])


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def close(got, a, b, dtype, few=False):
    """got = a · bᵀ of what the 8-bit operands stand for; few: at most 64 rows
    in the call.  Large products are compared on 64 of their rows."""
    if a.shape[0] * b.shape[0] * b.shape[1] > 1 << 28:
        rows = np.random.default_rng(0).permutation(a.shape[0])[:64]
        got, a = got[torch.from_numpy(rows).to(got.device)], a[rows]
    want, size = a @ b.T, np.abs(a) @ np.abs(b).T
    kb = -(-a.shape[1] // 128)
    eps = torch.finfo(DT[dtype]).eps / 2
    tol = np.abs(want) * eps + size * 2.0 ** -23 * (128 + kb) * (1 + eps) + torch.finfo(DT[dtype]).smallest_normal * eps
    if dtype != "f32" and few is not True:
        tol += O.dropped(a, b)
    err = np.abs(f64(got) - want)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())


# ---- blocks ----


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 128), (17, 200), (130, 64), (129, 257), (16, 1000)])
def test_rows(device, dtype, R, K):
    x = rand((R, K), dtype, R + K, 3.0)
    x[0] = 0
    if dtype == "f32":
        x[-1] *= 2.0 ** -120  # below the least block
    q, s, qt, st = fp8_quantize(x.to(device), transposed=True)
    for got_q, got_s, v in ((q, s, x.float().numpy()), (qt, st, x.float().numpy().T)):
        wq, ws = O.quantize_rows(np.ascontiguousarray(v))
        assert got_q.shape == (v.shape[0], -(-v.shape[1] // 128) * 128)
        assert (f64(got_s) == ws).all()
        assert (f64(got_q.float())[:, : v.shape[1]] == wq).all()
        assert (f64(got_q.float())[:, v.shape[1]:] == 0).all()
    alone = fp8_quantize(x.to(device))
    assert torch.equal(alone[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(alone[1], s)
    t_only = fp8_quantize(x.to(device), transposed=True, rows=False)
    assert torch.equal(t_only[0].view(torch.uint8), qt.view(torch.uint8)) and torch.equal(t_only[1], st)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 200), (2, 257, 129), (3, 64, 320)])
def test_tiles(device, dtype, shape):
    w = rand(shape, dtype, sum(shape), 2.0)
    h = Fp8Weight.quantize(w.to(device), transposed=True)
    qs = [O.quantize_tiles(m) for m in w.float().numpy().reshape(-1, *shape[-2:])]
    wq = np.stack([a for a, _ in qs]).reshape(shape)
    ws = np.stack([b for _, b in qs]).reshape(h.scale.shape)
    assert (f64(h.scale) == ws).all() and (f64(h.scale_t) == np.swapaxes(ws, -1, -2)).all()
    N, K = shape[-2:]
    for q, v, n in ((h.q, wq, K), (h.q_t, np.swapaxes(wq, -1, -2), N)):
        g = f64(q.float())
        assert (g[..., :n] == v).all() and (g[..., n:] == 0).all()
    held = np.stack([O.held_tiles(a, b) for a, b in qs]).reshape(shape)
    assert np.allclose(f64(h.dequantize()), held, rtol=2.0 ** -24, atol=0)
    src = h.q[..., :K].contiguous()
    back = Fp8Weight.from_quantized(src, h.scale, transposed=True)
    for a, b in ((back.q, h.q), (back.q_t, h.q_t)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(back.scale, h.scale) and torch.equal(back.scale_t, h.scale_t)


def test_a_nan_or_infinity_makes_its_block_nan(device):
    x = torch.ones(4, 300, device=device)
    x[1, 5] = float("nan")
    x[2, 130] = float("inf")
    y = fp8_linear(x, Fp8Weight.quantize(torch.ones(20, 300, device=device)))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[0]).all() and torch.isfinite(
        y[3]).all()


# ---- products ----

# (rows, N, K): few rows, tiles of 128, tiles of 256; sizes that fill no block
SIZES = [(1, 1, 1), (1, 100, 300), (3, 130, 128), (16, 64, 1000), (17, 33, 130), (64, 200, 2048), (65, 300, 129),
         (127, 129, 128), (130, 2690, 1000), (300, 126, 64), (515, 260, 384), (4200, 4100, 200)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,N,K", SIZES)
def test_linear(device, dtype, R, N, K):
    x, w = rand((R, K), dtype, R + 1, 0.5), rand((N, K), dtype, N + 2, 0.5)
    h = Fp8Weight.quantize(w.to(device))
    y = fp8_linear(x.to(device), h)
    assert y.dtype == x.dtype and y.shape == (R, N)
    a = O.held_rows(*O.quantize_rows(x.float().numpy()))
    b = O.held_tiles(*O.quantize_tiles(w.float().numpy()))
    close(y, a, b, dtype, R <= 64)
    assert torch.equal(fp8_linear(x.to(device), w.to(device)), y)  # (a tensor is rounded in the call)
    assert torch.equal(fp8_linear(x.to(device), h), y)


def held_cols(v):
    """v (R, C) rounded in blocks along its columns, as (C, R)."""
    return O.held_rows(*O.quantize_rows(np.ascontiguousarray(v.T)))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,N,K", [(1, 5, 3), (17, 130, 200), (129, 64, 300), (300, 257, 129), (520, 384, 256)])
def test_linear_gradients(device, dtype, R, N, K):
    x, w, dy = rand((R, K), dtype, 1, 0.3), rand((N, K), dtype, 2, 0.3), rand((R, N), dtype, 3, 0.3)
    xd, wd = x.to(device).requires_grad_(True), w.to(device).requires_grad_(True)
    y = fp8_linear(xd, wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.to(device))
    wh = O.held_tiles(*O.quantize_tiles(w.float().numpy()))
    dyn, xn = dy.float().numpy(), x.float().numpy()
    close(dx, O.held_rows(*O.quantize_rows(dyn)), np.ascontiguousarray(wh.T), dtype, R <= 64)
    close(dw, held_cols(dyn), held_cols(xn), dtype, N <= 64)
    # one gradient alone, and the frozen weight's, are the same bits
    only_w = fp8_linear(x.to(device), wd)
    assert torch.equal(torch.autograd.grad(only_w, wd, dy.to(device))[0], dw)
    only_x = fp8_linear(xd, w.to(device))
    assert torch.equal(torch.autograd.grad(only_x, xd, dy.to(device))[0], dx)
    frozen = fp8_linear(xd, Fp8Weight.quantize(w.to(device), transposed=True))
    assert torch.equal(torch.autograd.grad(frozen, xd, dy.to(device))[0], dx)
    assert torch.equal(frozen, y)


def test_linear_gradient_against_differences(device):
    # values on which every rounding is exact: the product is linear there
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.integers(-8, 9, (6, 130)).astype(np.float32))
    w = torch.from_numpy(rng.integers(-8, 9, (5, 130)).astype(np.float32))
    dy = torch.from_numpy(rng.integers(-8, 9, (6, 5)).astype(np.float32))
    for t in (x, w, dy):  # every block's largest value is 448 / 2^k times a power of two: 7, 14, ...
        t.clamp_(-7, 7)
    x[:, 0] = x[:, 128] = x[0] = 7.0
    w[0, 0] = w[0, 128] = 7.0
    dy[:, 0] = dy[0] = 7.0
    xd, wd = x.to(device).requires_grad_(True), w.to(device).requires_grad_(True)
    dx, dw = torch.autograd.grad(fp8_linear(xd, wd), (xd, wd), dy.to(device))
    f = lambda a, b: float((fp8_linear(a.to(device), b.to(device)).cpu() * dy).sum())
    for i, j in ((1, 3), (4, 127), (5, 129)):
        p, m = x.clone(), x.clone()
        p[i, j], m[i, j] = 3, -3
        assert (f(p, w) - f(m, w)) / 6 == float(dx[i, j])
    for i, j in ((1, 3), (4, 127), (2, 129)):
        p, m = w.clone(), w.clone()
        p[i, j], m[i, j] = 3, -3
        assert (f(x, p) - f(x, m)) / 6 == float(dw[i, j])


# ---- rows sorted by expert ----

COUNTS = [
    [3], [0, 5, 0, 1], [1] * 20, [16, 0, 17, 2], [0, 0, 0], [130, 1, 0, 129, 70], [5, 300, 0, 0, 2, 128, 256],
    [0] * 63 + [9] + [2] * 40,
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("extra", [0, 37])
def test_grouped(device, dtype, counts, extra):
    E, N, K = len(counts), 140, 260
    R = sum(counts) + extra
    off = np.concatenate([[0], np.cumsum(counts)])
    x, w, dy = rand((R, K), dtype, 1), rand((E, N, K), dtype, 2), rand((R, N), dtype, 3)
    h = Fp8Weight.quantize(w.to(device), transposed=True)
    xd = x.to(device).requires_grad_(True)
    offd = torch.from_numpy(off).to(torch.int32).to(device)
    y = fp8_grouped_linear(xd, h, offd)
    if R == 0:
        assert y.shape == (0, N)
        return
    (dx,) = torch.autograd.grad(y, xd, dy.to(device))
    a, da = O.held_rows(*O.quantize_rows(x.float().numpy())), O.held_rows(*O.quantize_rows(dy.float().numpy()))
    for e in range(E):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        b = O.held_tiles(*O.quantize_tiles(w[e].float().numpy()))
        close(y[lo:hi], a[lo:hi], b, dtype, R <= 64)
        close(dx[lo:hi], da[lo:hi], np.ascontiguousarray(b.T), dtype, R <= 64)
    assert (y[off[-1]:] == 0).all() and (dx[off[-1]:] == 0).all()


def test_grouped_ranges_are_clamped_to_the_rows(device):
    h = Fp8Weight.quantize(rand((3, 40, 64), "f32", 1).to(device))
    x = rand((200, 64), "f32", 2).to(device)
    want = fp8_grouped_linear(x, h, torch.tensor([0, 50, 50, 200], dtype=torch.int32, device=device))
    got = fp8_grouped_linear(x, h, torch.tensor([7, 50, 20, 1 << 30], dtype=torch.int32, device=device))
    assert torch.equal(got[:50], want[:50]) and torch.equal(got[50:], want[50:])


# ---- a layer of experts ----


def integers(device, B, T, C, F, E, dtype, seed=0):
    """A layer on which the mixed rows, their 8-bit form and the hidden rows
    are exact: whole numbers with 448 in every block (so its factors are 1)."""
    rng = np.random.default_rng(seed)
    x = rng.integers(-4, 5, (B, T, C)).astype(np.float32) * 2
    x[..., ::128] = 448.0
    key = rng.integers(-2, 3, (E, F, C)).astype(np.float32)
    key[:, ::128, ::128] = 448.0
    key[:, :, ::128] *= 1.0
    val = rng.normal(size=(E, C, F)).astype(np.float32)
    x_k = rng.integers(0, 3, (E, C)).astype(np.float32) / 2
    x_k[:, ::128] = 0
    to = lambda a: torch.from_numpy(a).to(DT[dtype])
    return to(x), to(x_k), to(key), to(val)


@pytest.mark.parametrize("B,T,C,F,E,k,dtype,gate", [
    (1, 1, 64, 128, 4, 2, "f16", 1.0), (5, 1, 128, 96, 8, 3, "bf16", 1.0), (2, 9, 192, 200, 3, 1, "f32", 1.0),
    (3, 40, 256, 384, 5, 4, "bf16", 1.0), (1, 130, 132, 160, 40, 8, "f16", 1.0),
    # gates that keep fp16 results in range (hidden values reach 448⁴)
    (1, 130, 132, 160, 40, 8, "f16", 2.0 ** -24), (2, 9, 128, 300, 6, 2, "f16", 2.0 ** -24),
    (1, 3, 64, 128, 4, 2, "f16", 2.0 ** -24)])
@pytest.mark.parametrize("prev,resid", [(False, False), (True, True)])
def test_experts(device, B, T, C, F, E, k, dtype, gate, prev, resid):
    x, x_k, key, val = integers(device, B, T, C, F, E, dtype)
    rng = np.random.default_rng(5)
    inds = torch.from_numpy(np.stack([rng.permutation(E)[:k] for _ in range(B * T)])).to(torch.int32).view(B, T, k)
    inds[-1, -1, 0] = -1  # an unrouted slot
    if k > 1:
        inds[0, 0, 1] = inds[0, 0, 0]  # one expert twice
    gates = torch.from_numpy(rng.random((B, T, k)) * gate).float()
    xp = x[:, -1].flip(0).clone() if prev else None
    res = rand((B, T, C), dtype, 9) if resid else None
    hk, hv = Fp8Weight.quantize(key.to(device)), Fp8Weight.quantize(val.to(device))
    d = lambda t: None if t is None else t.to(device)
    got = fp8_experts(d(x), d(inds), d(gates), d(x_k), hk, hv, x_prev=d(xp), residual=d(res))
    again = fp8_experts(d(x), d(inds), d(gates), d(x_k), hk, hv, x_prev=d(xp), residual=d(res))
    assert torch.equal(got, again)
    held = lambda w: [O.held_tiles(*O.quantize_tiles(m)) for m in w.float().numpy()]
    # more than 64 rows: with bf16 both products, with fp16 the value product come from the e4m3 instruction
    e4m3 = B * T * k > 64 and dtype != "f32"
    want, size, slack = O.experts(x.float().numpy(), inds.numpy(), gates.numpy(), x_k.float().numpy(), held(key),
                                  held(val), None if xp is None else xp.float().numpy(),
                                  None if res is None else f64(res), aligned=e4m3)
    eps = torch.finfo(DT[dtype]).eps / 2
    fb = -(-F // 128)
    # the value product's sums, then k fmas and the residual's sum in fp32, then one rounding
    mag = size + (0 if res is None else np.abs(f64(res)))
    tol = np.abs(want) * eps + mag * 2.0 ** -23 * (128 + fb + k + 1) * (1 + eps) + slack + 1e-30
    # a value from the largest one and half its step on (fp16: 65504 + 16) rounds to an infinity of that sign; one
    # whose tolerance reaches that border may fall on either side of it
    most = torch.finfo(DT[dtype]).max
    border = most + 2.0 ** np.floor(np.log2(most)) * eps
    g = f64(got)
    inf = np.isinf(g) & (g == np.sign(want) * np.inf)
    assert inf[np.abs(want) - tol >= border].all() and (np.abs(want) + tol >= border)[inf].all()
    err = np.abs(g - want)[~inf]
    assert (err <= tol[~inf]).all(), float((err / tol[~inf]).max())


def test_fp8_layer_run_of_routing_experts_and_decode(device):
    """A MoE layer in 8 bits behind each router: a prefill equals its tokens
    decoded one by one, and follows the 16-bit layer."""
    torch.manual_seed(0)
    cfg = RWKVConfig(n_embd=128, dim_ffn=256)
    moe = MoE_CMix(cfg, 0, 8, 2).to(device)
    with torch.no_grad():
        moe.expert_val.normal_(0, 0.06)
        moe.x_k.uniform_(0, 1)
    x = torch.randn(2, 6, 128, device=device)
    for router in (None, GroupRouter(128, 8, 2, n_groups=4, top_groups=2).to(device)):
        layer = Fp8MoE_CMix.from_moe(moe, router)
        out, aux, z = layer(x)
        assert out.shape == x.shape and torch.isfinite(out).all() and not out.requires_grad
        state = torch.zeros(2, 128, device=device)
        for t in range(6):
            step, state = channel_mixing_rnn(x[:, t], state, layer)
            # other tiles sum in another order: 2^-23 a term, and a hidden value on a border may round the other way
            assert (step - out[:, t]).abs().max() <= 2.0 ** -4 * out.abs().max()
        res = layer(x, residual=x)[0]
        assert (res - (x + out)).abs().max() <= 2.0 ** -22 * (x.abs() + out.abs()).max()
        if router is None:
            with torch.no_grad():
                ref, aux2, z2 = moe(x)
            assert torch.equal(aux, aux2) and torch.equal(z, z2)
            # three roundings of half a step 2^-4 in the product of two factors and a square
            assert (out - ref).abs().mean() <= 4 * 2.0 ** -4 * ref.abs().mean()


def test_streams_and_graphs(device):
    h = Fp8Weight.quantize(rand((200, 256), "bf16", 1).to(device))
    he = Fp8Weight.quantize(rand((4, 200, 256), "bf16", 1).to(device))
    off = torch.tensor([0, 10, 30, 30, 90], dtype=torch.int32, device=device)
    x = rand((90, 256), "bf16", 2).to(device)
    want = fp8_linear(x, h), fp8_grouped_linear(x, he, off)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fp8_linear(x, h), fp8_grouped_linear(x, he, off)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs on one stream, replayed in turns with eager calls of other sizes between
    graphs = []
    for fn in (lambda: fp8_linear(x, h), lambda: fp8_grouped_linear(x, he, off)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out, fn))
    for seed in range(3):
        x.copy_(rand((90, 256), "bf16", seed + 10))
        fp8_linear(torch.randn(700 + seed, 256, device=device), h)
        for g, out, fn in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out, fn in graphs:
            assert torch.equal(out, fn())


def test_strides_shapes_and_empty(device):
    w = rand((30, 96), "f16", 1).to(device)
    h = Fp8Weight.quantize(w, transposed=True)
    base = rand((12, 200), "f16", 2).to(device)
    want = fp8_linear(base[:, 3:99].contiguous(), h)
    assert torch.equal(fp8_linear(base[:, 3:99], h), want)           # rows that are not 16-byte aligned
    assert torch.equal(fp8_linear(base[::2, 3:99], h), want[::2])
    assert torch.equal(fp8_linear(base[:, 3:99].t().contiguous().t(), h), want)
    assert torch.equal(fp8_linear(base[:, 3:99].reshape(3, 4, 96), h), want.view(3, 4, 30))
    assert torch.equal(fp8_linear(base[0, 3:99], h), want[0])
    z = torch.zeros(0, 96, dtype=torch.float16, device=device, requires_grad=True)
    wt = w.clone().requires_grad_(True)
    dz, dw = torch.autograd.grad(fp8_linear(z, wt).sum(), (z, wt))
    assert dz.shape == (0, 96) and (dw == 0).all()
    assert fp8_linear(z.detach(), h).shape == (0, 30)
    # cotangents of other strides
    x = base[:, :96].detach().requires_grad_(True)
    y = fp8_linear(x, h)
    dy = rand((30, 12), "f16", 4).to(device)
    (a,) = torch.autograd.grad(y, x, dy.t(), retain_graph=True)
    (b,) = torch.autograd.grad(y, x, dy.t().contiguous(), retain_graph=True)
    (c,) = torch.autograd.grad(y, x, torch.ones((), dtype=torch.float16, device=device).expand(12, 30))
    assert torch.equal(a, b) and torch.isfinite(c).all()


def test_refusals(device):
    h = Fp8Weight.quantize(torch.zeros(8, 16, device=device))
    he = Fp8Weight.quantize(torch.zeros(2, 8, 16, device=device))
    x = torch.zeros(4, 16, device=device)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=device)
    xg = x.clone().requires_grad_(True)
    inds = torch.zeros(1, 4, 1, dtype=torch.int32, device=device)
    val = Fp8Weight.quantize(torch.zeros(2, 16, 8, device=device))
    ex = lambda x=x[None], inds=inds, gates=inds.float(), x_k=torch.zeros(2, 16, device=device), key=he, value=val, **k: \
        fp8_experts(x, inds, gates, x_k, key, value, **k)
    ex()
    for call, err in (
            (lambda: fp8_linear(x[:, :15], h), ValueError), (lambda: fp8_linear(x.double(), h), TypeError),
            (lambda: fp8_linear(x, he), ValueError), (lambda: fp8_linear(xg, h), ValueError),
            (lambda: fp8_grouped_linear(xg, he, off), ValueError), (lambda: fp8_grouped_linear(x, h, off), TypeError),
            (lambda: fp8_grouped_linear(x, he, off.long()), ValueError),
            (lambda: fp8_grouped_linear(x, he, off[:2]), ValueError),
            (lambda: fp8_grouped_linear(x[None], he, off), ValueError),
            (lambda: fp8_quantize(x[None]), ValueError), (lambda: Fp8Weight.quantize(x[0]), ValueError),
            (lambda: Fp8Weight.from_quantized(h.q, h.scale.t()[:0]), ValueError),
            (lambda: Fp8Weight.from_quantized(x, h.scale), TypeError),
            (lambda: ex(x=xg[None]), RuntimeError), (lambda: ex(inds=inds.long()), ValueError),
            (lambda: ex(value=he), ValueError), (lambda: ex(x_prev=x), ValueError),
            (lambda: ex(residual=x), ValueError), (lambda: ex(gates=torch.zeros(1, 4, 1)), ValueError)):
        with pytest.raises(err):
            call()


def test_a_layer_keeps_its_weights_through_casts(device):
    torch.manual_seed(1)
    moe = MoE_CMix(RWKVConfig(n_embd=64, dim_ffn=128), 0, 4, 2).to(device)
    with torch.no_grad():
        moe.expert_val.normal_(0, 0.1)
    layer = Fp8MoE_CMix.from_moe(moe)
    q, s = layer.key_q.clone(), layer.value_scale.clone()
    layer.half()
    assert layer.x_k.dtype == torch.float16 and layer.router.gate.weight.dtype == torch.float16
    assert torch.equal(layer.key_q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(layer.value_scale, s)
    out, _, _ = layer(torch.randn(1, 5, 64, device=device).half())
    assert out.dtype == torch.float16 and torch.isfinite(out).all()
    again = Fp8MoE_CMix.from_moe(moe).half()
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again.key_q.view(torch.uint8), layer.key_q.view(torch.uint8))


def test_offsets_past_32_bits(device):
    """x, its 8-bit form and the product lie past 4 GB: the last rows are the
    ones that they are on their own."""
    R, K, N = 2_200_000, 2048, 520
    x = torch.empty(R, K, dtype=torch.bfloat16, device=device).normal_()
    tail = x[-200:].clone()
    q, s, qt, st = fp8_quantize(x, transposed=True)
    q1, s1 = fp8_quantize(tail)
    assert q.numel() > 1 << 32
    assert torch.equal(q[-200:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[:, -200:], s1)
    last = R // 128 * 128 - 128  # the last whole block of rows
    qt1 = fp8_quantize(x[last:last + 128].clone(), transposed=True, rows=False)[0]
    assert torch.equal(qt[:, last:last + 128].contiguous().view(torch.uint8), qt1.view(torch.uint8))
    del q, s, qt, st
    h = Fp8Weight.quantize(rand((N, K), "bf16", 1).to(device))
    y = fp8_linear(x, h)
    assert torch.equal(y[-200:], fp8_linear(tail, h))
    he = Fp8Weight.quantize(rand((2, N, K), "bf16", 1).to(device))
    off = torch.tensor([0, 7, R - 100], dtype=torch.int32, device=device)
    y = fp8_grouped_linear(x, he, off)
    h1 = Fp8Weight.quantize(rand((2, N, K), "bf16", 1)[1].to(device))
    assert torch.equal(y[-200:-100], fp8_linear(tail[:100], h1)) and (y[-100:] == 0).all()


def test_gradients_in_a_graph(device):
    x = rand((150, 256), "bf16", 1).to(device).requires_grad_(True)
    w = rand((200, 256), "bf16", 2).to(device).requires_grad_(True)
    he = Fp8Weight.quantize(rand((3, 200, 256), "bf16", 3).to(device), transposed=True)
    off = torch.tensor([0, 40, 90, 150], dtype=torch.int32, device=device)
    dy = rand((150, 200), "bf16", 4).to(device)

    def step():
        a = torch.autograd.grad(fp8_linear(x, w), (x, w), dy)
        b = torch.autograd.grad(fp8_grouped_linear(x, he, off), x, dy)
        return (*a, *b)

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
            x.copy_(rand((150, 256), "bf16", seed + 20))
            dy.copy_(rand((150, 200), "bf16", seed + 30))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("N,K", [(2690, 1500), (2688, 1500), (2691, 300)])
def test_tiles_of_every_size_give_the_same_bits(device, dtype, N, K):
    """A row's sums take one order whatever tile holds it: 64 x 128 with 300 and
    1500 rows, 128 x 128 with 900, 192 x 256 with 3840 (16-bit results, K > 11
    blocks), and the last of these is held against the formula."""
    x, w = rand((3840, K), dtype, 1, 0.3), rand((N, K), dtype, 2, 0.3)
    h, xd = Fp8Weight.quantize(w.to(device)), x.to(device)
    all_rows = fp8_linear(xd, h)
    for r in (65, 300, 900, 1500):
        assert torch.equal(fp8_linear(xd[:r], h), all_rows[:r]), r
    assert torch.equal(fp8_linear(xd[3000:], h), all_rows[3000:])
    close(all_rows[:100], O.held_rows(*O.quantize_rows(x[:100].float().numpy())),
          O.held_tiles(*O.quantize_tiles(w.float().numpy())), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_grouped_tiles_of_every_size_give_the_same_bits(device, dtype):
    E, N, K = 9, 1281, 1500
    counts = [700, 0, 1, 900, 129, 128, 3, 2000, 400]
    off = np.concatenate([[0], np.cumsum(counts)])
    x, w = rand((off[-1] + 200, K), dtype, 1, 0.3).to(device), rand((E, N, K), dtype, 2, 0.3).to(device)
    h = Fp8Weight.quantize(w)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    y = fp8_grouped_linear(x, h, ints(off))
    assert (y[off[-1]:] == 0).all()
    for e in range(E):
        lo, hi = int(off[e]), int(off[e + 1])
        part = x[lo:hi] if hi - lo > 64 else x[lo:lo + 65]  # (up to 64 rows take the fp16 sums)
        one = ints([0] * (e + 1) + [hi - lo] * (E - e))
        assert torch.equal(fp8_grouped_linear(part, h, one)[:hi - lo], y[lo:hi]), e


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("C", [512, 1024])
def test_layers_of_every_size_give_the_same_bits(device, dtype, C):
    """Sequences of a large batch and the same ones in a small batch."""
    B, T, F, E, k = 40, 50, 1100, 8, 4
    x = rand((B, T, C), dtype, 1, 0.5).to(device)
    key, val = rand((E, F, C), dtype, 2, 0.05).to(device), rand((E, C, F), dtype, 3, 0.05).to(device)
    x_k = rand((E, C), dtype, 4, 0.5).to(device)
    gen = torch.Generator().manual_seed(5)
    inds = torch.rand(B, T, E, generator=gen).argsort(-1)[..., :k].to(torch.int32).to(device)
    gates = torch.rand(B, T, k, generator=gen).to(device)
    hk, hv = Fp8Weight.quantize(key), Fp8Weight.quantize(val)
    y = fp8_experts(x, inds, gates, x_k, hk, hv)
    # (hidden values of some 1e4 times values: part of the fp16 results lie past 65504)
    assert not y.isnan().any() and (dtype == "f16" or torch.isfinite(y).all())
    for b in (0, 17, 37):
        part = slice(b, b + 3)
        got = fp8_experts(x[part].contiguous(), inds[part].contiguous(), gates[part].contiguous(), x_k, hk, hv)
        assert torch.equal(got, y[part]), b


def test_what_the_backward_keeps(device):
    """The operands kept for a linear's backward can be kept elsewhere (saved
    tensor hooks), read twice, and are gone after the last backward."""
    x = rand((150, 256), "bf16", 1).to(device).requires_grad_(True)
    w = rand((200, 256), "f32", 2).to(device).requires_grad_(True)
    dy = rand((150, 200), "bf16", 4).to(device)
    y = fp8_linear(x, w)
    want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = fp8_linear(x, w)
    filler = torch.full((1 << 20,), 255, dtype=torch.uint8, device=device)  # (over what the call has freed)
    got = torch.autograd.grad(y, (x, w), dy)
    assert filler.min() == 255 and all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(torch.autograd.grad(fp8_linear(x, w.detach()), x, dy)[0], want[0])
    assert torch.equal(torch.autograd.grad(fp8_linear(x.detach(), w), w, dy)[0], want[1])


def test_the_layer_refuses_to_drop_a_gradient(device):
    torch.manual_seed(3)
    r = GroupRouter(64, 4, 2).to(device)
    key, val = rand((4, 96, 64), "bf16", 1).to(device), rand((4, 64, 96), "bf16", 2).to(device)
    m = Fp8MoE_CMix(r, torch.zeros(4, 64, device=device), Fp8Weight.quantize(key), Fp8Weight.quantize(val))
    x = rand((2, 3, 64), "bf16", 3).to(device)
    want = m(x)[0]
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(x.detach(), residual=x)
    with torch.no_grad():
        assert torch.equal(m(x)[0], want)


@pytest.mark.parametrize("train", [False, True])
def test_a_fused_layer_refuses_a_group_router(device, train):
    layer = MoE_CMix(RWKVConfig(n_embd=64, dim_ffn=128), 0, 4, 2).to(device)
    layer.router = GroupRouter(64, 4, 2).to(device)
    x = torch.randn(1, 3, 64, device=device, requires_grad=train)
    with torch.set_grad_enabled(train), pytest.raises(TypeError, match="GroupRouter"):
        layer(x)
