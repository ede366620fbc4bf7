"""Argument checks of the routing and 8-bit entry points, all on the host: no
call here reaches a launch."""
from __future__ import annotations

import copy
import ctypes

import pytest
import torch

from rwkv_mlx_amd import (Fp8MoE_CMix, Fp8Weight, GroupRouter, _lib as L, fp8_experts, fp8_grouped_linear, fp8_linear,
                          fp8_quantize, route_topk)

FAKE = 1 << 40


def route_desc(**kw):
    d = dict(rows=4, n_experts=16, top_k=2, n_groups=1, top_groups=1, dtype=L.F32, score=0, group_score=0, flags=0,
             scale=1.0, logits_stride=16)
    d.update(kw)
    return L.RouteDesc(*[d[n] for n, _ in L.RouteDesc._fields_])


def fp8_desc(**kw):
    d = dict(rows=4, n=8, k=16, groups=0, dtype=L.F32, block=L.FP8_TILES, stride=16)
    d.update(kw)
    return L.Fp8Desc(*[d[n] for n, _ in L.Fp8Desc._fields_])


ROUTE_BAD = [
    (dict(dtype=3), -3), (dict(rows=-1), -2), (dict(n_experts=0), -2), (dict(n_experts=513, logits_stride=513), -2),
    (dict(n_groups=3), -2), (dict(n_groups=0), -2), (dict(n_groups=4, top_groups=5), -2), (dict(top_groups=0), -2),
    (dict(logits_stride=15), -2), (dict(top_k=0), -7), (dict(top_k=17), -7), (dict(n_experts=64, top_k=33,
                                                                                logits_stride=64), -7),
    (dict(n_groups=4, top_groups=1, top_k=5), -7), (dict(score=2), -9), (dict(group_score=-1), -9),
    (dict(flags=2), -8),
]


@pytest.mark.parametrize("kw,want", ROUTE_BAD)
def test_route_refuses(kw, want):
    d = route_desc(**kw)
    p = FAKE
    assert L.lib().rwkvmoe_route(ctypes.byref(d), p, None, p, p, None) == want
    assert L.lib().rwkvmoe_route_backward(ctypes.byref(d), p, p, p, p, p, None) == want


def test_route_pointers():
    d = route_desc()
    fn, bwd = L.lib().rwkvmoe_route, L.lib().rwkvmoe_route_backward
    assert fn(None, FAKE, None, FAKE, FAKE, None) == -1
    assert fn(ctypes.byref(d), None, None, FAKE, FAKE, None) == -4
    assert fn(ctypes.byref(d), FAKE, None, None, FAKE, None) == -4
    assert fn(ctypes.byref(d), FAKE + 2, None, FAKE, FAKE, None) == -5
    assert fn(ctypes.byref(d), FAKE, FAKE + 1, FAKE, FAKE, None) == -5
    for i in range(5):
        a = [FAKE] * 5
        a[i] = None
        assert bwd(ctypes.byref(d), *a, None) == -4
    assert bwd(ctypes.byref(d), *[FAKE] * 4, FAKE + 8, None) == -5
    z = route_desc(rows=0)
    assert fn(ctypes.byref(z), None, None, None, None, None) == 0
    assert bwd(ctypes.byref(z), *[None] * 6) == 0


FP8_BAD = [(dict(dtype=5), -3), (dict(block=2), -9), (dict(rows=-1), -2), (dict(k=0), -2), (dict(k=(1 << 23) + 1), -2),
           (dict(groups=-1), -2), (dict(groups=1025), -2), (dict(rows=65535 * 128 + 1), -2)]


@pytest.mark.parametrize("kw,want", FP8_BAD)
def test_fp8_refuses(kw, want):
    d = fp8_desc(**kw)
    b = ctypes.c_size_t(0)
    lib = L.lib()
    assert lib.rwkvmoe_fp8_quantize(ctypes.byref(d), FAKE, FAKE, FAKE, None, None, None) == want
    assert lib.rwkvmoe_fp8_matmul(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == want
    assert lib.rwkvmoe_fp8_linear_workspace_bytes(ctypes.byref(d), ctypes.byref(b)) == want
    assert lib.rwkvmoe_fp8_linear(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == want


def test_fp8_pointers_and_workspace():
    lib = L.lib()
    d = fp8_desc()
    ref = ctypes.byref
    assert lib.rwkvmoe_fp8_quantize(None, FAKE, FAKE, FAKE, None, None, None) == -1
    assert lib.rwkvmoe_fp8_quantize(ref(d), FAKE, None, None, None, None, None) == -4
    assert lib.rwkvmoe_fp8_quantize(ref(d), FAKE, FAKE, None, None, None, None) == -4
    assert lib.rwkvmoe_fp8_quantize(ref(d), FAKE, FAKE, FAKE, FAKE, None, None) == -4
    assert lib.rwkvmoe_fp8_quantize(ref(d), FAKE + 2, FAKE, FAKE, None, None, None) == -5
    assert lib.rwkvmoe_fp8_quantize(ref(fp8_desc(stride=15)), FAKE, FAKE, FAKE, None, None, None) == -2
    assert lib.rwkvmoe_fp8_quantize(ref(fp8_desc(groups=2, block=0)), FAKE, FAKE, FAKE, None, None, None) == -2
    assert lib.rwkvmoe_fp8_layout(ref(fp8_desc(block=0)), FAKE, FAKE, FAKE, FAKE, None, None, None) == -9
    assert lib.rwkvmoe_fp8_layout(ref(d), FAKE, FAKE, FAKE + 8, FAKE, None, None, None) == -5
    assert lib.rwkvmoe_fp8_layout(ref(d), FAKE, FAKE, FAKE, FAKE, FAKE, None, None) == -4
    for i in (0, 1, 2, 3, 5):
        a = [FAKE] * 6
        a[i] = None
        assert lib.rwkvmoe_fp8_matmul(ref(d), *a, None) == -4
    g = fp8_desc(groups=3)
    assert lib.rwkvmoe_fp8_matmul(ref(g), FAKE, FAKE, FAKE, FAKE, None, FAKE, None) == -4
    assert lib.rwkvmoe_fp8_matmul(ref(fp8_desc(groups=3, block=0)), *[FAKE] * 6, None) == -9
    assert lib.rwkvmoe_fp8_matmul(ref(fp8_desc(n=0)), *[FAKE] * 6, None) == -2
    b = ctypes.c_size_t(0)
    assert lib.rwkvmoe_fp8_linear_workspace_bytes(ref(d), None) == -4
    assert lib.rwkvmoe_fp8_linear_workspace_bytes(ref(d), ref(b)) == 0 and b.value == 0
    d = fp8_desc(rows=65)
    assert lib.rwkvmoe_fp8_linear_workspace_bytes(ref(d), ref(b)) == 0 and b.value == 65 * 128 + 128 + 512
    lin = lambda desc, ws, n: lib.rwkvmoe_fp8_linear(ref(desc), FAKE, FAKE, FAKE, None, FAKE, ws, n, None)
    assert lin(d, None, b.value) == -6 and lin(d, FAKE, b.value - 1) == -6 and lin(d, FAKE + 16, b.value) == -6
    assert lin(fp8_desc(block=0), FAKE, 1 << 20) == -9 and lin(fp8_desc(stride=8), FAKE, 1 << 20) == -2
    assert lin(fp8_desc(rows=0), None, 0) == 0


def test_fp8_experts_checks():
    lib = L.lib()
    ref = ctypes.byref
    b = ctypes.c_size_t(0)

    def desc(**kw):
        d = dict(batch=2, seq_len=3, d_model=64, d_ffn=96, n_experts=4, top_k=2, lora_rank=1, dtype=L.F16, mode=0,
                 flags=0)
        d.update(kw)
        return L.Desc(*[d[n] for n, _ in L.Desc._fields_])

    size = lambda **kw: lib.rwkvmoe_fp8_experts_workspace_bytes(ref(desc(**kw)), ref(b))
    assert size() == 0 and b.value > 0
    need = b.value
    for kw, want in ((dict(d_model=66), -2), (dict(d_ffn=0), -2), (dict(n_experts=65), -2), (dict(top_k=5), -7),
                     (dict(dtype=7), -3), (dict(flags=L.HAS_BIAS), -8), (dict(batch=1 << 15, seq_len=1 << 12), -2)):
        assert size(**kw) == want, kw
    assert lib.rwkvmoe_fp8_experts_workspace_bytes(ref(desc()), None) == -4
    names = [n for n, _ in L.Fp8Experts._fields_][1:]

    def st(d=None, ws=FAKE, n=need, size=L.FP8_EXPERTS_SIZE, **kw):
        t = L.Fp8Experts(size, **{m: kw.get(m, FAKE) for m in names})
        return lib.rwkvmoe_fp8_experts_forward(ref(d or desc()), ref(t), ws, n, None)

    assert lib.rwkvmoe_fp8_experts_forward(ref(desc()), None, FAKE, need, None) == -1
    assert st(size=8) == -12 and st(ws=None) == -6 and st(n=need - 1) == -6 and st(ws=FAKE + 64) == -6
    for m in names:
        if m not in ("x_prev", "residual"):
            assert st(**{m: None}) == -4, m
    assert st(desc(flags=L.HAS_PREV), x_prev=None) == -8
    assert st(desc(flags=L.ADD_RESIDUAL), residual=None) == -8
    assert st(x=FAKE + 1) == -5 and st(key_q=FAKE + 8) == -5
    assert st(desc(batch=0), ws=None, n=0) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros(2, 8)
    for call in (lambda: route_topk(x, 2), lambda: fp8_quantize(x), lambda: Fp8Weight.quantize(x),
                 lambda: Fp8Weight.from_quantized(x.to(torch.float8_e4m3fn), torch.ones(1, 1)),
                 lambda: fp8_linear(x, torch.zeros(3, 8))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(TypeError):
        fp8_grouped_linear(x, x, torch.zeros(2, dtype=torch.int32))


def test_launches_stay_below_2_to_32_threads():
    """More rows than one launch has threads for are refused on the host."""
    lib, ref, b = L.lib(), ctypes.byref, ctypes.c_size_t(0)
    d = route_desc(rows=(1 << 26) - 63)
    assert lib.rwkvmoe_route(ref(d), FAKE, None, FAKE, FAKE, None) == -2
    assert lib.rwkvmoe_route_backward(ref(d), FAKE, FAKE, FAKE, FAKE, FAKE, None) == -2
    big = dict(k=8192, stride=8192)  # 64 slices: 2^18 workgroups of 16 rows are too many
    d = fp8_desc(rows=1 << 22, **big)
    assert lib.rwkvmoe_fp8_quantize(ref(d), FAKE, FAKE, FAKE, None, None, None) == -2
    assert lib.rwkvmoe_fp8_linear_workspace_bytes(ref(d), ref(b)) == -2
    assert lib.rwkvmoe_fp8_linear_workspace_bytes(ref(fp8_desc(rows=(1 << 22) - 64, **big)), ref(b)) == 0
    e = L.Desc()
    e.batch, e.seq_len, e.d_ffn, e.n_experts, e.top_k = 1, 1 << 22, 128, 8, 1
    for c in (4096, 8192):  # tokens x C / 4 threads
        e.d_model = c
        assert lib.rwkvmoe_fp8_experts_workspace_bytes(ref(e), ref(b)) == -2
    e.seq_len = (1 << 22) - 64
    e.d_model = 4096
    assert lib.rwkvmoe_fp8_experts_workspace_bytes(ref(e), ref(b)) == 0


def test_casts_leave_the_balance_bias_and_8_bit_weights_alone():
    """The bias adds up small steps: in bfloat16 1 + 0.001 is 1 again."""
    r = GroupRouter(8, 16, 2)
    r.balance_bias.fill_(1.0)
    for cast in (lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.type(torch.float64)):
        assert cast(r) is r and r.balance_bias.dtype == torch.float32 and r.gate.weight.dtype != torch.float32
        before = r.balance_bias.clone()
        r.update_balance(torch.zeros(4, 2, dtype=torch.int32), rate=1e-3)
        assert r.balance_bias[0] < before[0] and (r.balance_bias[1:] > before[1:]).all()
    e4m3 = lambda *s: torch.arange(16 * 128, dtype=torch.float32).remainder(100).view(1, 16, 128).to(
        torch.float8_e4m3fn)
    w = Fp8Weight((1, 16, 128), e4m3(), torch.full((1, 1, 1), 0.3))
    v = Fp8Weight((1, 128, 16), torch.zeros(1, 128, 128, dtype=torch.float8_e4m3fn), torch.ones(1, 1, 1))
    m = Fp8MoE_CMix(r, torch.zeros(1, 128), w, v)
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.type(torch.float64)):
        assert cast(m) is m and m.key_q.dtype == torch.float8_e4m3fn and m.key_scale.dtype == torch.float32
        assert torch.equal(m.key_q.view(torch.uint8), w.q.view(torch.uint8)) and m.key_scale.item() == w.scale.item()
        assert m.x_k.dtype != torch.float32


def test_fused_layers_refuse_a_group_router():
    """Their kernels route by the router's weight alone, after they have read its logit_bias."""
    r = GroupRouter(8, 4, 2)
    with pytest.raises(TypeError, match="Fp8MoE_CMix"):
        r.logit_bias
    assert set(r.state_dict()) == {"gate.weight", "balance_bias"} and copy.deepcopy(r).top_k == 2
