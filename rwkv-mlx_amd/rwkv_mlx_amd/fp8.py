"""Products in 8 bits: e4m3 operands with one fp32 scale for each block of 128.

  ``Fp8Weight``            a weight held in 8 bits (blocks of 128 x 128), or E of them
  ``fp8_linear``           x · wᵀ, x rounded in the call to 8 bits in blocks of 128
                           values of a row; w an Fp8Weight (frozen) or a trainable
                           tensor (rounded in the call; both gradients are 8-bit
                           products as well)
  ``fp8_grouped_linear``   the same for rows sorted by expert, E weights
  ``fp8_experts``          a layer of full ChannelMix experts (the reference's
                           rwkv_mlx/moe.py:218-234) on a given routing
  ``Fp8MoE_CMix``          ``MoE_CMix`` for inference with its experts in 8 bits

A block with a = max(|v|, 2^-100) is held as e4m3(v · fp32(448 / a)), rounded to
nearest even, and the scale fp32(a / 448).  A NaN or an infinity makes its
block NaN.  Products are summed in fp32 and rounded once.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .model import require_device

__all__ = ["Fp8Weight", "fp8_quantize", "fp8_linear", "fp8_grouped_linear", "fp8_experts", "Fp8MoE_CMix"]

BLOCK = 128


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _code(t: torch.Tensor, what: str) -> int:
    code = _lib.TORCH_DTYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: float32, float16 or bfloat16 expected, got {t.dtype}")
    return code


def _bytes(*shape, device):
    return torch.empty(*shape, dtype=torch.float8_e4m3fn, device=device)


def _f32(*shape, device):
    return torch.empty(*shape, dtype=torch.float32, device=device)


def _rows2d(x: torch.Tensor) -> torch.Tensor:
    """x (..., K) as rows (R, K) with unit stride along K, in place where that is so."""
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= x.shape[1]:
        return x
    return x.reshape(-1, x.shape[-1]).contiguous()


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _call(name: str, x: torch.Tensor, *args) -> None:
    _lib.launch(getattr(_lib.lib(), name), name, x.device, *args)


def fp8_quantize(x: torch.Tensor, transposed: bool = False, rows: bool = True):
    """x (R, K) in blocks of 128 values of a row: (q (R, 128·Kb) e4m3, zero
    from column K on, scales (Kb, R) fp32), Kb = ceil(K / 128).  With
    ``transposed`` also xᵀ in blocks of 128 values of a column of x: (q_t
    (K, 128·Rb), scales_t (Rb, K)); without ``rows`` that alone."""
    require_device(x, "fp8_quantize")
    if x.dim() != 2:
        raise ValueError(f"fp8_quantize expects (rows, columns), got {tuple(x.shape)}")
    x = _rows2d(x.detach())
    R, K = x.shape
    dev = x.device
    q = s = qt = st = None
    if rows:
        q, s = _bytes(R, _blocks(K) * BLOCK, device=dev), _f32(_blocks(K), R, device=dev)
    if transposed:
        qt, st = _bytes(K, _blocks(R) * BLOCK, device=dev), _f32(_blocks(R), K, device=dev)
    desc = _lib.fp8_desc(R, 0, K, 0, _code(x, "fp8_quantize"), _lib.FP8_ROWS, _stride(x))
    _call("rwkvmoe_fp8_quantize", x, desc, x.data_ptr(), _lib.ptr(q), _lib.ptr(s), _lib.ptr(qt),
          _lib.ptr(st))
    return tuple(t for t in (q, s, qt, st) if t is not None)


class Fp8Weight:
    """A weight (N, K), or E weights (E, N, K), held in 8 bits with one scale
    for each 128 x 128 block.  With ``transposed`` its transpose is held too,
    which the gradient of x reads.  It is not trained.

    q (.., N, 128·Kb) e4m3, zero from column K on; scale (.., Nb, Kb) fp32."""

    def __init__(self, shape, q, scale, q_t=None, scale_t=None):
        self.shape = tuple(shape)
        self.q, self.scale, self.q_t, self.scale_t = q, scale, q_t, scale_t

    @property
    def device(self) -> torch.device:
        return self.q.device

    @property
    def groups(self) -> int:
        return self.shape[0] if len(self.shape) == 3 else 0

    @classmethod
    def _empty(cls, shape, device, transposed):
        if len(shape) not in (2, 3) or min(shape) < 1:
            raise ValueError(f"Fp8Weight: (N, K) or (E, N, K) expected, got {tuple(shape)}")
        *lead, N, K = shape
        w = cls(shape, _bytes(*lead, N, _blocks(K) * BLOCK, device=device),
                _f32(*lead, _blocks(N), _blocks(K), device=device))
        if transposed:
            w.q_t = _bytes(*lead, K, _blocks(N) * BLOCK, device=device)
            w.scale_t = _f32(*lead, _blocks(K), _blocks(N), device=device)
        return w

    @classmethod
    def quantize(cls, w: torch.Tensor, transposed: bool = False) -> "Fp8Weight":
        """Rounds a weight (N, K) or (E, N, K) in float32, float16 or bfloat16."""
        require_device(w, "Fp8Weight.quantize")
        code = _code(w, "Fp8Weight.quantize")
        w = w.detach().contiguous()
        out = cls._empty(w.shape, w.device, transposed)
        N, K = w.shape[-2:]
        desc = _lib.fp8_desc(N, 0, K, out.groups, code, _lib.FP8_TILES, K)
        _call("rwkvmoe_fp8_quantize", w, desc, w.data_ptr(), out.q.data_ptr(), out.scale.data_ptr(),
              _lib.ptr(out.q_t), _lib.ptr(out.scale_t))
        return out

    @classmethod
    def from_quantized(cls, q: torch.Tensor, scale: torch.Tensor, transposed: bool = False) -> "Fp8Weight":
        """From a checkpoint's e4m3 values (.., N, K) and block scales
        (.., ceil(N / 128), ceil(K / 128)) fp32; a value stands for q · scale."""
        require_device(q, "Fp8Weight.from_quantized")
        if q.dtype != torch.float8_e4m3fn or q.dim() not in (2, 3):
            raise TypeError(f"Fp8Weight.from_quantized: q (N, K) or (E, N, K) in float8_e4m3fn expected, got "
                            f"{tuple(q.shape)} {q.dtype}")
        *lead, N, K = q.shape
        if scale.shape != (*lead, _blocks(N), _blocks(K)) or scale.device != q.device:
            raise ValueError(f"Fp8Weight.from_quantized: scales {(*lead, _blocks(N), _blocks(K))} on {q.device} "
                             f"expected, got {tuple(scale.shape)} on {scale.device}")
        q, scale = q.detach().contiguous(), scale.detach().to(torch.float32).contiguous()
        out = cls._empty(q.shape, q.device, transposed)
        desc = _lib.fp8_desc(0, N, K, out.groups, _lib.F32, _lib.FP8_TILES, K)
        _call("rwkvmoe_fp8_layout", q, desc, q.data_ptr(), scale.data_ptr(), out.q.data_ptr(),
              out.scale.data_ptr(), _lib.ptr(out.q_t), _lib.ptr(out.scale_t))
        return out

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the weight stands for."""
        *_, N, K = self.shape
        s = self.scale.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]
        return (self.q[..., :K].to(torch.float32) * s).to(dtype)


def _product(x, N, K, groups, code, q, scale, offsets, dtype):
    """x (R, K) rounded and multiplied with a weight in 8 bits: (R, N)."""
    R = x.shape[0]
    out = torch.empty(R, N, dtype=dtype, device=x.device)
    desc = _lib.fp8_desc(R, N, K, groups, code, _lib.FP8_TILES, _stride(x))
    nbytes = _lib.fp8_linear_bytes(R, N, K, groups, code)
    # (from torch's allocator: a captured graph keeps its own)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    _call("rwkvmoe_fp8_linear", x, desc, x.data_ptr(), q.data_ptr(), scale.data_ptr(),
          None if offsets is None else offsets.data_ptr(), out.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return out


class _FrozenFunction(torch.autograd.Function):
    """x · wᵀ with a frozen weight; d x = d y · w, d y rounded like x."""

    @staticmethod
    def forward(ctx, x, w, offsets):
        N, K = w.shape[-2:]
        ctx.w = w
        ctx.dtype = x.dtype
        ctx.save_for_backward(offsets)
        return _product(x, N, K, w.groups, _lib.TORCH_DTYPE_CODE[x.dtype], w.q, w.scale, offsets, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w = ctx.w
        N, K = w.shape[-2:]
        (offsets,) = ctx.saved_tensors
        dy = _rows2d(dy.to(ctx.dtype))
        return _product(dy, K, N, w.groups, _lib.TORCH_DTYPE_CODE[ctx.dtype], w.q_t, w.scale_t, offsets,
                        ctx.dtype), None, None


@lru_cache(maxsize=1024)
def _parts(*wanted):
    """(offsets, bytes) of 8-bit matrices in one allocation: for each (rows,
    columns, scales) its values and its scales, for None neither."""
    at, out = 0, []
    for part in wanted:
        if part is None:
            out += [None, None]
            continue
        rows, cols, scales = part
        for n in (rows * _blocks(cols) * BLOCK, scales * 4):
            out.append(at)
            at += -(-n // 256) * 256
    return out, at


def _alloc(device, *wanted):
    """One allocation for the matrices of ``_parts``, and their addresses."""
    offsets, n = _parts(*wanted)
    buf = torch.empty(n, dtype=torch.uint8, device=device)
    return buf, _at(buf, offsets)


def _at(buf: torch.Tensor, offsets):
    base = buf.data_ptr()
    return [None if o is None else base + o for o in offsets]


class _LinearFunction(torch.autograd.Function):
    """x · wᵀ with a trainable weight, all three products in 8 bits:
    y = x · wᵀ, d x = d y · w, d w = d yᵀ · x (both rounded in blocks along the
    rows, over which it sums).  The backward keeps the 8-bit operands."""

    @staticmethod
    def forward(ctx, x, w):
        R, K = x.shape
        N = w.shape[0]
        need_x, need_w = ctx.needs_input_grad
        Rb, Nb, Kb = _blocks(R), _blocks(N), _blocks(K)
        dev, xc, wc = x.device, _lib.TORCH_DTYPE_CODE[x.dtype], _lib.TORCH_DTYPE_CODE[w.dtype]
        w = w.contiguous()
        keep = ((K, N, Kb * Nb) if need_x else None, (K, R, Rb * K) if need_w else None)
        kept, back = _alloc(dev, *keep)
        tmp, ahead = _alloc(dev, (N, K, Nb * Kb), (R, K, Kb * R))
        _call("rwkvmoe_fp8_quantize", w, _lib.fp8_desc(N, 0, K, 0, wc, _lib.FP8_TILES, K), w.data_ptr(), *ahead[:2],
              *back[:2])
        _call("rwkvmoe_fp8_quantize", x, _lib.fp8_desc(R, 0, K, 0, xc, _lib.FP8_ROWS, _stride(x)), x.data_ptr(),
              *ahead[2:], *back[2:])
        y = torch.empty(R, N, dtype=x.dtype, device=dev)
        _call("rwkvmoe_fp8_matmul", x, _lib.fp8_desc(R, N, K, 0, xc, _lib.FP8_TILES, K), *ahead[2:], *ahead[:2], None,
              y.data_ptr())
        ctx.save_for_backward(kept)
        ctx.plan = (R, N, K, x.dtype, w.dtype, keep)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        R, N, K, xdt, wdt, keep = ctx.plan
        (kept,) = ctx.saved_tensors
        back = _at(kept, _parts(*keep)[0])
        need_x, need_w = ctx.needs_input_grad
        dy, dev = _rows2d(dy), dy.device
        tmp, g = _alloc(dev, (R, N, _blocks(N) * R) if need_x else None, (N, R, _blocks(R) * N) if need_w else None)
        _call("rwkvmoe_fp8_quantize", dy, _lib.fp8_desc(R, 0, N, 0, _code(dy, "fp8_linear"), _lib.FP8_ROWS, _stride(dy)),
              dy.data_ptr(), *g)
        dx = dw = None
        if need_x:
            dx = torch.empty(R, K, dtype=xdt, device=dev)
            _call("rwkvmoe_fp8_matmul", dy, _lib.fp8_desc(R, K, N, 0, _lib.TORCH_DTYPE_CODE[xdt], _lib.FP8_TILES, N),
                  *g[:2], *back[:2], None, dx.data_ptr())
        if need_w:
            dw = torch.empty(N, K, dtype=wdt, device=dev)
            _call("rwkvmoe_fp8_matmul", dy, _lib.fp8_desc(N, K, R, 0, _lib.TORCH_DTYPE_CODE[wdt], _lib.FP8_ROWS, R),
                  *g[2:], *back[2:], None, dw.data_ptr())
        return dx, dw


def _check_x(x, K, device, what):
    require_device(x, what)
    _code(x, what)
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"{what}: x (..., {K}) expected, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{what}: x is on {x.device}, the weight on {device}")


def fp8_linear(x: torch.Tensor, weight) -> torch.Tensor:
    """x (..., K) · weightᵀ: (..., N) in x's dtype.

    ``weight`` is an ``Fp8Weight`` (N, K), frozen, or a tensor (N, K) in
    float32, float16 or bfloat16, rounded in each call.  Differentiable in x
    (an Fp8Weight then needs to be ``transposed``) and in a weight tensor."""
    frozen = isinstance(weight, Fp8Weight)
    if len(weight.shape) != 2:
        raise ValueError(f"fp8_linear: a weight (N, K) expected, got {tuple(weight.shape)}")
    N, K = weight.shape
    _check_x(x, K, weight.device, "fp8_linear")
    x2 = _rows2d(x)
    grad = torch.is_grad_enabled()
    if x2.shape[0] == 0:  # no rows: no launch, and gradients of zeros
        y = x2.new_zeros(0, N)
        if grad and (x.requires_grad or (not frozen and weight.requires_grad)):
            y = y + x2.sum() * 0
            if not frozen:
                y = y + (weight.sum() * 0).to(y.dtype)
    elif frozen:
        if grad and x.requires_grad:
            if weight.q_t is None:
                raise ValueError("fp8_linear: the gradient of x reads the weight's transpose; lay the Fp8Weight out "
                                 "with transposed=True")
            y = _FrozenFunction.apply(x2, weight, None)
        else:
            y = _product(x2, N, K, 0, _lib.TORCH_DTYPE_CODE[x2.dtype], weight.q, weight.scale, None, x2.dtype)
    else:
        _code(weight, "fp8_linear")
        if min(weight.shape) < 1:
            raise ValueError(f"fp8_linear: a weight (N, K) expected, got {tuple(weight.shape)}")
        if grad and (x.requires_grad or weight.requires_grad):
            y = _LinearFunction.apply(x2, weight)
        else:
            w = Fp8Weight.quantize(weight)
            y = _product(x2, N, K, 0, _lib.TORCH_DTYPE_CODE[x2.dtype], w.q, w.scale, None, x2.dtype)
    return y.view(*x.shape[:-1], N)


def fp8_grouped_linear(x: torch.Tensor, weight: Fp8Weight, offsets: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] · weight[g]ᵀ for offsets[g] <= r < offsets[g + 1].

    x (R, K) sorted by expert, weight (E, N, K), offsets (E + 1) int32 on the
    device, ascending from 0 (the dispatch's offsets); rows at or past
    offsets[E] become 0.  Differentiable in x (``transposed`` weights)."""
    if not isinstance(weight, Fp8Weight) or not weight.groups:
        raise TypeError("fp8_grouped_linear: weight is an Fp8Weight (E, N, K)")
    E, N, K = weight.shape
    _check_x(x, K, weight.device, "fp8_grouped_linear")
    if x.dim() != 2:
        raise ValueError(f"fp8_grouped_linear: x (R, {K}) expected, got {tuple(x.shape)}")
    if offsets.dtype != torch.int32 or offsets.shape != (E + 1,) or offsets.device != x.device:
        raise ValueError(f"fp8_grouped_linear: offsets ({E + 1},) int32 on {x.device} expected, got "
                         f"{tuple(offsets.shape)} {offsets.dtype} on {offsets.device}")
    offsets = offsets.contiguous()
    x2 = _rows2d(x)
    if x2.shape[0] == 0:
        y = x2.new_zeros(0, N)
        return y + x2.sum() * 0 if x.requires_grad else y
    if torch.is_grad_enabled() and x.requires_grad:
        if weight.q_t is None:
            raise ValueError("fp8_grouped_linear: the gradient of x reads the weights' transposes; lay the Fp8Weight "
                             "out with transposed=True")
        return _FrozenFunction.apply(x2, weight, offsets)
    return _product(x2, N, K, E, _lib.TORCH_DTYPE_CODE[x2.dtype], weight.q, weight.scale, offsets, x2.dtype)


def fp8_experts(x: torch.Tensor, inds: torch.Tensor, gates: torch.Tensor, x_k: torch.Tensor, key: Fp8Weight,
                value: Fp8Weight, x_prev: torch.Tensor | None = None,
                residual: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = Σ_slots gates[t] · value_e(relu(key_e(x + (shift(x) - x) · x_k[e]))²)
    (+ residual) with e = inds[t, slot]: the full-expert layer of
    rwkv_mlx/moe.py:218-234 on a given routing, its products in 8 bits.

    x (B, T, C); inds (B, T, k) int32, an id outside 0..E-1 is an unrouted
    slot; gates (B, T, k); x_k (E, C); key an Fp8Weight (E, F, C), value
    (E, C, F); x_prev (B, C) the token before x[:, 0] (default: zeros).  E up
    to 64, k up to 8, C a multiple of 4.  For inference: it has no gradient."""
    require_device(x, "fp8_experts")
    code = _code(x, "fp8_experts")
    if x.dim() != 3:
        raise ValueError(f"fp8_experts: x (B, T, C) expected, got {tuple(x.shape)}")
    B, T, C = x.shape
    if len(key.shape) != 3 or key.shape[2] != C or value.shape != (key.shape[0], C, key.shape[1]):
        raise ValueError(f"fp8_experts: key (E, F, {C}) and value (E, {C}, F) expected, got {key.shape} and "
                         f"{value.shape}")
    E, F, _ = key.shape
    if inds.dim() != 3 or inds.shape[:2] != (B, T) or gates.shape != inds.shape or inds.dtype != torch.int32:
        raise ValueError(f"fp8_experts: inds (B, T, k) int32 and gates of that shape expected, got "
                         f"{tuple(inds.shape)} {inds.dtype} and {tuple(gates.shape)}")
    if x_k.numel() != E * C:
        raise ValueError(f"fp8_experts: x_k ({E}, {C}) expected, got {tuple(x_k.shape)}")
    if x_prev is not None and x_prev.shape != (B, C):
        raise ValueError(f"fp8_experts: x_prev ({B}, {C}) expected, got {tuple(x_prev.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"fp8_experts: residual {tuple(x.shape)} expected, got {tuple(residual.shape)}")
    dev = x.device
    others = [t for t in (inds, gates, x_k, x_prev, residual) if t is not None]
    if any(t.device != dev for t in (*others, key, value)):
        raise ValueError(f"fp8_experts: every operand has to be on {dev}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, *others)):
        raise RuntimeError("fp8_experts has no gradient: call it under torch.no_grad(), or train with MoE_CMix")
    out = torch.empty(B, T, C, dtype=x.dtype, device=dev)
    cast = lambda t: None if t is None else t.to(x.dtype).contiguous()
    x, x_k, x_prev, residual = x.contiguous(), cast(x_k), cast(x_prev), cast(residual)
    inds, gates = inds.contiguous(), gates.to(torch.float32).contiguous()
    flags = (_lib.HAS_PREV if x_prev is not None else 0) | (_lib.ADD_RESIDUAL if residual is not None else 0)
    desc, nbytes = _lib.fp8_experts_plan(B, T, C, F, E, inds.shape[2], 1, code, 0, flags)
    if B * T == 0:
        return out
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    t = _lib.Fp8Experts(_lib.FP8_EXPERTS_SIZE, *map(_lib.ptr, (
        x, x_prev, x_k, key.q, key.scale, value.q, value.scale, inds, gates, residual, out)))
    _call("rwkvmoe_fp8_experts_forward", x, ctypes.byref(desc), ctypes.byref(t), ws.data_ptr(), nbytes)
    return out


class Fp8MoE_CMix(nn.Module):
    """``MoE_CMix`` (rwkv_mlx/moe.py:170-242) for inference, its experts held
    in 8 bits: half the bytes of a 16-bit layer.  ``router`` is the layer's
    ``Router`` or a ``GroupRouter``.  Made with ``from_moe``; the weights are
    buffers (q, scale), the layer is not trained."""

    def __init__(self, router: nn.Module, x_k: torch.Tensor, key: Fp8Weight, value: Fp8Weight):
        super().__init__()
        self.router = router
        self.register_buffer("x_k", x_k.detach())
        self.n_experts, self.top_k = key.shape[0], router.top_k
        self._shapes = (key.shape, value.shape)
        for name, w in (("key", key), ("value", value)):
            self.register_buffer(f"{name}_q", w.q)
            self.register_buffer(f"{name}_scale", w.scale)

    @classmethod
    def from_moe(cls, layer: nn.Module, router: nn.Module | None = None) -> "Fp8MoE_CMix":
        """From a ``MoE_CMix`` on the GPU; `router` replaces the layer's."""
        return cls(layer.router if router is None else router, layer.x_k.reshape(layer.n_experts, -1),
                   Fp8Weight.quantize(layer.expert_key), Fp8Weight.quantize(layer.expert_val))

    def _apply(self, fn, recurse=True):
        # a cast (.half(), .to(dtype), .type(dtype)) is for the router and x_k: the weights move, as they are
        was = {n: self._buffers[n] for n in ("key_q", "key_scale", "value_q", "value_scale")}
        super()._apply(fn, recurse)
        for n, t in was.items():
            if self._buffers[n].dtype != t.dtype:
                self._buffers[n] = t.to(self._buffers[n].device)
        return self

    def forward(self, x: torch.Tensor, x_prev: torch.Tensor | None = None, residual: torch.Tensor | None = None):
        """(out, aux_loss, z_loss), as MoE_CMix's forward."""
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, x_prev, residual)):
            raise RuntimeError("Fp8MoE_CMix has no gradient: call it under torch.no_grad(), or train with MoE_CMix")
        with torch.no_grad():
            inds, gates, aux, z = self.router(x)
            key = Fp8Weight(self._shapes[0], self.key_q, self.key_scale)
            value = Fp8Weight(self._shapes[1], self.value_q, self.value_scale)
            out = fp8_experts(x, inds, gates, self.x_k, key, value, x_prev=x_prev, residual=residual)
        return out, aux, z

    def orthogonal_loss(self) -> torch.Tensor:
        """No orthogonality loss for full experts (moe.py:240-242)."""
        return torch.zeros((), dtype=torch.float32, device=self.x_k.device)
