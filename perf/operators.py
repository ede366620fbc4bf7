"""What is timed of the framework's expert routing and of its 8-bit products:
the operators next to the ChannelMix layers that a model with many experts, or
one whose frozen weights are held in 8 bits, is served and trained with.

Kinds of case
  route    ``route_topk``: the experts and weights of every token from the
           router's logits (sigmoid or softmax scores, a balance bias that
           only selects, groups of experts, renormalised weights); with
           `train` its gradient as well
  linear   ``fp8_linear``: x (16-bit or fp32) is rounded to e4m3 with a scale
           for each 128 values of a row, and multiplied with a weight that is
           held in e4m3 with a scale for each 128 x 128 block; with `train` the
           weight is a parameter in the compute dtype, rounded in the call, and
           the gradients of x and of the weight are 8-bit products as well
  grouped  ``fp8_grouped_linear``: the same product for rows that are sorted by
           expert, each range with its expert's weight; with `train` the
           gradient of x (the weights are frozen)
  experts  ``fp8_experts``: a whole layer of ChannelMix experts on a given
           routing: token shift, key product, relu squared, value product,
           weighted sum

An 8-bit block: a = max |v|, at least 2^-100; q = e4m3(v * fp32(448 / a)); it
stands for q * fp32(a / 448).  Activations are N(0, 1) with a few channels
twenty times as large, weights N(0, 1/sqrt(fan_in)), routing is skewed.
"""
import math
import sys
from pathlib import Path

import torch

_PKG = str(Path(__file__).resolve().parent.parent / "rwkv-mlx_amd")

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 128
E4M3_MAX = 448.0
LEAST = 2.0 ** -100


def _route(name, rows, experts, k, groups, top_groups, score, bias, train, dtype="f32", masked=0.0):
    c = dict(kind="route", rows=rows, experts=experts, top_k=k, groups=groups, top_groups=top_groups, score=score,
             bias=bias, train=train, dtype=dtype, masked=masked)
    return dict(c, name=name) if name else c


def _linear(name, rows, n, k, dtype, train=False):
    c = dict(kind="linear", rows=rows, n=n, k=k, dtype=dtype, train=train)
    return dict(c, name=name) if name else c


def _grouped(name, rows, groups, n, k, dtype, train=False):
    c = dict(kind="grouped", rows=rows, groups=groups, n=n, k=k, dtype=dtype, train=train)
    return dict(c, name=name) if name else c


def _experts(name, batch, seq, d_model, d_ffn, experts, top_k, dtype, step=False):
    c = dict(kind="experts", batch=batch, seq=seq, d_model=d_model, d_ffn=d_ffn, experts=experts, top_k=top_k,
             dtype=dtype, step=step)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a server's decode step routes 16 tokens over many experts: latency
        _route("route-step-16", 16, 256, 8, 8, 4, "sigmoid", True, False),
        # prefill: groups of experts, the balance bias selects
        _route("route-prefill", 16384, 256, 8, 8, 4, "sigmoid", True, False),
        # a training step of a softmax router over the framework's largest expert count, a ragged batch
        _route("route-train-softmax", 8191, 64, 4, 1, 1, "softmax", False, True),
        # a long training batch with groups, some experts masked out per token
        _route("route-train-groups", 65536, 160, 6, 8, 3, "sigmoid", True, True, masked=0.2),
        # one generated token through the wide layer's key weight: the weight's bytes
        _linear("linear-1", 1, 8192, 2048, "bf16"),
        # an odd prefill with sizes that fill no block
        _linear("linear-ragged", 509, 2690, 1000, "f16"),
        # the wide layer's key product on a large batch
        _linear("linear-wide", 16384, 8192, 2048, "bf16"),
        # a training step of one projection: both gradients
        _linear("linear-train", 4096, 4096, 1024, "bf16", train=True),
        # decode: a few rows for each of the experts, some with none
        _grouped("grouped-24", 24, 16, 4096, 1024, "bf16"),
        # fine-tuning through frozen experts: a ragged, skewed batch and its gradient
        _grouped("grouped-train", 8191, 32, 4096, 1024, "bf16", train=True),
        # a decode step of a small expert layer (dim_ffn 3.5x, the framework's default)
        _experts("experts-step-8", 8, 1, 768, 2688, 8, 2, "f16", step=True),
        # prefill of prompts of an odd length through 32 experts
        _experts("experts-prefill", 12, 677, 1024, 4096, 32, 4, "bf16"),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["route", "route", "linear", "linear", "grouped", "experts"])
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8, 5])
        experts = groups * max(2, log(8, 320) // groups)
        top_groups = groups if groups == 1 else rng.randint(1, groups)
        k = rng.randint(1, min(8, top_groups * (experts // groups)))
        rows = log(1, max(2, min(65536, 65536 * 160 // experts)))
        return _route(None, rows, experts, k, groups, top_groups, rng.choice(["sigmoid", "softmax"]),
                      rng.random() < 0.5, rng.random() < 0.5, rng.choice(["f32", "f32", "bf16", "f16"]),
                      rng.choice([0.0, 0.0, 0.3, 0.9]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "experts":
        d = rng.choice([512, 640, 768, 1024, 1280])
        f = 32 * log(32, 128)
        step = rng.random() < 0.4
        k = rng.choice([1, 2, 3, 4])
        batch, seq = (log(1, 64), 1) if step else (rng.randint(1, 6), log(3, 1050))
        return _experts(None, batch, seq, d, f, rng.randint(k, 40), k, dtype, step)
    n, k = log(100, 8192), log(64, 4096)
    train = rng.random() < 0.4
    rows = log(1, max(2, min(16384, 16384 * 8192 * 2048 // (3 * n * k))))
    if kind == "linear":
        return _linear(None, rows, n, k, dtype, train)
    groups = rng.randint(1, 48)
    while groups * n * k > 1 << 28:
        groups = (groups + 1) // 2
    return _grouped(None, min(rows, 9000), groups, n, k, dtype, train)


# ---- inputs -----------------------------------------------------------------


def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + sum(ord(ch) * (i + 1) for i, ch in enumerate(case["kind"])))
    return g


def _activations(g, rows, cols, dtype):
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.randint(cols, (max(1, cols // 128),), generator=g, device="cuda")
    x[:, loud] *= 20.0
    return x.to(dtype)


def _held_weight(g, groups, n, k):
    """(groups, n, k) e4m3 values and their (groups, n / 128, k / 128) fp32
    scales, both rounded up, as a checkpoint holds them."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    q = torch.empty(groups, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(groups, nb, kb, device="cuda")
    for i in range(groups):
        w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
        w[:n, :k] = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        t = w.view(nb, BLOCK, kb, BLOCK)
        a = t.abs().amax((1, 3)).clamp_min(LEAST)
        scale[i] = a / E4M3_MAX
        q[i] = (t * (E4M3_MAX / a)[:, None, :, None]).to(torch.float8_e4m3fn).view_as(w)[:n, :k]
    return q, scale


def _popularity(g, n):
    """Zipf shares of n experts, in a random order."""
    p = (torch.arange(n, device="cuda") + 1.0) ** -1.0
    return p[torch.randperm(n, generator=g, device="cuda")] / p.sum()


def _inputs(case, seed):
    g = _generator(case, seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "route":
        R, E = case["rows"], case["experts"]
        logits = torch.randn(R, E, generator=g, device="cuda") * 1.5
        if case["masked"]:
            gone = torch.rand(R, E, generator=g, device="cuda") < case["masked"]
            logits = logits.masked_fill(gone, -math.inf)
        s = {"logits": logits.to(dt)}
        s["bias"] = torch.randn(E, generator=g, device="cuda") * 0.1 if case["bias"] else None
        if case["train"]:
            s["d_gates"] = torch.randn(R, case["top_k"], generator=g, device="cuda")
        return s
    if kind == "linear":
        R, N, K = case["rows"], case["n"], case["k"]
        s = {"x": _activations(g, R, K, dt)}
        if case["train"]:
            s["w"] = (torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)).to(dt)
            s["dy"] = _activations(g, R, N, dt)
        else:
            q, scale = _held_weight(g, 1, N, K)
            s["q"], s["scale"] = q[0], scale[0]
        return s
    if kind == "grouped":
        R, G, N, K = case["rows"], case["groups"], case["n"], case["k"]
        s = {"x": _activations(g, R, K, dt)}
        s["q"], s["scale"] = _held_weight(g, G, N, K)
        ids = torch.multinomial(_popularity(g, G), R, replacement=True, generator=g)
        counts = (ids[:, None] == torch.arange(G, device="cuda")).sum(0)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        if case["train"]:
            s["dy"] = _activations(g, R, N, dt)
        return s
    B, T, C, F, E, k = (case[n] for n in ("batch", "seq", "d_model", "d_ffn", "experts", "top_k"))
    s = {"x": _activations(g, B * T, C, dt).view(B, T, C)}
    s["x_k"] = torch.rand(E, C, generator=g, device="cuda").to(dt)
    s["x_prev"] = _activations(g, B, C, dt) if case["step"] else None
    s["key"] = _held_weight(g, E, F, C)
    s["value"] = _held_weight(g, E, C, F)
    share = torch.rand(B * T, E, generator=g, device="cuda").log() / _popularity(g, E)  # (Gumbel-like draw)
    s["inds"] = share.sort(-1, descending=True).indices[:, :k].to(torch.int32).view(B, T, k).contiguous()
    s["gates"] = torch.randn(B, T, k, generator=g, device="cuda").softmax(-1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    state = {"case": case, **s}
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import rwkv_mlx_amd as R
        state["R"] = R
        # weights of a checkpoint, laid out once; fine-tuning also reads them transposed
        if "q" in s:
            state["weight"] = R.Fp8Weight.from_quantized(s["q"], s["scale"], transposed=case["train"])
        if case["kind"] == "experts":
            for n in ("key", "value"):
                state[n] = R.Fp8Weight.from_quantized(*s[n])
        for n in ("logits", "x", "w"):
            if n in s and case.get("train"):
                state[n] = s[n].requires_grad_(True)
    return state


# ---- the framework's operators ------------------------------------------------


def _run_own(s):
    c, R = s["case"], s["R"]
    kind = c["kind"]
    if kind == "route":
        inds, gates = R.route_topk(s["logits"], c["top_k"], bias=s["bias"], score=c["score"], n_groups=c["groups"],
                                   top_groups=c["top_groups"], group_score="top2", scale=2.5)
        if not c["train"]:
            return inds, gates
        (d_logits,) = torch.autograd.grad(gates, s["logits"], s["d_gates"])
        return inds, gates.detach(), d_logits
    if kind == "linear":
        if not c["train"]:
            return R.fp8_linear(s["x"], s["weight"])
        y = R.fp8_linear(s["x"], s["w"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return y.detach(), dx, dw
    if kind == "grouped":
        y = R.fp8_grouped_linear(s["x"], s["weight"], s["offsets"])
        if not c["train"]:
            return y
        (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
        return y.detach(), dx
    return R.fp8_experts(s["x"], s["inds"], s["gates"], s["x_k"], s["key"], s["value"], x_prev=s["x_prev"])


# ---- the plain form -----------------------------------------------------------


def _blocks(v, rows):
    """v (R, K) fp32, rounded to e4m3 in blocks of `rows` x 128 and back."""
    R, K = v.shape
    Rp, Kp = -(-R // rows) * rows, -(-K // BLOCK) * BLOCK
    t = torch.nn.functional.pad(v, (0, Kp - K, 0, Rp - R)).view(Rp // rows, rows, Kp // BLOCK, BLOCK)
    a = t.abs().amax((1, 3), keepdim=True).clamp_min(LEAST)
    q = (t * (E4M3_MAX / a)).to(torch.float8_e4m3fn).to(torch.float32)
    return (q * (a / E4M3_MAX)).view(Rp, Kp)[:R, :K]


def _held(q, scale):
    """What a weight held as e4m3 values and block scales stands for, fp32."""
    s = scale.repeat_interleave(BLOCK, 0)[: q.shape[0]].repeat_interleave(BLOCK, 1)[:, : q.shape[1]]
    return q.to(torch.float32) * s


def _plain_route(s):
    # in 64 bits: which expert is taken hangs on scores that lie close together
    c = s["case"]
    E, G, k = c["experts"], c["groups"], c["top_k"]
    l = s["logits"].to(torch.float64)
    gone = torch.isinf(l) & (l < 0)
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-l))
    else:
        top = l.amax(-1, keepdim=True)
        ex = torch.exp(l - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = ex.sum(-1, keepdim=True)
        score = ex / torch.where(total == 0, torch.ones_like(total), total)
    key = l if s["bias"] is None else score + s["bias"].to(torch.float64)
    key = key.masked_fill(gone, -math.inf)
    out = torch.zeros_like(gone)
    if G > 1:
        # a group counts as the sum of its two best experts that are left
        ranked = score if s["bias"] is None else score + s["bias"].to(torch.float64)
        two = ranked.masked_fill(gone, -math.inf).view(-1, G, E // G).sort(-1, descending=True).values[..., :2]
        best = torch.where(torch.isinf(two), torch.zeros_like(two), two).sum(-1)
        best = torch.where(torch.isinf(two[..., 0]), two[..., 0], best)
        groups = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter(-1, groups, True)
        out = ~keep.repeat_interleave(E // G, -1)
    # experts of other groups come after masked ones of the chosen groups
    rank = torch.where(torch.isinf(key), torch.full_like(key, -1e300), key)
    rank = rank.masked_fill(out, -math.inf)
    inds = rank.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    taken = score.gather(-1, inds).masked_fill(torch.isinf(key.gather(-1, inds)), 0.0)
    total = taken.sum(-1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    gates = taken / total * 2.5
    res = (inds.to(torch.int32), gates.to(torch.float32))
    if not c["train"]:
        return res
    dg = s["d_gates"].to(torch.float64) * 2.5 / total
    dg = dg - (dg * taken).sum(-1, keepdim=True) / total
    if c["score"] == "sigmoid":
        d = dg * taken * (1.0 - taken)
    else:  # (the sum over the softmax's other entries vanishes with the renormalisation)
        d = dg * taken
    return (*res, torch.zeros_like(l).scatter(-1, inds, d).to(s["logits"].dtype))


def _plain_linear(s):
    c = s["case"]
    x = s["x"].detach()
    xf = _blocks(x.to(torch.float32), 1)
    if not c["train"]:
        return (xf @ _held(s["q"], s["scale"]).t()).to(x.dtype)
    w = _blocks(s["w"].to(torch.float32), BLOCK)
    dy = s["dy"].to(torch.float32)
    y = (xf @ w.t()).to(x.dtype)
    dx = (_blocks(dy, 1) @ w).to(x.dtype)
    # both operands of the weight's gradient are rounded along the rows, over which it sums
    dw = (_blocks(dy.t(), 1) @ _blocks(x.to(torch.float32).t(), 1).t()).to(x.dtype)
    return y, dx, dw


def _plain_grouped(s):
    c = s["case"]
    x = s["x"].detach()
    xf = _blocks(x.to(torch.float32), 1)
    dyf = _blocks(s["dy"].to(torch.float32), 1) if c["train"] else None
    y = torch.empty(c["rows"], c["n"], dtype=x.dtype, device=x.device)
    dx = torch.empty_like(x)
    off = s["offsets"].tolist()
    for g in range(c["groups"]):
        a, b = off[g], off[g + 1]
        if a == b:
            continue
        w = _held(s["q"][g], s["scale"][g])
        y[a:b] = (xf[a:b] @ w.t()).to(x.dtype)
        if c["train"]:
            dx[a:b] = (dyf[a:b] @ w).to(x.dtype)
    return (y, dx) if c["train"] else y


def _plain_experts(s):
    c = s["case"]
    B, T, C, E, k = (c[n] for n in ("batch", "seq", "d_model", "experts", "top_k"))
    x = s["x"].to(torch.float32)
    first = torch.zeros(B, 1, C, device=x.device) if s["x_prev"] is None else s["x_prev"].to(torch.float32)[:, None]
    diff = (torch.cat([first, x[:, :-1]], 1) - x).view(B * T, C)
    x = x.view(B * T, C)
    inds = s["inds"].view(B * T, k)
    out = torch.zeros(B * T, C, device=x.device)
    for e in range(E):
        t, slot = (inds == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        mixed = x[t] + diff[t] * s["x_k"][e].to(torch.float32)
        h = _blocks(mixed, 1) @ _held(s["key"][0][e], s["key"][1][e]).t()
        h = torch.where(h > 0, h, torch.zeros_like(h))
        y = _blocks(h * h, 1) @ _held(s["value"][0][e], s["value"][1][e]).t()
        out[t] += y * s["gates"].view(B * T, k)[t, slot][:, None]
    return out.to(s["x"].dtype).view(B, T, C)


_PLAIN = {"route": _plain_route, "linear": _plain_linear, "grouped": _plain_grouped, "experts": _plain_experts}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    kind = case["kind"]
    size = DTYPES[case["dtype"]].itemsize
    if kind == "route":
        R, E, k = case["rows"], case["experts"], case["top_k"]
        nbytes = R * E * size + R * k * 8 + (4 * E if case["bias"] else 0)
        if case["train"]:  # the cotangent, and the logits' gradient
            nbytes += R * k * 4 + R * E * size
        return {"bytes": nbytes, "flops": R * E * (3 if case["train"] else 2)}
    if kind == "experts":
        N, C, F, E, k = case["batch"] * case["seq"], *(case[n] for n in ("d_model", "d_ffn", "experts", "top_k"))
        used = min(E, N * k)
        nbytes = 2 * N * C * size + (case["batch"] * C * size if case["step"] else 0) + 8 * N * k
        nbytes += used * (2 * F * C + C * size + 8 * -(-F // BLOCK) * -(-C // BLOCK))
        return {"bytes": nbytes, "flops": 4 * N * k * C * F}
    R, N, K = case["rows"], case["n"], case["k"]
    scales = 4 * -(-N // BLOCK) * -(-K // BLOCK)
    if kind == "linear":
        if case["train"]:  # x, w, dy read; y, dx, dw written
            return {"bytes": 2 * size * (R * K + R * N + N * K), "flops": 6 * R * N * K}
        return {"bytes": size * (R * K + R * N) + N * K + scales, "flops": 2 * R * N * K}
    used = min(case["groups"], R)
    nbytes = size * (R * K + R * N) + used * (N * K + scales) + 4 * (case["groups"] + 1)
    if case["train"]:
        nbytes += size * (R * K + R * N)
    return {"bytes": nbytes, "flops": (4 if case["train"] else 2) * R * N * K}


# ---- the definition in 64 bits --------------------------------------------------


def _e4m3(v):
    """Round to the nearest e4m3 value, ties to even (|v| < 464), in 64 bits."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    e = torch.where(v.abs() < torch.exp2(e), (e - 1).clamp_min(-6.0), e)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _exact_rows(v, transpose=False):
    """What v (fp32 values) stands for after blocks of 128 along its last axis
    (along its first with `transpose`), 64 bits.  A block's two factors are
    fp32 numbers by definition, and so is a value times its factor."""
    v = v.t() if transpose else v
    out = torch.empty(v.shape, dtype=torch.float64, device=v.device)
    for i in range(0, v.shape[1], BLOCK):
        b = v[:, i:i + BLOCK].to(torch.float32)
        a = b.to(torch.float64).abs().max(1, keepdim=True).values.clamp(min=LEAST)
        up, down = (E4M3_MAX / a).to(torch.float32), (a / E4M3_MAX).to(torch.float32)
        out[:, i:i + BLOCK] = _e4m3((b * up).to(torch.float64)) * down.to(torch.float64)
    return out.t() if transpose else out


def _exact_weight(q, scale):
    w = q.to(torch.float32).to(torch.float64)
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[i, j].to(torch.float64)
    return w


def _exact_route(case, s):
    E, G, k = case["experts"], case["groups"], case["top_k"]
    l = s["logits"].to(torch.float64)
    live = l > -math.inf
    l = l.clone().requires_grad_(case["train"])
    with torch.enable_grad():
        safe = torch.where(live, l, torch.full_like(l, -1e4))
        score = torch.sigmoid(safe) if case["score"] == "sigmoid" else torch.softmax(safe, -1)
        score = score * live
    with torch.no_grad():
        b = 0.0 if s["bias"] is None else s["bias"].to(torch.float64)
        order = s["logits"].to(torch.float64) if s["bias"] is None else score + b
        ok = torch.ones_like(live)
        if G > 1:
            v = (score + b).view(-1, G, E // G)
            lv = live.view(-1, G, E // G)
            one = torch.where(lv, v, torch.full_like(v, -math.inf)).max(-1)
            rest = lv.scatter(-1, one.indices[..., None], False)
            two = torch.where(rest, v, torch.full_like(v, -math.inf)).amax(-1)
            gs = torch.where(lv.any(-1), one.values + torch.where(rest.any(-1), two, torch.zeros_like(two)),
                             torch.full_like(two, -math.inf))
            # place of each group: how many are above it, or equal and before it
            above = (gs[:, None, :] > gs[:, :, None]) | (
                (gs[:, None, :] == gs[:, :, None])
                & (torch.arange(G, device=gs.device)[None, :] < torch.arange(G, device=gs.device)[:, None]))
            ok = (above.sum(-1) < case["top_groups"]).repeat_interleave(E // G, -1)
        picks = []
        at = torch.arange(E, device=l.device, dtype=torch.float64)
        for _ in range(k):  # the largest that is left; masked ones after all others; the lowest index of equals
            best = torch.where(ok & live, order, torch.full_like(order, -math.inf)).amax(-1, keepdim=True)
            cand = torch.where(torch.isinf(best) & (best < 0), ok, ok & live & (order == best))
            i = torch.where(cand, at, torch.full_like(order, 1e9)).amin(-1).long()
            picks.append(i)
            ok = ok.scatter(-1, i[:, None], False)
        inds = torch.stack(picks, -1)
    with torch.enable_grad():
        taken = score.gather(-1, inds)
        total = taken.sum(-1, keepdim=True)
        gates = 2.5 * taken / torch.where(total > 0, total, torch.ones_like(total))
    res = (inds.to(torch.int32), gates.detach())
    if not case["train"]:
        return res
    (d,) = torch.autograd.grad(gates, l, s["d_gates"].to(torch.float64))
    return (*res, d)


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(case, s)
    if kind == "linear":
        x = _exact_rows(s["x"])
        if not case["train"]:
            return x @ _exact_weight(s["q"], s["scale"]).t()
        N, K = s["w"].shape
        w = torch.empty(N, K, dtype=torch.float64, device="cuda")
        for i in range(0, N, BLOCK):  # a 128 x 128 block as one row of values
            for j in range(0, K, BLOCK):
                t = s["w"][i:i + BLOCK, j:j + BLOCK].to(torch.float32)
                a = t.to(torch.float64).abs().max().clamp(min=LEAST)
                up, down = (E4M3_MAX / a).to(torch.float32), (a / E4M3_MAX).to(torch.float32)
                w[i:i + BLOCK, j:j + BLOCK] = _e4m3((t * up).to(torch.float64)) * down.to(torch.float64)
        y = x @ w.t()
        dx = _exact_rows(s["dy"]) @ w
        dw = _exact_rows(s["dy"], True).t() @ _exact_rows(s["x"], True)
        return y, dx, dw
    if kind == "grouped":
        x = _exact_rows(s["x"])
        dy = _exact_rows(s["dy"]) if case["train"] else None
        y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        dx = torch.empty(case["rows"], case["k"], dtype=torch.float64, device="cuda")
        start = 0
        for g in range(case["groups"]):
            end = int(s["offsets"][g + 1])
            if end > start:
                w = _exact_weight(s["q"][g], s["scale"][g])
                y[start:end] = x[start:end] @ w.t()
                if case["train"]:
                    dx[start:end] = dy[start:end] @ w
            start = end
        return (y, dx) if case["train"] else y
    B, T, C, E, k = (case[n] for n in ("batch", "seq", "d_model", "experts", "top_k"))
    x = s["x"].to(torch.float32)
    prev = torch.zeros_like(x)
    prev[:, 1:] = x[:, :-1]
    if s["x_prev"] is not None:
        prev[:, 0] = s["x_prev"].to(torch.float32)
    x, prev = x.reshape(-1, C), prev.reshape(-1, C)
    flat, gates = s["inds"].reshape(-1).long(), s["gates"].reshape(-1).to(torch.float64)
    out = torch.zeros(B * T, C, dtype=torch.float64, device="cuda")
    for e in range(E):
        a = torch.nonzero(flat == e)[:, 0]
        if a.numel() == 0:
            continue
        t = a // k
        # the mix is an fp32 value by definition (it is rounded to e4m3 next), and so is the hidden one
        mixed = x[t] + (prev[t] - x[t]) * s["x_k"][e].to(torch.float32)
        h = (_exact_rows(mixed) @ _exact_weight(s["key"][0][e], s["key"][1][e]).t()).clamp(min=0.0) ** 2
        y = _exact_rows(h.to(torch.float32)) @ _exact_weight(s["value"][0][e], s["value"][1][e]).t()
        out.index_add_(0, t, y * gates[a, None])
    return out.view(B, T, C)
