"""Cases, plain forms and 64-bit definitions of the feed-forward operators.

The operators: products with 4-bit weights and group scales (``linear``, with a
residual, and ``swiglu``, gate and up rows with the activation), the same over
tokens sorted by expert (``experts``), the router's top-k with the sort of the
tokens by expert (``route``), and the way of the tokens to their experts and
back with the router's weights (``dispatch``, ``combine``), forward and, with
``train``, with their gradients.

A 4-bit matrix [n, k] is int32 ``codes`` [n, k / 8], ``scales`` [n, k / group]
and optionally uint8 ``zeros`` [n, k / group] (8 without them): weight
(q - zero) * scale.  A word holds eight consecutive weights; the even ones sit
in bits 0, 4, 8, 12 and the odd ones in bits 16, 20, 24, 28.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # The attention output product of one drafting row (16 heads of 128, width 2048), residual added.
        {"name": "linear_draft_1", "op": "linear", "tokens": 1, "k": 2048, "n": 2048, "group": 128, "zeros": False,
         "residual": True, "dtype": "bf16"},
        # The vocabulary head of one row: the largest single matrix a decode step reads.
        {"name": "linear_head_1", "op": "linear", "tokens": 1, "k": 4096, "n": 151936, "group": 128, "zeros": False,
         "residual": False, "dtype": "bf16"},
        # The down product of one verifying row with 8 drafts, finer groups with zero points.
        {"name": "linear_verify_9", "op": "linear", "tokens": 9, "k": 12288, "n": 4096, "group": 64, "zeros": True,
         "residual": True, "dtype": "bf16"},
        # Gate and up products of a decode step of 64 rows.
        {"name": "swiglu_batch_64", "op": "swiglu", "tokens": 64, "k": 4096, "n": 12288, "group": 128, "zeros": False,
         "residual": False, "dtype": "bf16"},
        # A ragged prefill chunk, fp16, the finest groups.
        {"name": "linear_prefill_4099", "op": "linear", "tokens": 4099, "k": 4096, "n": 12288, "group": 32,
         "zeros": True, "residual": False, "dtype": "f16"},
        # A decode step of 64 rows over 128 narrow experts, 8 per token: about 4 rows an expert.
        {"name": "experts_decode_64", "op": "experts", "tokens": 64, "experts": 128, "top_k": 8, "k": 2048, "n": 768,
         "group": 128, "zeros": False, "swiglu": True, "dtype": "bf16", "pad": 0},
        # The experts' down product of a prefill chunk.
        {"name": "experts_prefill_2050", "op": "experts", "tokens": 2050, "experts": 64, "top_k": 6, "k": 1536,
         "n": 2048, "group": 64, "zeros": False, "swiglu": False, "dtype": "bf16", "pad": 0},
        # Routing of a decode bucket whose last rows are padding (no expert).
        {"name": "route_decode_72", "op": "route", "tokens": 72, "experts": 128, "top_k": 8, "renormalize": True,
         "logits": "f32", "pad": 5, "train": False},
        # Routing of a training batch, with the gradient to the router's logits.
        {"name": "route_train_8192", "op": "route", "tokens": 8192, "experts": 128, "top_k": 8, "renormalize": True,
         "logits": "f32", "pad": 0, "train": True},
        # Tokens to their experts in a training batch and the gradient back.
        {"name": "dispatch_train_8192", "op": "dispatch", "tokens": 8192, "experts": 128, "top_k": 8, "width": 2048,
         "dtype": "bf16", "pad": 0, "train": True},
        # The experts' outputs of a decode step summed with their weights onto the residual.
        {"name": "combine_decode_64", "op": "combine", "tokens": 64, "experts": 128, "top_k": 8, "width": 2048,
         "dtype": "bf16", "pad": 3, "residual": True, "train": False},
        # The same in training, odd sizes, with the gradients of the experts' outputs and of the weights.
        {"name": "combine_train_4099", "op": "combine", "tokens": 4099, "experts": 60, "top_k": 4, "width": 4096,
         "dtype": "bf16", "pad": 0, "residual": False, "train": True},
    ]


MOST_BYTES = 300e6
MOST_FLOPS = 400e9


def draw(rng):
    def spread(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(lo, min(hi, int(round(v / step)) * step))

    op = rng.choice(["linear", "linear", "swiglu", "experts", "experts", "route", "dispatch", "combine"])
    while True:
        if op in ("linear", "swiglu"):
            group = rng.choice([32, 64, 128])
            case = {"op": op, "tokens": spread(1, 4096), "k": spread(512, 14336, group), "n": spread(256, 16384),
                    "group": group, "zeros": rng.random() < 0.4, "residual": op == "linear" and rng.random() < 0.5,
                    "dtype": rng.choice(["bf16", "bf16", "f16"])}
        elif op == "experts":
            group = rng.choice([32, 64, 128])
            experts = rng.choice([8, 16, 60, 64, 128, 160])
            case = {"op": op, "tokens": spread(1, 2048), "experts": experts,
                    "top_k": rng.randint(1, min(8, experts)), "k": spread(512, 4096, group),
                    "n": spread(256, 2048, 8), "group": group, "zeros": rng.random() < 0.4,
                    "swiglu": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "f16"]), "pad": 0}
            case["pad"] = rng.choice([0, 0, case["tokens"] // 8])
        else:
            experts = rng.choice([8, 16, 60, 64, 128, 160, 256])
            case = {"op": op, "tokens": spread(1, 8192), "experts": experts,
                    "top_k": rng.randint(1, min(8, experts))}
            case["pad"] = rng.choice([0, 0, case["tokens"] // 8])
            if op == "route":
                case.update(renormalize=rng.random() < 0.6, logits=rng.choice(["f32", "f32", "bf16"]))
            else:
                case.update(width=spread(256, 7168, 8), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
                if op == "combine":
                    case["residual"] = rng.random() < 0.5
            case["train"] = rng.random() < 0.5
        w = work(case)
        rows = case.get("experts", 1) * case["n"] * case["k"] if op == "experts" else 0
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and rows <= 300e6:
            return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _matrix(g, lead, n, k, group, zeros, dtype):
    """Random codes of a bell shape, scales of a trained matrix (rms of a weight about 0.02) and zero points around 8."""
    words = torch.zeros(*lead, n, k // 8, dtype=torch.int32, device="cuda")
    for i in range(8):
        q = torch.randn(*lead, n, k // 8, generator=g, device="cuda").mul_(2.7).round_().add_(8).clamp_(0, 15)
        words |= q.to(torch.int32) << (4 * (i // 2) + 16 * (i % 2))
    scales = (torch.rand(*lead, n, k // group, generator=g, device="cuda") + 0.5) * (0.02 / 2.7)
    z = None
    if zeros:
        z = torch.randint(6, 11, (*lead, n, k // group), generator=g, device="cuda").to(torch.uint8)
    return words, scales.to(dtype), z


def _logits(g, case):
    """Router logits: some experts are liked by most tokens; padding rows have no expert (-inf)."""
    t, e = case["tokens"], case["experts"]
    x = torch.randn(t, e, generator=g, device="cuda") + 0.7 * torch.randn(e, generator=g, device="cuda")
    if case["pad"]:
        x[t - case["pad"]:] = -math.inf
    return x


def _choose(logits, top_k):
    """Chosen experts [t, k] (-1: none): the largest logits, ties to the lowest index."""
    x = torch.where(logits != logits, -math.inf, logits.float())
    v, e = torch.sort(x, dim=1, descending=True, stable=True)
    v, e = v[:, :top_k], e[:, :top_k]
    return torch.where(v == -math.inf, -1, e).to(torch.int32)


def _sort(chosen, experts):
    """position [t, k] (-1: none), source [t k] (-1 past the last row) and offsets [e + 1] of the stable sort by expert."""
    flat = chosen.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=key.device)
    offsets[1:] = counts.cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=key.device)
    position = torch.where(flat < 0, -1, place).to(torch.int32).view(chosen.shape)
    source = torch.where(torch.arange(order.numel(), device=key.device) < offsets[-1], order, -1).to(torch.int32)
    return position, source, offsets


def prepare(case, seed):
    g = _gen(seed)
    op, t = case["op"], case["tokens"]
    s = {"case": case}
    if op in ("linear", "swiglu"):
        dt = DTYPES[case["dtype"]]
        rows = case["n"] * (2 if op == "swiglu" else 1)
        s["codes"], s["scales"], s["zeros"] = _matrix(g, (), rows, case["k"], case["group"], case["zeros"], dt)
        s["x"] = torch.randn(t, case["k"], generator=g, device="cuda").to(dt)
        s["residual"] = torch.randn(t, case["n"], generator=g, device="cuda").to(dt) if case["residual"] else None
        return s
    logits = _logits(g, case)
    if op == "route":
        s["logits"] = logits.to(DTYPES[case["logits"]]).requires_grad_(case["train"])
        s["grad"] = torch.randn(t, case["top_k"], generator=g, device="cuda") if case["train"] else None
        return s
    dt = DTYPES[case["dtype"]]
    chosen = _choose(logits, case["top_k"])
    s["position"], s["source"], s["offsets"] = _sort(chosen, case["experts"])
    total = t * case["top_k"]
    if op == "experts":
        rows = case["n"] * (2 if case["swiglu"] else 1)
        s["codes"], s["scales"], s["zeros"] = _matrix(g, (case["experts"],), rows, case["k"], case["group"],
                                                      case["zeros"], dt)
        x = torch.randn(t, case["k"], generator=g, device="cuda").to(dt)
        s["x"] = torch.where(s["source"][:, None] >= 0, x[(s["source"].long() // case["top_k"]).clamp(min=0)], 0)
        # The longest expert's rows: the plain form's batched product needs it as a size.
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        return s
    s["weights"] = torch.rand(t, case["top_k"], generator=g, device="cuda").add_(0.05)
    s["weights"] /= s["weights"].sum(1, keepdim=True)
    if op == "dispatch":
        s["x"] = torch.randn(t, case["width"], generator=g, device="cuda").to(dt).requires_grad_(case["train"])
        s["grad"] = torch.randn(total, case["width"], generator=g, device="cuda").to(dt) if case["train"] else None
        return s
    s["y"] = torch.randn(total, case["width"], generator=g, device="cuda").to(dt).requires_grad_(case["train"])
    s["weights"].requires_grad_(case["train"])
    s["residual"] = None
    if case["residual"]:
        s["residual"] = torch.randn(t, case["width"], generator=g, device="cuda").to(dt)
    s["grad"] = torch.randn(t, case["width"], generator=g, device="cuda").to(dt) if case["train"] else None
    return s


# -------------------------------------------------------------- plain form
def _unpack(codes, scales, zeros):
    """The weights in 32 bits [..., n, k]."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=codes.device, dtype=torch.int32)
    q = ((codes[..., None] >> shift) & 15).flatten(-2).float()
    group = q.shape[-1] // scales.shape[-1]
    q = q.unflatten(-1, (-1, group)) - (8.0 if zeros is None else zeros[..., None].float())
    return (q * scales[..., None].float()).flatten(-2)


def _silu_mul(g):
    a, b = g.chunk(2, dim=-1)
    return a / (1 + torch.exp(-a)) * b


def _plain_experts(s):
    case = s["case"]
    w = _unpack(s["codes"], s["scales"], s["zeros"])
    slot = torch.arange(s["most"], device="cuda")
    row = s["offsets"][:-1, None] + slot
    live = row < s["offsets"][1:, None]
    row = torch.where(live, row, 0).long()
    y = torch.bmm(s["x"].float()[row], w.transpose(1, 2))
    if case["swiglu"]:
        y = _silu_mul(y)
    out = torch.zeros(s["x"].shape[0] + 1, y.shape[-1], device="cuda")
    out[torch.where(live, row, s["x"].shape[0])] = y
    return out[:-1].to(s["x"].dtype)


def _plain(s):
    case = s["case"]
    op = case["op"]
    with torch.no_grad():
        if op in ("linear", "swiglu"):
            y = s["x"].float() @ _unpack(s["codes"], s["scales"], s["zeros"]).t()
            if op == "swiglu":
                y = _silu_mul(y)
            if s["residual"] is not None:
                y = y + s["residual"].float()
            return y.to(s["x"].dtype)
        if op == "experts":
            return _plain_experts(s)
        k = case["top_k"]
        if op == "route":
            x = s["logits"].float()
            chosen = _choose(x, k)
            at = chosen.clamp(min=0).long()
            live = chosen >= 0
            top = torch.where(live, x.gather(1, at), -math.inf)
            big = x.amax(1, keepdim=True)
            big = torch.where(big == -math.inf, 0, big)
            e = torch.exp(top - big)
            full = torch.exp(x - big)
            total = (e if case["renormalize"] else full).sum(1, keepdim=True)
            w = torch.where(live, e / torch.where(total > 0, total, 1), 0)
            position, source, offsets = _sort(chosen, case["experts"])
            out = {"weights": w, "experts": chosen, "position": position, "source": source, "offsets": offsets}
            if case["train"]:
                g = torch.where(live, s["grad"], 0)
                inner = (w * g).sum(1, keepdim=True)
                if case["renormalize"]:
                    d = torch.zeros_like(x)
                else:
                    d = -full / torch.where(total > 0, total, 1) * inner
                d = d.scatter_add(1, at, w * (g - inner) if case["renormalize"] else w * g)
                out["grad_logits"] = d.to(s["logits"].dtype)
            return out
        pos = s["position"].long()
        live = (pos >= 0)[..., None]
        src = s["source"].long()
        if op == "dispatch":
            out = {"y": torch.where(src[:, None] >= 0, s["x"][src.clamp(min=0) // k], 0)}
            if case["train"]:
                out["grad_x"] = torch.where(live, s["grad"].float()[pos.clamp(min=0)], 0).sum(1).to(s["x"].dtype)
            return out
        rows = torch.where(live, s["y"].float()[pos.clamp(min=0)], 0)
        y = (rows * s["weights"][..., None]).sum(1)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        out = {"y": y.to(s["y"].dtype)}
        if case["train"]:
            g = s["grad"].float()
            out["grad_weights"] = (rows * g[:, None, :]).sum(2)
            at = src.clamp(min=0)
            scaled = g[at // k] * s["weights"].reshape(-1)[at][:, None]
            out["grad_y"] = torch.where(src[:, None] >= 0, scaled, 0).to(s["y"].dtype)
        return out


# ------------------------------------------------------------- the calls
def _routing(s):
    from aspire_b200.moe import ExpertOrder

    return ExpertOrder(s["position"], s["source"], s["offsets"])


def _own(s):
    from aspire_b200 import moe, quant

    case = s["case"]
    op = case["op"]
    if op == "linear":
        return quant.w4_linear(s["x"], s["codes"], s["scales"], s["zeros"], residual=s["residual"])
    if op == "swiglu":
        return quant.w4_swiglu(s["x"], s["codes"], s["scales"], s["zeros"])
    if op == "experts":
        call = quant.w4_expert_swiglu if case["swiglu"] else quant.w4_expert_linear
        return call(s["x"], s["offsets"], s["codes"], s["scales"], s["zeros"])
    if op == "route":
        weights, experts, order = moe.moe_route(s["logits"], case["top_k"], renormalize=case["renormalize"])
        out = {"weights": weights.detach(), "experts": experts, "position": order.position, "source": order.source,
               "offsets": order.offsets}
        if case["train"]:
            out["grad_logits"] = torch.autograd.grad(weights, s["logits"], s["grad"])[0]
        return out
    if op == "dispatch":
        y = moe.moe_dispatch(s["x"], _routing(s))
        out = {"y": y.detach()}
        if case["train"]:
            out["grad_x"] = torch.autograd.grad(y, s["x"], s["grad"])[0]
        return out
    y = moe.moe_combine(s["y"], s["weights"], _routing(s), residual=s["residual"])
    out = {"y": y.detach()}
    if case["train"]:
        out["grad_y"], out["grad_weights"] = torch.autograd.grad(y, (s["y"], s["weights"]), s["grad"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------- work
def work(case):
    op, t = case["op"], case["tokens"]
    if op == "route":
        e, k = case["experts"], case["top_k"]
        size = 4 if case["logits"] == "f32" else 2
        b = t * e * size + t * k * (4 + 4 + 4 + 4) + 4 * (e + 1)
        if case["train"]:
            b += t * k * 4 + t * e * size
        return {"bytes": b, "flops": t * e * (6 if case["train"] else 4)}
    size = 4 if case["dtype"] == "f32" else 2
    if op in ("linear", "swiglu", "experts"):
        gated = op == "swiglu" or case.get("swiglu", False)
        rows = case["n"] * (2 if gated else 1)
        per = rows * case["k"] / 2 + rows * (case["k"] // case["group"]) * (3 if case["zeros"] else 2)
        m, count = t, 1
        if op == "experts":
            m = (t - case["pad"]) * case["top_k"]
            count = min(case["experts"], m)
        b = count * per + m * case["k"] * size + m * case["n"] * size * (2 if case.get("residual") else 1)
        return {"bytes": b, "flops": 2.0 * m * rows * case["k"]}
    k, d = case["top_k"], case["width"]
    live = (t - case["pad"]) * k
    if op == "dispatch":
        b = t * d * size + t * k * d * size + t * k * 8
        if case["train"]:
            b += live * d * size + t * d * size
        return {"bytes": b, "flops": live * d if case["train"] else 0}
    b = live * d * size + t * d * size * (2 if case["residual"] else 1) + t * k * 8
    f = 2.0 * live * d
    if case["train"]:
        # The gradients read the outputs' gradient and the experts' outputs once more and write theirs.
        b += t * d * size + live * d * size + t * k * d * size + t * k * 8
        f += 3.0 * live * d
    return {"bytes": b, "flops": f}


# ------------------------------------------------- the definition in 64 bits
def _exact_weight(codes, scales, zeros):
    """[..., n, k] in 64 bits, one weight of every eight at a time."""
    k = codes.shape[-1] * 8
    w = torch.empty(*codes.shape[:-1], k, dtype=torch.float64, device=codes.device)
    for i in range(8):
        w[..., i::8] = ((codes >> (4 * (i // 2) + 16 * (i % 2))) & 15).double()
    group = k // scales.shape[-1]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, -1)
    return (w - z).mul_(scales.double().repeat_interleave(group, -1))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op in ("linear", "swiglu"):
            x = s["x"].double()
            parts = []
            for at in range(0, s["codes"].shape[0], 8192):
                to = slice(at, at + 8192)
                w = _exact_weight(s["codes"][to], s["scales"][to], None if s["zeros"] is None else s["zeros"][to])
                parts.append(torch.matmul(w, x.t()))
            y = torch.cat(parts).t()
            if op == "swiglu":
                a = y[:, :case["n"]]
                y = a * torch.sigmoid(a) * y[:, case["n"]:]
            return y if s["residual"] is None else y + s["residual"].double()
        if op == "experts":
            ends = s["offsets"].tolist()
            y = torch.zeros(s["x"].shape[0], case["n"], dtype=torch.float64, device="cuda")
            for e in range(case["experts"]):
                if ends[e] == ends[e + 1]:
                    continue
                w = _exact_weight(s["codes"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e])
                o = s["x"][ends[e]:ends[e + 1]].double() @ w.t()
                if case["swiglu"]:
                    a = o[:, :case["n"]]
                    o = a * torch.sigmoid(a) * o[:, case["n"]:]
                y[ends[e]:ends[e + 1]] = o
            return y
        k, t = case["top_k"], case["tokens"]
        if op == "route":
            x = s["logits"].detach().double()
            live_rows = t - case["pad"]
            x = x[:live_rows]
            at = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
            v = x.gather(1, at)
            p = torch.softmax(x, 1)
            w = torch.softmax(v, 1) if case["renormalize"] else p.gather(1, at)
            full = torch.zeros(t, k, dtype=torch.float64, device="cuda")
            full[:live_rows] = w
            out = {"weights": full, "experts": None, "position": None, "source": None, "offsets": None}
            if case["train"]:
                g = s["grad"][:live_rows].double()
                d = torch.zeros(t, case["experts"], dtype=torch.float64, device="cuda")
                mean = (w * g).sum(1, keepdim=True)
                if case["renormalize"]:
                    d[:live_rows].scatter_(1, at, w * (g - mean))
                else:
                    chosen = torch.zeros_like(x).scatter_(1, at, g)
                    d[:live_rows] = p * (chosen - mean)
                out["grad_logits"] = d
            return out
        src = s["source"].long()
        n = int(s["offsets"][-1])
        tok = src[:n] // k
        if op == "dispatch":
            x = s["x"].detach().double()
            y = torch.zeros(t * k, case["width"], dtype=torch.float64, device="cuda")
            y[:n] = x[tok]
            out = {"y": y}
            if case["train"]:
                out["grad_x"] = torch.zeros_like(x).index_add_(0, tok, s["grad"][:n].double())
            return out
        rows = s["y"].detach()[:n].double()
        wt = s["weights"].detach().double().reshape(-1)[src[:n]]
        y = torch.zeros(t, case["width"], dtype=torch.float64, device="cuda")
        y.index_add_(0, tok, rows * wt[:, None])
        if s["residual"] is not None:
            y += s["residual"].double()
        out = {"y": y}
        if case["train"]:
            g = s["grad"].double()
            gy = torch.zeros(t * k, case["width"], dtype=torch.float64, device="cuda")
            gy[:n] = g[tok] * wt[:, None]
            gw = torch.zeros(t * k, dtype=torch.float64, device="cuda")
            gw[src[:n]] = (rows * g[tok]).sum(1)
            out.update(grad_y=gy, grad_weights=gw.view(t, k))
        return out
