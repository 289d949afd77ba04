"""Workloads of the routed-expert operators: routing, grouped products, SwiGLU with an 8-bit checkpoint, combination.

A case names one operator (``op``), its sizes, its element type and whether the backward pass runs too (``train``).
``run`` computes it in plain torch operations in 32 bits, or, with ``own`` set, through ``flare_b200.ops.experts``;
``exact`` computes it in 64 bits from the definition.  Layouts are those of ``flare_b200.ops.experts``:

* tokens are numbered slot-major, ``t = slot * tokens + b``; the experts of slot ``s`` are the groups ``s * E .. s * E + E - 1``;
* a routed token has ``top_k`` rows at most; rows are sorted by group, inside a group by token; ``offsets[g]`` is group ``g``'s first row;
* rows behind the last group (there are some where logits are masked) hold zeros.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
GROUP = 32  # columns that share one power-of-two scale in the 8-bit checkpoint


def listed():
    return [
        # a serving step of eight requests: the router of one layer, where latency counts
        dict(name="route decode", op="route", slots=1, tokens=8, experts=64, top_k=2, dtype="bf16", masked=False, train=False),
        # the head block of a token mixer: 12 heads with a bank of 8 experts each, 4096 samples
        dict(name="route heads", op="route", slots=12, tokens=4096, experts=8, top_k=2, dtype="bf16", masked=False, train=True),
        # a long padded batch over many experts, some of them masked out, the padding routed nowhere
        dict(name="route large masked", op="route", slots=1, tokens=131071, experts=128, top_k=4, dtype="fp32", masked=True, train=True),
        # serving: four tokens through the up projection of the experts that they chose (gathered from the tokens)
        dict(name="linear decode up", op="linear", slots=1, tokens=4, experts=16, top_k=2, width=512, out=4096, dtype="bf16", gather=True, masked=False, train=False),
        # serving: the same tokens through the down projection (rows already in group order)
        dict(name="linear decode down", op="linear", slots=1, tokens=4, experts=16, top_k=2, width=2048, out=512, dtype="bf16", gather=False, masked=False, train=False),
        # small odd groups, some of them empty, masked rows behind the last one
        dict(name="linear ragged", op="linear", slots=1, tokens=1001, experts=7, top_k=3, width=200, out=328, dtype="bf16", gather=True, masked=True, train=True),
        # the head block of a token mixer in training: 96 groups, the down projection, half precision
        dict(name="linear heads down", op="linear", slots=12, tokens=1365, experts=8, top_k=2, width=2048, out=512, dtype="fp16", gather=False, masked=False, train=True),
        # a full training batch through the up projection: 131072 rows over 32 experts
        dict(name="linear large up", op="linear", slots=1, tokens=65536, experts=32, top_k=2, width=512, out=4096, dtype="bf16", gather=True, masked=False, train=True),
        # the activation of that batch, with its 8-bit checkpoint and the backward pass that reads it
        dict(name="swiglu large", op="swiglu", rows=131072, width=2048, dtype="bf16", train=True),
        # an odd width and few rows
        dict(name="swiglu odd", op="swiglu", rows=1021, width=333, dtype="fp16", train=True),
        # the rows of that batch back to its tokens, with the weights' gradient
        dict(name="combine large", op="combine", slots=1, tokens=65536, experts=32, top_k=2, width=512, dtype="bf16", masked=False, train=True),
        # serving: five tokens of a wide model, four experts each
        dict(name="combine decode", op="combine", slots=1, tokens=5, experts=64, top_k=4, width=1024, dtype="fp32", masked=False, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    op = rng.choice(["route", "linear", "linear", "linear", "swiglu", "combine"])
    while True:
        c = dict(op=op)
        if op == "swiglu":
            c |= dict(rows=_log(rng, 1, 131072), width=_log(rng, 8, 4096))
        else:
            experts = rng.choice([1, 2, 3, 4, 7, 8, 16, 24, 32, 64, 128])
            slots = rng.choice([1, 1, 2, 5, 12])
            c |= dict(slots=slots, tokens=_log(rng, 1, 131072 // slots), experts=experts, top_k=rng.randint(1, min(4, experts)))
        if op == "linear":  # 16-byte rows
            c |= dict(width=8 * _log(rng, 1, 256), out=8 * _log(rng, 1, 512), gather=rng.random() < 0.5)
        if op == "combine":
            c["width"] = _log(rng, 1, 2048)
        c["dtype"] = rng.choice(["bf16", "fp16"] if op == "linear" else ["bf16", "fp16", "fp32"])
        if op != "swiglu":
            c["masked"] = rng.random() < 0.3
        c["train"] = rng.random() < 0.7
        w = work(c)
        # the plain form pads every group to the fullest one: its copies are bounded as well
        padded = 0 if op == "swiglu" else 4 * _rows(c) * (c.get("width", 1) + c.get("out", 1)) * min(6, c["experts"])
        weights = 12 * c["slots"] * c["experts"] * c["width"] * c["out"] if op == "linear" else 0
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and padded <= 24 << 30 and weights <= 4 << 30:
            return c


def _rows(case):
    return case["slots"] * case["tokens"] * case["top_k"]


def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op == "swiglu":
        n = case["rows"] * case["width"]
        if not case["train"]:
            return {"bytes": 3 * n * e, "flops": 6 * n}
        # forward: the input, the output and the checkpoint; backward: the output's gradient, the checkpoint, the input's gradient
        kept = 2 * n + 2 * case["rows"] * -(-case["width"] // GROUP)
        return {"bytes": 3 * n * e + kept + 3 * n * e + kept, "flops": 20 * n}
    t, r, g = case["slots"] * case["tokens"], _rows(case), case["slots"] * case["experts"]
    if op == "route":
        b = t * case["experts"] * e + r * 16 + 4 * (g + 1)
        return {"bytes": b + (t * case["experts"] * e + r * 12 if case["train"] else 0), "flops": t * case["experts"] * case["top_k"]}
    if op == "combine":
        n, y = r * case["width"] * e, t * case["width"] * e
        return {"bytes": n + y + 8 * r + (2 * n + y + 12 * r if case["train"] else 0), "flops": (6 if case["train"] else 2) * r * case["width"]}
    k, n = case["width"], case["out"]
    groups = min(g, r)  # the weights of a group that no row chose need not be read
    x = (t if case["gather"] else r) * k * e
    fwd = x + groups * (k * n + n) * e + r * n * e
    bwd = r * n * e + x + groups * k * n * e + x + g * (k * n + n) * e
    return {"bytes": fwd + (bwd if case["train"] else 0), "flops": (6 if case["train"] else 2) * r * k * n}


# ------------------------------------------------------------------ inputs
def _logits(case, gen):
    s, b, e = case["slots"], case["tokens"], case["experts"]
    popular = torch.randn(s, 1, e, generator=gen, device="cuda") * 0.7  # some experts are chosen more often than others
    x = torch.randn(s, b, e, generator=gen, device="cuda") * 1.5 + popular
    if case["masked"]:
        x = x.masked_fill(torch.rand(s, b, e, generator=gen, device="cuda") < 0.1, -math.inf)
        x[:, b - b // 16:] = -math.inf  # the padding of the batch
    return x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op, train = DTYPES[case["dtype"]], case["op"], case["train"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dt)

    s = {"case": dict(case)}
    if op == "swiglu":
        # rows of different magnitude, as experts' rows are
        size = torch.exp(torch.randn(case["rows"], 1, generator=gen, device="cuda"))
        s["x"] = normal(case["rows"], 2 * case["width"], scale=size).requires_grad_(train)
        s["dy"] = normal(case["rows"], case["width"])
        return s
    logits = _logits(case, gen)
    if op == "route":
        s["logits"] = logits.requires_grad_(train)
        s["dw"] = torch.randn(case["slots"], case["tokens"], case["top_k"], generator=gen, device="cuda")
        return s
    route = _route(logits, case["top_k"])
    s["route"] = route
    t, r, g, k = case["slots"] * case["tokens"], _rows(case), case["slots"] * case["experts"], case["width"]
    if op == "combine":
        s["weights"] = route["weights"].clone().requires_grad_(train)
        s["z"] = normal(r, k).requires_grad_(train)
        s["dy"] = normal(t, k)
        return s
    n = case["out"]
    s["cap"] = max(1, int((route["offsets"][1:] - route["offsets"][:-1]).max()))  # rows of the fullest group: the plain form pads to it
    s["x"] = normal(t if case["gather"] else r, k).requires_grad_(train)
    s["w"] = normal(g, k, n, scale=k ** -0.5).requires_grad_(train)
    s["b"] = normal(g, n, scale=0.1).requires_grad_(train)
    s["dy"] = normal(r, n)
    return s


# ------------------------------------------------------- the framework's calls
def _own(s):
    from flare_b200.ops.experts import ExpertRoute, combine_rows, grouped_linear, route_topk, swiglu

    case = s["case"]
    op, train = case["op"], case["train"]
    if op == "route":
        r = route_topk(s["logits"], case["top_k"])
        out = dict(r._asdict())
        if train:
            out["dlogits"], = torch.autograd.grad(r.weights, s["logits"], s["dw"])
        return out
    if op == "swiglu":
        y = swiglu(s["x"], checkpoint="e4m3" if train else None)
        return dict(y=y, dx=torch.autograd.grad(y, s["x"], s["dy"])[0]) if train else dict(y=y)
    route = ExpertRoute(**s["route"])
    if op == "combine":
        y = combine_rows(s["z"], route, s["weights"])
        if not train:
            return dict(y=y)
        dz, dw = torch.autograd.grad(y, (s["z"], s["weights"]), s["dy"])
        return dict(y=y, dz=dz, dw=dw)
    y = grouped_linear(s["x"], s["w"], s["b"], route=route) if case["gather"] else grouped_linear(s["x"], s["w"], s["b"], offsets=route.offsets)
    if not train:
        return dict(y=y)
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return dict(y=y, dx=dx, dw=dw, db=db)


# ------------------------------------------------------------- plain forms
def _route(logits, k):
    """Top-k softmax routing: ties go to the lowest expert, an expert at -inf is never chosen."""
    s, b, e = logits.shape
    val, idx = torch.sort(logits.detach().float(), dim=-1, descending=True, stable=True)
    val, idx = val[..., :k], idx[..., :k]
    live = val > -math.inf
    p = torch.exp(torch.where(live, val - torch.where(live[..., :1], val[..., :1], 0.0), -math.inf))
    w = torch.where(live, p / p.sum(-1, keepdim=True), 0.0)
    group = torch.where(live, idx + e * torch.arange(s, device=logits.device).view(s, 1, 1), s * e).reshape(-1)
    _, order = torch.sort(group, stable=True)
    counts = torch.zeros(s * e + 1, dtype=torch.int64, device=logits.device).index_add_(0, group, torch.ones_like(group))
    offsets = torch.cat([counts.new_zeros(1), counts[:-1].cumsum(0)])
    place = torch.arange(order.numel(), device=logits.device)
    rows = torch.where(place < offsets[-1], order // k, -1)
    row_of = torch.where(live.reshape(-1), torch.empty_like(place).scatter_(0, order, place), -1)
    i32 = torch.int32
    return dict(experts=torch.where(live, idx, -1).to(i32), weights=w, offsets=offsets.to(i32), rows=rows.to(i32), row_of=row_of.view(s, b, k).to(i32))


def _plain_route(s):
    logits, k = s["logits"], s["case"]["top_k"]
    out = _route(logits, k)
    if s["case"]["train"]:
        w = out["weights"]
        d = w * (s["dw"] - (w * s["dw"]).sum(-1, keepdim=True))
        at = torch.where(out["experts"] < 0, logits.shape[-1], out["experts"]).long()  # a place behind the experts for what was not chosen
        full = torch.zeros(*logits.shape[:2], logits.shape[2] + 1, device=d.device).scatter_(2, at, d)
        out["dlogits"] = full[..., :-1].to(logits.dtype)
    return out


def _quantised(x):
    """The values that the 8-bit checkpoint stands for: e4m3 with a power-of-two scale for each 32 columns (of either half)."""
    r, n = x.shape
    g = -(-n // GROUP)
    v = torch.nn.functional.pad(x, (0, g * GROUP - n)).view(r, g, GROUP)
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))  # amax = m * 2^e, m in [0.5, 1)
    shift = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)  # the largest lands in (224, 448]
    scale = torch.ldexp(torch.ones_like(m), shift)
    return ((v / scale).to(torch.float8_e4m3fn).float() * scale).view(r, g * GROUP)[:, :n]


def _plain_swiglu(s):
    x, h = s["x"].detach(), s["case"]["width"]
    up, gate = x[:, :h].float(), x[:, h:].float()
    out = dict(y=(up * gate * torch.sigmoid(gate)).to(x.dtype))
    if s["case"]["train"]:
        up, gate, dy = _quantised(up), _quantised(gate), s["dy"].float()
        sg = torch.sigmoid(gate)
        out["dx"] = torch.cat([dy * gate * sg, dy * up * sg * (1 + gate * (1 - sg))], 1).to(x.dtype)
    return out


def _plain_combine(s):
    z, w, r = s["z"].detach(), s["weights"].detach(), s["route"]
    t, k = s["dy"].shape[0], s["case"]["top_k"]
    at, w = r["row_of"].view(t, k).long(), w.view(t, k)
    picked = torch.where((at >= 0).unsqueeze(-1), z[at.clamp(min=0)].float(), 0.0)
    out = dict(y=(picked * w.unsqueeze(-1)).sum(1).to(z.dtype))
    if s["case"]["train"]:
        dy = s["dy"].float()
        out["dw"] = (picked * dy.unsqueeze(1)).sum(-1).view(s["weights"].shape)
        spot = torch.where(at >= 0, at, z.shape[0]).reshape(-1)  # one row behind the others takes what was not chosen
        dz = torch.zeros(z.shape[0] + 1, z.shape[1], device=z.device)
        dz[spot] = (w.unsqueeze(-1) * dy.unsqueeze(1)).reshape(t * k, -1)
        out["dz"] = dz[:-1].to(z.dtype)
    return out


def _plain_linear(s):
    """Every group padded to the fullest one, then one batched product."""
    case, r, cap = s["case"], s["route"], s["cap"]
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    g, k, n = w.shape
    off = r["offsets"].long()
    place = torch.arange(s["dy"].shape[0], device=x.device)
    group = torch.searchsorted(off[1:], place, right=True).clamp(max=g - 1)
    live = place < off[-1]
    spot = torch.where(live, group * cap + place - off[group], g * cap)

    def padded(v):
        return torch.zeros(g * cap + 1, v.shape[1], device=v.device).index_copy_(0, spot, v.float())[:-1].view(g, cap, -1)

    def packed(v):
        return torch.where(live.unsqueeze(1), v.reshape(g * cap, -1)[spot.clamp(max=g * cap - 1)], 0.0)

    xp = padded(x[r["rows"].long().clamp(min=0)] if case["gather"] else x)
    out = dict(y=packed(torch.bmm(xp, w.float()) + b.float().unsqueeze(1)).to(x.dtype))
    if case["train"]:
        dyp = padded(s["dy"])
        out["dw"] = torch.bmm(xp.transpose(1, 2), dyp).to(w.dtype)
        out["db"] = dyp.sum(1).to(b.dtype)
        dx = packed(torch.bmm(dyp, w.float().transpose(1, 2)))
        if case["gather"]:
            at = r["row_of"].view(x.shape[0], -1).long()
            dx = torch.where((at >= 0).unsqueeze(-1), dx[at.clamp(min=0)], 0.0).sum(1)
        out["dx"] = dx.to(x.dtype)
    return out


def run(state):
    if own:
        return _own(state)
    return {"route": _plain_route, "linear": _plain_linear, "swiglu": _plain_swiglu, "combine": _plain_combine}[state["case"]["op"]](state)


# ------------------------------------------------- the definitions, in 64 bits
def _e4m3(v):
    """Nearest value of 8 bits with 4 of exponent and 3 of mantissa, ties to even; |v| <= 448."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 4).clamp(min=-9).double())  # four significant bits; below 2^-6 the spacing stays 2^-9
    return torch.round(v / step) * step


def _exact_quantised(x):
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], GROUP):
        v = x[:, c:c + GROUP]
        top = v.abs().amax(1, keepdim=True)
        p = torch.floor(torch.log2(top.clamp(min=1e-300)))
        p = torch.where(torch.exp2(p) > top, p - 1, torch.where(torch.exp2(p + 1) <= top, p + 1, p))
        scale = torch.exp2(torch.where(top <= 1.75 * torch.exp2(p), p - 8, p - 7).clamp(min=-126))
        out[:, c:c + GROUP] = _e4m3(v / scale) * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, train = case["op"], case["train"]
    if op == "route":
        l64 = s["logits"].detach().double()
        sl, b, e = l64.shape
        left, picks = l64.clone(), []
        for _ in range(case["top_k"]):
            top = left.amax(-1, keepdim=True)
            first = torch.where(left == top, torch.arange(e, device=left.device), e).amin(-1, keepdim=True)
            picks.append(torch.where(torch.isneginf(top), -1, first))
            left = left.scatter(-1, first, -math.inf)
        experts = torch.cat(picks, -1)
        chosen = torch.where(experts >= 0, l64.gather(-1, experts.clamp(min=0)), -math.inf)
        w = torch.nan_to_num(torch.softmax(chosen, -1), nan=0.0)
        out = dict(experts=None, weights=w, offsets=None, rows=None, row_of=None)
        if train:
            dw = s["dw"].double()
            d = torch.zeros_like(l64)
            for j in range(case["top_k"]):
                mine = w[..., j] * (dw[..., j] - (w * dw).sum(-1))
                d.scatter_add_(-1, experts[..., j:j + 1].clamp(min=0), torch.where(experts[..., j] >= 0, mine, 0.0).unsqueeze(-1))
            out["dlogits"] = d
        return out
    if op == "swiglu":
        h = case["width"]
        up, gate = s["x"].detach().double().split(h, 1)
        out = dict(y=up * gate / (1 + torch.exp(-gate)))
        if train:
            up, gate, dy = _exact_quantised(up), _exact_quantised(gate), s["dy"].double()
            sg = 1 / (1 + torch.exp(-gate))
            out["dx"] = torch.cat([dy * gate * sg, dy * up * (sg + gate * sg * (1 - sg))], 1)
        return out
    route = s["route"]
    t, k = case["slots"] * case["tokens"], case["top_k"]
    if op == "combine":
        z, w, dy, at = s["z"].detach().double(), s["weights"].detach().double().view(t, k), s["dy"].double(), route["row_of"].view(t, k).long()
        y, dz, dw = torch.zeros_like(dy), torch.zeros_like(z), torch.zeros_like(w)
        for j in range(k):
            on = (at[:, j] >= 0).nonzero().squeeze(1)
            y[on] += w[on, j:j + 1] * z[at[on, j]]
            dz[at[on, j]] = w[on, j:j + 1] * dy[on]
            dw[on, j] = (z[at[on, j]] * dy[on]).sum(1)
        return dict(y=y, dz=dz, dw=dw.view(s["weights"].shape)) if train else dict(y=y)
    x, w, b, dy = (s[n].detach() for n in ("x", "w", "b", "dy"))
    off = route["offsets"].tolist()
    y = torch.zeros(dy.shape, dtype=torch.float64, device=x.device)
    dx, dw, db = (torch.zeros(v.shape, dtype=torch.float64, device=x.device) if train else None for v in (x, w, b))
    for g in range(w.shape[0]):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        at = route["rows"][lo:hi].long() if case["gather"] else torch.arange(lo, hi, device=x.device)
        xg, wg, dg = x[at].double(), w[g].double(), dy[lo:hi].double()
        y[lo:hi] = xg @ wg + b[g].double()
        if train:
            dx.index_add_(0, at, dg @ wg.t())
            dw[g] = xg.t() @ dg
            db[g] = dg.sum(0)
    return dict(y=y, dx=dx, dw=dw, db=db) if train else dict(y=y)
