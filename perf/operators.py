"""The operators that stand around the routed experts of a layer, as a user's program calls them, and their plain forms.

  route      the router's choice: scores of all experts -> ids and weights of each token's picks, and the gradient of the logits
  dispatch   the tokens' rows sorted by expert (sort and copy), and the gradient, which adds a token's rows up again
  combine    the experts' rows back to their tokens, weighted, and the gradients of rows and weights
  w4         products with 4-bit weights that have a scale (and a zero point) per group of columns: one matrix for all rows (a
             shared expert), or one per expert for the rows that are sorted by expert

listed() names the cases, draw() gives more of the same ranges, prepare() makes what the program holds before a call, run() is one
pass: with `own` through this repository's entry points, else in elementary torch operations.  exact() is the definition in 64 bits.

A case is
  op         route | dispatch | combine | w4
  T, topk, E tokens, picks per token, experts
  H          width of a row (dispatch, combine);  N, K, g: rows, columns and group of the 4-bit matrices (w4)
  dtype      of the rows (of the logits: route);  out: of what comes out (route: the weights; combine and w4: the rows)
  train      the backward pass too
  score, renorm, bias    route: sigmoid or softmax, weights divided by their sum, a bias per expert that only the choice sees
  zeros      w4: a zero point per group instead of 8
  experts    w4: one matrix per expert; `of` experts are routed over, E of them are here, rows of the others' picks have none
  pad        share of the tokens that are padding: ids of -1
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCALE = 2.5      # of the routing weights


def _route(name, T, E, topk, dtype="f32", out="f16", score="sigmoid", renorm=True, bias=True, train=False):
    return dict(name=name, op="route", T=T, E=E, topk=topk, dtype=dtype, out=out, score=score, renorm=renorm, bias=bias, train=train)


def _rows(name, op, T, E, topk, H, dtype="bf16", out="bf16", train=False, pad=0.0):
    return dict(name=name, op=op, T=T, E=E, topk=topk, H=H, dtype=dtype, out=out, train=train, pad=pad)


def _w4(name, T, N, K, g, dtype="f16", out="f16", zeros=False, experts=False, E=1, topk=1, of=1):
    return dict(name=name, op="w4", T=T, N=N, K=K, g=g, dtype=dtype, out=out, zeros=zeros, experts=experts, E=E, topk=topk, of=of)


def listed():
    return [
        # a decode batch: the choice of 8 of 256 experts, weights as the layer call takes them
        _route("route 32", 32, 256, 8),
        # a training step's tokens, with the gradient for the router
        _route("route 16384 train", 16384, 256, 8, out="f32", train=True),
        # a router that takes the softmax over all experts as it is, 16-bit logits, odd sizes
        _route("route 3001 softmax", 3001, 120, 6, dtype="bf16", out="bf16", score="softmax", renorm=False, bias=False, train=True),
        # a decode batch sorted by expert
        _rows("dispatch 32", "dispatch", 32, 256, 8, 6144, dtype="f16", out="f16"),
        # a training step, forward and backward
        _rows("dispatch 4096 train", "dispatch", 4096, 256, 8, 6144, train=True),
        # a decode batch back to its tokens, added in 32 bits
        _rows("combine 32", "combine", 32, 256, 8, 6144, dtype="f16", out="f32"),
        # a training step of the small layer's kind, ragged, a tenth of the tokens padding
        _rows("combine 5001 train", "combine", 5001, 64, 4, 1000, train=True, pad=0.1),
        # one token through the shared expert's gate and up rows: interactive decoding
        _w4("w4 1", 1, 4096, 6144, 128),
        # verification of speculated tokens through its down projection, zero points
        _w4("w4 8 down", 8, 6144, 2048, 64, dtype="bf16", out="bf16", zeros=True),
        # a full decode batch, fine groups, sums handed on in 32 bits
        _w4("w4 32", 32, 4096, 6144, 32, out="f32"),
        # a short prompt
        _w4("w4 512", 512, 4096, 6144, 128, dtype="bf16", out="bf16"),
        # a decode batch on one of eight expert-parallel ranks: 32 of 256 experts, most picks are other ranks'
        _w4("w4 experts", 32, 4096, 6144, 128, experts=True, E=32, topk=8, of=256),
    ]


def _log_between(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "dispatch", "combine", "w4", "w4"])
    if op == "route":
        E = _log_between(rng, 8, 512)
        topk = rng.randint(1, min(E, 10))
        score = rng.choice(["sigmoid", "sigmoid", "softmax"])
        T = min(_log_between(rng, 1, 16384), 16384 * 256 // E)
        return dict(op=op, T=T, E=E, topk=topk, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), out=rng.choice(["f32", "f16", "bf16"]), score=score,
                    renorm=rng.random() < 0.7, bias=score == "sigmoid" and rng.random() < 0.7, train=rng.random() < 0.5)
    if op in ("dispatch", "combine"):
        H = _log_between(rng, 64, 6144)
        if rng.random() < 0.7:
            H = (H + 63) // 64 * 64
        E = _log_between(rng, 8, 512)
        topk = rng.randint(1, 8)
        train = rng.random() < 0.5
        T = _log_between(rng, 1, 8192)
        while T * topk * H > 4096 * 8 * 6144:
            T = T * 3 // 4
        dtype = rng.choice(["bf16", "f16", "f32"])
        return dict(op=op, T=T, E=E, topk=topk, H=H, dtype=dtype, out=rng.choice([dtype, "f32"]) if op == "combine" else dtype, train=train,
                    pad=rng.choice([0.0, 0.0, 0.1]))
    g = rng.choice([32, 64, 128])
    experts = rng.random() < 0.4
    K = max(1, _log_between(rng, 256, 8192) // g) * g
    N = _log_between(rng, 64, 12288)
    if rng.random() < 0.7:
        N = (N + 15) // 16 * 16
    dtype = rng.choice(["f16", "bf16"])
    case = dict(op="w4", g=g, dtype=dtype, out=rng.choice([dtype, dtype, "f32"]), zeros=rng.random() < 0.5, experts=experts)
    if experts:
        E = _log_between(rng, 4, 64)
        while E * N * K > 32 * 4096 * 6144:
            E = max(4, E * 3 // 4)
            N = N * 3 // 4
        T = _log_between(rng, 1, 32)
        return dict(case, T=T, N=N, K=K, E=E, topk=rng.randint(1, 4), of=E * rng.choice([1, 1, 4]))
    T = _log_between(rng, 1, 512)
    while N * K > 2 * 4096 * 6144 or T * N * K > 512 * 4096 * 6144:
        N = N * 3 // 4
    return dict(case, T=T, N=N, K=K, E=1, topk=1, of=1)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _picks(case, gen, over):
    """distinct experts of each token, as a router's choice has them: popular ones among them; padding tokens have none"""
    T, topk = case["T"], case["topk"]
    logits = torch.randn(T, over, generator=gen, device="cuda") + 0.5 * torch.randn(over, generator=gen, device="cuda")
    sel = logits.argsort(1, descending=True)[:, :topk].contiguous()
    if case.get("pad"):
        sel[torch.rand(T, generator=gen, device="cuda") < case["pad"]] = -1
    return sel


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    T, E, topk = case["T"], case["E"], case["topk"]
    dt, out = TYPES[case["dtype"]], TYPES[case["out"]]
    s = dict(case=case, gen=gen)
    if case["op"] == "route":
        s["logits"] = (1.5 * f(T, E)).to(dt).requires_grad_(case["train"])
        s["bias"] = 0.2 * f(E) if case["bias"] else None
        s["drw"] = f(T, topk).to(out)
    elif case["op"] == "dispatch":
        s["sel"] = _picks(case, gen, E)
        s["x"] = f(T, case["H"]).to(dt).requires_grad_(case["train"])
        s["dxs"] = f(T * topk, case["H"]).to(dt) if case["train"] else None
    elif case["op"] == "combine":
        s["sel"] = _picks(case, gen, E)
        s["y"] = f(T * topk, case["H"]).to(dt).requires_grad_(case["train"])
        w = torch.softmax(f(T, topk), 1) * SCALE
        s["rw"] = w.to(torch.float32 if case["train"] else torch.float16).requires_grad_(case["train"])
        s["dout"] = f(T, case["H"]).to(out) if case["train"] else None
        if own:                                  # the order is what the program has from sorting before the experts' products
            from nestquant_b200 import routing
            s["order"] = routing.sort_picks(s["sel"], E)
        else:
            s["order"] = _plain_order(s["sel"], E)
    else:
        N, K, g = case["N"], case["K"], case["g"]
        lead = (E,) if case["experts"] else ()
        s["q"] = torch.randint(0, 256, lead + (N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)      # two columns a byte, the even one low
        s["scales"] = (0.01 * (0.5 + torch.rand(lead + (N, K // g), generator=gen, device="cuda"))).to(dt)
        s["zeros"] = torch.randint(4, 12, lead + (N, K // g), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["start"] = None
        rows = T
        if case["experts"]:
            sel = _picks(case, gen, case["of"])
            sizes = torch.bincount(sel.flatten(), minlength=case["of"])[:E]
            s["start"] = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).int()
            rows = T * topk
        s["x"] = f(rows, K).to(dt)
        s["w"] = None
        if own:                                  # the matrices as the program keeps them, laid out once when they are loaded
            from nestquant_b200 import w4
            s["w"] = w4.W4(s["q"], s["scales"], s["zeros"])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)[s["case"]["op"]](s)


def _own_route(s):
    from nestquant_b200 import routing
    c = s["case"]
    sel, rw = routing.route(s["logits"], c["topk"], score=c["score"], bias=s["bias"], renorm=c["renorm"], scale=SCALE, dtype=TYPES[c["out"]])
    if not c["train"]:
        return sel, rw
    return sel, rw, torch.autograd.grad(rw, s["logits"], s["drw"])[0]


def _own_dispatch(s):
    from nestquant_b200 import routing
    order = routing.sort_picks(s["sel"], s["case"]["E"])
    xs = routing.dispatch(s["x"], order)
    if not s["case"]["train"]:
        return order.start, order.pos, xs
    return order.start, order.pos, xs, torch.autograd.grad(xs, s["x"], s["dxs"])[0]


def _own_combine(s):
    from nestquant_b200 import routing
    out = routing.combine(s["y"], s["order"], s["rw"], dtype=TYPES[s["case"]["out"]])
    if not s["case"]["train"]:
        return out
    return out, *torch.autograd.grad(out, (s["y"], s["rw"]), s["dout"])


def _own_w4(s):
    return s["w"](s["x"], start=s["start"], dtype=TYPES[s["case"]["out"]])


_run_own = {"route": _own_route, "dispatch": _own_dispatch, "combine": _own_combine, "w4": _own_w4}


def _plain_route(s):
    c, dt = s["case"], TYPES[s["case"]["out"]]
    k, wide = c["topk"], s["logits"].detach()
    key = wide if s["bias"] is None else 1 / (1 + torch.exp(-wide.double())) + s["bias"].double()      # 64 bits: which expert wins a near tie
    sel = key.sort(dim=1, descending=True, stable=True)[1][:, :k].contiguous()
    full, drw = wide.float(), s["drw"].float()
    picked = full.gather(1, sel)
    if c["score"] == "sigmoid":
        p = 1 / (1 + torch.exp(-picked))
    else:
        e = torch.exp(full - full.amax(1, keepdim=True))
        every = e / e.sum(1, keepdim=True)
        p = every.gather(1, sel)
    total = p.sum(1, keepdim=True)
    rw = (SCALE * (p / total if c["renorm"] else p)).to(dt)
    if not c["train"]:
        return sel, rw
    dp = SCALE * ((drw - (drw * p).sum(1, keepdim=True) / total) / total if c["renorm"] else drw)
    grad = torch.zeros_like(full)
    if c["score"] == "sigmoid":
        grad.scatter_(1, sel, dp * p * (1 - p))
    else:
        grad.scatter_(1, sel, dp)
        grad = every * (grad - (dp * p).sum(1, keepdim=True))
    return sel, rw, grad.to(wide.dtype)


def _plain_order(sel, E):
    flat = sel.flatten()
    bins = torch.where((flat >= 0) & (flat < E), flat, E)
    perm = bins.argsort(stable=True)
    pos = torch.empty_like(perm)
    pos[perm] = torch.arange(perm.numel(), device=perm.device)
    start = torch.searchsorted(bins[perm], torch.arange(E + 1, device=perm.device))
    return perm, pos.view(sel.shape), start, bins < E


def _plain_dispatch(s):
    c, x = s["case"], s["x"].detach()
    perm, pos, start, live = _plain_order(s["sel"], c["E"])
    xs = torch.where(live[perm][:, None], x[perm // c["topk"]], 0)
    if not c["train"]:
        return start.int(), pos.int(), xs
    dx = torch.where(live.view(pos.shape)[:, :, None], s["dxs"][pos].float(), 0).sum(1).to(x.dtype)
    return start.int(), pos.int(), xs, dx


def _plain_combine(s):
    c, y, rw = s["case"], s["y"].detach(), s["rw"].detach().float()
    _, pos, _, live = s["order"]
    live = live.view(pos.shape)
    rows = torch.where(live[:, :, None], y[pos].float(), 0)
    rw = torch.where(live, rw, 0)
    out = (rows * rw[:, :, None]).sum(1).to(TYPES[c["out"]])
    if not c["train"]:
        return out
    dout = s["dout"].float()
    dy = torch.empty_like(y)
    dy[pos.flatten()] = (rw[:, :, None] * dout[:, None]).to(y.dtype).flatten(0, 1)
    return out, dy, (rows * dout[:, None]).sum(2).to(s["rw"].dtype)


def _weights(s, wide):
    """the matrices, in `wide` bits: (q - zero) * scale, group by group"""
    q, g = s["q"], s["case"]["g"]
    w = torch.stack([q & 15, q >> 4], -1).to(wide).view(*q.shape[:-1], -1, g)
    zero = 8 if s["zeros"] is None else s["zeros"].to(wide)[..., None]
    return ((w - zero) * s["scales"].to(wide)[..., None]).flatten(-2)


def _plain_w4(s):
    c = s["case"]
    w, x, out = _weights(s, torch.float32), s["x"].float(), TYPES[c["out"]]
    if not c["experts"]:
        return (x @ w.T).to(out)
    # a token picks an expert once at most: T places for each expert, the last one for rows without one
    place = torch.arange(x.shape[0], device=x.device)
    e = torch.searchsorted(s["start"].long(), place, right=True) - 1
    at = torch.where(e < c["E"], e * c["T"] + place - s["start"].long()[e], c["E"] * c["T"])
    wide = x.new_zeros(c["E"] * c["T"] + 1, c["K"])
    wide[at] = x
    y = x.new_zeros(c["E"] * c["T"] + 1, c["N"])
    y[:-1] = torch.bmm(wide[:-1].view(c["E"], c["T"], -1), w.transpose(1, 2)).flatten(0, 1)
    return torch.where((e < c["E"])[:, None], y[at], 0).to(out)


_run_plain = {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "w4": _plain_w4}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        l = s["logits"].detach().double()
        key = l if s["bias"] is None else torch.sigmoid(l) + s["bias"].double()
        picked = torch.zeros_like(l).scatter_(1, key.sort(dim=1, descending=True, stable=True)[1][:, :case["topk"]], 1.0) > 0
        order = key.masked_fill(~picked, -math.inf).sort(dim=1, descending=True, stable=True)[1][:, :case["topk"]]
        l.requires_grad_(True)
        score = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, 1)
        w = torch.where(picked, score, 0)
        w = SCALE * (w / w.sum(1, keepdim=True) if case["renorm"] else w)
        rw = w.gather(1, order)
        if not case["train"]:
            return None, rw.detach()
        return None, rw.detach(), torch.autograd.grad(rw, l, s["drw"].double())[0]
    if case["op"] in ("dispatch", "combine"):
        T, topk, E = case["T"], case["topk"], case["E"]
        sel = s["sel"].flatten().tolist()
        ranked = sorted(range(T * topk), key=lambda i: (sel[i] if 0 <= sel[i] < E else E, i))
        n = sum(0 <= e < E for e in sel)
        at = torch.tensor(ranked, device="cuda")
        token, lives = at // topk, torch.arange(T * topk, device="cuda") < n
    if case["op"] == "dispatch":
        x = s["x"].detach().double()
        xs = x[token] * lives[:, None]
        if not case["train"]:
            return None, None, xs
        return None, None, xs, torch.zeros_like(x).index_add_(0, token[:n], s["dxs"][:n].double())
    if case["op"] == "combine":
        y, w = s["y"].detach().double(), s["rw"].detach().double().flatten()[at]
        out = torch.zeros(T, case["H"], device="cuda", dtype=torch.float64).index_add_(0, token[:n], y[:n] * w[:n, None])
        if not case["train"]:
            return out
        d = s["dout"].double()[token]
        drw = torch.zeros(T * topk, device="cuda", dtype=torch.float64)
        drw[at[:n]] = torch.einsum("ph,ph->p", y[:n], d[:n])
        return out, d * (w * lives)[:, None], drw.view(T, topk)
    q, g, K = s["q"], case["g"], case["K"]
    col = torch.arange(K, device="cuda")
    scale, zero = s["scales"].double(), s["zeros"]
    x = s["x"].double()

    def product(rows, q, scale, zero):
        # group by group: the sum over its columns, then its scale
        y = torch.zeros(rows.shape[0], q.shape[0], device="cuda", dtype=torch.float64)
        for j in range(K // g):
            c = col[j * g:(j + 1) * g]
            n = ((q[:, c // 2].int() >> (4 * (c % 2)).int()) & 15).double() - (8 if zero is None else zero[:, j:j + 1].double())
            y += rows[:, c] @ n.T * scale[:, j]
        return y

    if not case["experts"]:
        return product(x, q, scale, zero)
    bounds = s["start"].tolist()
    y = torch.zeros(x.shape[0], case["N"], device="cuda", dtype=torch.float64)
    for e in range(case["E"]):
        if bounds[e] < bounds[e + 1]:
            y[bounds[e]:bounds[e + 1]] = product(x[bounds[e]:bounds[e + 1]], q[e], scale[e], None if zero is None else zero[e])
    return y


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    T, E, topk, a, b = case["T"], case["E"], case["topk"], SIZE[case["dtype"]], SIZE[case["out"]]
    P = T * topk
    if case["op"] == "route":
        fwd = T * E * a + P * (8 + b) + (4 * E if case["bias"] else 0)
        bwd = P * b + T * E * a if case["train"] else 0            # the logits are there already
        return dict(bytes=fwd + bwd, flops=T * E * (8 + (4 if case["train"] else 0)))
    if case["op"] == "dispatch":
        n = T * case["H"] * a
        fwd, bwd = 12 * P + 4 * (E + 1) + n * (1 + topk), n * (1 + topk) if case["train"] else 0
        return dict(bytes=fwd + bwd, flops=P * case["H"] if case["train"] else 0)
    if case["op"] == "combine":
        H = case["H"]
        live = 1 - case["pad"]
        w = 4 if case["train"] else 2
        fwd = P * H * a * live + T * H * b + P * (4 + w)
        bwd = T * H * b + P * H * a + P * w if case["train"] else 0          # the experts' rows are there already
        return dict(bytes=fwd + bwd, flops=P * H * (6 if case["train"] else 2))
    N, K, g = case["N"], case["K"], case["g"]
    one = N * K / 2 + N * (K // g) * (2 + (1 if case["zeros"] else 0))
    if not case["experts"]:
        return dict(bytes=one + T * K * a + T * N * b, flops=2 * T * N * K)
    hit = E * (1 - (1 - topk / case["of"]) ** T)                 # experts with a row
    live = P * E / case["of"]
    return dict(bytes=one * hit + live * K * a + P * N * b, flops=2 * live * N * K)
