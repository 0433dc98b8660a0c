"""The operators of an expert layer over atoms, as measurable cases.

A layer whose weights depend on the atom: the residual is added and the row normalised (rms_norm,
with an 8-bit form for serving), a gate or the atom's species chooses experts (route, group_plan),
every row is multiplied by its experts' weights (grouped_linear, each direction, and in 8 bits), and
the experts' rows are joined (expert_combine).

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program has in
hand before the call, run() makes one pass, in elementary torch operations or (own) through the
framework, exact() is the same result in 64 bits.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E4M3_MAX, SCALE_MIN = 448.0, 2.0 ** -126
OPS = ("norm", "route", "linear", "combine")
SPECIES = (9143, 10286, 4571)              # H, C and O of the 24,000-atom liquid


def _experts():
    """The framework's module of these operators."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "face-mlip_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from face_amd import experts
    return experts


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # the invariants of one 21-atom molecule (9 C columns, C = 96) normalised in an MD step: latency
        _norm("norm_molecule21_c96", 21, 864, "f32", residual=False),
        # residual stream and norm of a 24,000-atom liquid, C = 160, trained in 32 bits: both directions
        _norm("norm_train_24k_c160", 24000, 1440, "f32", grad=True),
        # the same of 100,000 atoms, C = 256, served: 16-bit rows, normalised rows leave in 8 bits
        _norm("norm_q8_100k_c256", 100000, 2304, "bf16", q8=True),
        # the gate of one molecule, two of eight experts, and the grouping of its rows: latency
        _route("route_molecule21", 21, 8, 2),
        # the gate of 100,000 atoms over 64 experts, some closed to a species, both directions
        _route("route_train_100k", 100000, 64, 4, species=True, renorm=False, grad=True),
        # the readout's last layer of one molecule by species, SiLU on its input, an odd width: both directions
        _linear("linear_molecule21_c96", 21, 1, 3, 192, 97, "f32", silu=True, grad=True, species=True),
        # the readout's first layer by species, 24,000 atoms, C = 160, trained in 32 bits
        _linear("linear_train_24k_c160", 24000, 1, 3, 1440, 320, "f32", grad=True, species=True),
        # the same layer at C = 256 as two of eight learned experts, 100,000 atoms, trained in 16 bits
        _linear("linear_train_100k_c256", 100000, 2, 8, 2304, 512, "bf16", grad=True),
        # that layer served in 8 bits
        _linear("linear_q8_100k_c256", 100000, 2, 8, 2304, 512, "bf16", q8=True),
        # one atom through two of 64 wide experts: a single row, bound by the weights
        _linear("linear_one_atom", 1, 2, 64, 2048, 2048, "bf16"),
        # the experts' rows of one molecule joined and added to the residual: latency
        _combine("combine_molecule21_c96", 21, 2, 96, "f32"),
        # the same of 100,000 atoms and 16 bits, both directions
        _combine("combine_train_100k_c256", 100000, 2, 512, "bf16", grad=True),
    ]


def _norm(name, rows, width, dtype, residual=True, grad=False, q8=False):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "grad": grad,
            "q8": q8}


def _route(name, rows, experts, k, species=False, renorm=True, grad=False, dtype="f32"):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "k": k, "species": species, "renorm": renorm,
            "grad": grad, "dtype": dtype}


def _linear(name, rows, k, experts, n_in, n_out, dtype, silu=False, grad=False, q8=False, species=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "experts": experts, "n_in": n_in, "n_out": n_out,
            "dtype": dtype, "silu": silu, "grad": grad, "q8": q8, "species": species}


def _combine(name, rows, k, width, dtype, grad=False):
    return {"name": name, "op": "combine", "rows": rows, "k": k, "width": width, "dtype": dtype, "grad": grad}


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: atoms from one to 100,000, widths of a model's readout, odd ones too."""
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(OPS + ("linear", "linear"))
        rows, dtype, grad = _log(rng, 1, 100000), rng.choice(list(TYPES)), rng.random() < 0.5
        if op == "norm":
            c = _norm(None, rows, _log(rng, 16, 4096), dtype, rng.random() < 0.7, grad)
            c["q8"] = not grad and rng.random() < 0.5
        elif op == "route":
            experts = _log(rng, 2, 128)
            k = rng.randint(1, min(8, experts))
            # one expert's weight over itself is one: no gradient
            c = _route(None, rows, experts, k, rng.random() < 0.5, k > 1 and rng.random() < 0.5, grad, dtype)
        elif op == "combine":
            c = _combine(None, rows, rng.randint(1, 8), _log(rng, 16, 2304), dtype, grad)
        else:
            species = rng.random() < 0.4
            c = _linear(None, rows, 1 if species else rng.randint(1, 4), 3 if species else _log(rng, 4, 64),
                        _log(rng, 16, 2304), _log(rng, 16, 2304), dtype, False, grad, False, species)
            c["silu"] = rng.random() < 0.4
            c["q8"] = not grad and not c["silu"] and rng.random() < 0.4
        del c["name"]
        if _cost(c) <= most:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    op, n = case["op"], case["rows"]
    z = SIZE[case["dtype"]]
    if op == "norm":
        f = case["width"]
        parts = (1 + 2 * case["residual"]) * z + (1 if case["q8"] else z)            # x, residual, sum; the result
        b = n * f * parts + f * z + (4 * n if case["q8"] else 0)
        if case["grad"]:
            b += n * f * z * (3 + case["residual"]) + 2 * f * z                       # s, dy, ds in; dx and dw out
        return {"bytes": b, "flops": n * f * (6 + 10 * case["grad"])}
    if op == "route":
        e, k = case["experts"], case["k"]
        b = n * e * z + n * k * 8 + n * k * 4 + 4 * (e + 1) + n * k * 4               # logits; experts, weights, plan
        b += (4 * n + 3 * e) * case["species"]
        if case["grad"]:
            b += 2 * n * e * z + n * k * 12
        return {"bytes": b, "flops": n * e * (5 + k)}
    if op == "combine":
        f, k = case["width"], case["k"]
        b = n * k * f * z + 2 * n * f * z + 4 * n * k
        if case["grad"]:
            b += 2 * n * k * f * z + n * f * z + 8 * n * k
        return {"bytes": b, "flops": 2 * n * k * f * (1 + 2 * case["grad"])}
    a, e, ki, fo = n * case["k"], case["experts"], case["n_in"], case["n_out"]
    e = min(e, a)                                                                     # experts with rows
    rows = a if case["silu"] else n                                                   # a hidden row per slot
    if case["q8"]:
        return {"bytes": rows * (ki + 4) + e * fo * (ki + 4) + a * (fo * z + 4), "flops": 2 * a * ki * fo}
    b = rows * ki * z + e * fo * (ki + 1) * z + a * (fo * z + 4)
    if case["grad"]:
        b += a * fo * z + 2 * rows * ki * z + 2 * e * fo * (ki + 1) * z
    return {"bytes": b, "flops": 2 * a * ki * fo * (3 if case["grad"] else 1)}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, n, op = TYPES[case["dtype"]], case["rows"], case["op"]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {"case": case}
    if op == "norm":
        f = case["width"]
        s["x"] = normal(n, f)
        s["w"] = (1 + 0.1 * torch.randn(f, generator=g, device=DEV)).to(t)
        if case["residual"]:
            s["r"] = normal(n, f, scale=3.0)
        if case["grad"]:
            s["dy"], s["ds"] = normal(n, f), (normal(n, f) if case["residual"] else None)
        return s
    if op == "route":
        e = case["experts"]
        s["logits"] = normal(n, e, scale=1.5)
        if case["species"]:
            s["group"] = _species(n, g).to(torch.int32)
            s["allowed"] = torch.rand(len(SPECIES), e, generator=g, device=DEV) < 0.8
            s["allowed"][:, 0] = True
        if case["grad"]:
            s["dweight"] = normal(n, case["k"], dtype=torch.float32)
        return s
    if op == "combine":
        f, k = case["width"], case["k"]
        s["y"], s["r"] = normal(n * k, f), normal(n, f)
        s["weight"] = torch.softmax(torch.randn(n, k, generator=g, device=DEV), 1)
        if case["grad"]:
            s["dout"] = normal(n, f)
        return s
    k, e, ki, fo = case["k"], case["experts"], case["n_in"], case["n_out"]
    if case["species"]:
        expert = _species(n, g).view(n, 1)
    else:
        bias = 0.7 * torch.randn(e, generator=g, device=DEV)                          # some experts draw more rows
        expert = torch.topk(bias + torch.randn(n, e, generator=g, device=DEV), k, 1).indices
    # the plan a program keeps as long as its grouping stands: the slots by expert, and where each expert's begin
    flat = expert.reshape(-1)
    s["order"] = torch.sort(flat, stable=True).indices.to(torch.int32)
    counts = torch.bincount(flat, minlength=e)
    s["ptr"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    s["used"], s["most"] = counts.nonzero()[:, 0], int(counts.max())
    rows = n * k if case["silu"] else n
    if case["q8"]:
        s["x"], s["xs"] = _to_e4m3(normal(rows, ki, dtype=torch.float32))
        s["w"], s["ws"] = _to_e4m3(normal(e, fo, ki, scale=ki ** -0.5, dtype=torch.float32))
        return s
    s["x"], s["w"], s["b"] = normal(rows, ki), normal(e, fo, ki, scale=ki ** -0.5), normal(e, fo, scale=0.1)
    if case["grad"]:
        s["dy"] = normal(n * k, fo)
    return s


def _species(n, g):
    p = torch.tensor(SPECIES, device=DEV, dtype=torch.float32)
    return torch.multinomial(p, n, replacement=True, generator=g)


def _to_e4m3(v):
    """(values in 8 bits, scale of each row): the row's largest magnitude becomes the type's largest."""
    scale = (v.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (v / scale[..., None]).to(torch.float8_e4m3fn), scale


# ----------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _RUN_OWN[state["case"]["op"]](state)
    with torch.no_grad():
        return _RUN_PLAIN[state["case"]["op"]](state)


def _norm_plain(s):
    c = s["case"]
    t = s["x"].dtype
    a = s["x"] if not c["residual"] else (s["x"].float() + s["r"].float()).to(t)
    x, w = a.float(), s["w"].float()
    rstd = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    y = x * rstd * w
    out = {"s": a} if c["residual"] else {}
    if c["q8"]:
        out["q"], out["scale"] = _to_e4m3(y)
        return out
    out["y"] = y.to(t)
    if c["grad"]:
        dy = s["dy"].float()
        gw = dy * w
        dx = rstd * gw - x * rstd.pow(3) * (gw * x).mean(1, keepdim=True)
        if s["ds"] is not None:
            dx = dx + s["ds"].float()
        out["dx"], out["dw"] = dx.to(t), (dy * x * rstd).sum(0).to(t)
    return out


def _route_plain(s):
    c = s["case"]
    n, e, k = c["rows"], c["experts"], c["k"]
    l = s["logits"].float()
    if c["species"]:
        l = l.masked_fill(~s["allowed"][s["group"].long()], -math.inf)
    top, at = torch.sort(l, dim=1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    fits = top > -math.inf
    ex = torch.exp(l - top[:, :1])
    p = ex / ex.sum(1, keepdim=True)
    w = torch.where(fits, p.gather(1, at), 0.0)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    expert = torch.where(fits, at, -1).to(torch.int32)
    flat = expert.reshape(-1)
    flat = torch.where(flat < 0, e, flat)
    order = torch.sort(flat, stable=True).indices.to(torch.int32)
    counts = (flat[:, None] == torch.arange(e, device=DEV, dtype=torch.int32)).sum(0)
    ptr = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    out = {"expert": expert, "weight": w, "order": order, "ptr": ptr}
    if c["grad"]:
        g = torch.where(fits, s["dweight"], 0.0)
        mean = (w * g).sum(1, keepdim=True)
        if c["renorm"]:
            d = torch.zeros_like(l).scatter_add_(1, at, w * (g - mean))
        else:
            d = p * (torch.zeros_like(l).scatter_add_(1, at, g) - mean)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _linear_plain(s):
    """The rows of every expert that has some, padded to the most that one has, and one batched product."""
    c = s["case"]
    used, ki, fo, k, most = s["used"], c["n_in"], c["n_out"], c["k"], s["most"]
    order, begin, end = s["order"].long(), s["ptr"].long()[used], s["ptr"].long()[used + 1]
    e, a = used.numel(), order.numel()
    group = torch.bucketize(torch.arange(a, device=DEV), end, right=True)
    place = group * most + torch.arange(a, device=DEV) - begin[group]                 # row of the padded blocks
    row = order if c["silu"] else torch.div(order, k, rounding_mode="floor")
    x, w = s["x"].float(), s["w"][used].float()
    if c["q8"]:
        x, w = x * s["xs"][:, None], w * s["ws"][used][:, :, None]
    h = x * torch.sigmoid(x) if c["silu"] else x
    xp = x.new_zeros(e * most, ki).index_copy_(0, place, h[row]).view(e, most, ki)
    yp = torch.bmm(xp, w.transpose(1, 2))
    if c["q8"]:
        y = yp.view(e * most, fo)[place]
        return {"y": torch.empty_like(y).index_copy_(0, order, y).to(TYPES[c["dtype"]])}
    y = (yp + s["b"][used].float()[:, None]).view(e * most, fo)[place]
    t = s["x"].dtype
    out = {"y": torch.empty_like(y).index_copy_(0, order, y).to(t)}
    if c["grad"]:
        dyp = x.new_zeros(e * most, fo).index_copy_(0, place, s["dy"].float()[order]).view(e, most, fo)
        dxp = torch.bmm(dyp, w).view(e * most, ki)[place]
        dx = torch.empty_like(dxp).index_copy_(0, order, dxp)
        if c["silu"]:
            sg = torch.sigmoid(x)
            dx = dx * (sg * (1 + x * (1 - sg)))
        else:
            dx = dx.view(c["rows"], k, ki).sum(1)
        out["dx"] = dx.to(t)
        dw = torch.bmm(dyp.transpose(1, 2).contiguous(), xp).to(t)
        out["dw"] = torch.zeros_like(s["w"]).index_copy_(0, used, dw)
        out["db"] = torch.zeros_like(s["b"]).index_copy_(0, used, dyp.sum(1).to(t))
    return out


def _combine_plain(s):
    c = s["case"]
    n, k, f = c["rows"], c["k"], c["width"]
    t = s["y"].dtype
    y, w = s["y"].float().view(n, k, f), s["weight"]
    out = {"out": (s["r"].float() + (w[:, :, None] * y).sum(1)).to(t)}
    if c["grad"]:
        d = s["dout"].float()
        out["dy"] = (w[:, :, None] * d[:, None]).view(n * k, f).to(t)
        out["dweight"] = (y * d[:, None]).sum(2)
    return out


def _leaf(t):
    return t.detach().requires_grad_(True)


def _norm_own(s):
    E, c = _experts(), s["case"]
    r = s.get("r")
    if c["q8"]:
        o = E.rms_norm_q8(s["x"], s["w"], EPS, residual=r)
        return dict(zip(("q", "scale", "s"), o))
    if not c["grad"]:
        o = E.rms_norm(s["x"], s["w"], EPS, residual=r)
        return {"y": o} if r is None else {"y": o[0], "s": o[1]}
    x, w = _leaf(s["x"]), _leaf(s["w"])
    if r is None:
        y = E.rms_norm(x, w, EPS)
        dx, dw = torch.autograd.grad([y], [x, w], [s["dy"]])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y, a = E.rms_norm(x, w, EPS, residual=r)
    dx, dw = torch.autograd.grad([y, a], [x, w], [s["dy"], s["ds"]])
    return {"y": y.detach(), "s": a.detach(), "dx": dx, "dw": dw}


def _route_own(s):
    E, c = _experts(), s["case"]
    l = _leaf(s["logits"]) if c["grad"] else s["logits"]
    expert, weight = E.route(l, c["k"], allowed=s.get("allowed"), group=s.get("group"), renormalise=c["renorm"])
    plan = E.group_plan(expert, c["experts"])
    out = {"expert": expert, "weight": weight.detach(), "order": plan.order, "ptr": plan.ptr}
    if c["grad"]:
        out["dlogits"], = torch.autograd.grad([weight], [l], [s["dweight"]])
    return out


def _linear_own(s):
    E, c = _experts(), s["case"]
    plan = E.GroupPlan(s["ptr"], s["order"], c["rows"], c["k"])
    if c["q8"]:
        return {"y": E.grouped_linear_q8(s["x"], s["xs"], s["w"], s["ws"], plan, dtype=TYPES[c["dtype"]])}
    op = "silu" if c["silu"] else None
    if not c["grad"]:
        return {"y": E.grouped_linear(s["x"], s["w"], plan, bias=s["b"], x_op=op)}
    x, w, b = _leaf(s["x"]), _leaf(s["w"]), _leaf(s["b"])
    y = E.grouped_linear(x, w, plan, bias=b, x_op=op)
    dx, dw, db = torch.autograd.grad([y], [x, w, b], [s["dy"]])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _combine_own(s):
    E, c = _experts(), s["case"]
    if not c["grad"]:
        return {"out": E.expert_combine(s["y"], s["weight"], residual=s["r"])}
    y, w = _leaf(s["y"]), _leaf(s["weight"])
    o = E.expert_combine(y, w, residual=s["r"])
    dy, dw = torch.autograd.grad([o], [y, w], [s["dout"]])
    return {"out": o.detach(), "dy": dy, "dweight": dw}


_RUN_PLAIN = {"norm": _norm_plain, "route": _route_plain, "linear": _linear_plain, "combine": _combine_plain}
_RUN_OWN = {"norm": _norm_own, "route": _route_own, "linear": _linear_own, "combine": _combine_own}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _norm64, "route": _route64, "linear": _linear64, "combine": _combine64}[case["op"]](s, case)


def _norm64(s, c):
    a = s["x"].double()
    out = {}
    if c["residual"]:
        a = (a + s["r"].double()).to(s["x"].dtype).double()     # the sum is held in the rows' type, by definition
        out["s"] = a
    x = a.requires_grad_(True) if c["grad"] else a
    w = s["w"].double().requires_grad_(c["grad"])
    with torch.set_grad_enabled(c["grad"]):
        y = x / torch.sqrt((x * x).sum(1, keepdim=True) / c["width"] + EPS) * w
    if c["q8"]:
        scale = torch.clamp_min(y.abs().amax(1) / E4M3_MAX, SCALE_MIN)
        return {**out, "q": (y / scale[:, None]).to(torch.float8_e4m3fn).double(), "scale": scale}
    if c["grad"]:
        outs, ups = [y], [s["dy"].double()]
        if c["residual"]:
            outs, ups = outs + [x], ups + [s["ds"].double()]
        with torch.enable_grad():
            out["dx"], out["dw"] = torch.autograd.grad(outs, [x, w], ups)
    out["y"] = y.detach()
    return {k: v.detach() for k, v in out.items()}


def _route64(s, c):
    l = s["logits"].double()
    if c["species"]:
        l = torch.where(s["allowed"][s["group"].long()], l, torch.full_like(l, -math.inf))
    with torch.enable_grad():
        l.requires_grad_(c["grad"])
        at = torch.sort(l.detach(), dim=1, descending=True, stable=True).indices[:, :c["k"]]
        fits = l.detach().gather(1, at) > -math.inf
        p = torch.softmax(l, 1)
        w = torch.where(fits, p.gather(1, at), 0.0)
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
        out = {"expert": None, "weight": w.detach(), "order": None, "ptr": None}
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad([w], [l], [s["dweight"].double()])
    return out


def _linear64(s, c):
    """Expert by expert."""
    ptr = s["ptr"].tolist()
    n, k = c["rows"], c["k"]
    x, w = s["x"].double(), s["w"]
    if c["q8"]:
        x = x * s["xs"].double()[:, None]
    sg = torch.sigmoid(x) if c["silu"] else None
    h = x * sg if c["silu"] else x
    y = x.new_zeros(n * k, c["n_out"])
    dx = torch.zeros_like(x)
    dw, db = [], []
    for e in range(c["experts"]):
        a = s["order"][ptr[e]:ptr[e + 1]].long()
        row = a if c["silu"] else a // k
        we = w[e].double()
        if c["q8"]:
            y[a] = h[row] @ (we * s["ws"][e].double()[:, None]).t()
            continue
        y[a] = h[row] @ we.t() + s["b"][e].double()
        if c["grad"]:
            d = s["dy"][a].double()
            dx.index_add_(0, row, d @ we)
            dw.append(d.t() @ h[row])
            db.append(d.sum(0))
    if not c["grad"]:
        return {"y": y}
    if c["silu"]:
        dx = dx * (sg + x * sg * (1 - sg))
    return {"y": y, "dx": dx, "dw": torch.stack(dw), "db": torch.stack(db)}


def _combine64(s, c):
    n, k, f = c["rows"], c["k"], c["width"]
    w, y = s["weight"].double(), s["y"].double().view(n, k, f)
    out = {"out": s["r"].double() + torch.matmul(w[:, None], y)[:, 0]}
    if c["grad"]:
        d = s["dout"].double()
        out["dy"] = (w[:, :, None] * d[:, None, :]).reshape(n * k, f)
        out["dweight"] = torch.matmul(y, d[:, :, None])[:, :, 0]
    return out
