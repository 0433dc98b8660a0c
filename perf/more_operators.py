"""More operators of layers over atom rows, as measurable cases.

What a model built of the expert layer needs around it: rows of a table by species or pair of species, with
the gradient summed in a fixed order (embed), the layer norm with the residual, trained and served (layer_norm,
layer_norm_q8), rows laid out by expert and joined again (expert_dispatch, expert_return), the gated activation
(gated_silu), and rows kept in 8 bits for the backward (pack_rows, unpack_rows, keep8).

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
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E4M3_MAX, SCALE_MIN, BLOCK = 448.0, 2.0 ** -126, 32
OPS = ("norm", "embed", "sort", "gate", "pack")


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
        # the same of 100,000 atoms, C = 256, in 16 bits, normalised rows kept in 8 bits between the directions
        _norm("norm_keep8_100k_c256", 100000, 2304, "bf16", grad=True, keep8=True),
        # the species rows of one molecule, trained: latency of both directions
        _embed("embed_molecule21_c96", 21, 3, 96, "f32", grad=True),
        # the species rows of 100,000 atoms, three species: gradients that share their rows 30,000 times
        _embed("embed_species_100k_c256", 100000, 3, 256, "bf16", grad=True),
        # rows for the neighbour pairs of a crystal's many elements (119 squared), a million pairs, trained
        _embed("embed_pairs_1m", 1000000, 14161, 64, "f32", grad=True),
        # the rows of one molecule to two of eight experts and back: latency
        _sort("sort_molecule21_c96", 21, 2, 8, 96, "f32"),
        # the same of 100,000 atoms, C = 256, some choices closed, both directions
        _sort("sort_train_100k_c256", 100000, 2, 8, 2304, "bf16", closed=True, grad=True),
        # the hidden rows of one molecule through the gate, an odd width: latency of both directions
        _gate("gate_molecule21", 42, 97, "f32", grad=True),
        # hidden rows of 100,000 atoms through two experts, trained in 16 bits, inputs kept in 8 bits
        _gate("gate_keep8_100k", 200000, 512, "bf16", grad=True, keep8=True),
        # the input rows of a layer of 24,000 atoms kept in 8 bits and read again
        _pack("pack_24k_c160", 24000, 1440, "f32"),
        # the same of 100,000 atoms, C = 256, in 16 bits
        _pack("pack_100k_c256", 100000, 2304, "bf16"),
    ]


def _norm(name, rows, width, dtype, residual=True, grad=False, q8=False, keep8=False):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "grad": grad,
            "q8": q8, "keep8": keep8}


def _embed(name, rows, vocab, width, dtype, grad=False):
    return {"name": name, "op": "embed", "rows": rows, "vocab": vocab, "width": width, "dtype": dtype, "grad": grad}


def _sort(name, rows, k, experts, width, dtype, closed=False, grad=False):
    return {"name": name, "op": "sort", "rows": rows, "k": k, "experts": experts, "width": width, "dtype": dtype,
            "closed": closed, "grad": grad}


def _gate(name, rows, width, dtype, grad=False, keep8=False):
    return {"name": name, "op": "gate", "rows": rows, "width": width, "dtype": dtype, "grad": grad, "keep8": keep8}


def _pack(name, rows, width, dtype):
    return {"name": name, "op": "pack", "rows": rows, "width": width, "dtype": dtype}


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: atoms from one to 100,000 (pairs to a million), widths of a model's readout, odd ones too."""
    most = max(_cost(c) for c in listed())
    while True:
        op, dtype, grad = rng.choice(OPS), rng.choice(list(TYPES)), rng.random() < 0.6
        if op == "norm":
            c = _norm(None, _log(rng, 1, 100000), _log(rng, 16, 4096), dtype, rng.random() < 0.7, grad)
            c["q8"] = not grad and rng.random() < 0.4
            # rows of 32 bits are kept as they are: what rounds to 8 bits after a norm hangs on its last bits
            c["keep8"] = grad and dtype != "f32" and rng.random() < 0.5
        elif op == "embed":
            c = _embed(None, _log(rng, 1, 1000000), _log(rng, 2, 20000), _log(rng, 8, 2304), dtype, grad)
        elif op == "sort":
            experts = _log(rng, 2, 64)
            c = _sort(None, _log(rng, 1, 100000), rng.randint(1, min(4, experts)), experts, _log(rng, 16, 2304), dtype,
                      rng.random() < 0.5, grad)
        elif op == "gate":
            c = _gate(None, _log(rng, 1, 200000), _log(rng, 8, 2304), dtype, grad, grad and rng.random() < 0.5)
        else:
            c = _pack(None, _log(rng, 1, 100000), _log(rng, 16, 4096), dtype)
        del c["name"]
        if _cost(c) <= most:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    op, n, f = case["op"], case["rows"], case["width"]
    z = SIZE[case["dtype"]]
    kept = 1 + 1 / BLOCK                                                             # bytes of a value in 8 bits
    if op == "norm":
        parts = (1 + 2 * case["residual"]) * z + (1 if case["q8"] else z)            # x, residual, sum; the result
        b = n * f * parts + 2 * f * z + (4 * n if case["q8"] else 0)
        if case["grad"]:                                                             # rows, dy, ds in; dx, dw, db out
            rows = 2 * kept if case["keep8"] else z                                  # kept ones are written and read
            b += n * f * (rows + z * (2 + case["residual"])) + 4 * f * z
        return {"bytes": b, "flops": n * f * (8 + 14 * case["grad"])}
    if op == "embed":
        used = min(case["vocab"], n)
        b = used * f * z + n * f * z + 4 * n
        if case["grad"]:
            b += n * f * z + case["vocab"] * f * z + 4 * n
        return {"bytes": b, "flops": n * f * (1 + case["grad"])}
    if op == "sort":
        a = n * case["k"]
        b = n * f * z + a * f * z + 4 * a                                            # dispatch
        b += a * f * z + 2 * n * f * z + 8 * a                                       # return
        if case["grad"]:
            b += a * f * z + n * f * z + 4 * a                                       # dx
            b += n * f * z + 2 * a * f * z + 12 * a                                  # dout, y; dy, dweight
        return {"bytes": b, "flops": a * f * (2 + 4 * case["grad"])}
    if op == "gate":
        b = 3 * n * f * z
        if case["grad"]:
            b += 2 * n * f * (2 * kept if case["keep8"] else z) + 3 * n * f * z
        return {"bytes": b, "flops": n * f * (6 + 12 * case["grad"])}
    return {"bytes": 2 * n * f * (z + kept), "flops": 4 * n * f}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, n, f, op = TYPES[case["dtype"]], case["rows"], case["width"], case["op"]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {"case": case}
    if op == "norm":
        s["x"] = (torch.randn(n, f, generator=g, device=DEV) + 0.3).to(t)             # invariants have a mean
        s["w"] = (1 + 0.1 * torch.randn(f, generator=g, device=DEV)).to(t)
        s["b"] = normal(f, scale=0.1)
        if case["residual"]:
            s["r"] = normal(n, f, scale=3.0)
        if case["grad"]:
            s["dy"], s["ds"] = normal(n, f), (normal(n, f) if case["residual"] else None)
    elif op == "embed":
        v = case["vocab"]
        s["table"], s["scale"] = normal(v, f), math.sqrt(f)
        # some entries are frequent, most are rare
        p = torch.exp(1.5 * torch.randn(v, generator=g, device=DEV))
        s["index"] = torch.multinomial(p, n, replacement=True, generator=g).to(torch.int32)
        if case["grad"]:
            s["dy"] = normal(n, f)
    elif op == "sort":
        k, e = case["k"], case["experts"]
        bias = 0.7 * torch.randn(e, generator=g, device=DEV)                          # some experts draw more rows
        logits = bias + torch.randn(n, e, generator=g, device=DEV)
        top, expert = torch.topk(logits, k, 1)
        s["weight"] = torch.softmax(top, 1)
        if case["closed"]:                                                            # a choice that could not be filled
            shut = torch.rand(n, k, generator=g, device=DEV) < 0.05
            expert = torch.where(shut, e, expert)
            s["weight"] = torch.where(shut, 0.0, s["weight"])
        # the plan that route and group_plan leave in hand: the slots by expert, and where each expert's begin
        flat = expert.reshape(-1)
        s["order"] = torch.sort(flat, stable=True).indices.to(torch.int32)
        counts = torch.bincount(flat, minlength=e + 1)[:e]
        s["ptr"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["x"], s["r"], s["y"] = normal(n, f), normal(n, f), normal(n * k, f)
        if case["grad"]:
            s["dxs"], s["dout"] = normal(n * k, f), normal(n, f)
    elif op == "gate":
        s["x"] = normal(n, 2 * f, scale=1.5)
        if case["grad"]:
            s["dy"] = normal(n, f)
    else:
        spread = torch.exp(0.7 * torch.randn(f, generator=g, device=DEV))             # columns of other sizes
        s["x"] = (torch.randn(n, f, generator=g, device=DEV) * spread).to(t)
    return s


# ----------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _RUN_OWN[state["case"]["op"]](state)
    with torch.no_grad():
        return _RUN_PLAIN[state["case"]["op"]](state)


def _kept_plain(v):
    """float32 rows as 8 bits hold them: e4m3 with a power of two for each 32 columns, the least that keeps the
    largest magnitude within 448."""
    f = v.shape[-1]
    pad = -f % BLOCK
    b = torch.nn.functional.pad(v, (0, pad)).unflatten(-1, (-1, BLOCK))
    bits = b.abs().amax(-1, keepdim=True).view(torch.int32)
    e = ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000)).clamp_min(1)              # exponent + 127
    up, down = (e << 23).view(torch.float32), ((254 - e) << 23).view(torch.float32)
    return ((b * down).to(torch.float8_e4m3fn).float() * up).flatten(-2)[..., :f]


def _norm_plain(s):
    c = s["case"]
    t = s["x"].dtype
    a = s["x"] if not c["residual"] else (s["x"].float() + s["r"].float()).to(t)
    x, w, b = a.float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(xc.square().mean(1, keepdim=True) + EPS)
    xh = xc * rstd
    y = xh * w + b
    out = {"s": a} if c["residual"] else {}
    if c["q8"]:
        scale = (y.abs().amax(1) / E4M3_MAX).clamp_min(SCALE_MIN)
        out["q"], out["scale"] = (y / scale[:, None]).to(torch.float8_e4m3fn), scale
        return out
    out["y"] = y.to(t)
    if c["grad"]:
        if c["keep8"]:
            xh = _kept_plain(xh)
        dy = s["dy"].float()
        gw = dy * w
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        if s["ds"] is not None:
            dx = dx + s["ds"].float()
        out["dx"], out["dw"], out["db"] = dx.to(t), (dy * xh).sum(0).to(t), dy.sum(0).to(t)
    return out


def _embed_plain(s):
    c = s["case"]
    t, i = s["table"].dtype, s["index"].long()
    out = {"y": (s["table"][i].float() * s["scale"]).to(t)}
    if c["grad"]:
        dy = s["dy"].float()
        if c["vocab"] <= 64:                                                          # few entries: one product
            one = (torch.arange(c["vocab"], device=DEV)[:, None] == i[None]).float()
            d = one @ dy
        else:
            d = dy.new_zeros(c["vocab"], c["width"]).index_add_(0, i, dy)
        out["dtable"] = (d * s["scale"]).to(t)
    return out


def _sort_plain(s):
    c = s["case"]
    n, k, f = c["rows"], c["k"], c["width"]
    t, a, order = s["x"].dtype, n * k, s["order"].long()
    open_ = torch.arange(a, device=DEV) < s["ptr"][-1]                                # places of an expert
    row = torch.div(order, k, rounding_mode="floor")
    out = {"xs": torch.where(open_[:, None], s["x"][row], 0)}
    place = torch.empty_like(order)
    place[order] = torch.arange(a, device=DEV)
    fits = open_[place].view(n, k, 1)
    w = s["weight"][:, :, None]
    y = torch.where(fits, s["y"][place].view(n, k, f).float(), 0.0)
    out["out"] = (s["r"].float() + (w * y).sum(1)).to(t)
    if c["grad"]:
        out["dx"] = torch.where(fits, s["dxs"][place].view(n, k, f).float(), 0.0).sum(1).to(t)
        d = s["dout"].float()
        dy = (w * d[:, None]).view(a, f).to(t)
        out["dy"] = torch.where(open_[:, None], dy[order], 0)
        out["dweight"] = (y * d[:, None]).sum(2)
    return out


def _gate_plain(s):
    c = s["case"]
    n, f = c["rows"], c["width"]
    t = s["x"].dtype
    x = s["x"].float().view(n, 2, f)
    out = {"y": (x[:, 0] * torch.sigmoid(x[:, 0]) * x[:, 1]).to(t)}
    if c["grad"]:
        if c["keep8"]:
            x = _kept_plain(x)
        a, b, d = x[:, 0], x[:, 1], s["dy"].float()
        sg = torch.sigmoid(a)
        out["dx"] = torch.cat([d * b * (sg * (1 + a * (1 - sg))), d * a * sg], 1).to(t)
    return out


def _pack_plain(s):
    return {"x": _kept_plain(s["x"].float()).to(s["x"].dtype)}


def _leaf(t):
    return t.detach().requires_grad_(True)


def _norm_own(s):
    E, c = _experts(), s["case"]
    r = s.get("r")
    if c["q8"]:
        o = E.layer_norm_q8(s["x"], s["w"], s["b"], EPS, residual=r)
        return dict(zip(("q", "scale", "s"), o))
    if not c["grad"]:
        o = E.layer_norm(s["x"], s["w"], s["b"], EPS, residual=r)
        return {"y": o} if r is None else {"y": o[0], "s": o[1]}
    x, w, b = _leaf(s["x"]), _leaf(s["w"]), _leaf(s["b"])
    if r is None:
        y = E.layer_norm(x, w, b, EPS, keep8=c["keep8"])
        dx, dw, db = torch.autograd.grad([y], [x, w, b], [s["dy"]])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    y, a = E.layer_norm(x, w, b, EPS, residual=r, keep8=c["keep8"])
    dx, dw, db = torch.autograd.grad([y, a], [x, w, b], [s["dy"], s["ds"]])
    return {"y": y.detach(), "s": a.detach(), "dx": dx, "dw": dw, "db": db}


def _embed_own(s):
    E, c = _experts(), s["case"]
    if not c["grad"]:
        return {"y": E.embed(s["table"], s["index"], s["scale"])}
    table = _leaf(s["table"])
    y = E.embed(table, s["index"], s["scale"])
    d, = torch.autograd.grad([y], [table], [s["dy"]])
    return {"y": y.detach(), "dtable": d}


def _sort_own(s):
    E, c = _experts(), s["case"]
    plan = E.GroupPlan(s["ptr"], s["order"], c["rows"], c["k"])
    if not c["grad"]:
        return {"xs": E.expert_dispatch(s["x"], plan), "out": E.expert_return(s["y"], plan, s["weight"], residual=s["r"])}
    x, y, w = _leaf(s["x"]), _leaf(s["y"]), _leaf(s["weight"])
    xs = E.expert_dispatch(x, plan)
    o = E.expert_return(y, plan, w, residual=s["r"])
    dx, dy, dw = torch.autograd.grad([xs, o], [x, y, w], [s["dxs"], s["dout"]])
    return {"xs": xs.detach(), "out": o.detach(), "dx": dx, "dy": dy, "dweight": dw}


def _gate_own(s):
    E, c = _experts(), s["case"]
    if not c["grad"]:
        return {"y": E.gated_silu(s["x"])}
    x = _leaf(s["x"])
    y = E.gated_silu(x, keep8=c["keep8"])
    dx, = torch.autograd.grad([y], [x], [s["dy"]])
    return {"y": y.detach(), "dx": dx}


def _pack_own(s):
    E = _experts()
    q, scale = E.pack_rows(s["x"])
    return {"x": E.unpack_rows(q, scale, s["x"].dtype)}


_RUN_PLAIN = {"norm": _norm_plain, "embed": _embed_plain, "sort": _sort_plain, "gate": _gate_plain, "pack": _pack_plain}
_RUN_OWN = {"norm": _norm_own, "embed": _embed_own, "sort": _sort_own, "gate": _gate_own, "pack": _pack_own}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm64, "embed": _embed64, "sort": _sort64, "gate": _gate64, "pack": _pack64}[case["op"]](s, case)


def _kept64(v):
    n, f = v.shape
    m = -(-f // BLOCK)
    full = v.new_zeros(n, m * BLOCK)
    full[:, :f] = v
    blocks = full.view(n, m, BLOCK)
    part, e = torch.frexp(blocks.abs().max(2, keepdim=True).values)                   # top = part 2^e, part in [1/2, 1)
    e = torch.where(part <= 0.875, e - 9, e - 8).clamp(min=-126)                      # 448 = 0.875 2^9
    unit = torch.pow(torch.full_like(part, 2.0), e)
    return ((blocks / unit).to(torch.float8_e4m3fn).double() * unit).view(n, -1)[:, :f]


def _norm64(s, c):
    t = s["x"].dtype
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    out = {}
    if c["residual"]:
        x = (x + s["r"].double()).to(t).double()                # the sum is held in the rows' type, by definition
        out["s"] = x
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    xh = (x - mean) / sd
    y = xh * w + b
    if c["q8"]:
        scale = torch.clamp_min(y.abs().amax(1) / E4M3_MAX, SCALE_MIN)
        return {**out, "q": (y / scale[:, None]).to(torch.float8_e4m3fn).double(), "scale": scale}
    out["y"] = y
    if c["grad"]:
        if c["keep8"]:
            xh = _kept64(xh)
        dy, f = s["dy"].double(), c["width"]
        g = dy * w
        # the gradient's parts along the row of ones and along the normalised row are taken out
        dx = (g - (g.sum(1, keepdim=True) + xh * (g * xh).sum(1, keepdim=True)) / f) / sd
        out["dx"] = dx if s["ds"] is None else dx + s["ds"].double()
        out["dw"], out["db"] = (dy * xh).sum(0), dy.sum(0)
    return out


def _embed64(s, c):
    i = s["index"].long()
    out = {"y": s["table"].double().index_select(0, i) * s["scale"]}
    if c["grad"]:
        d = torch.zeros(c["vocab"], c["width"], dtype=torch.float64, device=DEV)
        out["dtable"] = d.index_add_(0, i, s["dy"].double()) * s["scale"]
    return out


def _sort64(s, c):
    n, k, f = c["rows"], c["k"], c["width"]
    m = int(s["ptr"][-1])
    a = s["order"][:m].long()                                                         # the slots of an expert
    i = a // k
    x, w = s["x"].double(), s["weight"].double().reshape(-1)[a]
    xs, o, y = x.new_zeros(n * k, f), s["r"].double(), s["y"][:m].double()
    xs[:m] = x[i]
    out = {"xs": xs, "out": o.index_add(0, i, y * w[:, None])}
    if c["grad"]:
        d = s["dout"].double()[i]
        dy, dw = torch.zeros_like(xs), x.new_zeros(n * k)
        dy[:m] = d * w[:, None]
        dw[a] = (d * y).sum(1)
        out["dx"] = torch.zeros_like(x).index_add_(0, i, s["dxs"][:m].double())
        out["dy"], out["dweight"] = dy, dw.view(n, k)
    return out


def _gate64(s, c):
    f = c["width"]
    x = s["x"].double()
    a, b = x[:, :f], x[:, f:]
    out = {"y": a / (1 + torch.exp(-a)) * b}
    if c["grad"]:
        if c["keep8"]:
            a, b = _kept64(a), _kept64(b)
        d, p = s["dy"].double(), 1 / (1 + torch.exp(-a))
        out["dx"] = torch.cat([d * b * (p + a * p * (1 - p)), d * a * p], 1)
    return out


def _pack64(s, c):
    return {"x": _kept64(s["x"].double())}
