"""Operators of an expert layer over atoms: layers whose weights depend on the atom.

The readout of a FACE model is a norm, linear layers and a residual, the same weights for every
atom. Here the weights are chosen per atom, by its species or by a learned gate (for models built of these
operators: the FACE model itself calls none of them):

    y, s = rms_norm(x, w, eps, residual=r)                s = x + r and its normalised rows
    expert, weight = route(gate, k)                        the k experts of every atom (or its species)
    plan = group_plan(expert, n_experts)                   the rows of each expert
    u = grouped_linear(y, W1, plan, bias=b1)               one row per (atom, choice)
    v = grouped_linear(u, W2, plan, bias=b2, x_op="silu")
    out = expert_combine(v, weight, residual=s)            the choices joined

and, for serving in 8 bits, rms_norm_q8 and quantize_rows in front of grouped_linear_q8.

Rows are float32, bfloat16 or float16 (all tensors of a call alike, gate weights and scales float32); sums,
softmax and norm statistics are float32. Every operator launches the kernels of
libface_hip.so on torch's current stream of its tensors' device, allocates its results and workspaces with torch and never
synchronises; none has a CPU path. They differentiate once, in training too: all of their floating
inputs take gradients, except those of the 8-bit forms. Forward-mode derivatives are refused. Forward and backward are captured into a graph together,
as with torch's own operators on leaves of which no eager graph is alive (fresh ones, by detach().requires_grad_()).
"""
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import call, ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_E4M3 = torch.float8_e4m3fn
_X_OPS = {None: 0, "silu": 1}
MAX_WIDTH = 65536                   # widest row of rms_norm and quantize_rows
MAX_EXPERTS, MAX_K = 1024, 16       # of route; group_plan takes as many groups


def _fail(name, why):
    raise ValueError(f"{name}: {why}")


def _dtype(name, t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        _fail(name, f"float32, bfloat16 or float16 rows, got {t.dtype}")
    return code


def _no_tangents(name, *ts):
    """The kernels see a tensor's values alone: the tangent of a dual tensor would be dropped in silence."""
    if getattr(forward_ad, "_current_level", 0) >= 0:            # else no tensor has one
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name}: no forward-mode derivatives")


def _check(name, ref, **tensors):
    """Every tensor on ref's HIP device, and none with a tangent."""
    _no_tangents(name, ref, *tensors.values())
    _lib.require_gpu(ref, *tensors.values())
    for k, t in tensors.items():
        if t is not None and t.device != ref.device:
            _fail(name, f"{k} is on {t.device}, the rows are on {ref.device}")


def _rows(t, width):
    """t as (rows, width) with unit column stride and rows one after the other: a view where its
    strides allow one, else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if t.stride(1) == 1 and t.stride(0) >= width:
        return t
    return t.clone(memory_format=torch.contiguous_format)


_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(t, name, label, *args):
    """Call entry point `name` with args and the current stream of t's device, as the current device."""
    idx = t.device.index
    if idx == _get_device():
        call(name, *args, _lib.stream_of(t), label=label)
    else:
        with torch.cuda.device(idx):
            call(name, *args, _lib.stream_of(t), label=label)


def _once(name, *grads):
    """A backward that is itself recorded, or whose incoming gradients have tangents, would need second derivatives."""
    _no_tangents(name + "'s gradient", *grads)
    if torch.is_grad_enabled():
        raise NotImplementedError("the expert layer's operators differentiate once (create_graph=False)")


def _like(t):
    """A dense tensor of t's shape and type (half the host time of torch.empty(t.shape, ...))."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _work(n_bytes, device):
    return torch.empty(n_bytes, dtype=torch.uint8, device=device) if n_bytes else None


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ----------------------------------------------------------------------------- norm
def _norm_args(name, x, w, eps, residual):
    code = _dtype(name, x)
    if x.dim() < 1 or w.dim() != 1 or x.shape[-1] != w.shape[0]:
        _fail(name, f"x (..., F) and w (F), got {tuple(x.shape)} and {tuple(w.shape)}")
    if not 1 <= x.shape[-1] <= MAX_WIDTH:
        _fail(name, f"rows of 1 to {MAX_WIDTH} columns, got {x.shape[-1]}")
    if w.dtype != x.dtype:
        _fail(name, f"w of the rows' type {x.dtype}, got {w.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        _fail(name, f"residual like x, {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    if not 0 <= eps < float("inf"):
        _fail(name, f"eps >= 0, got {eps}")
    _check(name, x, w=w, residual=residual)
    return code


def _norm_fwd(code, x, w, eps, r, q8):
    """(y, s) or (q, scale, s); s is None without a residual."""
    F = x.shape[-1]
    x2, w = _rows(x, F), w.contiguous()
    r2 = None if r is None else _rows(r, F)
    N = x2.shape[0]
    s = None if r is None else _like(x)
    y = None if q8 else _like(x)
    q = torch.empty(x.shape, dtype=_E4M3, device=x.device) if q8 else None
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if q8 else None
    _launch(x, "face_rms_norm_fwd", "rms_norm_fwd", x2.data_ptr(), x2.stride(0), ptr(r2), F if r2 is None else r2.stride(0),
            N, F, code, w.data_ptr(), eps, ptr(y), ptr(s), ptr(q), ptr(scale))
    return (q, scale, s) if q8 else (y, s)


class RMSNorm(torch.autograd.Function):
    """Keeps only the rows it normalised: the backward forms their statistics again as it reads them."""

    @staticmethod
    def forward(ctx, x, w, eps, r):
        y, s = _norm_fwd(_DTYPES[x.dtype], x, w, eps, r, False)
        ctx.save_for_backward(x if s is None else s, w)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    def backward(ctx, dy, ds=None):
        _once("rms_norm", dy, ds)
        need_x, need_w, _, need_r = ctx.needs_input_grad
        if dy is None and ds is None:
            return None, None, None, None
        s, w = ctx.saved_tensors
        F, code = s.shape[-1], _DTYPES[s.dtype]
        s2, w = _rows(s, F), w.contiguous()
        N = s2.shape[0]
        if dy is not None:
            dy = _rows(dy, F)
        if ds is not None:
            ds = _rows(ds, F)
        dx = _like(s) if need_x or need_r else None
        dw = work = None
        need = 0
        if need_w:
            dw = torch.empty_like(w)
            need = _lib.lib().face_rms_norm_bwd_work(N, F)
            work = _work(need, s.device)
        _launch(s, "face_rms_norm_bwd", "rms_norm_bwd", s2.data_ptr(), s2.stride(0), ptr(dy), F if dy is None else dy.stride(0),
                ptr(ds), F if ds is None else ds.stride(0), N, F, code, w.data_ptr(), ctx.eps, ptr(dx), ptr(dw), ptr(work), need)
        return dx if need_x else None, dw, None, dx if need_r else None


def rms_norm(x, w, eps=1e-6, residual=None):
    """x (..., F), w (F) -> x w / sqrt(mean(x^2) + eps) over the last axis. With residual (like x): (that of
    s, s) for s = x + residual, rounded to the rows' type before it is normalised. F <= MAX_WIDTH; the squares of a
    row are summed in float32."""
    eps = float(eps)
    code = _norm_args("rms_norm", x, w, eps, residual)
    if _wants_grad(x, w, residual):
        return RMSNorm.apply(x, w, eps, residual)
    y, s = _norm_fwd(code, x, w, eps, residual, False)
    return y if s is None else (y, s)


@torch.no_grad()
def rms_norm_q8(x, w, eps=1e-6, residual=None):
    """rms_norm whose normalised rows leave in 8 bits, for serving: (q (..., F) float8_e4m3fn, scale (...)
    float32), and s with a residual. A row stands for q * scale, its largest magnitude for 448 * scale (scale
    >= 2^-126); a row with a NaN gets a NaN scale. No gradients."""
    eps = float(eps)
    code = _norm_args("rms_norm_q8", x, w, eps, residual)
    q, scale, s = _norm_fwd(code, x, w, eps, residual, True)
    return (q, scale) if s is None else (q, scale, s)


@torch.no_grad()
def quantize_rows(x, x_op=None):
    """x (..., F) -> (q float8_e4m3fn, scale (...) float32) of op(x), x_op None or "silu", each row scaled as in
    rms_norm_q8: hidden rows between two 8-bit layers, or weights (G, n, k) laid out once. No gradients."""
    code = _dtype("quantize_rows", x)
    if x_op not in _X_OPS:
        _fail("quantize_rows", f"x_op None or 'silu', got {x_op!r}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        _fail("quantize_rows", f"rows of 1 to {MAX_WIDTH} columns, got {tuple(x.shape)}")
    _check("quantize_rows", x)
    F = x.shape[-1]
    x2 = _rows(x, F)
    q = torch.empty(x.shape, dtype=_E4M3, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _launch(x, "face_quantize_rows", "quantize_rows", x2.data_ptr(), x2.stride(0), x2.shape[0], F, code, _X_OPS[x_op],
            q.data_ptr(), scale.data_ptr())
    return q, scale


# ----------------------------------------------------------------------------- gate and grouping
def _route_fwd(logits, k, allowed, group, renorm):
    N, E = logits.shape
    l2 = _rows(logits, E)
    expert = torch.empty(N, k, dtype=torch.int32, device=logits.device)
    weight = torch.empty(N, k, dtype=torch.float32, device=logits.device)
    _launch(logits, "face_route_fwd", "route_fwd", l2.data_ptr(), l2.stride(0), N, E, k, _DTYPES[logits.dtype], ptr(allowed),
            ptr(group), 0 if allowed is None else allowed.shape[0], int(renorm), expert.data_ptr(), weight.data_ptr())
    return expert, weight


class Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, allowed, group, renorm):
        expert, weight = _route_fwd(logits, k, allowed, group, renorm)
        ctx.save_for_backward(logits, allowed, group, expert, weight)
        ctx.k, ctx.renorm = k, renorm
        ctx.mark_non_differentiable(expert)
        ctx.set_materialize_grads(False)
        return expert, weight

    @staticmethod
    def backward(ctx, _, dweight):
        _once("route", dweight)
        if dweight is None:
            return None, None, None, None, None
        logits, allowed, group, expert, weight = ctx.saved_tensors
        N, E = logits.shape
        l2, dweight = _rows(logits, E), dweight.contiguous()
        dl = torch.empty(N, E, dtype=logits.dtype, device=logits.device)
        _launch(logits, "face_route_bwd", "route_bwd", l2.data_ptr(), l2.stride(0), N, E, ctx.k, _DTYPES[logits.dtype],
                ptr(allowed), ptr(group), 0 if allowed is None else allowed.shape[0], int(ctx.renorm), expert.data_ptr(),
                weight.data_ptr(), dweight.data_ptr(), dl.data_ptr())
        return dl, None, None, None, None


def route(logits, k, allowed=None, group=None, renormalise=True):
    """logits (N, E) -> (expert (N, k) int32, weight (N, k) float32): the k largest logits of a row in
    descending order, ties to the lower expert, and their softmax weights, over the chosen experts
    (renormalise) or over all that are open to the row.

    allowed (G, E) bool opens experts to rows by group (N,) int32 (a species, say; without group G = 1, the same
    for all); a row whose group lies outside [0, G) has none. A logit of -inf closes its expert too. What a row
    cannot fill has expert -1 and weight 0. A NaN counts as the largest logit and makes the row's weights NaN.
    Differentiable in the logits through the weights. E <= MAX_EXPERTS, k <= min(E, MAX_K)."""
    _dtype("route", logits)
    if logits.dim() != 2:
        _fail("route", f"logits (N, E), got {tuple(logits.shape)}")
    N, E = logits.shape
    k = int(k)
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_K):
        _fail("route", f"1 <= k <= min(E, {MAX_K}) and E <= {MAX_EXPERTS}, got k = {k}, E = {E}")
    if allowed is None:
        if group is not None:
            _fail("route", "group without allowed")
    else:
        if allowed.dtype != torch.bool or allowed.dim() != 2 or allowed.shape[1] != E or allowed.shape[0] < 1:
            _fail("route", f"allowed (G, {E}) bool, got {tuple(allowed.shape)} {allowed.dtype}")
        if group is None:
            if allowed.shape[0] != 1:
                _fail("route", "allowed of several groups needs group (N,)")
        elif group.dtype != torch.int32 or group.shape != (N,):
            _fail("route", f"group ({N},) int32, got {tuple(group.shape)} {group.dtype}")
    _check("route", logits, allowed=allowed, group=group)
    allowed = None if allowed is None else allowed.contiguous()
    group = None if group is None else group.contiguous()
    if _wants_grad(logits):
        return Route.apply(logits, k, allowed, group, bool(renormalise))
    return _route_fwd(logits, k, allowed, group, renormalise)


class GroupPlan:
    """Slots 0 .. rows * k - 1, slot i * k + j the j-th choice of row i, sorted by group: order (rows * k,) int32,
    and ptr (G + 1,) int32, where each group's begin in it; the slots behind ptr[G] belong to none.

    Made by group_plan, or from tensors that a program keeps (rows that stay grouped: species). Ranges
    and slots are bounds-checked on the device: what lies outside is left out. Each slot has one place in
    order; rows of a slot that has none are not written."""

    __slots__ = ("ptr", "order", "rows", "k")

    def __init__(self, ptr, order, rows, k=1):
        rows, k = int(rows), int(k)
        if k < 1 or rows < 0 or rows * k >= 1 << 31:
            _fail("GroupPlan", f"rows >= 0, k >= 1 and rows * k < 2^31, got {rows} and {k}")
        for name, t in (("ptr", ptr), ("order", order)):
            if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                _fail("GroupPlan", f"{name}: a contiguous int32 vector, got {tuple(t.shape)} {t.dtype}")
        if ptr.shape[0] < 2 or order.shape[0] != rows * k:
            _fail("GroupPlan", f"ptr (G + 1,) and order ({rows * k},), got {tuple(ptr.shape)} and {tuple(order.shape)}")
        if ptr.device != order.device:
            _fail("GroupPlan", f"ptr on {ptr.device}, order on {order.device}")
        self.ptr, self.order, self.rows, self.k = ptr, order, rows, k

    @property
    def n_groups(self):
        return self.ptr.shape[0] - 1

    @property
    def slots(self):
        return self.rows * self.k


@torch.no_grad()
def group_plan(expert, n_groups):
    """expert (N,) or (N, k) int32 (int64 too), the group of every row or of each of its k choices -> GroupPlan: a
    stable sort of the slots by group; values outside [0, n_groups) belong to none. n_groups <= MAX_EXPERTS."""
    n_groups = int(n_groups)
    if expert.dim() not in (1, 2) or expert.dim() == 2 and expert.shape[1] < 1:
        _fail("group_plan", f"expert (N,) or (N, k), got {tuple(expert.shape)}")
    if not 1 <= n_groups <= MAX_EXPERTS:
        _fail("group_plan", f"1 <= n_groups <= {MAX_EXPERTS}, got {n_groups}")
    if expert.dtype == torch.int64:
        expert = expert.clamp(-1, n_groups).to(torch.int32)
    elif expert.dtype != torch.int32:
        _fail("group_plan", f"int32 or int64 groups, got {expert.dtype}")
    _check("group_plan", expert)
    e = expert.contiguous()
    slots = e.numel()
    if slots >= 1 << 31:
        _fail("group_plan", f"fewer than 2^31 slots, got {slots}")
    p = torch.empty(n_groups + 1, dtype=torch.int32, device=e.device)
    order = torch.empty(slots, dtype=torch.int32, device=e.device)
    need = _lib.lib().face_group_plan_work(slots, n_groups)
    work = _work(need, e.device)
    _launch(e, "face_group_plan", "group_plan", e.data_ptr(), slots, n_groups, p.data_ptr(), order.data_ptr(), ptr(work), need)
    return GroupPlan(p, order, e.shape[0], 1 if e.dim() == 1 else e.shape[1])


# ----------------------------------------------------------------------------- products by group
def _weights(w):
    """w (G, n, k) with unit last stride and rows one after the other."""
    if w.stride(2) != 1 and w.shape[2] > 1 or w.stride(1) < w.shape[2] or w.stride(0) < 0:
        w = w.clone(memory_format=torch.contiguous_format)
    return w


def _div(plan, rows):
    """Slots per row of an operand."""
    return 1 if rows == plan.slots else plan.k


def _linear_args(name, x, w, plan, bias, out_dtype):
    if not isinstance(plan, GroupPlan):
        _fail(name, f"plan: a GroupPlan, got {type(plan).__name__}")
    if x.dim() != 2 or w.dim() != 3 or w.shape[2] != x.shape[1] or w.shape[1] < 1 or w.shape[2] < 1:
        _fail(name, f"x (rows, k) and w (G, n, k), got {tuple(x.shape)} and {tuple(w.shape)}")
    if w.shape[0] != plan.n_groups:
        _fail(name, f"w of the plan's {plan.n_groups} groups, got {w.shape[0]}")
    if x.shape[0] not in (plan.rows, plan.slots):
        _fail(name, f"x of {plan.rows} rows or {plan.slots} slots, got {x.shape[0]}")
    if w.dtype != x.dtype:
        _fail(name, f"w of the rows' type {x.dtype}, got {w.dtype}")
    if bias is not None and (bias.shape != w.shape[:2] or bias.dtype != out_dtype):
        _fail(name, f"bias {tuple(w.shape[:2])} {out_dtype}, got {tuple(bias.shape)} {bias.dtype}")


def _linear_fwd(x, w, plan, bias, op):
    G, n, k = w.shape
    x2, w, b = _rows(x, k), _weights(w), None if bias is None else bias.contiguous()
    y = torch.empty(plan.slots, n, dtype=x.dtype, device=x.device)
    _launch(x, "face_grouped_linear", "grouped_linear_fwd", x2.data_ptr(), x2.stride(0), _div(plan, x.shape[0]), op,
            w.data_ptr(), w.stride(1), w.stride(0), ptr(b), n, plan.ptr.data_ptr(), plan.order.data_ptr(), plan.slots, G, n, k,
            _DTYPES[x.dtype], y.data_ptr(), n)
    return y


class GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, p, order, plan, op):
        y = _linear_fwd(x, w, plan, bias, op)
        ctx.save_for_backward(x, w, p, order)
        ctx.plan, ctx.op = plan, op
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    def backward(ctx, dy):
        _once("grouped_linear", dy)
        if dy is None:
            return (None,) * 7
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x, w, p, order = ctx.saved_tensors
        dtype, dev, code = x.dtype, x.device, _DTYPES[x.dtype]
        G, n, k = w.shape
        slots = order.shape[0]
        div = _div(ctx.plan, x.shape[0])
        x2, dy, w2 = _rows(x, k), _rows(dy, n), _weights(w)
        dx = _like(x) if need_x else None
        db = torch.empty(G, n, dtype=dtype, device=dev) if need_b else None

        def launch(k, op, dx, dw, db):
            need = _lib.lib().face_grouped_linear_bwd_work(slots, n, k, code, div, dx is not None, dw is not None, db is not None)
            work = _work(need, dev)
            _launch(x, "face_grouped_linear_bwd", "grouped_linear_bwd", x2.data_ptr(), x2.stride(0), div, op, dy.data_ptr(),
                    dy.stride(0), w2.data_ptr(), w2.stride(1), w2.stride(0), p.data_ptr(), order.data_ptr(), slots, G, n, k, code,
                    ptr(dx), ptr(dw), ptr(db), ptr(work), need)

        if need_w or not need_b:
            dw = torch.empty(G, n, k, dtype=dtype, device=dev) if need_w else None
            launch(k, ctx.op, dx, dw, db)
        else:                                        # db comes with dw: that of eight columns, not of all
            dw = None
            if need_x:
                launch(k, ctx.op, dx, None, None)
            few = min(k, 8)
            launch(few, 0, None, torch.empty(G, n, few, dtype=dtype, device=dev), db)
        return dx, dw, db, None, None, None, None


def grouped_linear(x, w, plan, bias=None, x_op=None):
    """y (plan.slots, n), y[a] = op(x[row(a)]) w[g]^T + bias[g] for the slots a of group g, 0 for slots of no group.

    x (plan.rows, k), each row multiplied by the weights of all its choices, or (plan.slots, k), a row per
    slot; w (G, n, k), bias (G, n); x_op "silu" applies SiLU to x as it loads. float32 rows: products as of
    exact three-way bfloat16 splits (float32 accuracy); 16-bit rows: one product each, or with SiLU two, of its
    rounding to the rows' type and of the rest; sums in float32 (over a shared row's choices too). Differentiable in x, w and bias; gradients are
    bitwise reproducible."""
    code_op = _X_OPS.get(x_op)
    if code_op is None:
        _fail("grouped_linear", f"x_op None or 'silu', got {x_op!r}")
    _dtype("grouped_linear", x)
    _linear_args("grouped_linear", x, w, plan, bias, x.dtype)
    _check("grouped_linear", x, w=w, bias=bias, plan=plan.ptr)
    if _wants_grad(x, w, bias):
        return GroupedLinear.apply(x, w, bias, plan.ptr, plan.order, plan, code_op)
    return _linear_fwd(x, w, plan, bias, code_op)


@torch.no_grad()
def grouped_linear_q8(x, x_scale, w, w_scale, plan, bias=None, dtype=torch.bfloat16):
    """grouped_linear of 8-bit operands, for serving: x float8_e4m3fn with x_scale (rows of x,), w (G, n, k)
    float8_e4m3fn with w_scale (G, n), as rms_norm_q8 and quantize_rows make them; y[a] = x_scale w_scale
    sum_k(x w) + bias, in `dtype` (bias too). A float32 result sums the exact products, at half the rate; for 16-bit
    results the matrix instruction cuts each of 64 neighbouring products below 2^-13 of the largest. No gradients."""
    name = "grouped_linear_q8"
    if x.dtype != _E4M3:
        _fail(name, f"float8_e4m3fn rows, got {x.dtype}")
    if dtype not in _DTYPES:
        _fail(name, f"dtype float32, bfloat16 or float16, got {dtype}")
    _linear_args(name, x, w, plan, bias, dtype)
    G, n, k = w.shape
    for what, t, shape in (("x_scale", x_scale, (x.shape[0],)), ("w_scale", w_scale, (G, n))):
        if t.shape != shape or t.dtype != torch.float32:
            _fail(name, f"{what} {shape} float32, got {tuple(t.shape)} {t.dtype}")
    _check(name, x, w=w, bias=bias, plan=plan.ptr, x_scale=x_scale, w_scale=w_scale)
    x2, w2 = _rows(x, k), _weights(w)
    xs, ws, b = x_scale.contiguous(), w_scale.contiguous(), None if bias is None else bias.contiguous()
    y = torch.empty(plan.slots, n, dtype=dtype, device=x.device)
    _launch(x, "face_grouped_linear_q8", "grouped_linear_q8", x2.data_ptr(), x2.stride(0), xs.data_ptr(),
            _div(plan, x.shape[0]), w2.data_ptr(), w2.stride(1), w2.stride(0), ws.data_ptr(), ptr(b), n, plan.ptr.data_ptr(),
            plan.order.data_ptr(), plan.slots, G, n, k, _DTYPES[dtype], y.data_ptr(), n)
    return y


# ----------------------------------------------------------------------------- join
def _combine_fwd(y, weight, residual):
    N, k = weight.shape
    F = y.shape[1]
    y2, w = _rows(y, F), weight.contiguous()
    r = None if residual is None else _rows(residual, F)
    out = torch.empty(N, F, dtype=y.dtype, device=y.device)
    _launch(y, "face_expert_combine_fwd", "expert_combine_fwd", y2.data_ptr(), y2.stride(0), w.data_ptr(), ptr(r),
            F if r is None else r.stride(0), N, k, F, _DTYPES[y.dtype], out.data_ptr())
    return out


class ExpertCombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weight, residual):
        ctx.save_for_backward(y, weight)
        return _combine_fwd(y, weight, residual)

    @staticmethod
    def backward(ctx, dout):
        _once("expert_combine", dout)
        need_y, need_w, need_r = ctx.needs_input_grad
        dy = dw = None
        if need_y or need_w:
            y, weight = ctx.saved_tensors
            N, k = weight.shape
            F = y.shape[1]
            if need_y:
                dy = torch.empty(N * k, F, dtype=y.dtype, device=y.device)
            if need_w:
                dw = torch.empty(N, k, dtype=torch.float32, device=y.device)
            y2, w, d = _rows(y, F), weight.contiguous(), _rows(dout, F)
            _launch(y, "face_expert_combine_bwd", "expert_combine_bwd", d.data_ptr(), d.stride(0), y2.data_ptr(), y2.stride(0),
                    w.data_ptr(), N, k, F, _DTYPES[y.dtype], ptr(dy), ptr(dw))
        return dy, dw, dout if need_r else None


def expert_combine(y, weight, residual=None):
    """out (N, F) = residual + sum_j weight[:, j] y[i k + j]: the rows of every atom's k choices joined.
    y (N k, F), weight (N, k) float32, residual (N, F) like y or None. Differentiable in all three."""
    name = "expert_combine"
    _dtype(name, y)
    if y.dim() != 2 or weight.dim() != 2 or weight.shape[1] < 1 or y.shape[1] < 1 or \
            y.shape[0] != weight.shape[0] * weight.shape[1]:
        _fail(name, f"y (N k, F) and weight (N, k), got {tuple(y.shape)} and {tuple(weight.shape)}")
    if weight.dtype != torch.float32:
        _fail(name, f"float32 weights, got {weight.dtype}")
    if residual is not None and (residual.shape != (weight.shape[0], y.shape[1]) or residual.dtype != y.dtype):
        _fail(name, f"residual ({weight.shape[0]}, {y.shape[1]}) {y.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    _check(name, y, weight=weight, residual=residual)
    if _wants_grad(y, weight, residual):
        return ExpertCombine.apply(y, weight, residual)
    return _combine_fwd(y, weight, residual)
