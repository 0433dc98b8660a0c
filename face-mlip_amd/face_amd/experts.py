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

Around it, for whole models of such layers:

    x = embed(table, species, scale)                       rows of a table, by species or pair of species
    y, s = layer_norm(x, w, b, eps, residual=r)            the norm with the mean taken out, and layer_norm_q8
    xs = expert_dispatch(y, plan)                          rows laid out by expert, for code of the user's own
    h = gated_silu(u)                                      silu of one half of the hidden rows times the other
    out = expert_return(v, plan, weight, residual=s)       such rows joined in the order of the atoms

and training in less memory: layer_norm, gated_silu and grouped_linear with keep8=True keep what their backward reads in
8 bits (pack_rows, unpack_rows).

Rows are float32, bfloat16 or float16 (all tensors of a call alike, gate weights and scales float32); sums,
softmax and norm statistics are float32. Every operator launches the kernels of
libface_hip.so on torch's current stream of its tensors' device, allocates its results and workspaces with torch and never
synchronises; none has a CPU path. They differentiate once, in training too: all of their floating
inputs take gradients, except those of the 8-bit forms for serving and of pack_rows. Forward-mode derivatives are refused. Forward and backward are captured into a graph together,
as with torch's own operators on leaves of which no eager graph is alive (fresh ones, by detach().requires_grad_()).
"""
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import call, ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_X_OPS = {None: 0, "silu": 1}
MAX_WIDTH = 65536                   # widest row of the norms, quantize_rows and embed
MAX_PACKED = 1 << 28                # of pack_rows, gated_silu and rows by expert
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
    strides = t.stride()
    if len(strides) != 2:
        t = t.reshape(-1, width)
        strides = t.stride()
    if strides[1] == 1 and strides[0] >= width:
        return t
    return t.clone(memory_format=torch.contiguous_format)


_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream, _recorded = _lib._raw_stream, torch.is_grad_enabled


def _launch(t, name, label, *args):
    """Call entry point `name` with args and the current stream of t's device, as the current device."""
    idx, L = t.get_device(), _lib._lib
    if idx != _get_device():
        with torch.cuda.device(idx):
            call(name, *args, _lib.stream_of(t), label=label)
    elif L is None or _raw_stream is None or _lib._timing is not None or _lib._order is not None:
        call(name, *args, _lib.stream_of(t), label=label)
    else:                                        # what call() does where nobody listens, in half its host time
        code = getattr(L, name)(*args, _raw_stream(idx))
        if code:
            _lib.fail(name, code)


def _once(name, *grads):
    """A backward that is itself recorded, or whose incoming gradients have tangents, would need second derivatives."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents(name + "'s gradient", *grads)
    if _recorded():
        raise NotImplementedError("the expert layer's operators differentiate once (create_graph=False)")


def _like(t):
    """A dense tensor of t's shape and type (half the host time of torch.empty(t.shape, ...))."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=4096)
def _work_size(name, *sizes):
    """Workspace of a call, by its sizes alone."""
    return getattr(_lib.lib(), name)(*sizes)


def _work(n_bytes, device):
    return torch.empty(n_bytes, dtype=torch.uint8, device=device) if n_bytes else None


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ----------------------------------------------------------------------------- norm
def _norm_args(name, x, w, eps, residual, b=None):
    code = _dtype(name, x)
    if x.dim() < 1 or w.dim() != 1 or x.shape[-1] != w.shape[0]:
        _fail(name, f"x (..., F) and w (F), got {tuple(x.shape)} and {tuple(w.shape)}")
    if not 1 <= x.shape[-1] <= MAX_WIDTH:
        _fail(name, f"rows of 1 to {MAX_WIDTH} columns, got {x.shape[-1]}")
    if w.dtype != x.dtype:
        _fail(name, f"w of the rows' type {x.dtype}, got {w.dtype}")
    if b is not None and (b.shape != w.shape or b.dtype != x.dtype):
        _fail(name, f"b like w, {tuple(w.shape)} {x.dtype}, got {tuple(b.shape)} {b.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        _fail(name, f"residual like x, {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    if not 0 <= eps < float("inf"):
        _fail(name, f"eps >= 0, got {eps}")
    _check(name, x, w=w, b=b, residual=residual)
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


def _layer_norm_fwd(code, x, w, b, eps, r, q8=False, grad=False, keep8=False):
    """(y, s, kept): kept holds what the backward reads, (mean, rstd), (q, block scales, rstd) or nothing. y is
    (q, scale) with q8; s is None without a residual."""
    F = x.shape[-1]
    x2, w = _rows(x, F), w.contiguous()
    r2 = None if r is None else _rows(r, F)
    b = None if b is None else b.contiguous()
    N, dev = x2.shape[0], x.device
    s = None if r is None else _like(x)
    y = None if q8 else _like(x)
    q = torch.empty(x.shape, dtype=_E4M3, device=dev) if q8 or keep8 else None
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if q8 else None
    block = _work(N * _blocks(F), dev) if keep8 else None
    stat = torch.empty((1 if keep8 else 2) * N, dtype=torch.float32, device=dev) if grad else None
    rstd = ptr(stat)
    mean = None if stat is None or keep8 else rstd + 4 * N
    _launch(x, "face_layer_norm_rows_fwd", "layer_norm_fwd", x2.data_ptr(), x2.stride(0), ptr(r2),
            F if r2 is None else r2.stride(0), N, F, code, w.data_ptr(), ptr(b), eps, ptr(y), ptr(s), ptr(q), ptr(scale),
            ptr(block), mean, rstd)
    return (q, scale) if q8 else y, s, (q, block, stat) if keep8 else (stat,)


# The backward passes run in a thread of their own, where a line of Python takes two to three times as long (gated_silu of
# 42 x 194, both directions: 60 us against 75): what the forward knows they take from ctx.
class LayerNorm(torch.autograd.Function):
    """Keeps the rows it normalised and each one's mean and rstd; with keep8 the normalised rows in 8 bits and rstd."""

    @staticmethod
    def forward(ctx, x, w, b, eps, r, keep8):
        code, F = _DTYPES[x.dtype], w.shape[0]
        y, s, kept = _layer_norm_fwd(code, x, w, b, eps, r, grad=True, keep8=keep8)
        ctx.save_for_backward(w, *kept, *(() if keep8 else (x if s is None else s,)))
        N = x.numel() // F
        ctx.known = N, F, code, keep8, _work_size("face_layer_norm_rows_bwd_work", N, F)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    def backward(ctx, dy, ds=None):
        _once("layer_norm", dy, ds)
        need_x, need_w, need_b, _, need_r, _ = ctx.needs_input_grad
        some = dy if dy is not None else ds
        if some is None:
            return None, None, None, None, None, None
        N, F, code, keep8, need = ctx.known
        if keep8:
            w, q, block, stat = ctx.saved_tensors
            mean, s, ld = None, None, F
        else:
            w, stat, s = ctx.saved_tensors
            s = _rows(s, F)
            mean, ld, q, block = stat.data_ptr() + 4 * N, s.stride(0), None, None
        w = w.contiguous()
        dx = _like(some) if need_x or need_r else None
        dw = _like(w) if need_w else None
        db = _like(w) if need_b else None
        work = None
        if need_w or need_b:
            work = _work(need, some.device)
        else:
            need = 0
        if dy is not None:
            dy = _rows(dy, F)
        if ds is not None:
            ds = _rows(ds, F)
        _launch(some, "face_layer_norm_rows_bwd", "layer_norm_bwd", ptr(s), ld, ptr(q), ptr(block), mean, stat.data_ptr(), ptr(dy),
                F if dy is None else dy.stride(0), ptr(ds), F if ds is None else ds.stride(0), N, F, code, w.data_ptr(), ptr(dx),
                ptr(dw), ptr(db), ptr(work), need)
        return dx if need_x else None, dw, db, None, dx if need_r else None, None


def layer_norm(x, w, b=None, eps=1e-5, residual=None, keep8=False):
    """x (..., F), w (F), b (F) or None -> (x - mean) w / sqrt(var + eps) + b over the last axis, var the mean square of
    x - mean. With residual (like x): (that of s, s) for s = x + residual, rounded to the rows' type before it is
    normalised. F <= MAX_WIDTH; sums in float32. keep8: the backward reads the normalised rows as 8 bits hold them
    (pack_rows), 1.03 bytes a value, in place of s."""
    eps = float(eps)
    code = _norm_args("layer_norm", x, w, eps, residual, b)
    if _wants_grad(x, w, b, residual):
        return LayerNorm.apply(x, w, b, eps, residual, bool(keep8))
    y, s, _ = _layer_norm_fwd(code, x, w, b, eps, residual)
    return y if s is None else (y, s)


@torch.no_grad()
def layer_norm_q8(x, w, b=None, eps=1e-5, residual=None):
    """layer_norm whose rows leave in 8 bits, for serving, as those of rms_norm_q8: (q, scale), and s with a residual.
    No gradients."""
    eps = float(eps)
    code = _norm_args("layer_norm_q8", x, w, eps, residual, b)
    y, s, _ = _layer_norm_fwd(code, x, w, b, eps, residual, q8=True)
    return y if s is None else (*y, s)


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


# ----------------------------------------------------------------------------- rows kept in 8 bits
def _row_count(name, x):
    if x.numel() >= x.shape[-1] << 31:
        _fail(name, f"fewer than 2^31 rows, got {tuple(x.shape)}")


def _blocks(F):
    """Scales of a kept row: one for each 32 columns."""
    return (F + 31) // 32


def _pack(x):
    F = x.shape[-1]
    x2 = _rows(x, F)
    q = torch.empty(x.shape, dtype=_E4M3, device=x.device)
    scale = torch.empty(*x.shape[:-1], _blocks(F), dtype=_E8M0, device=x.device)
    _launch(x, "face_pack_rows", "pack_rows", x2.data_ptr(), x2.stride(0), x2.shape[0], F, _DTYPES[x.dtype], q.data_ptr(),
            scale.data_ptr())
    return q, scale


def _unpack(q, scale, dtype):
    F = q.shape[-1]
    q2, s2 = _rows(q, F), _rows(scale, scale.shape[-1])
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    _launch(q, "face_unpack_rows", "unpack_rows", q2.data_ptr(), q2.stride(0), s2.data_ptr(), s2.stride(0), q2.shape[0], F,
            _DTYPES[dtype], x.data_ptr())
    return x


@torch.no_grad()
def pack_rows(x):
    """x (..., F) -> (q (..., F) float8_e4m3fn, scale (..., ceil(F / 32)) float8_e8m0fnu): rows as a backward pass
    keeps them in 8 bits, 1.03 bytes a value. Each 32 columns share a power of two, the least (>= 2^-126) that
    keeps their largest magnitude within 448: a value is off by at most 2^-4 of itself or 2^-17 of the block's
    largest (2^-136 where that is below 2^-118). A NaN or an infinity is kept as NaN and leaves the others as they are. No gradients."""
    _dtype("pack_rows", x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_PACKED:
        _fail("pack_rows", f"rows of 1 to {MAX_PACKED} columns, got {tuple(x.shape)}")
    _row_count("pack_rows", x)
    _check("pack_rows", x)
    return _pack(x)


@torch.no_grad()
def unpack_rows(q, scale, dtype=torch.bfloat16):
    """The values that (q, scale) of pack_rows stand for, in `dtype`; one past its largest is that. No gradients."""
    name = "unpack_rows"
    if q.dtype != _E4M3 or q.dim() < 1 or not 1 <= q.shape[-1] <= MAX_PACKED:
        _fail(name, f"float8_e4m3fn rows of 1 to {MAX_PACKED} columns, got {tuple(q.shape)} {q.dtype}")
    if dtype not in _DTYPES:
        _fail(name, f"dtype float32, bfloat16 or float16, got {dtype}")
    _row_count(name, q)
    shape = (*q.shape[:-1], _blocks(q.shape[-1]))
    if scale.shape != shape or scale.dtype != _E8M0:
        _fail(name, f"scale {shape} float8_e8m0fnu, got {tuple(scale.shape)} {scale.dtype}")
    _check(name, q, scale=scale)
    return _unpack(q, scale, dtype)


# ----------------------------------------------------------------------------- gated activation
def _gated_fwd(x, keep8=False):
    F = x.shape[-1] // 2
    x2 = _rows(x, 2 * F)
    N = x2.shape[0]
    y = x.new_empty((*x.shape[:-1], F))
    q = _work(N * 2 * F, x.device) if keep8 else None
    scale = _work(N * 2 * _blocks(F), x.device) if keep8 else None
    _launch(x, "face_gated_silu_fwd", "gated_silu_fwd", x2.data_ptr(), x2.stride(0), N, F, _DTYPES[x.dtype], y.data_ptr(), ptr(q),
            ptr(scale))
    return y, q, scale


class GatedSiLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, keep8):
        y, q, scale = _gated_fwd(x, keep8)
        if keep8:
            ctx.save_for_backward(q, scale)
        else:
            ctx.save_for_backward(x)
        F = y.shape[-1]
        ctx.known = y.numel() // F, F, _DTYPES[x.dtype], keep8, x.is_contiguous()
        return y

    @staticmethod
    def backward(ctx, dy):
        _once("gated_silu", dy)
        N, F, code, keep8, dense = ctx.known
        ld, ld_dy = 2 * F, F
        if not dy.is_contiguous():
            dy = _rows(dy, F)
            ld_dy = dy.stride(0)
        x = q = scale = None
        if keep8:
            q, scale = ctx.saved_tensors
            dx = dy.new_empty((*dy.shape[:-1], ld))
        else:
            x, = ctx.saved_tensors
            dx = torch.empty_like(x) if dense else _like(x)
            if not dense:
                x = _rows(x, ld)
                ld = x.stride(0)
        _launch(dx, "face_gated_silu_bwd", "gated_silu_bwd", ptr(x), ld, ptr(q), ptr(scale), dy.data_ptr(), ld_dy, N, F, code,
                dx.data_ptr())
        return dx, None


def gated_silu(x, keep8=False):
    """x (..., 2 F) -> silu(x[..., :F]) x[..., F:], the hidden rows between two products whose first makes gates and
    values side by side. keep8: the backward reads x as 8 bits hold it (pack_rows, each half in blocks of its own)
    in place of x, written as the forward reads it. Differentiable in x."""
    _dtype("gated_silu", x)
    if x.dim() < 1 or x.shape[-1] % 2 or not 2 <= x.shape[-1] <= 2 * MAX_PACKED:
        _fail("gated_silu", f"x (..., 2 F), F <= {MAX_PACKED}, got {tuple(x.shape)}")
    _row_count("gated_silu", x)
    _check("gated_silu", x)
    if _wants_grad(x):
        return GatedSiLU.apply(x, bool(keep8))
    return _gated_fwd(x)[0]


# ----------------------------------------------------------------------------- rows of a table
def _embed_fwd(table, index, factor, keys):
    V, F = table.shape
    t2, i = _rows(table, F), index.contiguous()
    y = table.new_empty((*index.shape, F))
    key = None
    wide = i.dtype == torch.int64
    if keys:
        key = torch.empty(i.shape, dtype=torch.int32, device=i.device) if wide else i
    _launch(table, "face_embed_fwd", "embed_fwd", t2.data_ptr(), t2.stride(0), i.data_ptr(), int(wide), i.numel(), V, F,
            _DTYPES[table.dtype], factor, y.data_ptr(), key.data_ptr() if keys and wide else None)
    return y, key


class Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, factor):
        y, key = _embed_fwd(table, index, factor, True)
        ctx.save_for_backward(key)
        V, F = table.shape
        N = key.numel()
        ctx.known = N, V, F, _DTYPES[table.dtype], factor, _work_size("face_embed_bwd_work", N, V, F)
        return y

    @staticmethod
    def backward(ctx, dy):
        _once("embed", dy)
        key, = ctx.saved_tensors
        N, V, F, code, factor, need = ctx.known
        ld = F
        if not dy.is_contiguous():
            dy = _rows(dy, F)
            ld = dy.stride(0)
        dt = dy.new_empty((V, F))
        work = _work(need, dy.device)
        _launch(dt, "face_embed_bwd", "embed_bwd", key.data_ptr(), dy.data_ptr(), ld, N, V, F, code, factor, dt.data_ptr(), ptr(work),
                need)
        return dt, None, None


def embed(table, index, scale=1.0):
    """table (V, F), index (...) int32 or int64 -> (..., F): scale times the table's rows, zeros where an index lies outside
    [0, V): the rows of every atom's species, or of every pair's. F <= MAX_WIDTH. Differentiable in the table: a
    dense gradient, each row's sum in float32 in a fixed order, rounded once."""
    name = "embed"
    _dtype(name, table)
    if table.dim() != 2 or not 1 <= table.shape[1] <= MAX_WIDTH or not 1 <= table.shape[0] < (1 << 31) - 1:
        _fail(name, f"table (V, F) with 1 <= V < 2^31 - 1 and 1 <= F <= {MAX_WIDTH}, got {tuple(table.shape)}")
    if index.dtype not in (torch.int32, torch.int64):
        _fail(name, f"int32 or int64 index, got {index.dtype}")
    if index.numel() >= 1 << 31:
        _fail(name, f"fewer than 2^31 rows, got {index.numel()}")
    if isinstance(scale, torch.Tensor):
        _fail(name, "scale: a number, got a tensor (no gradient would reach it)")
    factor = float(scale)
    _check(name, table, index=index)
    if _wants_grad(table):
        return Embed.apply(table, index, factor)
    return _embed_fwd(table, index, factor, False)[0]


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
    def forward(ctx, x, w, bias, p, order, plan, op, keep8):
        y = _linear_fwd(x, w, plan, bias, op)
        ctx.save_for_backward(w, p, order, *(_pack(x) if keep8 else (x,)))
        ctx.plan, ctx.op = plan, op
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    def backward(ctx, dy):
        _once("grouped_linear", dy)
        if dy is None:
            return (None,) * 8
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        w, p, order, *x = ctx.saved_tensors
        x = x[0] if len(x) == 1 else _unpack(*x, w.dtype)
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
        return dx, dw, db, None, None, None, None, None


def grouped_linear(x, w, plan, bias=None, x_op=None, keep8=False):
    """y (plan.slots, n), y[a] = op(x[row(a)]) w[g]^T + bias[g] for the slots a of group g, 0 for slots of no group.

    x (plan.rows, k), each row multiplied by the weights of all its choices, or (plan.slots, k), a row per
    slot; w (G, n, k), bias (G, n); x_op "silu" applies SiLU to x as it loads. float32 rows: products as of
    exact three-way bfloat16 splits (float32 accuracy); 16-bit rows: one product each, or with SiLU two, of its
    rounding to the rows' type and of the rest; sums in float32 (over a shared row's choices too). Differentiable in x, w and bias; gradients are
    bitwise reproducible. keep8: the backward reads x as 8 bits hold it (pack_rows) in place of x."""
    code_op = _X_OPS.get(x_op)
    if code_op is None:
        _fail("grouped_linear", f"x_op None or 'silu', got {x_op!r}")
    _dtype("grouped_linear", x)
    _linear_args("grouped_linear", x, w, plan, bias, x.dtype)
    _check("grouped_linear", x, w=w, bias=bias, plan=plan.ptr)
    if _wants_grad(x, w, bias):
        return GroupedLinear.apply(x, w, bias, plan.ptr, plan.order, plan, code_op, bool(keep8))
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


# ----------------------------------------------------------------------------- rows by expert and back
def _by_rows(slots, k, F):
    """Whether rows are read once and written to their k places, which takes the order's inverse first, or gathered by
    the order, read k times. bf16, k = 2, us: 2^25 elements out gathered 21, by rows 22; 2^26 of 2304 columns 40 / 37, 2^28 182 /
    148, but of 96 columns 213 / 226."""
    return k > 1 and F >= 256 and slots * F >= 1 << 26


def _dispatch_fwd(x, p, order, k):
    F, slots = x.shape[1], order.shape[0]
    x2 = _rows(x, F)
    place = torch.empty_like(order) if _by_rows(slots, k, F) else None
    xs = x.new_empty((slots, F))
    _launch(x, "face_expert_dispatch", "expert_dispatch", x2.data_ptr(), x2.stride(0), k, p.data_ptr(), order.data_ptr(), ptr(place),
            x.shape[0], p.shape[0] - 1, F, _DTYPES[x.dtype], xs.data_ptr())
    return xs, place


class ExpertDispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, order, k):
        xs, place = _dispatch_fwd(x, p, order, k)
        ctx.save_for_backward(p, order, place)
        ctx.k, ctx.rows = k, x.shape[0]
        return xs

    @staticmethod
    def backward(ctx, dxs):
        _once("expert_dispatch", dxs)
        p, order, place = ctx.saved_tensors
        return _return_fwd(dxs, p, order, place, None, None, ctx.rows, ctx.k)[0], None, None, None


def expert_dispatch(x, plan):
    """xs (plan.slots, F): the rows of x laid out by group, xs[i] = x[row(plan.order[i])], zeros at the places of no
    group, behind plan.ptr[G]: rows of one expert one after the other, for code of the user's own, or an exchange.
    x (plan.rows, F), each row to the places of all its choices, or (plan.slots, F), a row per slot. Differentiable in x."""
    name = "expert_dispatch"
    _dtype(name, x)
    if not isinstance(plan, GroupPlan):
        _fail(name, f"plan: a GroupPlan, got {type(plan).__name__}")
    if x.dim() != 2 or x.shape[0] not in (plan.rows, plan.slots) or not 1 <= x.shape[1] <= MAX_PACKED:
        _fail(name, f"x of {plan.rows} rows or {plan.slots} slots and 1 to {MAX_PACKED} columns, got {tuple(x.shape)}")
    _check(name, x, plan=plan.ptr)
    k = _div(plan, x.shape[0])
    if _wants_grad(x):
        return ExpertDispatch.apply(x, plan.ptr, plan.order, k)
    return _dispatch_fwd(x, plan.ptr, plan.order, k)[0]


def _return_fwd(y, p, order, place, weight, residual, N, k):
    """(out, place): place, the inverse of the plan's order, is made here if it is None."""
    F = y.shape[1]
    y2, w = _rows(y, F), None if weight is None else weight.contiguous()
    r = None if residual is None else _rows(residual, F)
    placed = place is not None
    if not placed:
        place = torch.empty_like(order)
    out = y.new_empty((N, F))
    _launch(y, "face_expert_return_fwd", "expert_return_fwd", y2.data_ptr(), y2.stride(0), p.data_ptr(), order.data_ptr(),
            place.data_ptr(), int(placed), ptr(w), ptr(r), F if r is None else r.stride(0), N, k, p.shape[0] - 1, F,
            _DTYPES[y.dtype], out.data_ptr())
    return out, place


class ExpertReturn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weight, residual, p, order, rows, k):
        out, place = _return_fwd(y, p, order, None, weight, residual, rows, k)
        # without a gradient of the weights the backward reads no row of y
        ctx.save_for_backward(y if weight is not None and ctx.needs_input_grad[1] else None, weight, p, order, place)
        ctx.known = rows, k, y.shape[1], p.shape[0] - 1, _DTYPES[y.dtype]
        return out

    @staticmethod
    def backward(ctx, dout):
        _once("expert_return", dout)
        need_y, need_w, need_r = ctx.needs_input_grad[:3]
        dy = dw = None
        if need_y or need_w:
            y, weight, p, order, place = ctx.saved_tensors
            N, k, F, G, code = ctx.known
            if need_y:
                dy = dout.new_empty((N * k, F))
            if need_w:
                dw = dout.new_empty((N, k), dtype=torch.float32)
            d2, w = _rows(dout, F), None if weight is None else weight.contiguous()
            y2 = _rows(y, F) if need_w else None
            _launch(dout, "face_expert_return_bwd", "expert_return_bwd", d2.data_ptr(), d2.stride(0), ptr(y2),
                    F if y2 is None else y2.stride(0), p.data_ptr(), order.data_ptr(), place.data_ptr(), ptr(w), N, k, G, F, code,
                    ptr(dy), ptr(dw))
        return dy, dw, dout if need_r else None, None, None, None, None


def expert_return(y, plan, weight=None, residual=None):
    """out (plan.rows, F) = residual + the sum of a row's choices, weight[i, j] y[place of slot i k + j]: rows laid out by
    expert_dispatch joined in the order of the rows. y (plan.slots, F), weight (plan.rows, plan.k) float32 or None (ones),
    residual (plan.rows, F) like y or None. Slots of no group add nothing, and their rows of y are not read. Differentiable
    in y, weight and residual."""
    name = "expert_return"
    _dtype(name, y)
    if not isinstance(plan, GroupPlan):
        _fail(name, f"plan: a GroupPlan, got {type(plan).__name__}")
    if y.dim() != 2 or y.shape[0] != plan.slots or not 1 <= y.shape[1] <= MAX_PACKED:
        _fail(name, f"y of {plan.slots} slots and 1 to {MAX_PACKED} columns, got {tuple(y.shape)}")
    if weight is not None and (weight.shape != (plan.rows, plan.k) or weight.dtype != torch.float32):
        _fail(name, f"weight ({plan.rows}, {plan.k}) float32, got {tuple(weight.shape)} {weight.dtype}")
    if residual is not None and (residual.shape != (plan.rows, y.shape[1]) or residual.dtype != y.dtype):
        _fail(name, f"residual ({plan.rows}, {y.shape[1]}) {y.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    _check(name, y, plan=plan.ptr, weight=weight, residual=residual)
    if _wants_grad(y, weight, residual):
        return ExpertReturn.apply(y, weight, residual, plan.ptr, plan.order, plan.rows, plan.k)
    return _return_fwd(y, plan.ptr, plan.order, None, weight, residual, plan.rows, plan.k)[0]
