"""Layer norm, rows kept in 8 bits, the gated activation, rows of a table and rows by expert, against their definitions in
64 bits.

Tolerances. u(T) is half a step of type T relative to the value (float32 2^-24, bfloat16 2^-8, float16 2^-11,
e4m3 2^-4). A sum of m terms formed in float32 is off by at most m u sum|terms|. A lane adds at most 64
values of a row, its lanes and waves at most 16 more: 80 steps. A result of T adds u(T) of itself.
"""
import math
import sys

import pytest
import torch

from face_amd import experts as ex

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16, E4M3, E8M0 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [F32, BF16, F16]
U32 = 2.0 ** -24
STEPS = 80


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def u(t):
    return {F32: U32, BF16: 2.0 ** -8, F16: 2.0 ** -11, E4M3: 2.0 ** -4}[t]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def near(got, want, bound, what=""):
    """|got - want| <= bound + u(T) |want|, element by element; want and bound in 64 bits."""
    d = got.double() - want
    lim = bound + u(got.dtype) * (want.abs() + bound) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    bad = ~(d.abs() <= lim)
    assert not bad.any(), (what, int(bad.sum()), (d.abs() / lim).nan_to_num(1e9).max().item())


def leaf(t):
    return t.detach().requires_grad_(True)


# ----------------------------------------------------------------------------- kept rows, by the definition
def kept64(v):
    """(what 8 bits hold, the scale's exponent) of 64-bit rows (..., F)."""
    F = v.shape[-1]
    m = -(-F // 32)
    b = torch.zeros(*v.shape[:-1], m * 32, dtype=torch.float64, device=v.device)
    b[..., :F] = v
    b = b.unflatten(-1, (m, 32))
    top = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(-1, keepdim=True)
    part, e = torch.frexp(top)                                       # top = part 2^e, part in [1/2, 1)
    e = torch.where(part <= 0.875, e - 9, e - 8).clamp(min=-126)     # 448 = 0.875 2^9
    e = torch.where(top == 0, -126, e)
    unit = ((e.long() + 1023) << 52).view(torch.float64)             # 2^e, exactly
    q = (b / unit).to(E4M3).double()
    q = torch.where(torch.isfinite(b), q, math.nan)
    top = torch.finfo(F32).max                                       # 256 2^120 passes it
    return (q * unit).clamp(-top, top).flatten(-2)[..., :F], e[..., 0]


# ----------------------------------------------------------------------------- layer norm
def ln64(x, r, w, b, eps):
    """s, h, rstd and the bound of h's error in float32."""
    s = x.double() if r is None else (x.double() + r.double()).to(x.dtype).double()
    mean = s.mean(-1, keepdim=True)
    d = s - mean
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    h = d * rstd
    # the mean is rounded once and corrected by the sum of the differences; the root halves the error of the squares
    eh = U32 * (rstd * (mean.abs() + (STEPS + 2) * d.abs().mean(-1, keepdim=True)) + (STEPS / 2 + 8) * h.abs())
    return s, h, rstd, eh


def ln_grads(h, eh, rstd, w, dy, ds):
    """dx, dw, db by the formula, with bounds, from h that is off by eh."""
    g = dy * w
    mg, mgh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - mg - h * mgh)
    emgh = (STEPS + 4) * U32 * (g * h).abs().mean(-1, keepdim=True) + (g.abs() * eh).mean(-1, keepdim=True)
    lim = rstd * (4 * U32 * g.abs() + (STEPS + 4) * U32 * g.abs().mean(-1, keepdim=True) + (h.abs() + eh) * emgh + eh * mgh.abs())
    lim = lim + (STEPS / 2 + 12) * U32 * rstd * (g.abs() + mg.abs() + (h * mgh).abs())
    if ds is not None:
        dx = dx + ds
        lim = lim + 2 * U32 * ds.abs()
    rows = dy.shape[0]
    dw, db = (dy * h).sum(0), dy.sum(0)
    ew = (rows + 8) * U32 * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0)
    return (dx, lim), (dw, ew), (db, (rows + 8) * U32 * dy.abs().sum(0))


LN_WIDTHS = [1, 7, 8, 96, 130, 257, 300, 520, 864, 1440, 2304, 4097, 6200, 9000, 16384, 16400, 65536]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", LN_WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_both_directions(dtype, F, residual):
    for rows in (1, 5, 67):
        say("layer_norm", dtype, F, residual, rows)
        g = gen(F + rows)
        x, w, b = rand(g, rows, F, dtype=dtype), (1 + 0.2 * rand(g, F)).to(dtype), rand(g, F, dtype=dtype, scale=0.3)
        x = (x.float() + 0.5).to(dtype)
        r = rand(g, rows, F, dtype=dtype, scale=3.0) if residual else None
        dy, ds = rand(g, rows, F, dtype=dtype), rand(g, rows, F, dtype=dtype)
        s, h, rstd, eh = ln64(x, r, w, b, 1e-5)
        leaves = [leaf(t) for t in ((x, w, b, r) if residual else (x, w, b))]
        out = ex.layer_norm(*leaves[:3], 1e-5, residual=leaves[3] if residual else None)
        y, gs = out if residual else (out, None)
        want = h * w.double() + b.double()
        near(y, want, eh * w.double().abs() + 3 * U32 * (h * w.double()).abs(), "y")
        if residual:
            assert torch.equal(gs.double(), s)
        grads = torch.autograd.grad([y] + ([gs] if residual else []), leaves, [dy] + ([ds] if residual else []))
        for what, got, (want, lim) in zip(("dx", "dw", "db"), grads,
                                          ln_grads(h, eh, rstd, w.double(), dy.double(), ds.double() if residual else None)):
            near(got, want, lim, what)
        if residual:
            assert torch.equal(grads[3], grads[0])
        with torch.no_grad():                                        # the same rows without gradients
            o = ex.layer_norm(x, w, b, 1e-5, residual=r)
        assert torch.equal(o[0] if residual else o, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [1, 7, 31, 33, 96, 130, 300, 864, 2304, 4097, 16384, 16400])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_kept_in_8_bits(dtype, F, residual):
    for rows in (1, 67):
        say("layer_norm keep8", dtype, F, residual, rows)
        g = gen(F + rows + 1)
        x, w, b = rand(g, rows, F, dtype=dtype), (1 + 0.2 * rand(g, F)).to(dtype), rand(g, F, dtype=dtype, scale=0.3)
        r = rand(g, rows, F, dtype=dtype, scale=3.0) if residual else None
        dy, ds = rand(g, rows, F, dtype=dtype), rand(g, rows, F, dtype=dtype)
        s, h, rstd, eh = ln64(x, r, w, b, 1e-5)
        leaves = [leaf(t) for t in ((x, w, b, r) if residual else (x, w, b))]
        out = ex.layer_norm(*leaves[:3], 1e-5, residual=leaves[3] if residual else None, keep8=True)
        y = out[0] if residual else out
        grads = torch.autograd.grad(list(out) if residual else [out], leaves, [dy, ds] if residual else [dy])
        with torch.no_grad():                                        # the forward is the same
            o = ex.layer_norm(x, w, b, 1e-5, residual=r)
        assert torch.equal(o[0] if residual else o, y)
        # a value within its error of a border of 8 bits may fall on either side of it
        hk = kept64(h)[0]
        ek = torch.maximum((kept64(h + eh)[0] - hk).abs(), (kept64(h - eh)[0] - hk).abs())
        for what, got, (want, lim) in zip(("dx", "dw", "db"), grads,
                                          ln_grads(hk, ek, rstd, w.double(), dy.double(), ds.double() if residual else None)):
            near(got, want, lim, what)


@pytest.mark.parametrize("keep8", [False, True])
def test_layer_norm_gradient_against_differences(keep8):
    g = gen(0)
    x, r, w, b = rand(g, 9, 300), rand(g, 9, 300), 1 + 0.2 * rand(g, 300), rand(g, 300)
    dy, ds = rand(g, 9, 300), rand(g, 9, 300)
    leaves = [leaf(t) for t in (x, r, w, b)]
    y, s = ex.layer_norm(leaves[0], leaves[2], leaves[3], 1e-3, residual=leaves[1], keep8=keep8)
    grads = torch.autograd.grad([y, s], leaves, [dy, ds])

    def loss(x, r, w, b):
        s = x + r
        d = s - s.mean(-1, keepdim=True)
        y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-3) * w + b
        return (y * dy.double()).sum() + (s * ds.double()).sum()

    for i, t in enumerate(leaves):
        v = rand(g, *t.shape).double()
        at = [z.detach().double() for z in leaves]
        hi, lo = list(at), list(at)
        hi[i], lo[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
        want = (loss(*hi) - loss(*lo)) / 2e-5
        got = (grads[i].double() * v).sum()
        # central differences: 1e-10 of the third derivative, far below the float32 bound of a sum of 2700 terms of order 3;
        # values of 8 bits are off by 2^-4 each way, 2^-4 sqrt(2700) of such terms with 5 times that for the tail
        tol = 5 * 2.0 ** -4 * 3 * 2700 ** 0.5 if keep8 and i != 3 else 2700 * 3 * 100 * U32
        assert abs(got - want) <= tol, (i, got.item(), want.item())


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_of_unusual_rows(dtype):
    g = gen(3)
    F = 200
    x = rand(g, 8, F, dtype=dtype)
    x[1] = 0.0
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = 3.0                                                       # no spread: y = b
    w, b = (1 + 0.2 * rand(g, F)).to(dtype), rand(g, F, dtype=dtype)
    l = [leaf(t) for t in (x, w, b)]
    y = ex.layer_norm(*l, 1e-5)
    dy = rand(g, 8, F, dtype=dtype)
    dx, dw, db = torch.autograd.grad([y], l, [dy])
    assert torch.equal(y[1], b) and torch.equal(y[4], b)
    for rows in (y, dx):
        assert rows[2].isnan().all() and rows[3].isnan().any()
        assert rows[[0, 1, 4, 5, 6, 7]].isfinite().all()
    good = [0, 1, 4, 5, 6, 7]
    l2 = [leaf(t) for t in (x[good], w, b)]
    assert torch.equal(ex.layer_norm(*l2, 1e-5), y[good])
    assert dw.isnan().all() and db.isfinite().all()
    # a mean a thousand times the spread, in float32: as exact as the mean's own rounding
    far = (rand(g, 5, 1440) + 1000.0)
    s, h, rstd, eh = ln64(far, None, torch.ones(1440, device=DEV), None, 1e-5)
    near(ex.layer_norm(far, torch.ones(1440, device=DEV), None, 1e-5), h, eh + 3 * U32 * h.abs())


def test_layer_norm_strides_and_missing_gradients():
    g = gen(4)
    big, wide = rand(g, 40, 500), rand(g, 300)
    x = big[::2, 3:303]                                              # rows 1000 apart, off alignment
    dy = rand(g, 300, 20).t()                                        # columns one after the other
    w, b = 1 + 0.1 * wide, rand(g, 600)[::2]
    base = [leaf(t.contiguous()) for t in (x, w, b)]
    want_y = ex.layer_norm(*base, 1e-5)
    want = torch.autograd.grad([want_y], base, [dy.contiguous()])
    l = [leaf(x), leaf(w), leaf(b)]
    y = ex.layer_norm(*l, 1e-5)
    assert torch.equal(y, want_y)
    for a, c in zip(torch.autograd.grad([y], l, [dy]), want):
        assert torch.equal(a, c)
    for only in range(3):                                            # each gradient alone is the same one
        l = [leaf(t) if i == only else t.detach() for i, t in enumerate((x, w, b))]
        a, = torch.autograd.grad([ex.layer_norm(*l, 1e-5)], [l[only]], [dy])
        assert torch.equal(a, want[only])
    # only the sum's gradient arrives, or only that of the norm
    r = rand(g, 20, 300)
    l = [leaf(t) for t in (x, w, b, r)]
    y, s = ex.layer_norm(*l[:3], 1e-5, residual=l[3])
    dx, dw = torch.autograd.grad([s], [l[0], l[1]], [dy], retain_graph=True, allow_unused=True)
    assert torch.equal(dx, dy) and not dw.any()
    # a row, no row, three axes, no bias
    one = ex.layer_norm(x[0], w, b, 1e-5)
    assert torch.equal(one, want_y[0])
    l = [leaf(torch.empty(0, 300, device=DEV)), leaf(w), leaf(b)]
    dx, dw, db = torch.autograd.grad([ex.layer_norm(*l, 1e-5)], l, [torch.empty(0, 300, device=DEV)])
    assert dx.shape == (0, 300) and not dw.any() and not db.any()
    assert torch.equal(ex.layer_norm(x.reshape(4, 5, 300), w, b, 1e-5).view(20, 300), want_y)
    assert torch.equal(ex.layer_norm(x, w, None, 1e-5), ex.layer_norm(x, w, torch.zeros_like(b), 1e-5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [1, 7, 96, 864, 2304, 4097, 16400, 65536])
def test_layer_norm_q8(dtype, F):
    say("layer_norm_q8", dtype, F)
    g = gen(F)
    x, r = rand(g, 5, F, dtype=dtype), rand(g, 5, F, dtype=dtype)
    w, b = (1 + 0.2 * rand(g, F)).to(dtype), rand(g, F, dtype=dtype, scale=0.3)
    s, h, rstd, eh = ln64(x, r, w, b, 1e-5)
    q, scale, s8 = ex.layer_norm_q8(x, w, b, 1e-5, residual=r)
    assert torch.equal(s8.double(), s)
    y = h * w.double() + b.double()
    ey = eh * w.double().abs() + 4 * U32 * y.abs() + 3 * U32 * (h * w.double()).abs()
    top = y.abs().amax(-1)
    near(scale, torch.clamp_min(top / 448, 2.0 ** -126), ey.amax(-1) / 448 + 2 * U32 * top / 448, "scale")
    # a value is its rounding to 8 bits: half a step 2^-4 of it, or of the smallest normal
    back = q.double() * scale.double()[:, None]
    lim = ey + 2.0 ** -4 * (y.abs() + ey) * (1 + 8 * U32) + 2.0 ** -10 * scale.double()[:, None]
    assert ((back - y).abs() <= lim).all()
    q2, scale2 = ex.layer_norm_q8(s8, w, b, 1e-5)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale2, scale)


# ----------------------------------------------------------------------------- pack
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [1, 7, 8, 31, 32, 33, 63, 97, 130, 257, 864, 1440, 2304, 10001])
def test_pack_rows(dtype, F):
    """Bit for bit: a scale is a power of two, so that only the rounding to 8 bits is left."""
    for rows in (1, 3, 130):
        say("pack", dtype, F, rows)
        g = gen(F + rows)
        x = rand(g, rows, F, dtype=dtype) * torch.exp(2 * rand(g, rows, F)).to(dtype)
        x[rows // 2, F // 2:] = 0.0
        q, scale = ex.pack_rows(x)
        want, e = kept64(x.double())
        assert q.shape == x.shape and q.dtype == E4M3 and scale.dtype == E8M0 and scale.shape == (rows, -(-F // 32))
        assert torch.equal(scale.view(torch.uint8).long(), (e + 127).clamp_min(1).long())
        back = ex.unpack_rows(q, scale, F32)
        assert torch.equal(back.double(), want)
        # half a step of e4m3's subnormals, 2^-10 of a scale that is less than 1/224 of the block's largest: 2^-17.8 of that
        assert ((back.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -17 * x.double().abs().amax()).all()
        for t in (BF16, F16):
            assert torch.equal(ex.unpack_rows(q, scale, t), want.clamp(-torch.finfo(t).max, torch.finfo(t).max).to(t))


def test_pack_unusual_values():
    F = 100
    x = torch.zeros(9, F, device=DEV)
    x[1, 3], x[1, 40], x[1, 41] = math.nan, math.inf, -math.inf
    x[1, 4], x[1, 42] = 1.0, -2.0
    x[2] = 448.0
    x[3] = 449.0                                                     # past 448: the next power
    x[4] = torch.finfo(F32).max
    x[5] = 1e-40                                                     # below the least scale's range
    x[6] = 2.0 ** -126 * 448
    x[7] = -2.0 ** -126 * 449
    x[8, 99] = 3.0                                                   # a last block of four columns
    q, scale = ex.pack_rows(x)
    want, e = kept64(x.double())
    back = ex.unpack_rows(q, scale, F32).double()
    assert torch.equal(back.isnan(), want.isnan()) and back[1].isnan().sum() == 3
    assert torch.equal(ex.unpack_rows(q, scale, BF16)[4].double(), torch.full((F,), torch.finfo(BF16).max, device=DEV).double())
    bad = back.nan_to_num(0) != want.nan_to_num(0)
    assert not bad.any(), (back[bad], want[bad])
    assert back[1, 4] == 1 and back[1, 42] == -2
    # fp16's own largest, kept as 65536
    h = torch.full((2, 40), 65504.0, dtype=F16, device=DEV)
    h[1] = -65504.0
    q, scale = ex.pack_rows(h)
    assert torch.equal(ex.unpack_rows(q, scale, F16), h)
    assert (ex.unpack_rows(q, scale, F32).abs() == 65536).all()
    # every byte of a scale that other code may have written
    q = torch.ones(256, 3, device=DEV).to(E4M3)
    s = torch.arange(256, dtype=torch.uint8, device=DEV).view(256, 1).view(E8M0)
    got = ex.unpack_rows(q, s, F32)[:, 0].double()
    assert got[255].isnan()
    assert torch.equal(got[:255], (torch.arange(896, 1151, device=DEV) << 52).view(torch.float64))       # 2^-127 .. 2^127


def test_pack_strides_and_empty():
    g = gen(9)
    big = rand(g, 30, 400)
    x = big[::3, 5:138]
    q, scale = ex.pack_rows(x)
    q2, scale2 = ex.pack_rows(x.contiguous())
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale.view(torch.uint8), scale2.view(torch.uint8))
    qs, ss = torch.empty(10, 200, device=DEV).to(E4M3), torch.empty(10, 9, dtype=torch.uint8, device=DEV).view(E8M0)
    qs[:, 1:134], ss[:, 2:7] = q, scale
    assert torch.equal(ex.unpack_rows(qs[:, 1:134], ss[:, 2:7], F32), ex.unpack_rows(q, scale, F32))
    q, scale = ex.pack_rows(big.view(5, 6, 400))
    assert q.shape == (5, 6, 400) and scale.shape == (5, 6, 13)
    q, scale = ex.pack_rows(torch.empty(0, 70, device=DEV))
    assert ex.unpack_rows(q, scale).shape == (0, 70)
    q, scale = ex.pack_rows(big[0])
    assert scale.shape == (13,) and ex.unpack_rows(q, scale).shape == (400,)


# ----------------------------------------------------------------------------- gated activation
def gate64(a, b, dy=None):
    sg = 1 / (1 + torch.exp(-a))
    y = a * sg * b
    if dy is None:
        return y
    return torch.cat([dy * b * sg * (1 + a * (1 - sg)), dy * a * sg], -1)


def near_gate(y, dx, x, xk, dy, what):
    F = y.shape[-1]
    a, b = x[..., :F].double(), x[..., F:].double()
    # the sigmoid's two corrected steps are within 4 u, two products more; beyond 87 what is left out is below 2^-119
    near(y, gate64(a, b), 8 * U32 * gate64(a, b).abs() + 2.0 ** -119 * b.abs(), what + " y")
    a, b = xk[..., :F].double(), xk[..., F:].double()
    d = dy.double()
    sg = 1 / (1 + torch.exp(-a))
    mag = torch.cat([(d * b).abs() * sg * (1 + a.abs() * (1 - sg)), (d * a).abs() * sg], -1)
    tail = 2.0 ** -119 * torch.cat([(d * b).abs(), d.abs()], -1)
    near(dx, gate64(a, b, d), 12 * U32 * mag + tail, what + " dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [1, 7, 8, 31, 33, 97, 160, 320, 512, 1001, 2304])
@pytest.mark.parametrize("keep8", [False, True])
def test_gated_silu(dtype, F, keep8):
    for rows in (1, 5, 130):
        say("gated", dtype, F, keep8, rows)
        g = gen(F + rows)
        x, dy = rand(g, rows, 2 * F, dtype=dtype, scale=2.0), rand(g, rows, F, dtype=dtype)
        if F > 4:
            x[0, :4] = torch.tensor([200.0, -200.0, 88.0, -88.0], device=DEV)
        l = leaf(x)
        y = ex.gated_silu(l, keep8=keep8)
        dx, = torch.autograd.grad([y], [l], [dy])
        xk = kept64(x.double().view(rows, 2, F))[0].reshape(rows, 2 * F) if keep8 else x
        near_gate(y, dx, x, xk, dy, f"{dtype} {F}")
        assert torch.equal(ex.gated_silu(x), y)


def test_gated_silu_strides_values_and_differences():
    g = gen(11)
    big = rand(g, 60, 300)
    x, dy = big[::2, 7:201], rand(g, 97, 30).t()
    for keep8 in (False, True):
        l, c = leaf(x), leaf(x.contiguous())
        y, yc = ex.gated_silu(l, keep8), ex.gated_silu(c, keep8)
        assert torch.equal(y, yc)
        assert torch.equal(torch.autograd.grad([y], [l], [dy])[0], torch.autograd.grad([yc], [c], [dy.contiguous()])[0])
    # a gradient that is one number, broadcast
    l = leaf(x)
    dx, = torch.autograd.grad([ex.gated_silu(l).sum()], [l])
    near_gate(ex.gated_silu(x), dx, x, x, torch.ones(30, 97, device=DEV), "sum")
    # values that are not finite stay in their row, and of a kept row in their column and its partner
    for keep8 in (False, True):
        bad = x.contiguous().clone()
        bad[3, 5], bad[4, 100], bad[5, 6] = math.nan, math.inf, -math.inf
        l, ok = leaf(bad), leaf(x.contiguous())
        y, yo = ex.gated_silu(l, keep8), ex.gated_silu(ok, keep8)
        dx, = torch.autograd.grad([y], [l], [dy])
        do, = torch.autograd.grad([yo], [ok], [dy])
        same = torch.ones(30, 194, dtype=torch.bool, device=DEV)
        for i, j in ((3, 5), (4, 3), (5, 6)):
            same[i, j] = same[i, j + 97] = False
        if not keep8:                                                # a block without its largest may have another scale
            assert torch.equal(dx[same], do[same])
        assert dx[same].isfinite().all() and torch.equal(y[same[:, :97]], yo[same[:, :97]])
    assert ex.gated_silu(torch.empty(0, 6, device=DEV)).shape == (0, 3)
    assert ex.gated_silu(rand(g, 6)).shape == (3,) and ex.gated_silu(rand(g, 2, 3, 8)).shape == (2, 3, 4)
    l = leaf(rand(g, 20, 60))
    d = rand(g, 20, 30)
    got, = torch.autograd.grad([ex.gated_silu(l)], [l], [d])
    v, at = rand(g, 20, 60).double(), l.detach().double()
    f = lambda t: (gate64(t[:, :30], t[:, 30:]) * d.double()).sum()
    want = (f(at + 1e-5 * v) - f(at - 1e-5 * v)) / 2e-5
    # 1200 terms of order 3, each off by 12 u; the differences by 1e-10 of the third derivative
    assert abs((got.double() * v).sum() - want) <= 1200 * 3 * 12 * U32 + 1e-6


# ----------------------------------------------------------------------------- products whose rows are kept
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("silu", [False, True])
def test_grouped_linear_kept_in_8_bits(dtype, silu):
    """The same products on the rows that 8 bits hold, bit for bit; the forward on the rows themselves."""
    g = gen(12)
    N, k, G, ki, n = 300, 2, 5, 97, 65
    plan = ex.group_plan(torch.randint(-1, G, (N, k), generator=g, device=DEV), G)
    rows = N * k if silu else N
    x, w, b = rand(g, rows, ki, dtype=dtype), rand(g, G, n, ki, dtype=dtype, scale=0.1), rand(g, G, n, dtype=dtype)
    dy = rand(g, N * k, n, dtype=dtype)
    op = "silu" if silu else None
    l = [leaf(t) for t in (x, w, b)]
    y = ex.grouped_linear(l[0], l[1], plan, bias=l[2], x_op=op, keep8=True)
    got = torch.autograd.grad([y], l, [dy], retain_graph=True)
    assert torch.equal(y, ex.grouped_linear(x, w, plan, bias=b, x_op=op))
    x8 = ex.unpack_rows(*ex.pack_rows(x), dtype)
    c = [leaf(t) for t in (x8, w, b)]
    want = torch.autograd.grad([ex.grouped_linear(c[0], c[1], plan, bias=c[2], x_op=op)], c, [dy])
    for a, o in zip(got, want):
        assert torch.equal(a, o)
    for i in range(3):
        a, = torch.autograd.grad([y], [l[i]], [dy], retain_graph=True)
        assert torch.equal(a, want[i])
    with torch.no_grad():                                            # what is kept is a copy: the rows may change
        l[0].add_(1.0)
    assert torch.equal(torch.autograd.grad([y], [l[1]], [dy])[0], want[1])


# ----------------------------------------------------------------------------- rows of a table
def check_embed(table, index, scale, dy):
    V, F = table.shape
    i = index.reshape(-1).long()
    inside = (i >= 0) & (i < V)
    at = torch.where(inside, i, 0)
    t = leaf(table)
    y = ex.embed(t, index, scale)
    want = torch.where(inside[:, None], table.double()[at] * scale, 0.0)
    assert y.shape == (*index.shape, F) and y.dtype == table.dtype
    # the factor is rounded to float32, then one product
    near(y.reshape(-1, F), want, 2 * U32 * want.abs(), "y")
    d, = torch.autograd.grad([y], [t], [dy], retain_graph=True)
    assert d.shape == table.shape and d.dtype == table.dtype
    at = torch.where(inside, i, V)
    d2 = dy.reshape(-1, F).double()
    sums = torch.zeros(V + 1, F, dtype=torch.float64, device=DEV).index_add_(0, at, d2)[:V] * scale
    mags = torch.zeros(V + 1, F, dtype=torch.float64, device=DEV).index_add_(0, at, d2.abs())[:V] * abs(scale)
    count = torch.bincount(at, minlength=V + 1)[:V, None].double()
    near(d, sums, (count + 3) * U32 * mags, "dtable")
    assert not d[count[:, 0] == 0].any()
    assert torch.equal(torch.autograd.grad([y], [t], [dy])[0], d)    # the same bits every time
    assert torch.equal(ex.embed(table, index, scale), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,F", [(1, 1, 1), (1, 5, 96), (21, 3, 96), (21, 119, 7), (64, 2, 8), (65, 3, 2304), (300, 20000, 40),
                                   (512, 17, 130), (513, 17, 130), (700, 3, 33), (4096, 40, 65), (4097, 300, 64), (5000, 16, 520),
                                   (9000, 255, 96), (9000, 256, 97), (3000, 70000, 24), (30000, 70000, 24), (40000, 14161, 64),
                                   (100000, 3, 256), (900, 70000, 40), (2048, 9, 70), (2049, 9, 70), (50000, 20, 600), (20000, 17, 2304), (200000, 1000, 16)])
def test_embed(dtype, N, V, F):
    say("embed", dtype, N, V, F)
    g = gen(N + V + F)
    table, dy = rand(g, V, F, dtype=dtype), rand(g, N, F, dtype=dtype)
    p = torch.exp(1.5 * rand(g, V))
    index = torch.multinomial(p, N, replacement=True, generator=g)
    check_embed(table, index.to(torch.int32), math.sqrt(F), dy)
    out = torch.rand(N, generator=g, device=DEV) < 0.2
    index = torch.where(out, torch.randint(-3, V + 5, (N,), generator=g, device=DEV), index)
    check_embed(table, index, 1.0, dy)                               # some outside, int64


def test_embed_runs_of_every_length():
    """Sorted rows in shares of 16: runs that end within a share, fill some, go on over a few or over thousands."""
    g = gen(5)
    V, F = 60, 40
    for lengths in ([1] * 60, [16] * 60, [15, 17] * 30, [32, 1, 31] * 20, [100, 3, 129, 128, 127] * 12, [8000, 1, 1, 500] * 15,
                    [0, 0, 4000, 0, 130, 144, 145] * 8, [60000] + [0] * 58 + [7]):
        index = torch.cat([torch.full((n,), v, device=DEV) for v, n in enumerate(lengths)])
        if index.numel() <= 2048:
            index = index.repeat(2048 // index.numel() + 2)
        index = index[torch.randperm(index.numel(), generator=g, device=DEV)]
        say("runs", index.numel())
        check_embed(rand(g, V, F), index.to(torch.int32), 0.5, rand(g, index.numel(), F))


def test_embed_shapes_strides_and_far_indices():
    g = gen(6)
    big = rand(g, 80, 200)
    table = big[::2, 3:133]
    for N in (30, 7000):                                             # nothing sorted, sorted
        index = torch.randint(0, 40, (N, 2), generator=g, device=DEV)
        dy = rand(g, 130, 2, N).permute(2, 1, 0)
        check_embed(table, index, -2.0, dy)
        check_embed(table, index[:, 0], 1.0, dy[:, 0])               # every other index
        a, = torch.autograd.grad([ex.embed(t := leaf(table), index).sum()], [t])         # a broadcast gradient
        near(a, torch.bincount(index.reshape(-1), minlength=40)[:, None].double().expand(40, 130),
             torch.zeros(1, dtype=torch.float64, device=DEV))
        none = torch.full((N,), -1, device=DEV, dtype=torch.int32)
        d, = torch.autograd.grad([ex.embed(t := leaf(table), none)], [t], [dy[:, 0]])
        assert not d.any() and not ex.embed(table, none).any()
    far = torch.tensor([1 << 40, -(1 << 40), (1 << 32) + 1, 2, (1 << 31), -1], device=DEV)
    check_embed(table, far, 1.0, rand(g, 6, 130))                    # 64-bit indices that a cut to 32 would bring back
    check_embed(table, torch.empty(0, dtype=torch.int32, device=DEV), 1.0, rand(g, 0, 130))
    check_embed(table, torch.tensor(7, device=DEV), 1.0, rand(g, 130))
    # a row that is not finite is its entry's alone
    for N in (30, 7000):
        index = torch.randint(0, 40, (N,), generator=g, device=DEV)
        dy = rand(g, N, 130)
        dy[5, 3] = math.nan
        d, = torch.autograd.grad([ex.embed(t := leaf(table), index)], [t], [dy])
        assert d.isnan().sum() == 1 and d[index[5], 3].isnan()


def test_embed_of_millions():
    """Segments of the sort that are longer than what is loaded at once, three passes."""
    g = gen(7)
    N, V = 5000003, 70001
    index = (torch.rand(N, generator=g, device=DEV) ** 3 * V).to(torch.int32)
    check_embed(rand(g, V, 9), index, 1.0, rand(g, N, 9))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows_in_both_directions(dtype, keep8):
    none = lambda *s: torch.empty(0, *s, dtype=dtype, device=DEV)
    w, b = torch.ones(7, dtype=dtype, device=DEV), torch.ones(7, dtype=dtype, device=DEV)
    l = [leaf(none(7)), leaf(w), leaf(b), leaf(none(7))]
    y, s = ex.layer_norm(l[0], l[1], l[2], residual=l[3], keep8=keep8)
    dx, dw, db, dr = torch.autograd.grad([y, s], l, [none(7), none(7)])
    assert dx.shape == dr.shape == (0, 7) and not dw.any() and not db.any()
    l = leaf(none(6))
    assert torch.autograd.grad([ex.gated_silu(l, keep8)], [l], [none(3)])[0].shape == (0, 6)
    plan = ex.group_plan(torch.empty(0, 2, dtype=torch.int32, device=DEV), 3)
    l = [leaf(none(5)), leaf(torch.ones(3, 4, 5, dtype=dtype, device=DEV))]
    dx, dw = torch.autograd.grad([ex.grouped_linear(*l, plan, keep8=keep8)], l, [none(4)])
    assert dx.shape == (0, 5) and not dw.any()


# ----------------------------------------------------------------------------- rows by expert
def sort_case(g, N, k, G, F, dtype, closed=0.1):
    e = torch.randint(0, G, (N, k), generator=g, device=DEV)
    e = torch.where(torch.rand(N, k, generator=g, device=DEV) < closed, -1, e)
    return ex.group_plan(e, G), rand(g, N, k).softmax(1) * (e >= 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,G,F", [(0, 2, 3, 8), (1, 1, 1, 1), (1, 3, 2, 96), (21, 2, 8, 96), (50, 5, 3, 257), (301, 8, 64, 513),
                                     (4096, 2, 8, 40), (5000, 3, 8, 300), (9000, 1, 3, 800), (3000, 4, 16, 4100)])
@pytest.mark.parametrize("by_rows", [False, True])
def test_rows_by_expert_and_back(dtype, N, k, G, F, by_rows, monkeypatch):
    say("sort", dtype, N, k, G, F, by_rows)
    monkeypatch.setattr(ex, "_by_rows", lambda *a: by_rows)          # either way at every size
    g = gen(N + k + F)
    plan, weight = sort_case(g, N, k, G, F, dtype)
    slots, m = N * k, int(plan.ptr[-1])
    x, r, ys = rand(g, N, F, dtype=dtype), rand(g, N, F, dtype=dtype), rand(g, slots, F, dtype=dtype)
    ys[m:] = math.nan                                                # of no group: not read
    a = plan.order[:m].long()
    i = torch.div(a, k, rounding_mode="floor")
    lx = leaf(x)
    xs = ex.expert_dispatch(lx, plan)
    assert torch.equal(xs[:m], x[i]) and not xs[m:].any() and xs.shape == (slots, F)
    assert torch.equal(ex.expert_dispatch(x, plan), xs)
    dxs = rand(g, slots, F, dtype=dtype)
    dxs[m:] = math.nan
    dx, = torch.autograd.grad([xs], [lx], [dxs])
    zero = torch.zeros(N, F, dtype=torch.float64, device=DEV)
    near(dx, zero.index_add(0, i, dxs[:m].double()), k * U32 * zero.index_add(0, i, dxs[:m].double().abs()), "dx")
    # back, with weights and residual, and without
    w = weight.double().reshape(-1)[a][:, None]
    y64 = ys[:m].double()
    ly, lw, lr = leaf(ys), leaf(weight), leaf(r)
    out = ex.expert_return(ly, plan, lw, residual=lr)
    near(out, r.double() + zero.index_add(0, i, y64 * w),
         (k + 2) * U32 * (r.double().abs() + zero.index_add(0, i, (y64 * w).abs())), "out")
    dout = rand(g, N, F, dtype=dtype)
    dy, dw, dr = torch.autograd.grad([out], [ly, lw, lr], [dout])
    d = dout.double()[i]
    near(dy[:m], d * w, U32 * (d * w).abs(), "dy")
    assert not dy[m:].any() and torch.equal(dr, dout)
    want, mag = torch.zeros(2, slots, dtype=torch.float64, device=DEV)
    want[a], mag[a] = (d * y64).sum(1), (d * y64).abs().sum(1)
    near(dw.reshape(-1), want, (F / 16 + 24) * U32 * mag, "dweight")
    ly = leaf(ys)
    bare = ex.expert_return(ly, plan)
    near(bare, zero.index_add(0, i, y64), k * U32 * zero.index_add(0, i, y64.abs()), "ones")
    dy, = torch.autograd.grad([bare], [ly], [dout])
    assert torch.equal(dy[:m], dout[i]) and not dy[m:].any()
    # a row per slot
    z = rand(g, slots, F, dtype=dtype)
    lz = leaf(z)
    zs = ex.expert_dispatch(lz, plan)
    assert torch.equal(zs[:m], z[a]) and not zs[m:].any()
    dz, = torch.autograd.grad([zs], [lz], [dxs])
    assert torch.equal(dz[a], dxs[:m])
    other = torch.ones(slots, dtype=torch.bool, device=DEV)
    other[a] = False
    assert not dz[other].any()


@pytest.mark.parametrize("N,F", [(40, 33), (3000, 700), (9000, 20)])
@pytest.mark.parametrize("by_rows", [False, True])
def test_rows_by_a_kept_plan_of_some_slots(N, F, by_rows, monkeypatch):
    """Plans that a program keeps: places that name no slot, slots that have none, ends past the order."""
    monkeypatch.setattr(ex, "_by_rows", lambda *a: by_rows)
    g = gen(N)
    k, slots = 2, 2 * N
    perm = torch.randperm(slots, generator=g, device=DEV).to(torch.int32)
    gone = torch.zeros(slots, dtype=torch.bool, device=DEV)
    gone[::7] = True
    order = torch.where(gone, torch.tensor([-1, slots, slots + 9, -(1 << 31)], device=DEV, dtype=torch.int32)[perm.long() % 4], perm)
    for ends in ([0, 10, slots - 5], [0, 3, slots + 1000], [0, 0, 0], [0, 5, -4]):
        plan = ex.GroupPlan(torch.tensor(ends, dtype=torch.int32, device=DEV), order, N, k)
        m = max(0, min(ends[-1], slots))
        at = torch.arange(slots, device=DEV)
        ok = (at < m) & ~gone
        x, ys, r = rand(g, N, F), rand(g, slots, F), rand(g, N, F)
        ys[~ok] = math.nan
        lx, ly = leaf(x), leaf(ys)
        xs = ex.expert_dispatch(lx, plan)
        row = torch.where(ok, order, 0).long()
        want = torch.where(ok[:, None], x[row // k], 0.0)
        assert torch.equal(xs, want)
        w = leaf(rand(g, N, k))
        out = ex.expert_return(ly, plan, w, residual=r)
        y0 = torch.where(ok[:, None], ys, 0.0).double()
        slot = torch.zeros(slots, F, dtype=torch.float64, device=DEV).index_add_(0, row, y0)
        per = slot.view(N, k, F) * w.detach().double()[:, :, None]
        near(out, r.double() + per.sum(1), 4 * U32 * (r.double().abs() + per.abs().sum(1)))
        dout, dxs = rand(g, N, F), rand(g, slots, F)
        dy, dw, dx = torch.autograd.grad([out, xs], [ly, w, lx], [dout, dxs])
        wd = torch.where(ok[:, None], (w.detach().reshape(-1)[row][:, None] * dout[row // k]), 0.0)
        assert torch.equal(dy, wd)
        near(dw, (slot.view(N, k, F) * dout.double()[:, None]).sum(2),
             (F / 16 + 24) * U32 * (slot.view(N, k, F) * dout.double()[:, None]).abs().sum(2))
        d0 = torch.where(ok[:, None], dxs, 0.0).double()
        want = torch.zeros(N, F, dtype=torch.float64, device=DEV).index_add_(0, row // k, d0)
        near(dx, want, 2 * U32 * torch.zeros_like(want).index_add_(0, row // k, d0.abs()))


def test_rows_by_expert_strides_and_some_gradients():
    g = gen(8)
    N, k, F = 60, 2, 130
    plan, weight = sort_case(g, N, k, 4, F, F32)
    big = rand(g, 130, 400)
    x, ys, r = big[:120:2, 3:133], big[:120, 200:330], rand(g, F, N).t()
    wt = torch.cat([weight, weight], 1)[:, :2]
    dxs, dout = rand(g, F, N * k).t(), rand(g, F, N).t()
    assert torch.equal(ex.expert_dispatch(x, plan), ex.expert_dispatch(x.contiguous(), plan))
    full = None
    for only in (None, 0, 1, 2):
        l = [leaf(t) if only in (None, i) else t.detach() for i, t in enumerate((ys, wt, r))]
        out = ex.expert_return(l[0], plan, l[1], residual=l[2])
        got = torch.autograd.grad([out], [t for t in l if t.requires_grad], [dout])
        if only is None:
            c = [leaf(t.contiguous()) for t in (ys, wt, r)]
            o2 = ex.expert_return(c[0], plan, c[1], residual=c[2])
            full = torch.autograd.grad([o2], c, [dout.contiguous()])
            assert torch.equal(out, o2) and all(torch.equal(a, b) for a, b in zip(got, full))
        else:
            assert torch.equal(got[0], full[only])
    l, c = leaf(x), leaf(x.contiguous())
    a, = torch.autograd.grad([ex.expert_dispatch(l, plan)], [l], [dxs])
    b, = torch.autograd.grad([ex.expert_dispatch(c, plan)], [c], [dxs.contiguous()])
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_operands_that_lie_by_columns(dtype):
    """Operands whose rows are not one after the other are copied for the call: the same results as of the copies."""
    g = gen(15)
    cols = lambda n, f: rand(g, f, n, dtype=dtype).t()
    plan, weight = sort_case(g, 40, 2, 4, 66, dtype)
    index = torch.randint(0, 40, (90,), generator=g, device=DEV)
    w, b = rand(g, 66, dtype=dtype), rand(g, 66, dtype=dtype)
    wt = weight.t().contiguous().t()
    x, r, ys, dy, dys, d3 = cols(40, 66), cols(40, 66), cols(80, 66), cols(40, 66), cols(80, 66), cols(90, 66)
    lin = rand(g, 4, 5, 66, dtype=dtype)
    calls = [(lambda x, r: ex.layer_norm(x, w, b, residual=r)[0], (x, r), dy),
             (lambda x, r: ex.layer_norm(x, w, b, residual=r, keep8=True)[0], (x, r), dy),
             (lambda x: ex.gated_silu(x), (x,), cols(40, 33)), (lambda x: ex.gated_silu(x, True), (x,), cols(40, 33)),
             (lambda x: ex.embed(x, index, 2.0), (x,), d3), (lambda x: ex.expert_dispatch(x, plan), (x,), dys),
             (lambda y, v, r: ex.expert_return(y, plan, v, residual=r), (ys, wt, r), dy),
             (lambda x: ex.grouped_linear(x, lin, plan, keep8=True), (x,), cols(80, 5))]
    for i, (f, operands, d) in enumerate(calls):
        say("columns", dtype, i)
        l, c = [leaf(t) for t in operands], [leaf(t.contiguous()) for t in operands]
        y, yc = f(*l), f(*c)
        assert torch.equal(y, yc), i
        got = torch.autograd.grad([y], l, [d])
        for a, o in zip(got, torch.autograd.grad([yc], c, [d.contiguous()])):
            assert torch.equal(a, o), i
    for a, o in zip(ex.pack_rows(x), ex.pack_rows(x.contiguous())):
        assert torch.equal(a.view(torch.uint8), o.view(torch.uint8))


def test_gradients_against_differences():
    """Rows of a table, rows by expert and back: linear in each operand, so that a difference of any length is exact in 64 bits;
    what is left is float32's rounding of sums of m terms."""
    g = gen(14)
    N, k, F = 70, 2, 50
    plan, weight = sort_case(g, N, k, 4, F, F32)
    m = int(plan.ptr[-1])
    a = plan.order[:m].long()
    i = a // k
    index = torch.randint(-1, 6, (N,), generator=g, device=DEV)
    table, ys, r = rand(g, 6, F), rand(g, N * k, F), rand(g, N, F)
    d1, d2, d3 = rand(g, N, F), rand(g, N * k, F), rand(g, N, F)

    def loss(table, ys, weight, r):
        y = torch.where(index[:, None] >= 0, table[index.clamp_min(0)], 0.0) * 3.0
        xs = torch.zeros(N * k, F, dtype=torch.float64, device=DEV)
        xs[:m] = y[i]
        out = r.index_add(0, i, ys[:m] * weight.reshape(-1)[a][:, None])
        return (y * d1.double()).sum() + (xs * d2.double()).sum() + (out * d3.double()).sum()

    l = [leaf(t) for t in (table, ys, weight, r)]
    y = ex.embed(l[0], index, 3.0)
    xs = ex.expert_dispatch(y, plan)
    out = ex.expert_return(l[1], plan, l[2], residual=l[3])
    grads = torch.autograd.grad([y, xs, out], l, [d1, d2, d3])
    for j, t in enumerate(l):
        v = rand(g, *t.shape).double()
        at = [z.detach().double() for z in l]
        hi, lo = list(at), list(at)
        hi[j], lo[j] = at[j] + v, at[j] - v
        want = (loss(*hi) - loss(*lo)) / 2
        # a gradient's element is a sum of at most 3 N terms of order 3 x 3, each direction's element of order 3
        n = t.numel()
        assert abs((grads[j].double() * v).sum() - want) <= 3 * N * U32 * 27 * n ** 0.5 * 10, j


# ----------------------------------------------------------------------------- together
class Layer:
    """Species rows, norm, rows by expert, one product per expert, the gate, a product by group, and back."""

    def __init__(self, g, V=4, C=48, G=3, H=40, dtype=F32):
        self.G, self.H = G, H
        self.p = [t.to(dtype) for t in (rand(g, V, C), 1 + 0.1 * rand(g, C), 0.1 * rand(g, C), rand(g, G, 2 * H, C, scale=C ** -0.5),
                                        rand(g, G, C, H, scale=H ** -0.5))]

    def __call__(self, p, species, r, plan, weight, keep8=False):
        table, w, b, W1, W2 = p
        x = ex.embed(table, species, 1.5)
        y, s = ex.layer_norm(x, w, b, 1e-5, residual=r, keep8=keep8)
        xs = ex.expert_dispatch(y, plan)
        own = self.identity(plan)
        u = ex.grouped_linear(xs, W1, own, keep8=keep8)
        v = ex.grouped_linear(ex.gated_silu(u, keep8=keep8), W2, own, keep8=keep8)
        return ex.expert_return(v, plan, weight, residual=s)

    def identity(self, plan):
        """Rows that already lie by expert: each slot is its own place."""
        return ex.GroupPlan(plan.ptr, torch.arange(plan.slots, dtype=torch.int32, device=DEV), plan.slots)

    def plain(self, p, species, r, expert, weight):
        table, w, b, W1, W2 = p
        x = table[species.long()] * 1.5
        s = x + r
        d = s - s.mean(-1, keepdim=True)
        y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * w + b
        out = s
        for j in range(expert.shape[1]):
            e = expert[:, j].clamp_min(0).long()
            h = torch.matmul(W1[e], y[:, :, None])[:, :, 0]
            h = h[:, :self.H] * torch.sigmoid(h[:, :self.H]) * h[:, self.H:]
            o = torch.matmul(W2[e], h[:, :, None])[:, :, 0]
            out = out + torch.where(expert[:, j:j + 1] >= 0, weight[:, j:j + 1] * o, 0.0)
        return out


def layer_case(N, dtype=F32, seed=0):
    g = gen(seed)
    layer = Layer(g, dtype=dtype)
    species = torch.randint(0, 4, (N,), generator=g, device=DEV, dtype=torch.int32)
    expert = torch.randint(-1, 3, (N, 2), generator=g, device=DEV)
    weight = rand(g, N, 2).softmax(1)
    return layer, species, rand(g, N, 48, dtype=dtype), expert, weight, rand(g, N, 48, dtype=dtype)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("N", [1, 21, 3000])
def test_layer_end_to_end(N, keep8):
    layer, species, r, expert, weight, dout = layer_case(N)
    plan = ex.group_plan(expert, 3)
    l = [leaf(t) for t in (*layer.p, r, weight)]
    out = layer(l[:5], species, l[5], plan, l[6], keep8)
    got = torch.autograd.grad([out], l, [dout])
    c = [leaf(t.double()) for t in (*layer.p, r, weight)]
    want_out = layer.plain(c[:5], species, c[5], expert, c[6])
    want = torch.autograd.grad([want_out], c, [dout.double()])
    # Seven operators, each off by at most 100 u of its values relative to their norm, slopes of at most 3 each: 2100 u, with
    # a factor of 10 for cancellation in a norm. In 8 bits four of them read values off by 2^-4 at most, 2^-4 / sqrt 3 on average.
    off = lambda a, b: ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()
    assert off(out, want_out) <= 21000 * U32
    for i, (a, b) in enumerate(zip(got, want)):
        assert off(a, b) <= (4 * 3 * 2.0 ** -4 / 3 ** 0.5 if keep8 else 21000 * U32), (i, off(a, b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keep8", [False, True])
def test_layer_in_two_captured_graphs(dtype, keep8):
    """Forward and backward captured twice and replayed in turn with new inputs, eager work between; every replay
    equals the eager result."""
    layer, species0, r0, expert, weight0, dout = layer_case(2500, dtype)
    g = gen(21)
    plan = ex.group_plan(expert, 3)

    def step(species, r, weight):
        l = [leaf(t) for t in (*layer.p, r, weight)]
        out = layer(l[:5], species, l[5], plan, l[6], keep8)
        return [out.detach()] + list(torch.autograd.grad([out], l, [dout]))

    held = []
    for _ in range(2):
        species, r, weight = species0.clone(), r0.clone(), weight0.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(species, r, weight)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            outs = step(species, r, weight)
        held.append((cg, species, r, weight, outs))
    for turn in range(4):
        for cg, species, r, weight, outs in held:
            species.copy_(torch.randint(-1, 5, species.shape, generator=g, device=DEV))
            r.copy_(rand(g, *r.shape))
            weight.copy_(rand(g, *weight.shape).softmax(1))
            cg.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step(species, r, weight)):
                assert torch.equal(a, b), turn


@pytest.mark.parametrize("N,V", [(300, 4), (6000, 40), (9000, 3)])
def test_embed_in_a_graph(N, V):
    """The table's gradient replayed, few rows, sorted, few entries: indices that change between replays."""
    g = gen(N)
    table, dy = rand(g, V, 70), rand(g, N, 70)
    index = torch.randint(0, V, (N,), generator=g, device=DEV)

    def step():
        t = leaf(table)
        return torch.autograd.grad([ex.embed(t, index, 2.0)], [t], [dy])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    cg = torch.cuda.CUDAGraph()
    with torch.cuda.graph(cg):
        out = step()
    for _ in range(4):
        index.copy_(torch.randint(-2, V + 2, (N,), generator=g, device=DEV))
        cg.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_other_streams_and_two_calls_at_once():
    layer, species, r, expert, weight, dout = layer_case(3000)
    plan = ex.group_plan(expert, 3)

    def step():
        l = [leaf(t) for t in (*layer.p, r, weight)]
        out = layer(l[:5], species, l[5], plan, l[6], True)
        return [out.detach()] + list(torch.autograd.grad([out], l, [dout]))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_second_derivatives_and_tangents_of_gradients_are_refused():
    g = gen(0)
    plan = ex.group_plan(torch.zeros(4, dtype=torch.int32, device=DEV), 1)
    x, w = rand(g, 4, 8).requires_grad_(True), torch.ones(8, device=DEV)
    i = torch.zeros(4, dtype=torch.int32, device=DEV)
    for out in (ex.layer_norm(x, w), ex.layer_norm(x, w, keep8=True), ex.gated_silu(x), ex.gated_silu(x, True), ex.embed(x, i),
                ex.expert_dispatch(x, plan), ex.expert_return(x, plan), ex.grouped_linear(x, rand(g, 1, 3, 8), plan, keep8=True)):
        with pytest.raises(NotImplementedError, match="differentiate once"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_an_operand_changed_before_its_backward_is_noticed():
    g = gen(1)
    x, w = rand(g, 6, 8), torch.ones(8, device=DEV)
    i = torch.zeros(6, dtype=torch.int32, device=DEV)
    plan = ex.group_plan(torch.zeros(6, dtype=torch.int32, device=DEV), 1)
    for f, changed in ((lambda l: ex.layer_norm(l * 1, w), w), (lambda l: ex.embed(l, i), i),
                       (lambda l: ex.expert_dispatch(l, plan), plan.order), (lambda l: ex.expert_return(l, plan), plan.ptr)):
        l = leaf(x)
        out = f(l)
        changed.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), l)


# ----------------------------------------------------------------------------- far rows
@pytest.mark.parametrize("keep8", [False, True])
def test_rows_past_two_to_the_31_elements(keep8):
    """The last rows of operands of 2^31 elements and more, against the same rows alone."""
    N, F = 1 << 20, 2056
    g = gen(2)
    base = rand(g, 4096, F, dtype=BF16)
    x = base.repeat(N // 4096, 1)
    tail = slice(N - 3000, N)
    w, b = (1 + 0.1 * rand(g, F)).to(BF16), rand(g, F, dtype=BF16)
    say("norm")
    l, t = leaf(x), leaf(x[tail])
    y, yt = ex.layer_norm(l, w, b, keep8=keep8), ex.layer_norm(t, w, b, keep8=keep8)
    assert torch.equal(y[tail], yt)
    dx, = torch.autograd.grad([y], [l], [x])
    dt, = torch.autograd.grad([yt], [t], [x[tail]])
    assert torch.equal(dx[tail], dt)
    del y, dx
    say("gate")
    y, yt = ex.gated_silu(l, keep8), ex.gated_silu(t, keep8)
    assert torch.equal(y[tail], yt)
    dx, = torch.autograd.grad([y], [l], [x[:, :F // 2]])
    dt, = torch.autograd.grad([yt], [t], [x[tail, :F // 2]])
    assert torch.equal(dx[tail], dt)
    del y, dx
    if keep8:
        say("pack")
        q, scale = ex.pack_rows(x)
        q2, scale2 = ex.pack_rows(x[tail])
        assert torch.equal(q[tail].view(torch.uint8), q2.view(torch.uint8))
        assert torch.equal(ex.unpack_rows(q, scale)[tail], ex.unpack_rows(q2, scale2))
        return
    say("embed")
    for V in (3, 4096):                                              # few entries, sorted
        index = torch.arange(N, device=DEV, dtype=torch.int32) % V
        lt = leaf(base[:V])
        y = ex.embed(lt, index)
        assert torch.equal(y[tail], base[index[tail].long()])
        d, = torch.autograd.grad([y], [lt], [x])
        del y
        if V == 4096:                                                # 256 equal rows each: exact in float32
            assert torch.equal(d, (base.double() * 256).to(BF16))
    say("by expert")
    order = torch.arange(N - 1, -1, -1, dtype=torch.int32, device=DEV)
    for k in (1, 2):
        plan = ex.GroupPlan(torch.tensor([0, N], dtype=torch.int32, device=DEV), order, N // k, k)
        xs = ex.expert_dispatch(x[:N // k], plan)
        assert torch.equal(xs[tail], x[(order[tail] // k).long()]) and torch.equal(xs[:3000], x[(order[:3000] // k).long()])
        out = ex.expert_return(xs, plan)
        assert torch.equal(out[-3000:], (k * x[:N // k][-3000:].float()).to(BF16))
        del xs, out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [901, 904])
def test_large_calls_give_the_rows_of_small_ones(dtype, F):
    """Past 256 MB rows are read and written by other accesses, whole pieces and cut ones: bit for bit the same rows, and sums
    over all rows within their bound."""
    g = gen(F)
    N = 48001 if dtype != F32 else 24001
    x, r, dy, ds = (rand(g, N, F, dtype=dtype) for _ in range(4))
    w, b = (1 + 0.1 * rand(g, F)).to(dtype), rand(g, F, dtype=dtype)
    parts = (slice(0, 700), slice(N - 700, N))

    def same(big, f):
        for p in parts:
            for a, c in zip(big, f(p)):
                assert torch.equal(a[p].view(torch.uint8), c.view(torch.uint8))

    for keep8 in (False, True):
        say("norm", dtype, F, keep8)

        def norm(p):
            l = [leaf(t) for t in (x[p], r[p], w, b)]
            y, s = ex.layer_norm(l[0], l[2], l[3], residual=l[1], keep8=keep8)
            return (y.detach(), s.detach(), *torch.autograd.grad([y, s], l, [dy[p], ds[p]]))

        out = norm(slice(0, N))
        same(out[:4], lambda p: norm(p)[:4])
        d = dy.double()
        near(out[5], d.sum(0), (N + 8) * U32 * d.abs().sum(0), "db")
        if not keep8:
            s, h, rstd, eh = ln64(x, r, w, b, 1e-5)
            near(out[4], (d * h).sum(0), (N + 8) * U32 * (d * h).abs().sum(0) + (d.abs() * eh).sum(0), "dw")
            del s, h, rstd, eh
        del d
        say("gate", dtype, F, keep8)
        M = N // 2
        z = torch.stack([x[:M], r[:M]], 1).reshape(M, 2 * F).repeat(3, 1)
        dz = dy[:M].repeat(3, 1)
        parts = (slice(0, 700), slice(3 * M - 700, 3 * M))

        def gate(p):
            l = leaf(z[p])
            y = ex.gated_silu(l, keep8)
            return y.detach(), torch.autograd.grad([y], [l], [dz[p]])[0]

        same(gate(slice(0, 3 * M)), gate)
        parts = (slice(0, 700), slice(N - 700, N))
    say("norm in 8 bits, pack")
    same(ex.layer_norm_q8(x, w, b, residual=r), lambda p: ex.layer_norm_q8(x[p], w, b, residual=r[p]))
    z = torch.cat([x, r, dy, ds])
    parts = (slice(0, 700), slice(4 * N - 700, 4 * N))
    same(ex.pack_rows(z), lambda p: ex.pack_rows(z[p]))
    q, scale = ex.pack_rows(z)
    same([ex.unpack_rows(q, scale, dtype)], lambda p: [ex.unpack_rows(q[p], scale[p], dtype)])
    say("by expert")
    k = 2
    plan, weight = sort_case(g, N, k, 5, F, dtype)
    m = int(plan.ptr[-1])
    at, i = plan.order[:m].long(), plan.order[:m].long() // k
    lx, ly, lw = leaf(x), leaf(z[:N * k]), leaf(weight)
    xs = ex.expert_dispatch(lx, plan)
    assert torch.equal(xs[:m], x[i]) and not xs[m:].any()
    out = ex.expert_return(ly, plan, lw, residual=r)
    dx, dys, dw = torch.autograd.grad([xs, out], [lx, ly, lw], [z[N * k:], dy])
    v = torch.zeros(N * k, F, dtype=dtype, device=DEV)
    v[at] = z[:m]                                                    # by slot, summed as the join does
    want = r.float()
    for j in range(k):
        want = torch.addcmul(want, weight[:, j:j + 1], v.view(N, k, F)[:, j].float())
    near(out, want.double(), 4 * U32 * (r.double().abs() + v.view(N, k, F).double().abs().sum(1)), "out")
    v.zero_()
    v[at] = z[N * k:][:m]
    near(dx, v.view(N, k, F).double().sum(1), 2 * U32 * v.view(N, k, F).double().abs().sum(1), "dx")
    wd = weight.reshape(-1)[at][:, None] * dy[i].float()
    assert torch.equal(dys[:m], wd.to(dtype)) and not dys[m:].any()
    say("embed")
    for V in (5, 3000):
        index = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
        check_embed(x[:V].contiguous(), index, 1.0, dy)


@pytest.mark.parametrize("keep8", [False, True])
def test_more_rows_than_one_dimension_of_a_grid(keep8):
    """Hundreds of millions of narrow rows, more workgroups than a grid takes side by side: the last rows are those of a
    small call."""
    g = gen(4)
    N = 71000003
    base = rand(g, 4099, 2, dtype=BF16)
    x = base.repeat(N // 4099 + 1, 1)[:N]
    tail = slice(N - 5000, N)
    w, b = rand(g, 2, dtype=BF16), rand(g, 2, dtype=BF16)
    say("norm")
    l, t = leaf(x), leaf(x[tail])
    y, yt = ex.layer_norm(l, w, b, 1e-2, keep8=keep8), ex.layer_norm(t, w, b, 1e-2, keep8=keep8)
    assert torch.equal(y[tail], yt)
    dx, = torch.autograd.grad([y], [l], [x])
    dt, = torch.autograd.grad([yt], [t], [x[tail]])
    assert torch.equal(dx[tail], dt)
    del y, dx
    say("by expert")
    order = torch.arange(N - 1, -1, -1, dtype=torch.int32, device=DEV)
    plan = ex.GroupPlan(torch.tensor([0, N], dtype=torch.int32, device=DEV), order, N)
    xs = ex.expert_dispatch(x, plan)
    assert torch.equal(xs[tail], x[:5000].flip(0)) and torch.equal(xs[:5000], x[tail].flip(0))
    out = ex.expert_return(xs, plan)
    assert torch.equal(out, x)
    del xs, out, order, plan
    say("gate")
    z = x.repeat(4, 1)
    tail = slice(4 * N - 5000, 4 * N)
    l, t = leaf(z), leaf(z[tail])
    y, yt = ex.gated_silu(l, keep8), ex.gated_silu(t, keep8)
    assert torch.equal(y[tail], yt)
    dx, = torch.autograd.grad([y], [l], [y.detach()])
    dt, = torch.autograd.grad([yt], [t], [yt.detach()])
    assert torch.equal(dx[tail], dt)
    del y, dx
    say("pack")
    q, scale = ex.pack_rows(z)
    q2, scale2 = ex.pack_rows(z[tail])
    assert torch.equal(q[tail].view(torch.uint8), q2.view(torch.uint8))
    assert torch.equal(ex.unpack_rows(q, scale)[tail], ex.unpack_rows(q2, scale2))


def test_a_table_of_millions_of_entries():
    """Few rows of it: every other entry's gradient is zero."""
    g = gen(5)
    V, F = 9000001, 3
    table, index = rand(g, V, F), torch.randint(0, V, (300,), generator=g, device=DEV)
    index[:40] = V - 1
    check_embed(table, index, 2.0, rand(g, 300, F))
    index = torch.randint(0, V, (900,), generator=g, device=DEV)
    check_embed(table, index, 2.0, rand(g, 900, F))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_wide_embedding_gradient(dtype):
    """Rows of many column tiles, and of a width that no lane's piece divides."""
    g = gen(3)
    for N, V, F in ((2000, 100, 1111), (600, 30, 65536), (300, 5, 65535)):
        say("wide", dtype, N, V, F)
        index = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
        check_embed(rand(g, V, F, dtype=dtype), index, 1.0, rand(g, N, F, dtype=dtype))
