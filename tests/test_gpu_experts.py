"""The expert layer's operators against their definitions in 64 bits.

Tolerances. u(T) is half a step of type T relative to the value (float32 2^-24, bfloat16 2^-8, float16 2^-11,
e4m3 2^-4). A sum of m terms formed in float32 is off by at most m u sum|terms|; a matrix instruction cuts its
addends, so each of its steps counts for a whole step, 2 u. A result of T adds u(T) of itself, float16
below its smallest normal 2^-25, e4m3 2^-10 of the row's scale.
"""
import math
import sys

import pytest
import torch

from face_amd import experts as ex

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
TYPES = [F32, BF16, F16]
U32 = 2.0 ** -24


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


# ----------------------------------------------------------------------------- norm
def norm64(x, r, w, eps):
    s = x.double() if r is None else (x.double() + r.double()).to(x.dtype).double()
    return s, s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w.double()


def norm_terms(F):
    """Rounding steps of a normalised value: a lane's and the lanes' additions halved by the square root,
    and six more operations."""
    return (64 + 16) / 2 + 6


WIDTHS = [1, 7, 8, 96, 257, 300, 864, 1440, 2304, 4097, 16400, 65536]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_both_directions(dtype, F, residual):
    say("rms_norm", dtype, F, residual)
    for rows in (1, 5, 67):
        g = gen(F + rows)
        x, w = rand(g, rows, F, dtype=dtype), (1 + 0.2 * rand(g, F)).to(dtype)
        r = rand(g, rows, F, dtype=dtype, scale=3.0) if residual else None
        dy, ds = rand(g, rows, F, dtype=dtype), rand(g, rows, F, dtype=dtype)
        s, y = norm64(x, r, w, 1e-5)
        leaves = [t.requires_grad_(True) for t in ((x, w, r) if residual else (x, w))]
        out = ex.rms_norm(x, w, 1e-5, residual=r)
        got, gs = out if residual else (out, x)
        near(got, y, norm_terms(F) * U32 * y.abs(), "y")
        if residual:
            assert torch.equal(gs.double(), s)
        grads = torch.autograd.grad([got] + ([gs] if residual else []), leaves, [dy] + ([ds] if residual else []))
        # the formula's gradient
        rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
        gw = dy.double() * w.double()
        m = (gw * s).mean(-1, keepdim=True)
        dx = rstd * (gw - s * rstd ** 2 * m)
        mag = rstd * (gw.abs() + s.abs() * rstd ** 2 * (gw * s).abs().mean(-1, keepdim=True))
        lim = 3 * (norm_terms(F) + 4) * U32 * mag
        if residual:
            dx = dx + ds.double()
            lim = lim + 2 * U32 * ds.double().abs()
        near(grads[0], dx, lim, "dx")
        dw_terms = dy.double() * s * rstd
        near(grads[1], dw_terms.sum(0), (rows + norm_terms(F) + 8) * U32 * dw_terms.abs().sum(0), "dw")
        if residual:
            assert torch.equal(grads[2], grads[0])
        # without gradients the same kernel gives the same rows
        with torch.no_grad():
            o = ex.rms_norm(x, w, 1e-5, residual=r)
        assert torch.equal(o[0] if residual else o, got)


def test_rms_norm_gradient_against_differences():
    g = gen(0)
    x, r, w = rand(g, 9, 300), rand(g, 9, 300), 1 + 0.2 * rand(g, 300)
    dy, ds = rand(g, 9, 300), rand(g, 9, 300)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, s = ex.rms_norm(x, w, 1e-3, residual=r)
    grads = torch.autograd.grad([y, s], leaves, [dy, ds])

    def loss(x, r, w):
        s, y = (x + r), None
        y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-3) * w
        return (y * dy.double()).sum() + (s * ds.double()).sum()

    for i, t in enumerate(leaves):
        v = rand(g, *t.shape).double()
        at = [z.detach().double() for z in leaves]
        hi, lo = list(at), list(at)
        hi[i], lo[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
        want = (loss(*hi) - loss(*lo)) / 2e-5
        got = (grads[i].double() * v).sum()
        assert abs(got - want) <= 1e-5 * (grads[i].double() * v).abs().sum()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [1, 7, 96, 864, 2304, 4097, 65536])
def test_q8_rows(dtype, F):
    say("q8", dtype, F)
    g = gen(F)
    x, r, w = rand(g, 33, F, dtype=dtype), rand(g, 33, F, dtype=dtype), (1 + 0.2 * rand(g, F)).to(dtype)
    x[3], r[3] = 0, 0                                    # a row of zeros
    x[4], r[4] = 2.0 ** -24, 0                           # tiny values
    for res in (None, r):
        out = ex.rms_norm_q8(x, w, 1e-6, residual=res)
        s, y = norm64(x, res, w, 1e-6)
        if res is not None:
            assert torch.equal(out[2].double(), s)
        check_q8(out[0], out[1], y, norm_terms(F) * U32)
    q, scale = ex.quantize_rows(x)
    check_q8(q, scale, x.double(), 0.0)
    q, scale = ex.quantize_rows(x, "silu")
    check_q8(q, scale, torch.nn.functional.silu(x.double()), 4 * U32)


def check_q8(q, scale, y, rel):
    want = (y.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    near(scale, want, (rel + 2 * U32) * want, "scale")
    got = q.double() * scale.double()[..., None]
    lim = y.abs() * (2.0 ** -4 + 4 * rel + 8 * U32) + scale.double()[..., None] * 2.0 ** -10 * (1 + 1e-5)
    assert bool(((got - y).abs() <= lim).all())
    assert bool((q.float().abs() <= 448).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_unusual_rows(dtype):
    """Strides, odd addresses, leading axes, no rows, and values at the ends of the range."""
    g = gen(3)
    w = (1 + 0.2 * rand(g, 97)).to(dtype)
    base = rand(g, 20, 200, dtype=dtype)
    for x in (base[:, 1:98], base[::2, 3:100], base[:, :97].t().contiguous().t(), base[:1, :97].expand(20, 97),
              base[:, 5:102].view(4, 5, 97), base[0, :97], base[:, ::2][:, :97]):
        y = ex.rms_norm(x, w)
        assert y.shape == x.shape and torch.equal(y, ex.rms_norm(x.clone(memory_format=torch.contiguous_format), w))
        q, s = ex.rms_norm_q8(x, w, residual=x)[:2]
        q1, s1 = ex.rms_norm_q8(x.contiguous(), w, residual=x.contiguous())[:2]
        assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)
    x = base[:0, :97].requires_grad_(True)
    wl = w.clone().requires_grad_(True)
    y, s = ex.rms_norm(x, wl, residual=base[:0, :97])
    gx, gw = torch.autograd.grad([y.sum() + s.sum()], [x, wl])
    assert y.shape == (0, 97) and gx.shape == (0, 97) and torch.equal(gw, torch.zeros_like(gw))
    assert ex.rms_norm_q8(base[:0, :97], w)[1].shape == (0,)
    # a NaN or an infinity stays in its row; zeros stay zeros, without eps NaN as 0 / 0
    x = rand(g, 6, 97, dtype=dtype)
    x[1, 5], x[2, 7], x[3] = math.nan, math.inf, 0
    y = ex.rms_norm(x, w)
    assert y[1].isnan().all() and y[2, 7].isnan() and bool((y[3] == 0).all())
    ok = ex.rms_norm(x[[0, 4, 5]], w)
    assert torch.equal(y[[0, 4, 5]], ok)
    assert ex.rms_norm(x, w, 0.0)[3].isnan().all()
    q, s = ex.rms_norm_q8(x, w)
    assert s[1].isnan() and q[1].float().isnan().all() and torch.isfinite(s[[0, 3, 4, 5]]).all()


# ----------------------------------------------------------------------------- gate
def route64(l, k, allowed, group, renorm, dw):
    """(expert, weight, dlogits) in 64 bits: a stable sort, softmax, and the formula's gradient."""
    l = l.double()
    if allowed is not None:
        gi = torch.zeros(l.shape[0], dtype=torch.long, device=l.device) if group is None else group.long()
        inside = (gi >= 0) & (gi < allowed.shape[0])
        open_ = allowed[gi.clamp(0, allowed.shape[0] - 1)] & inside[:, None]
        l = l.masked_fill(~open_, -math.inf)
    top, at = torch.sort(l, dim=1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    fits = top > -math.inf
    first = torch.where(fits[:, :1], top[:, :1], 0.0)
    p = torch.exp(l - first)
    p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    w = torch.where(fits, p.gather(1, at), 0.0)
    if renorm:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    gsel = torch.where(fits, dw.double(), 0.0)
    mean = (w * gsel).sum(1, keepdim=True)
    up = torch.zeros_like(l).scatter_add_(1, at, gsel)
    if renorm:
        d = torch.zeros_like(l).scatter_add_(1, at, w * (gsel - mean))
        mag = torch.zeros_like(l).scatter_add_(1, at, w * (gsel.abs() + (w * gsel.abs()).sum(1, keepdim=True)))
    else:
        d = p * (up - mean)
        mag = p * (up.abs() + (w * gsel.abs()).sum(1, keepdim=True))
    return torch.where(fits, at, -1).to(torch.int32), w, d, mag


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (8, 2), (16, 16), (17, 3), (64, 4), (100, 8), (256, 5), (257, 2), (1024, 16)])
def test_route(dtype, E, k):
    say("route", dtype, E, k)
    for N in (0, 1, 5, 301):
        g = gen(E + N)
        l = rand(g, N, E, dtype=dtype, scale=2.0)
        if N > 4:
            l[1] = 0                                     # ties throughout
            l[2] = -math.inf                             # nothing open
            l[3, ::2] = -math.inf
            l[4] = torch.finfo(dtype).min                # the lowest finite value is a logit like others
        allowed = torch.rand(3, E, generator=g, device=DEV) < 0.5
        allowed[2] = False                               # a species without experts
        group = torch.randint(-1, 4, (N,), generator=g, device=DEV, dtype=torch.int32)
        dw = rand(g, N, k)
        for a, gr in ((None, None), (allowed, group), (allowed[:1], None)):
            for renorm in (True, False):
                e64, w64, d64, mag = route64(l, k, a, gr, renorm, dw)
                x = l.detach().requires_grad_(True)
                e, w = ex.route(x, k, allowed=a, group=gr, renormalise=renorm)
                assert torch.equal(e, e64) and e.dtype == torch.int32
                # exp: two steps, and its argument's rounding, up to 30 of it; the sum's additions
                near(w, w64, (E / 16 + 50) * U32 * w64 + 1e-38, "weight")
                d, = torch.autograd.grad(w, x, dw)
                near(d, d64, 3 * (E / 16 + 60) * U32 * mag + 1e-38, "dlogits")
                e1, w1 = ex.route(l, k, allowed=a, group=gr, renormalise=renorm)
                assert torch.equal(e1, e) and torch.equal(w1, w)


def test_route_of_nan_infinity_and_strides():
    g = gen(5)
    l = rand(g, 8, 24)
    l[1, 3], l[2, 4], l[3, 5] = math.nan, math.inf, -math.inf
    l[4, 0], l[4, 1] = -0.0, 0.0
    l[4, 2:] = -1.0
    e, w = ex.route(l, 2)
    assert e[1, 0] == 3 and w[1].isnan().all() and e[2, 0] == 4 and w[2].isnan().all()
    assert e[4].tolist() == [0, 1] and w[4].tolist() == [0.5, 0.5]
    rows = [0, 3, 4, 5, 6, 7]
    e1, w1 = ex.route(l[rows], 2)
    assert torch.equal(e1, e[rows]) and torch.equal(w1, w[rows])
    wide = rand(g, 8, 60)
    for v in (wide[:, 7:31], wide[:, ::2], wide[:, :8].t(), wide[:1].expand(8, 60)):
        e, w = ex.route(v, 3)
        e1, w1 = ex.route(v.clone(memory_format=torch.contiguous_format), 3)
        assert torch.equal(e, e1) and torch.equal(w, w1)
    # an expanded upstream gradient
    x = wide.clone().requires_grad_(True)
    _, w = ex.route(x, 3, renormalise=False)
    d, = torch.autograd.grad(w.sum(), x)
    *_, d64, mag = route64(wide, 3, None, None, False, torch.ones_like(w))
    near(d, d64, 200 * U32 * mag)


def test_route_gradient_against_differences():
    g = gen(6)
    l, dw = rand(g, 12, 20), rand(g, 12, 4)
    for renorm in (True, False):
        x = l.clone().requires_grad_(True)
        e, w = ex.route(x, 4, renormalise=renorm)
        d, = torch.autograd.grad(w, x, dw)
        v = rand(g, 12, 20).double()

        def loss(z):
            p = torch.softmax(z, 1).gather(1, e.long())
            return ((p / p.sum(1, keepdim=True) if renorm else p) * dw.double()).sum()
        want = (loss(l.double() + 1e-5 * v) - loss(l.double() - 1e-5 * v)) / 2e-5
        assert abs((d.double() * v).sum() - want) <= 1e-5 * (d.double() * v).abs().sum()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [6, 64, 300])
def test_route_gradient_of_rows_that_are_not_finite(dtype, E):
    """A NaN or an infinity among a row's logits or upstream gradients reaches the experts that its weights depend on, and
    no other: closed ones, and (renormalised) those not chosen, have a gradient of exactly 0."""
    g = gen(E)
    k = 2
    l, dw = rand(g, 40, E, dtype=dtype), rand(g, 40, k)
    allowed = torch.rand(1, E, generator=g, device=DEV) < 0.5
    allowed[0, :2], allowed[0, 2] = True, False
    l[0, 1], l[1, 0], l[2, 3:], l[3, 2] = math.nan, math.inf, -math.inf, math.nan
    dw[4, 0], dw[5, 1], dw[6] = math.inf, math.nan, -math.inf
    odd = torch.arange(40, device=DEV) < 7
    for a in (None, allowed):
        open_ = (l > -math.inf) | l.isnan()
        if a is not None:
            open_ &= a
        for renorm in (True, False):
            say("gradient of odd rows", dtype, E, a is not None, renorm)
            x = l.clone().requires_grad_(True)
            e, w = ex.route(x, k, allowed=a, renormalise=renorm)
            d, = torch.autograd.grad(w, x, dw)
            got = torch.zeros_like(open_).scatter_(1, e.clamp_min(0).long(), e >= 0)
            reached = got if renorm else open_
            assert bool((d[~reached] == 0).all())
            assert bool(torch.isfinite(d[~odd]).all())
            # the mean of the upstream gradients over the weights is not finite in these rows, and no reached one escapes it
            hit = [0, 1, 4, 5, 6] + ([3] if a is None else [])
            for i in hit:
                assert not torch.isfinite(d[i][reached[i]]).any(), i
            ok = torch.autograd.grad(ex.route(x, k, allowed=a, renormalise=renorm)[1][7:], x, dw[7:])[0]
            assert torch.equal(ok[7:], d[7:])


# ----------------------------------------------------------------------------- grouping
@pytest.mark.parametrize("slots", [0, 1, 63, 64, 513, 4096, 4097, 70001, 5000000])
@pytest.mark.parametrize("G", [1, 3, 64, 1024])
def test_group_plan(slots, G):
    say("plan", slots, G)
    g = gen(slots + G)
    e = torch.randint(-2, G + 2, (slots,), generator=g, device=DEV, dtype=torch.int32)
    p = ex.group_plan(e, G)
    check_plan(p, e, G)
    assert p.rows == slots and p.k == 1 and p.n_groups == G
    far = e.long()
    far[far < 0] = -(1 << 40)
    far[far >= G] = (1 << 32) + G // 2                   # low words that look like groups
    q = ex.group_plan(far, G)
    assert torch.equal(q.ptr, p.ptr) and torch.equal(q.order, p.order)
    if slots:
        check_plan(ex.group_plan(torch.full_like(e, G - 1), G), torch.full_like(e, G - 1), G)
        check_plan(ex.group_plan(torch.full_like(e, -1), G), torch.full_like(e, -1), G)


def check_plan(p, e, G):
    c = torch.where((e >= 0) & (e < G), e, G).reshape(-1).long()
    assert torch.equal(p.order.long(), torch.sort(c, stable=True).indices)
    n = torch.bincount(c, minlength=G + 1)[:G]
    assert torch.equal(p.ptr.long(), torch.cat([n.new_zeros(1), n.cumsum(0)]))


def test_group_plan_of_choices():
    e = torch.tensor([[1, 0], [-1, 1], [0, 0]], dtype=torch.int32, device=DEV)
    for v in (e, e.t().contiguous().t(), e.long()):
        p = ex.group_plan(v, 2)
        assert (p.rows, p.k, p.slots) == (3, 2, 6)
        assert p.order.tolist() == [1, 4, 5, 0, 3, 2] and p.ptr.tolist() == [0, 3, 5]


# ----------------------------------------------------------------------------- products
def linear64(x, w, expert, bias, silu, dy=None):
    """(y, sum of the terms' magnitudes, dx and its terms, dw and its terms, db) by slots, in 64 bits. expert (N, k)."""
    N, k = expert.shape
    G, n, ki = w.shape
    e = expert.reshape(-1).long()
    per = x.shape[0] == N * k
    rows = torch.arange(N * k, device=DEV) // (1 if per else k)
    x64, w64 = x.double(), w.double()
    sg = torch.sigmoid(x64)
    h = x64 * sg if silu else x64
    y = torch.zeros(N * k, n, dtype=torch.float64, device=DEV)
    ay = torch.zeros_like(y)
    d = torch.zeros(N * k, ki, dtype=torch.float64, device=DEV)
    ad = torch.zeros_like(d)
    dw, adw = torch.zeros_like(w64), torch.zeros_like(w64)
    db, adb = torch.zeros(G, n, dtype=torch.float64, device=DEV), torch.zeros(G, n, dtype=torch.float64, device=DEV)
    for i in range(G):
        a = (e == i).nonzero()[:, 0]
        if not len(a):
            continue
        ha = h[rows[a]]
        y[a], ay[a] = ha @ w64[i].t(), ha.abs() @ w64[i].abs().t()
        if bias is not None:
            y[a] += bias[i].double()
            ay[a] += bias[i].double().abs()
        if dy is not None:
            g = dy[a].double()
            d[a], ad[a] = g @ w64[i], g.abs() @ w64[i].abs()
            if silu:
                # s (1 + z (1 - s)) crosses zero at z = -1.28: its error is 8 u of s (1 + |z| (1 - s)), a step or two
                # each of s, of 1 - s, of the product and of the sum, not of its value; ad counts both in units of
                # steps(T, 1) > 8 u
                sa, za = sg[rows[a]], x64[rows[a]]
                d[a] *= sa * (1 + za * (1 - sa))
                ad[a] *= sa * (1 + za.abs() * (1 - sa))
            dw[i], adw[i] = g.t() @ ha, g.abs().t() @ ha.abs()
            db[i], adb[i] = g.sum(0), g.abs().sum(0)
    return y, ay, d, ad, dw, adw, db, adb


def steps(dtype, m):
    """Steps of 2 u of a sum of m products: one per 16 of a matrix instruction (six instructions for float32,
    whose dropped limb products are another step), the joins and the epilogue."""
    return 2 * U32 * ((6 if dtype == F32 else 1) * (m / 16 + 1) + 16)


def check_linear(N, k, G, ki, n, dtype, per=False, silu=False, bias=True, expert=None, seed=0, grads=True, x=None, w=None):
    g = gen(seed + N + 7 * ki + n)
    if expert is None:
        expert = torch.randint(0, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
    x = rand(g, N * k if per else N, ki, dtype=dtype) if x is None else x
    w = rand(g, G, n, ki, dtype=dtype, scale=ki ** -0.5) if w is None else w
    b = rand(g, G, n, dtype=dtype) if bias else None
    dy = rand(g, N * k, n, dtype=dtype)
    plan = ex.group_plan(expert, G)
    y64, ay, d64, ad, dw64, adw, db64, adb = linear64(x, w, expert, b, silu, dy)
    op = "silu" if silu else None
    ls = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = ex.grouped_linear(x, w, plan, bias=b, x_op=op)
    # silu on load: four steps of float32, and the rounding to a 16-bit operand
    pre = (0 if not silu else 4 * U32 + (0 if dtype == F32 else u(dtype)))
    near(y, y64, (steps(dtype, ki) + pre) * ay, "y")
    with torch.no_grad():
        assert torch.equal(ex.grouped_linear(x, w, plan, bias=b, x_op=op), y)
    if grads:
        out = torch.autograd.grad(y, ls, dy)
        lim = (steps(dtype, n) + 8 * U32) * ad
        if per or k == 1:
            near(out[0], d64, lim, "dx")
        else:                                            # each choice's part rounded, then their sum
            part = (lim + u(dtype) * (d64.abs() + lim)).view(N, k, ki).sum(1)
            tiny = k * 2.0 ** -25 if dtype == F16 else 0.0
            near(out[0], d64.view(N, k, ki).sum(1), part + k * U32 * ad.view(N, k, ki).sum(1) + tiny, "dx")
        m = N * k
        # silu(x) as a float16 operand: below 2^-14 the type's values are 2^-24 apart, so its rounding is off by up to 2^-25
        # whatever its size, times |dy|. (A silu of 3.9e-6 in a group of one slot is 2^-25 / 3.9e-6 = 0.8 % off, 15 u.)
        sub = 2.0 ** -25 * adb[:, :, None] if silu and dtype == F16 else 0.0
        near(out[1], dw64, (steps(dtype, m) + pre) * adw + sub, "dw")
        if bias:
            near(out[2], db64, m * U32 * adb, "db")
        again = torch.autograd.grad(ex.grouped_linear(x, w, plan, bias=b, x_op=op), ls, dy)
        assert all(torch.equal(p, q) for p, q in zip(out, again))
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,G,ki,n", [(1, 1, 1, 1, 1), (1, 2, 64, 96, 40), (21, 1, 3, 192, 97), (21, 2, 8, 33, 65),
                                        (64, 3, 5, 864, 192), (130, 1, 2, 31, 129), (333, 4, 16, 257, 31),
                                        (1344, 1, 3, 96, 385), (2000, 2, 7, 130, 513), (5000, 1, 3, 200, 520),
                                        (9000, 2, 3, 72, 257)])
def test_grouped_linear(dtype, N, k, G, ki, n):
    say("grouped_linear", dtype, N, k, G, ki, n)
    check_linear(N, k, G, ki, n, dtype)
    check_linear(N, k, G, ki, n, dtype, per=True, silu=True, bias=False)
    check_linear(N, k, G, ki, n, dtype, silu=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,G,ki,n", [(513, 1, 96, 97), (600, 3, 1440, 320), (900, 1, 520, 264), (1600, 16, 512, 512),
                                      (1600, 3, 257, 130), (2500, 2, 2304, 512)])
def test_weight_gradient_by_shares_or_by_group(dtype, N, G, ki, n):
    """Sizes on both sides of the choice between shares of the slots and a workgroup per group; groups of equal size, and
    all slots but one in the last group."""
    say("shares", dtype, N, G, ki, n)
    check_linear(N, 1, G, ki, n, dtype)
    e = torch.full((N, 1), G - 1, dtype=torch.int32, device=DEV)
    e[N // 3] = 0
    check_linear(N, 1, G, ki, n, dtype, expert=e, silu=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,ki,n", [(30, 2, 5, 17), (700, 1, 200, 97), (20000, 2, 2304, 256)])
def test_bias_gradient_alone(dtype, N, k, ki, n):
    """Frozen weights with a trained bias, with and without rows that take gradients: no weight gradient is formed, nor room
    for one."""
    G = 64
    g = gen(ki)
    e = torch.randint(-1, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
    e[e == 3] = 4                                        # a group without slots
    plan = ex.group_plan(e, G)
    x, w, dy = rand(g, N, ki, dtype=dtype), rand(g, G, n, ki, dtype=dtype, scale=n ** -0.5), rand(g, N * k, n, dtype=dtype)
    b = rand(g, G, n, dtype=dtype).requires_grad_(True)
    i = torch.where(e < 0, G, e).reshape(-1).long()
    want = torch.zeros(G + 1, n, dtype=torch.float64, device=DEV).index_add_(0, i, dy.double())[:G]
    mag = torch.zeros(G + 1, n, dtype=torch.float64, device=DEV).index_add_(0, i, dy.double().abs())[:G]
    for op in (None, "silu"):
        say("bias alone", dtype, N, op)
        y = ex.grouped_linear(x, w, plan, bias=b, x_op=op)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        db, = torch.autograd.grad(y, b, dy)
        if ki > 2000:
            assert torch.cuda.max_memory_allocated() - before < w.numel() * w.element_size()
        near(db, want, N * k * U32 * mag, "db")
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        d, db1 = torch.autograd.grad(ex.grouped_linear(xl, w, plan, bias=b, x_op=op), [xl, b], dy)
        d0, _, _ = torch.autograd.grad(ex.grouped_linear(xl, wl, plan, bias=b, x_op=op), [xl, wl, b], dy)
        assert torch.equal(db1, db) and torch.equal(d, d0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 300, 20000])
def test_grouped_linear_of_thousands_of_groups(dtype, N):
    """A plan that a program made itself, of more groups than group_plan takes, most of them without rows."""
    G, ki, n = 5000, 24, 17
    g = gen(N)
    e = torch.randint(0, G, (N,), generator=g, device=DEV)
    x, w, b = rand(g, N, ki, dtype=dtype), rand(g, G, n, ki, dtype=dtype), rand(g, G, n, dtype=dtype)
    dy = rand(g, N, n, dtype=dtype)
    c = torch.bincount(e, minlength=G)
    plan = ex.GroupPlan(torch.cat([c.new_zeros(1), c.cumsum(0)]).int(), torch.sort(e, stable=True).indices.int(), N)
    ls = [t.requires_grad_(True) for t in (x, w, b)]
    y = ex.grouped_linear(x, w, plan, bias=b)
    dx, dw, db = torch.autograd.grad(y, ls, dy)
    x64, w64, d64 = x.detach().double(), w.detach().double()[e], dy.double()
    t = w64 * x64[:, None]
    bias = b.detach().double()[e]
    near(y, t.sum(2) + bias, steps(dtype, ki) * (t.abs().sum(2) + bias.abs()), "y")
    t = w64 * d64[:, :, None]
    near(dx, t.sum(1), steps(dtype, n) * t.abs().sum(1), "dx")
    t = d64[:, :, None] * x64[:, None]
    z = torch.zeros(G, n, ki, dtype=torch.float64, device=DEV)
    near(dw, z.index_add(0, e, t), steps(dtype, N) * z.index_add(0, e, t.abs()), "dw")
    near(db, z[:, :, 0].index_add(0, e, d64), N * U32 * z[:, :, 0].index_add(0, e, d64.abs()), "db")


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_linear_uneven_groups(dtype):
    """Groups without rows, one with all, slots of no group, a group of one row."""
    g = gen(1)
    for N in (40, 3000):
        for lo, hi in ((0, 1), (4, 5), (-1, 7), (2, 4), (-3, 0)):
            e = torch.randint(lo, hi, (N, 2), generator=g, device=DEV, dtype=torch.int32)
            e[N // 2, 1] = 5
            say("uneven", dtype, N, lo, hi)
            y = check_linear(N, 2, 6, 70, 260, dtype, expert=e)
            none = ((e < 0) | (e > 5)).reshape(-1)
            assert bool((y[none] == 0).all())
    # nothing anywhere
    e = torch.full((10, 1), -1, dtype=torch.int32, device=DEV)
    check_linear(10, 1, 4, 16, 16, dtype, expert=e)
    x, w = torch.zeros(0, 16, device=DEV, dtype=dtype, requires_grad=True), rand(g, 4, 8, 16, dtype=dtype).requires_grad_(True)
    y = ex.grouped_linear(x, w, ex.group_plan(e[:0], 4))
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert y.shape == (0, 8) and dx.shape == (0, 16) and bool((dw == 0).all())


def test_grouped_linear_float32_accuracy():
    """All three limbs enter: the error's norm stays below 1e-6 of the result's, where a product without the
    lowest limbs (2^-17 of each factor) would be 4e-6 off."""
    for N, k, G, ki, n in ((700, 1, 3, 1440, 320), (24000, 1, 3, 96, 64), (30, 2, 4, 512, 64)):
        g = gen(ki)
        e = torch.randint(0, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
        x, w, dy = rand(g, N, ki), rand(g, G, n, ki), rand(g, N * k, n)
        y64, _, d64, _, dw64, *_ = linear64(x, w, e, None, False, dy)
        x.requires_grad_(True), w.requires_grad_(True)
        y = ex.grouped_linear(x, w, ex.group_plan(e, G))
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        for a, b in ((y, y64), (dx, d64.view(N, k, ki).sum(1)), (dw, dw64)):
            assert (a.double() - b).norm() < 1e-6 * b.norm()


@pytest.mark.parametrize("dtype", TYPES)
def test_silu_of_far_values(dtype):
    """SiLU and its slope over the types' whole range: x sigmoid(x) falls to 0 on the left and is x on the right, the slope 0
    and 1; an infinity gives what the formula gives, NaN or itself. Left of -87 both are 0: |x| e^x < 87 e^-87 = 2^-118.9 there,
    the only difference that the 8-bit rows (scales down to 2^-126) could show."""
    far = [-104.0, -100.0, -90.0, -81.0, -80.5, -80.0, -79.5, -20.0, 0.0, 20.0, 79.5, 80.0, 80.5, 81.0, 90.0, 104.0, 1000.0, -1000.0,
           6e4, -6e4, math.inf, -math.inf, math.nan]
    far += [] if dtype == F16 else [v * 10.0 ** e for e in (10, 20, 30, 35, 38) for v in (-3.0, 3.0)]
    x = torch.tensor(far, device=DEV).to(dtype)[:, None]
    N = x.shape[0]
    x64 = x.double()
    sg = torch.sigmoid(x64)
    for reps in (1, 100):                                # few slots, and tiles of many
        say("far values", dtype, reps)
        xs = x.repeat(reps, 1).requires_grad_(True)
        plan = ex.group_plan(torch.arange(N, device=DEV).repeat(reps), N)
        w = torch.ones(N, 1, 1, device=DEV, dtype=dtype, requires_grad=True)
        y = ex.grouped_linear(xs, w, plan, x_op="silu")
        dy = torch.zeros(N * reps, 1, device=DEV, dtype=dtype)
        dy[:N] = 1
        d, dw = torch.autograd.grad(y, [xs, w], dy)
        want, slope = (x64 * sg)[:, 0], (sg * (1 + x64 * (1 - sg)))[:, 0]
        ok = torch.isfinite(want)
        pre = 4 * U32 + (0 if dtype == F32 else u(dtype))                     # as in check_linear
        # below 2^-126 a float32 product may be cut: 2^-126 |x|, and 2^-25 of a float16 operand
        tiny = 2.0 ** -126 * x64[:, 0].abs().clamp_max(1e4) + (2.0 ** -25 if dtype == F16 else 0.0)
        for got in (y[:N, 0], y[-N:, 0]):
            near(got[ok], want[ok], ((steps(dtype, 1) + pre) * want.abs() + tiny)[ok], "silu")
            assert torch.equal(got[~ok].double().nan_to_num(7.0), want[~ok].nan_to_num(7.0))
        fin = torch.isfinite(slope)
        mag = (sg * (1 + x64.abs() * (1 - sg)))[:, 0]
        near(d[:N, 0][fin], slope[fin], ((steps(dtype, 1) + 8 * U32) * mag + tiny)[fin], "slope")
        assert d[:N, 0][~fin].isnan().all()
        one = torch.autograd.grad(ex.grouped_linear(xs[:N], w, ex.group_plan(torch.arange(N, device=DEV), N), x_op="silu"), w,
                                  dy[:N])[0][:, 0, 0]
        near(one[ok], want[ok], ((steps(dtype, 1) + pre) * want.abs() + tiny)[ok], "dw")
    q, scale = ex.quantize_rows(x, "silu")
    left = x64 < -87
    assert bool(((x64 * sg)[left & ok[:, None]].abs() < 2.0 ** -118.9).all())
    check_q8(q[ok], scale[ok], torch.where(left, 0.0, x64 * sg)[ok], 4 * U32)


def test_grouped_linear_gradient_against_differences():
    g = gen(9)
    e = torch.randint(-1, 3, (15, 2), generator=g, device=DEV, dtype=torch.int32)
    x, w, b, dy = rand(g, 15, 20), rand(g, 3, 9, 20, scale=0.3), rand(g, 3, 9), rand(g, 30, 9)
    ls = [t.requires_grad_(True) for t in (x, w, b)]
    out = torch.autograd.grad(ex.grouped_linear(x, w, ex.group_plan(e, 3), bias=b, x_op="silu"), ls, dy)

    def loss(x, w, b):
        y, *_ = linear64(x, w, e, b, True)
        return (y * dy.double()).sum()

    for i in range(3):
        v = rand(g, *ls[i].shape).double()
        hi, lo = [t.detach().double() for t in ls], [t.detach().double() for t in ls]
        hi[i], lo[i] = hi[i] + 1e-5 * v, lo[i] - 1e-5 * v
        want = (loss(*hi) - loss(*lo)) / 2e-5
        assert abs((out[i].double() * v).sum() - want) <= 1e-5 * (out[i].double() * v).abs().sum()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,G,ki,n", [(1, 2, 3, 40, 24), (50, 4, 8, 257, 31), (700, 3, 4, 96, 130), (3000, 4, 8, 256, 192)])
def test_input_gradient_of_shared_rows_is_rounded_once(dtype, N, k, G, ki, n):
    """A row's choices are summed in 32 bits: one rounding to the rows' type, in the result."""
    g = gen(N + k)
    e = torch.randint(-1, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
    plan = ex.group_plan(e, G)
    w, dy = rand(g, G, n, ki, dtype=dtype, scale=n ** -0.5), rand(g, N * k, n, dtype=dtype)
    for silu in (False, True):
        say("shared rows", dtype, N, k, silu)
        x = rand(g, N, ki, dtype=dtype).requires_grad_(True)
        d, = torch.autograd.grad(ex.grouped_linear(x, w, plan, x_op="silu" if silu else None), x, dy)
        _, _, d64, ad, *_ = linear64(x.detach(), w, e, None, silu, dy)
        lim = (steps(dtype, n) + 8 * U32) * ad + k * U32 * ad
        near(d, d64.view(N, k, ki).sum(1), lim.view(N, k, ki).sum(1), "dx")


def test_input_gradient_whose_parts_pass_the_types_largest():
    """Choices whose parts pass float16's 65504 and cancel: 300 * 250 - 300 * 240."""
    x = torch.zeros(40, 8, device=DEV, dtype=F16, requires_grad=True)
    w = torch.tensor([250.0, -240.0], device=DEV, dtype=F16).view(2, 1, 1).expand(2, 1, 8)
    plan = ex.group_plan(torch.tensor([[0, 1]], device=DEV).expand(40, 2), 2)
    d, = torch.autograd.grad(ex.grouped_linear(x, w, plan), x, torch.full((80, 1), 300.0, device=DEV, dtype=F16))
    assert bool((d == 3000).all())


# Sizes (N, G, ki, n) that take tiles of 128 x 64 (the first four, in both directions) and 128 x 128 (the next three in one
# direction, the last two in both) of 16-bit rows on 256 CUs: sums that end within a chunk of 64, groups that end within a
# tile, last columns of 8 to 128; both operands whole chunks of 16 bytes, one of them or neither.
LARGE = [(24000, 3, 264, 320), (24000, 3, 320, 319), (24000, 3, 257, 264), (24000, 3, 319, 257), (24000, 3, 136, 200),
         (24000, 3, 200, 135), (24000, 3, 135, 200), (12000, 3, 520, 520), (16000, 3, 2304, 392)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,G,ki,n", LARGE)
def test_large_tiles(dtype, N, G, ki, n):
    say("large tiles", dtype, N, ki, n)
    g = gen(ki)
    e = torch.randint(-1, G, (N, 1), generator=g, device=DEV, dtype=torch.int32)
    check_linear(N, 1, G, ki, n, dtype, expert=e)
    check_linear(N, 1, G, ki, n, dtype, expert=e, silu=True, bias=False)
    if ki < 300:                                          # odd addresses of either operand
        wide, ww = rand(g, N, ki + 9, dtype=dtype), rand(g, G, n, ki + 8, dtype=dtype, scale=ki ** -0.5)
        check_linear(N, 1, G, ki, n, dtype, expert=e, x=wide[:, 1:ki + 1].detach(), w=ww[..., :ki].detach())
        check_linear(N, 1, G, ki, n, dtype, expert=e, x=wide[:, :ki].detach(), w=ww[..., 1:ki + 1].detach())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,k,G,ki,n", [(1, 1, 1, 1, 1), (21, 2, 3, 192, 97), (40, 1, 3, 2048, 300), (700, 1, 3, 1440, 320),
                                        (3000, 2, 4, 257, 65)] + [(N, 1, G, ki, n) for N, G, ki, n in LARGE])
def test_silu_on_load_adds_no_rounding(dtype, N, k, G, ki, n):
    """silu of 16-bit rows enters the products in two limbs, h = T(s) and T(s - h): off by u^2 of it (2^-16, 2^-22), and in
    float16, whose values are 2^-24 apart at the least, by 2^-25 whatever its size. One limb would be off by u."""
    say("two limbs", dtype, N, k, ki, n)
    g = gen(N + ki)
    e = torch.randint(-1, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
    plan = ex.group_plan(e, G)
    x, w = rand(g, N * k, ki, dtype=dtype), rand(g, G, n, ki, dtype=dtype, scale=ki ** -0.5)
    dy = rand(g, N * k, n, dtype=dtype)
    y64, ay, _, _, dw64, adw, _, adb = linear64(x, w, e, None, True, dy)
    w.requires_grad_(True)
    y = ex.grouped_linear(x, w, plan, x_op="silu")
    dw, = torch.autograd.grad(y, w, dy)
    pre = 4 * U32 + u(dtype) ** 2
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    sums = torch.cat([w.detach().double().abs().sum(2), torch.zeros(1, n, device=DEV).double()])
    rows = sums[torch.where(e < 0, G, e).reshape(-1).long()]
    near(y, y64, (steps(dtype, 2 * ki) + pre) * ay + tiny * rows, "y")
    near(dw, dw64, (steps(dtype, 2 * N * k) + pre) * adw + tiny * adb[:, :, None], "dw")
    if min(ki, n) > 90 and N > 20:
        # the norm of the error: that of the result's rounding, uniform within a step, u / sqrt 3 of a value at the most
        for got, want in ((y, y64), (dw, dw64)):
            assert (got.double() - want).norm() <= 1.02 * (want.to(dtype).double() - want).norm()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_products_of_many_slots(dtype):
    """The forward and the input gradient of a hundred thousand slots, one row each and two of a row."""
    N, G, ki, n = 100300, 6, 1544, 656
    g = gen(18)
    w = rand(g, G, n, ki, dtype=dtype, scale=ki ** -0.5)
    for k, rows in ((1, N), (2, N // 2)):
        e = torch.randint(-1, 5, (rows, k), generator=g, device=DEV, dtype=torch.int32)
        plan = ex.group_plan(e, G)
        x, dy = rand(g, rows, ki, dtype=dtype).requires_grad_(True), rand(g, rows * k, n, dtype=dtype)
        y = ex.grouped_linear(x, w, plan)
        d, = torch.autograd.grad(y, x, dy)
        y64, ay, d64, ad, *_ = linear64(x.detach(), w, e, None, False, dy)
        near(y, y64, steps(dtype, ki) * ay, "y")
        lim = (steps(dtype, n) + k * U32) * ad.view(rows, k, ki).sum(1)
        near(d, d64.view(rows, k, ki).sum(1), lim, "dx")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weight_gradient_of_many_slots(dtype):
    """Tiles of 256 x 256: a hundred thousand slots in uneven groups, one of them empty, and slots of none."""
    N, G, ki, n = 100300, 6, 1544, 656
    g = gen(8)
    e = torch.randint(-1, 4, (N,), generator=g, device=DEV, dtype=torch.int32)
    e[:30000] = 5
    plan = ex.group_plan(e, G)
    x, w = rand(g, N, ki, dtype=dtype), rand(g, G, n, ki, dtype=dtype).requires_grad_(True)
    b, dy = rand(g, G, n, dtype=dtype).requires_grad_(True), rand(g, N, n, dtype=dtype)
    dw, db = torch.autograd.grad(ex.grouped_linear(x, w, plan, bias=b), [w, b], dy)
    for i in range(G):
        a = e == i
        xa, da, m = x[a].double(), dy[a].double(), int(a.sum())
        near(dw[i], da.t() @ xa, steps(dtype, m) * (da.abs().t() @ xa.abs()), f"dw {i}")
        near(db[i], da.sum(0), m * U32 * da.abs().sum(0), f"db {i}")
    again = torch.autograd.grad(ex.grouped_linear(x, w, plan, bias=b), [w, b], dy)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [50, 4000])
def test_grouped_linear_strides(dtype, N):
    """Row strides, odd addresses, column-major and expanded operands and gradients."""
    g = gen(N)
    e = torch.randint(0, 3, (N, 1), generator=g, device=DEV, dtype=torch.int32)
    wide, ww = rand(g, N, 200, dtype=dtype), rand(g, 4, 300, 200, dtype=dtype, scale=0.1)
    for x, w in ((wide[:, 1:100], ww[1:, 5:275, 3:102]), (wide[:, :99].t().contiguous().t(), ww[:3, :, :99]),
                 (wide[:1, :99].expand(N, 99), ww[:1, :270, :99].expand(3, 270, 99)),
                 (wide[:, ::2][:, :99], ww[:3, :, :99].transpose(1, 2).contiguous().transpose(1, 2)),
                 (wide[:, :99], ww.view(4, 300, 200)[:3, ::2, :99])):
        check_linear(N, 1, 3, 99, w.shape[1], dtype, expert=e, x=x.detach(), w=w.detach())
    x, w = wide[:, :99].detach().clone().requires_grad_(True), ww[:3, :270, :99].detach().clone().requires_grad_(True)
    plan = ex.group_plan(e, 3)
    a = torch.autograd.grad(ex.grouped_linear(x, w, plan).sum(), [x, w])
    b = torch.autograd.grad(ex.grouped_linear(x, w, plan), [x, w], torch.ones(N, 270, device=DEV, dtype=dtype))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("N", [40, 5000])
def test_grouped_linear_values_that_are_not_finite(N):
    """Infinities and NaN stay in their rows and their group, and float32 values past bfloat16's largest are products
    like others."""
    g = gen(2)
    e = (torch.arange(N, device=DEV, dtype=torch.int32) % 3)[:, None]
    plan = ex.group_plan(e, 3)
    for dtype in TYPES:
        x, w = rand(g, N, 80, dtype=dtype), rand(g, 3, 300, 80, dtype=dtype)
        ok = ex.grouped_linear(x, w, plan)
        bx = x.clone()
        bx[4, 7], bx[5, 9], bx[6, 3] = math.nan, math.inf, -math.inf
        y = ex.grouped_linear(bx, w, plan)
        rest = [i for i in range(N) if i not in (4, 5, 6)]
        assert torch.equal(y[rest], ok[rest]) and y[4].isnan().all()
        assert torch.equal(y[5], math.inf * w[2, :, 9].sign()) and torch.equal(y[6], -math.inf * w[0, :, 3].sign())
        bw = w.clone()
        bw[1, 11, 5] = math.inf
        y = ex.grouped_linear(x, bw, plan)
        want = ok.clone()
        want[1::3, 11] = math.inf * x[1::3, 5].sign()
        assert torch.equal(y, want)
        # weights of a group without rows are not looked at
        none = torch.cat([w, torch.full_like(w[:1], math.nan)])
        assert torch.equal(ex.grouped_linear(x, none, ex.group_plan(e, 4)), ok)
        # gradients: a NaN in dy reaches its row and its group only
        dy = rand(g, N, 300, dtype=dtype)
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        good = torch.autograd.grad(ex.grouped_linear(xl, wl, plan), [xl, wl], dy)
        dy[7, 13] = math.nan
        d, dw = torch.autograd.grad(ex.grouped_linear(xl, wl, plan), [xl, wl], dy)
        assert d[7].isnan().all() and torch.equal(d[:7], good[0][:7]) and torch.equal(d[8:], good[0][8:])
        assert dw[1, 13].isnan().all() and torch.equal(dw[0], good[1][0]) and torch.equal(dw[2], good[1][2])
    big = 3.4e38                                          # bfloat16 ends at 3.39e38
    x, w = torch.zeros(N, 80, device=DEV), torch.zeros(3, 300, 80, device=DEV)
    x[:, 3], w[:, :, 3] = big, 0.5
    assert bool((ex.grouped_linear(x, w, plan) == torch.tensor(big, device=DEV) * 0.5).all())


@pytest.mark.parametrize("N,G,ki,n", [(21, 3, 300, 97), (21, 3, 33, 65), (100, 3, 2048, 2048), (700, 3, 1440, 320), (3000, 3, 96, 70),
                                      (12000, 3, 520, 330)])
def test_float32_values_past_the_range_of_bfloat16(N, G, ki, n):
    """Products of fp32 values past bfloat16's largest (3.39e38), in one row and column or everywhere, and of infinities and
    NaN everywhere, in every tile and direction: as plain float32 products, whose sums of m terms are off by m u of them."""
    say("past bfloat16", N, G, ki, n)
    g = gen(N + ki)
    e = torch.randint(0, G, (N, 1), generator=g, device=DEV, dtype=torch.int32)
    plan = ex.group_plan(e, G)
    big = lambda *s: (3.395e38 + 5e35 * torch.rand(*s, generator=g, device=DEV)) * (torch.randint(0, 2, s, generator=g, device=DEV) * 2 - 1)
    tiny = lambda *s: rand(g, *s, scale=2.0 ** -100)
    for where in ("rows", "weights", "all"):
        x, w, dy = rand(g, N, ki), rand(g, G, n, ki), tiny(N, n)
        if where == "rows":
            x, w = tiny(N, ki), tiny(G, n, ki)
            x[N // 2, ki // 3], x[0, 0], dy[N // 3, n // 2] = 3.4e38, -3.4e38, 3.4e38
        elif where == "weights":
            x, w = tiny(N, ki), tiny(G, n, ki)
            w[G - 1, n // 2, ki // 2] = w[0, 0, 0] = 3.4e38
        else:
            x, w = big(N, ki), tiny(G, n, ki) if N > 100 else tiny(G, n, ki) * 2.0 ** -20
        y64, ay, d64, ad, dw64, adw, *_ = linear64(x, w, e, None, False, dy)
        x.requires_grad_(True), w.requires_grad_(True)
        y = ex.grouped_linear(x, w, plan)
        d, dw = torch.autograd.grad(y, [x, w], dy)
        for got, want, terms, m, what in ((y, y64, ay, ki, "y"), (d, d64, ad, n, "dx"), (dw, dw64, adw, N, "dw")):
            assert bool(torch.isfinite(got).all()), (where, what)
            near(got, want, (m * U32 + steps(F32, m)) * terms + 2.0 ** -126, (where, what))
    for v in (math.nan, math.inf):
        x, w, dy = torch.full((N, ki), v, device=DEV), rand(g, G, n, ki), rand(g, N, n)
        dy[:, 0], w[:, 0] = dy[:, 0].abs(), w[:, 0].abs()                  # a column whose infinities agree
        y64, _, d64, *_ = linear64(x, w, e, None, False, torch.full_like(dy, v))
        x.requires_grad_(True), w.requires_grad_(True)
        y = ex.grouped_linear(x, w, plan)
        dw64 = linear64(x.detach(), w.detach(), e, None, False, dy)[4]
        dw, = torch.autograd.grad(y, w, dy)
        d, = torch.autograd.grad(ex.grouped_linear(x, w, plan), x, torch.full_like(dy, v))
        for got, want in ((y, y64), (d, d64), (dw, dw64)):
            assert torch.equal(got.double().nan_to_num(7.0), want.nan_to_num(7.0)), v


def test_float32_values_that_are_not_finite_cost_a_bounded_time():
    """A diverged step: every value NaN or infinite takes some ten times a finite step's time, where sums formed again one by
    one take hundreds."""
    g = gen(1)
    N, G, ki, n = 24000, 3, 1440, 320
    plan = ex.group_plan(torch.randint(0, G, (N,), generator=g, device=DEV, dtype=torch.int32), G)
    w, dy = rand(g, G, n, ki).requires_grad_(True), rand(g, N, n)

    def ms(v):
        x = (rand(g, N, ki) if v is None else torch.full((N, ki), v, device=DEV)).requires_grad_(True)
        up = dy if v is None else torch.full_like(dy, v)
        best = math.inf
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            torch.autograd.grad(ex.grouped_linear(x, w, plan), [x, w], up)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    fine = ms(None)
    for v in (math.nan, math.inf):
        t = ms(v)
        say("ms: finite", fine, "of", v, t)
        assert t < 60 * fine


def test_plans_that_name_no_slot_are_bounded():
    """Ranges and slots outside the plan are left out: no access outside the operands."""
    g = gen(4)
    x, w = rand(g, 8, 32), rand(g, 3, 20, 32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    plan = ex.GroupPlan(i32(-5, 4, 3, 99), i32(0, 1, -7, 3, 1 << 30, 5, 6, 7), 8)
    y = ex.grouped_linear(x, w, plan)
    assert torch.equal(y[0], ex.grouped_linear(x[:1], w, ex.GroupPlan(i32(0, 1, 1, 1), i32(0), 1))[0])
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    for t in torch.autograd.grad(ex.grouped_linear(xl, wl, plan), [xl, wl], torch.ones_like(y)):
        assert t.shape
    # every group claims all slots: more pieces than the workspace of the weight gradient has places
    n = 4000
    x, w = rand(g, n, 16).requires_grad_(True), rand(g, 3, 8, 16).requires_grad_(True)
    p = torch.zeros(4, dtype=torch.int32, device=DEV)
    p[1::2] = n
    plan = ex.GroupPlan(p, torch.arange(n, dtype=torch.int32, device=DEV), n)
    torch.autograd.grad(ex.grouped_linear(x, w, plan).sum(), [x, w])
    torch.cuda.synchronize()


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("N,k,G,ki,n", [(1, 1, 1, 1, 1), (1, 2, 64, 96, 40), (21, 2, 8, 33, 65), (64, 3, 5, 864, 192),
                                        (333, 4, 16, 257, 31), (5000, 1, 3, 200, 520), (9000, 2, 3, 72, 257)])
def test_grouped_linear_q8(out, N, k, G, ki, n):
    say("q8 linear", out, N, k, G, ki, n)
    g = gen(N + ki)
    e = torch.randint(-1, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
    plan = ex.group_plan(e, G)
    for per in (False, True):
        q, xs = ex.quantize_rows(rand(g, N * k if per else N, ki))
        wq, ws = ex.quantize_rows(rand(g, G, n, ki))
        b = rand(g, G, n, dtype=out) if per else None
        y = ex.grouped_linear_q8(q, xs, wq, ws, plan, bias=b, dtype=out)
        x64, w64 = q.double() * xs.double()[:, None], wq.double() * ws.double()[..., None]
        y64, ay, *_ = linear64(x64, w64, e, b, False)
        # float32: exact products, a step of the instruction per 16 of them, and the scales. 16 bits: the e4m3
        # instruction cuts each of 64 products below 2^-13 of the largest (the products of a step, or the sum so
        # far), which is at most ay: 2^-13 of a mean product for each, and of ay for each of ki / 64 sums
        cut = 0.0 if out == F32 else 2.0 ** -13 * (1 + math.ceil(ki / 64))
        near(y, y64, (2 * U32 * (ki / 16 + 16) + cut) * ay, "y")
        assert y.dtype == out and bool((y.view(N, k, n)[e < 0] == 0).all())
    # columns of a wider matrix, at an odd address
    wide = torch.zeros(N, ki + 9, device=DEV, dtype=E4M3)
    q, xs = ex.quantize_rows(rand(g, N, ki))
    wide[:, 5:5 + ki] = q
    assert torch.equal(ex.grouped_linear_q8(wide[:, 5:5 + ki], xs, wq, ws, plan, dtype=out),
                       ex.grouped_linear_q8(q, xs, wq, ws, plan, dtype=out))


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("N,G,ki,n", [(24000, 3, 272, 320), (24000, 3, 136, 264), (24000, 3, 144, 200), (24000, 3, 200, 135),
                                      (12000, 3, 528, 520), (16000, 3, 2304, 392)])
def test_large_tiles_q8(out, N, G, ki, n):
    """Tiles of 128 x 64 and 128 x 128 in 8 bits: chunks of 128, whole or not, either operand at an odd address."""
    say("large tiles q8", out, N, ki, n)
    g = gen(ki)
    e = torch.randint(-1, G, (N, 1), generator=g, device=DEV, dtype=torch.int32)
    plan = ex.group_plan(e, G)
    q, xs = ex.quantize_rows(rand(g, N, ki))
    wq, ws = ex.quantize_rows(rand(g, G, n, ki))
    b = rand(g, G, n, dtype=out)
    y = ex.grouped_linear_q8(q, xs, wq, ws, plan, bias=b, dtype=out)
    y64, ay, *_ = linear64(q.double() * xs.double()[:, None], wq.double() * ws.double()[..., None], e, b, False)
    # 16 bits: each of a step's 64 products cut below 2^-13 of the largest of them, which is at most the terms' sum
    cut = 0.0 if out == F32 else 2.0 ** -13 * math.ceil(ki / 64)
    near(y, y64, (2 * U32 * (ki / 16 + 16) + cut) * ay, "y")
    assert bool((y[e[:, 0] < 0] == 0).all())
    wide, ww = torch.zeros(N, ki + 16, device=DEV, dtype=E4M3), torch.zeros(G, n, ki + 16, device=DEV, dtype=E4M3)
    for at, bt in ((5, 0), (0, 3), (16, 16)):
        wide[:, at:at + ki], ww[..., bt:bt + ki] = q, wq
        assert torch.equal(ex.grouped_linear_q8(wide[:, at:at + ki], xs, ww[..., bt:bt + ki], ws, plan, bias=b, dtype=out), y)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("N,n", [(40, 64), (3000, 512), (24000, 320), (24000, 200)])
def test_q8_sums_of_one_sign(out, N, n):
    """The cut of the 8-bit instruction goes by the products of a step, not by the sum so far: a sum of 2304 positive products
    keeps its digits. Operands in [1/2, 1], so that no product is below a quarter of a step's largest: the cut, 2^-13 of that
    largest for each, is at most 2^-11 of each product. By the sum so far it would be up to 64 2^-13 of it in each of 36 steps."""
    g = gen(n)
    q = (0.5 + 0.5 * torch.rand(N, 2304, generator=g, device=DEV)).to(E4M3)
    wq = (0.5 + 0.5 * torch.rand(1, n, 2304, generator=g, device=DEV)).to(E4M3)
    ones, plan = torch.ones(N, device=DEV), ex.group_plan(torch.zeros(N, dtype=torch.int32, device=DEV), 1)
    y = ex.grouped_linear_q8(q, ones, wq, torch.full((1, n), 2.0 ** -5, device=DEV), plan, dtype=out)
    want = q.double() @ wq[0].double().t() / 32
    near(y, want, (2 * U32 * (2304 / 16 + 16) + (0.0 if out == F32 else 2.0 ** -11)) * want, "y")


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("N,n", [(3, 5), (2000, 300)])
def test_grouped_linear_q8_of_far_scales(out, N, n):
    """Scales whose product leaves float32's range while the result does not: sums of 0 stay 0, tiny and huge ones keep
    their digits."""
    k = 48
    plan = ex.group_plan(torch.zeros(N, dtype=torch.int32, device=DEV), 1)
    fill = lambda v, *shape: torch.full(shape, v, device=DEV).to(E4M3)
    for xv, wv, xs, ws in ((448.0, 416.0, 1.2345 * 2.0 ** -70, 1.7 * 2.0 ** -72), (2.0 ** -9, 3 * 2.0 ** -9, 1.3 * 2.0 ** 90, 1.1 * 2.0 ** 40),
                           (448.0, 0.0, 2.0 ** 100, 2.0 ** 40), (0.0, 448.0, 2.0 ** 40, 2.0 ** 100), (448.0, 448.0, 2.0 ** 100, 1.1 * 2.0 ** -120),
                           (448.0, 448.0, 1.3 * 2.0 ** -120, 2.0 ** 110)):
        y = ex.grouped_linear_q8(fill(xv, N, k), torch.full((N,), xs, device=DEV), fill(wv, 1, n, k), torch.full((1, n), ws, device=DEV),
                                 plan, dtype=out)
        f32 = lambda v: torch.tensor(v, dtype=F32).double().item()
        want = torch.full((N, n), k * xv * wv * f32(xs) * f32(ws), device=DEV, dtype=torch.float64)
        # equal products, whose partial sums are whole multiples below 2^24 of one: exact; three roundings of scales
        near(y, want, 3 * U32 * want.abs(), f"{xs:.3g} {ws:.3g}")


def test_rows_past_two_to_the_31_elements():
    """Rows of x, y and the gradient whose offsets pass 32 bits."""
    N, n = 70000, 33000
    g = gen(1)
    e = (torch.arange(N, device=DEV) % 2).to(torch.int32)
    plan = ex.group_plan(e, 2)
    x, w = rand(g, N, 16, dtype=BF16), rand(g, 2, n, 16, dtype=BF16)
    y = ex.grouped_linear(x, w, plan)
    rows = torch.tensor([0, 1, 35001, N - 2, N - 1], device=DEV)
    want = torch.stack([x[r].double() @ w[int(e[r])].double().t() for r in rows])
    mag = torch.stack([x[r].double().abs() @ w[int(e[r])].double().abs().t() for r in rows])
    near(y[rows], want, steps(BF16, 16) * mag)
    s = ex.rms_norm(y, torch.ones(n, device=DEV, dtype=BF16))
    _, y64 = norm64(y[rows], None, torch.ones(n, device=DEV), 1e-6)
    near(s[rows], y64, norm_terms(n) * U32 * y64.abs())
    del s
    xl = x.clone().requires_grad_(True)
    d, = torch.autograd.grad(ex.grouped_linear(xl, w, plan), xl, y)
    want = torch.stack([y[r].double() @ w[int(e[r])].double() for r in rows])
    mag = torch.stack([y[r].double().abs() @ w[int(e[r])].double().abs() for r in rows])
    near(d[rows], want, steps(BF16, n) * mag)
    out = ex.expert_combine(y, torch.full((N, 1), 2.0, device=DEV))
    assert torch.equal(out[rows], 2 * y[rows])


def test_gradients_past_two_to_the_31_elements():
    """Offsets that pass 32 bits in the backwards: the weight gradient's and the norm's rows, the join's slots."""
    N, n = 70000, 33000
    g = gen(2)
    e = (torch.arange(N, device=DEV) % 2).to(torch.int32)
    plan = ex.group_plan(e, 2)
    x, w = rand(g, N, 16, dtype=BF16), rand(g, 2, n, 16, dtype=BF16).requires_grad_(True)
    b = torch.zeros(2, n, device=DEV, dtype=BF16, requires_grad=True)
    dy = rand(g, N, n, dtype=BF16)
    for op in (None, "silu"):                             # staged without and through registers
        say("weight gradient past 2^31", op)
        dw, db = torch.autograd.grad(ex.grouped_linear(x, w, plan, bias=b, x_op=op), [w, b], dy)
        cols = torch.tensor([0, 1, 16500, n - 2, n - 1], device=DEV)
        h = x.double() * (torch.sigmoid(x.double()) if op else 1)
        pre = (4 * U32 + u(BF16)) if op else 0
        for i in range(2):
            da, ha = dy[i::2, cols].double(), h[i::2]
            near(dw[i, cols], da.t() @ ha, (steps(BF16, N) + pre) * (da.abs().t() @ ha.abs()), f"dw {i}")
            near(db[i, cols], da.sum(0), N * U32 * da.abs().sum(0), f"db {i}")
    # x rows past 2^31, gathered by the weight gradient
    wt = rand(g, 2, 8, n, dtype=BF16, scale=0.01).requires_grad_(True)
    up = rand(g, N, 8, dtype=BF16)
    dw, = torch.autograd.grad(ex.grouped_linear(dy, wt, plan), wt, up)
    for i in range(2):
        da, ha = up[i::2].double(), dy[i::2, cols].double()
        near(dw[i][:, cols], da.t() @ ha, steps(BF16, N) * (da.abs().t() @ ha.abs()), f"dw of wide rows {i}")
    del dw, db
    say("norm past 2^31")
    rows = torch.tensor([0, 1, 35001, N - 2, N - 1], device=DEV)
    wn = torch.ones(n, device=DEV, dtype=BF16, requires_grad=True)
    xs = dy.detach().requires_grad_(True)
    up = torch.ones(1, 1, device=DEV, dtype=BF16).expand(N, n)
    d, dwn = torch.autograd.grad(ex.rms_norm(xs, wn, 1e-5), [xs, wn], up)
    s = dy[rows].double()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    m = s.mean(-1, keepdim=True)
    mag = rstd * (1 + s.abs() * rstd ** 2 * s.abs().mean(-1, keepdim=True))
    near(d[rows], rstd * (1 - s * rstd ** 2 * m), 3 * (norm_terms(n) + 4) * U32 * mag, "dx")
    rstd = 1 / torch.sqrt(torch.stack([(dy[i:i + 10000].double() ** 2).mean(1) for i in range(0, N, 10000)]).reshape(-1, 1) + 1e-5)
    t = dy[:, cols].double() * rstd
    near(dwn[cols], t.sum(0), (N + norm_terms(n) + 8) * U32 * t.abs().sum(0), "dw")
    del d, xs, up
    say("join past 2^31")
    y, wc = dy.detach().requires_grad_(True), rand(g, N // 2, 2).requires_grad_(True)
    dout = rand(g, N // 2, n, dtype=BF16)
    gy, gw = torch.autograd.grad(ex.expert_combine(y, wc), [y, wc], dout)
    at, j = rows // 2, rows % 2
    near(gy[rows], wc.detach().double()[at, j][:, None] * dout[at].double(), torch.zeros((), device=DEV).double(), "dy")
    t = dy[rows].double() * dout[at].double()
    near(gw[at, j], t.sum(1), (n + 8) * U32 * t.abs().sum(1), "dweight")


# ----------------------------------------------------------------------------- join
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,F", [(0, 2, 8), (1, 1, 1), (21, 2, 96), (50, 3, 257), (301, 8, 512), (40, 20, 700),
                                   (17, 5, 5000), (1000, 2, 33)])
def test_expert_combine(dtype, N, k, F):
    say("combine", dtype, N, k, F)
    g = gen(N + k)
    y, w, r = rand(g, N * k, F, dtype=dtype), rand(g, N, k), rand(g, N, F, dtype=dtype)
    dout = rand(g, N, F, dtype=dtype)
    y64, w64 = y.double().view(N, k, F), w.double()
    for res in (None, r):
        ls = [t.detach().requires_grad_(True) for t in (y, w, res) if t is not None]
        out = ex.expert_combine(ls[0], ls[1], residual=ls[2] if res is not None else None)
        want = (w64[:, :, None] * y64).sum(1) + (0 if res is None else res.double())
        mag = (w64[:, :, None] * y64).abs().sum(1) + (0 if res is None else res.double().abs())
        near(out, want, (k + 1) * U32 * mag, "out")
        gr = torch.autograd.grad(out, ls, dout)
        near(gr[0], (w64[:, :, None] * dout.double()[:, None]).view(N * k, F), torch.zeros((), device=DEV).double(), "dy")
        t = y64 * dout.double()[:, None]
        near(gr[1], t.sum(2), (F + 8) * U32 * t.abs().sum(2), "dweight")
        if res is not None:
            assert torch.equal(gr[2], dout)
        with torch.no_grad():
            assert torch.equal(ex.expert_combine(y, w, residual=res), out)
        only, = torch.autograd.grad(ex.expert_combine(y, ls[1], residual=res), ls[1:2], dout)
        assert torch.equal(only, gr[1])


def test_expert_combine_strides_and_broadcast():
    g = gen(1)
    wide, w = rand(g, 40, 300), rand(g, 2, 20).t()
    for y in (wide[:, 3:100], wide[:, ::3][:, :97], wide[:1, :97].expand(40, 97)):
        a = ex.expert_combine(y, w, residual=wide[:20, 7:104])
        b = ex.expert_combine(y.contiguous(), w.contiguous(), residual=wide[:20, 7:104].contiguous())
        assert torch.equal(a, b)
    y, wl = wide[:, :97].clone().requires_grad_(True), w.clone().requires_grad_(True)
    a = torch.autograd.grad(ex.expert_combine(y, wl).sum(), [y, wl])
    b = torch.autograd.grad(ex.expert_combine(y, wl), [y, wl], torch.ones(20, 97, device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # one weight for all rows
    s = torch.ones(1, 1, device=DEV, requires_grad=True)
    d, = torch.autograd.grad(ex.expert_combine(wide, s.expand(20, 2)).sum(), s)
    assert abs(d.item() - wide.double().sum().item()) <= 1e-5 * wide.double().abs().sum().item()


# ----------------------------------------------------------------------------- together
class _Layer:
    """A pre-norm expert layer: gate on the normalised rows, two products by expert, the residual."""

    def __init__(self, g, C, H, E, k, dtype):
        self.k, self.E = k, E
        self.p = [(1 + 0.1 * rand(g, C)).to(dtype), rand(g, E, C, dtype=dtype, scale=C ** -0.5),
                  rand(g, E, H, C, dtype=dtype, scale=C ** -0.5), rand(g, E, H, dtype=dtype, scale=0.1),
                  rand(g, E, C, H, dtype=dtype, scale=H ** -0.5), rand(g, E, C, dtype=dtype, scale=0.1)]

    def __call__(self, x, r, allowed=None, group=None):
        w, gate, w1, b1, w2, b2 = self.p
        y, s = ex.rms_norm(x, w, 1e-6, residual=r)
        expert, weight = ex.route(y @ gate.t(), self.k, allowed=allowed, group=group)
        plan = ex.group_plan(expert, self.E)
        u_ = ex.grouped_linear(y, w1, plan, bias=b1)
        v = ex.grouped_linear(u_, w2, plan, bias=b2, x_op="silu")
        return ex.expert_combine(v, weight, residual=s)

    def plain(self, x, r, ps, expert, allowed=None, group=None):
        """The same in 64 bits, dense over the experts, with the choices that were made."""
        w, gate, w1, b1, w2, b2 = ps
        s = x + r
        y = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6) * w
        l = y @ gate.t()
        at = expert.clamp_min(0).long()
        p = torch.where(expert >= 0, torch.exp(l.gather(1, at)), 0.0)
        p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
        out = s
        for j in range(self.k):
            for e in range(self.E):
                m = (expert[:, j] == e).double() * p[:, j]
                h = torch.nn.functional.silu(y @ w1[e].t() + b1[e])
                out = out + m[:, None] * (h @ w2[e].t() + b2[e])
        return out


def _layer_case(dtype=F32, N=300):
    g = gen(11)
    layer = _Layer(g, 48, 72, 5, 2, dtype)
    x, r = rand(g, N, 48, dtype=dtype), rand(g, N, 48, dtype=dtype)
    allowed = torch.tensor([[1, 1, 1, 0, 0], [0, 0, 1, 1, 1], [0, 0, 0, 0, 1], [0, 0, 0, 0, 0]], dtype=torch.bool, device=DEV)
    group = torch.randint(0, 4, (N,), generator=g, device=DEV, dtype=torch.int32)
    return layer, x, r, allowed, group, rand(g, N, 48, dtype=dtype)


def test_expert_layer_end_to_end():
    """The operators as one layer, forward and backward, species that open some, one or no experts."""
    layer, x, r, allowed, group, dout = _layer_case()
    leaves = [x.requires_grad_(True), r.requires_grad_(True)] + [p.requires_grad_(True) for p in layer.p]
    out = layer(x, r, allowed, group)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        y, _ = ex.rms_norm(x, layer.p[0], 1e-6, residual=r)
        expert, _ = ex.route(y @ layer.p[1].t(), 2, allowed=allowed, group=group)
    ls = [t.detach().double().requires_grad_(True) for t in leaves]
    want = layer.plain(ls[0], ls[1], ls[2:], expert)
    wg = torch.autograd.grad(want, ls, dout.double())
    assert (out.double() - want).norm() < 1e-6 * want.norm()
    for a, b, n in zip(grads, wg, ("x", "r", "w", "gate", "w1", "b1", "w2", "b2")):
        assert (a.double() - b).norm() < 3e-6 * b.norm(), n
    none = group == 3
    assert torch.equal(out[none], (x + r)[none])          # no expert: the residual alone


def test_expert_layer_in_8_bits():
    """The serving chain: its result is that of the float32 chain up to the roundings of two 8-bit operands per
    product. A product of K terms with two independent relative errors of at most 2^-4 each (uniform within a
    step: rms 2^-4 / sqrt(3) at most) is off by at most sqrt(2) 2^-4 / sqrt(3) = 0.051 of the terms' norm, which is the
    result's for random operands; two products and the step of silu between them: 0.11."""
    layer, x, r, _, _, _ = _layer_case()
    w, gate, w1, b1, w2, b2 = layer.p
    q1, s1 = ex.quantize_rows(w1)
    q2, s2 = ex.quantize_rows(w2)
    y, s = ex.rms_norm(x, w, 1e-6, residual=r)
    expert, weight = ex.route(y @ gate.t(), 2)
    plan = ex.group_plan(expert, 5)
    full = ex.expert_combine(ex.grouped_linear(ex.grouped_linear(y, w1, plan, bias=b1), w2, plan, bias=b2, x_op="silu"), weight)
    q, sc, s8 = ex.rms_norm_q8(x, w, 1e-6, residual=r)
    assert torch.equal(s8, s)
    u8 = ex.grouped_linear_q8(q, sc, q1, s1, plan, bias=b1, dtype=F32)
    h, hs = ex.quantize_rows(u8, "silu")
    out = ex.expert_combine(ex.grouped_linear_q8(h, hs, q2, s2, plan, bias=b2, dtype=F32), weight)
    assert (out - full).norm() < 0.11 * full.norm()


def test_other_streams_and_two_calls_at_once():
    """Two layers on two streams at once, and tensors made on another stream than the one they are used on."""
    layer, x, r, allowed, group, _ = _layer_case(N=3000)
    want = layer(x, r, allowed, group)
    want2 = layer(r, x, allowed, group)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for st, a, b in ((s1, x, r), (s2, r, x)):
            with torch.cuda.stream(st):
                got.append(layer(a, b, allowed, group))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want2 if i % 2 else want)
    leaf = x.detach().requires_grad_(True)
    ref, = torch.autograd.grad(layer(leaf, r).sum(), leaf)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        out = layer(leaf, r).sum()
    s2.wait_stream(s1)
    with torch.cuda.stream(s2):
        g2, = torch.autograd.grad(out, leaf)
    torch.cuda.synchronize()
    assert torch.equal(g2, ref)


def test_two_captured_graphs():
    """Forward and backward captured twice and replayed in turn with new inputs, eager work between; every replay
    equals the eager result."""
    layer, x0, r0, allowed, group, dout = _layer_case(N=2500)
    g = gen(21)

    def step(x, r):
        leaves = [x.detach().requires_grad_(True)] + [p.detach().requires_grad_(True) for p in layer.p]
        keep, layer.p = layer.p, leaves[1:]
        out = layer(leaves[0], r, allowed, group)
        layer.p = keep
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dout))

    held = []
    for _ in range(2):
        x, r = x0.clone(), r0.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(x, r)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            outs = step(x, r)
        held.append((cg, x, r, outs))
    for turn in range(4):
        for cg, x, r, outs in held:
            x.copy_(rand(g, *x.shape))
            r.copy_(rand(g, *r.shape))
            cg.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step(x, r)):
                assert torch.equal(a, b), turn


def test_a_recorded_backward_is_refused():
    """Second derivatives would be dropped in silence: a backward with create_graph raises, in every operator."""
    g = gen(0)
    x, w = rand(g, 4, 8).requires_grad_(True), rand(g, 2, 4).softmax(1).requires_grad_(True)
    plan = ex.group_plan(torch.zeros(4, dtype=torch.int32, device=DEV), 1)
    for out in (ex.rms_norm(x, torch.ones(8, device=DEV)), ex.route(x, 2)[1], ex.grouped_linear(x, rand(g, 1, 3, 8), plan),
                ex.expert_combine(x, rand(g, 2, 2)), ex.expert_combine(x.detach(), w[:, :2])):
        leaf = x if out.grad_fn.next_functions[0][0] is not None else w
        with pytest.raises(NotImplementedError, match="differentiate once"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)


def test_tangents_of_gradients_are_refused():
    """Forward over reverse: a gradient that comes with a tangent raises in every operator's backward, and calls without
    one give what they give outside a dual level."""
    g = gen(3)
    x, plan = rand(g, 4, 8).requires_grad_(True), ex.group_plan(torch.zeros(4, dtype=torch.int32, device=DEV), 1)
    w, m, c = rand(g, 8), rand(g, 1, 3, 8), rand(g, 2, 2)
    ops = [lambda: ex.rms_norm(x, w), lambda: ex.route(x, 2)[1], lambda: ex.grouped_linear(x, m, plan), lambda: ex.expert_combine(x, c)]
    for f in ops:
        ones = torch.ones_like(f())
        want, = torch.autograd.grad(f(), x, ones)
        with torch.autograd.forward_ad.dual_level():
            got, = torch.autograd.grad(f(), x, ones)
            assert torch.equal(got, want)
            with pytest.raises(NotImplementedError, match="gradient: no forward-mode"):
                torch.autograd.grad(f(), x, torch.autograd.forward_ad.make_dual(ones, ones))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ex.rms_norm(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()), w)


def test_gradients_of_some_operands():
    """Every subset of the leaves: the gradients that all leaves together get, and nothing for the others."""
    import itertools
    g = gen(12)
    N, k, F, G = 40, 2, 96, 5
    e = torch.randint(-1, G, (N, k), generator=g, device=DEV, dtype=torch.int32)
    plan = ex.group_plan(e, G)
    for dtype in TYPES:
        r = lambda *s: rand(g, *s, dtype=dtype)
        cases = [(lambda x, w, q: ex.rms_norm(x, w, 1e-5, residual=q), [r(N, F), r(F), r(N, F)], [r(N, F), r(N, F)]),
                 (lambda x, w, b: (ex.grouped_linear(x, w, plan, bias=b, x_op="silu"),), [r(N, F), r(G, 33, F), r(G, 33)], [r(N * k, 33)]),
                 (lambda y, c, q: (ex.expert_combine(y, c, residual=q),), [r(N * k, F), rand(g, N, k), r(N, F)], [r(N, F)])]
        for f, ops, ups in cases:
            fresh = lambda on: [t.detach().requires_grad_(i in on) for i, t in enumerate(ops)]
            ls = fresh((0, 1, 2))
            full = torch.autograd.grad(f(*ls), ls, ups)
            for m in (1, 2):
                for on in itertools.combinations(range(3), m):
                    ls = fresh(on)
                    for i, d in zip(on, torch.autograd.grad(f(*ls), [ls[j] for j in on], ups)):
                        assert torch.equal(d, full[i]) and d.dtype == ops[i].dtype, (dtype, on)
        x, w, q = (t.detach().requires_grad_(True) for t in cases[0][1])
        _, s = ex.rms_norm(x, w, residual=q)
        d = torch.autograd.grad(s, [x, w, q], cases[0][2][0])                # of the sum alone
        assert torch.equal(d[0], cases[0][2][0]) and torch.equal(d[2], d[0]) and not d[1].any()


def test_one_tensor_twice_and_backward_twice():
    """The same leaf as two operands, the same weights in two products, and a backward run again on a kept graph."""
    g = gen(5)
    x, w = rand(g, 70, 40).requires_grad_(True), rand(g, 40).requires_grad_(True)
    dy, ds = rand(g, 70, 40), rand(g, 70, 40)
    both = torch.autograd.grad(ex.rms_norm(x, w, 1e-5, residual=x), [x, w], [dy, ds])
    r = x.detach().clone().requires_grad_(True)
    apart = torch.autograd.grad(ex.rms_norm(x, w, 1e-5, residual=r), [x, r, w], [dy, ds])
    assert torch.equal(both[0], apart[0] + apart[1]) and torch.equal(both[1], apart[2])
    x.grad = r.grad = None
    torch.autograd.backward(ex.rms_norm(x, w, 1e-5, residual=r), [dy, ds])
    assert x.grad.data_ptr() != r.grad.data_ptr() and torch.equal(x.grad, apart[0]) and torch.equal(r.grad, apart[1])

    plan = ex.group_plan(torch.randint(0, 3, (70, 1), generator=g, device=DEV, dtype=torch.int32), 3)
    m = rand(g, 3, 40, 40, scale=0.2).requires_grad_(True)
    u = ex.grouped_linear(x, m, plan)
    v = ex.grouped_linear(u, m, plan, x_op="silu")
    once = torch.autograd.grad(v, [x, m, u], dy, retain_graph=True)
    again = torch.autograd.grad(v, [x, m, u], dy)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    d1, = torch.autograd.grad(ex.grouped_linear(x, m, plan), m, once[2])
    d2, = torch.autograd.grad(ex.grouped_linear(u.detach(), m, plan, x_op="silu"), m, dy)
    assert torch.equal(once[1], d1 + d2) or torch.equal(once[1], d2 + d1)
    with torch.autograd.set_multithreading_enabled(False):
        u = ex.grouped_linear(x, m, plan)
        one = torch.autograd.grad(ex.grouped_linear(u, m, plan, x_op="silu"), [x, m, u], dy)
    assert all(torch.equal(a, b) for a, b in zip(once, one))

    weight = torch.softmax(rand(g, 35, 2), 1).requires_grad_(True)
    y = rand(g, 70, 40).requires_grad_(True)
    d = rand(g, 35, 40)
    gy, = torch.autograd.grad(ex.expert_combine(y, weight, residual=y[:35]), y, d)
    a, b = torch.autograd.grad(ex.expert_combine(y, weight, residual=r[:35]), [y, r], d)
    assert torch.equal(gy, a + b)


def test_an_operand_changed_before_its_backward_is_noticed():
    """What the backward reads is what the forward read: torch's version check covers operands, results and plans."""
    g = gen(6)
    x, m = rand(g, 12, 8).requires_grad_(True), rand(g, 2, 8, 8).requires_grad_(True)
    plan = ex.group_plan(torch.arange(12, device=DEV) % 2, 2)
    r = rand(g, 12, 8)
    y, s = ex.rms_norm(x, torch.ones(8, device=DEV), residual=r)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    y = ex.grouped_linear(x, m, plan)
    plan.order.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), m)
