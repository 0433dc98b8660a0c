"""What the row operators beside the expert layer refuse, before anything reaches a device: no GPU calls."""
import pytest
import torch

from face_amd import _lib
from face_amd import experts as ex

X = torch.zeros(4, 8)
W = torch.ones(8)
I = torch.zeros(4, dtype=torch.int32)
PLAN = ex.GroupPlan(torch.tensor([0, 4], dtype=torch.int32), torch.arange(4, dtype=torch.int32), 4)
Q, S = X.to(torch.float8_e4m3fn), torch.ones(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)


def bad(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def test_host_tensors_are_refused():
    for f in (lambda: ex.layer_norm(X, W), lambda: ex.layer_norm_q8(X, W), lambda: ex.pack_rows(X), lambda: ex.unpack_rows(Q, S),
              lambda: ex.gated_silu(X), lambda: ex.embed(X, I), lambda: ex.expert_dispatch(X, PLAN),
              lambda: ex.expert_return(X, PLAN), lambda: ex.grouped_linear(X, torch.zeros(1, 3, 8), PLAN, keep8=True)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


def test_tangents_are_refused():
    dual, level = torch.autograd.forward_ad.make_dual, torch.autograd.forward_ad.dual_level
    with level():
        d = lambda t: dual(t, torch.ones_like(t))
        for f in (lambda: ex.layer_norm(d(X), W), lambda: ex.layer_norm(X, d(W)), lambda: ex.layer_norm(X, W, d(W)),
                  lambda: ex.layer_norm(X, W, residual=d(X)), lambda: ex.layer_norm_q8(d(X), W), lambda: ex.pack_rows(d(X)),
                  lambda: ex.gated_silu(d(X)), lambda: ex.embed(d(X), I), lambda: ex.expert_dispatch(d(X), PLAN),
                  lambda: ex.expert_return(d(X), PLAN), lambda: ex.expert_return(X, PLAN, d(torch.ones(4, 1))),
                  lambda: ex.expert_return(X, PLAN, residual=d(X))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()


def test_layer_norm_refusals():
    for f in (ex.layer_norm, ex.layer_norm_q8):
        bad("float32, bfloat16 or float16", f, X.double(), W.double())
        bad("x .* and w", f, X, torch.ones(7))
        bad("rows' type", f, X, W.half())
        bad("b like w", f, X, W, torch.ones(7))
        bad("b like w", f, X, W, W.half())
        bad("residual like x", f, X, W, W, residual=torch.zeros(3, 8))
        bad("eps >= 0", f, X, W, W, -1.0)
        bad("eps >= 0", f, X, W, W, float("nan"))
        bad("columns", f, torch.zeros(4, 0), torch.ones(0))
        bad("columns", f, torch.zeros(1, 65537), torch.ones(65537))


def test_kept_rows_refusals():
    bad("float32, bfloat16 or float16", ex.pack_rows, X.double())
    bad("columns", ex.pack_rows, torch.zeros(3, 0))
    bad("columns", ex.pack_rows, torch.tensor(1.0))
    bad("float8_e4m3fn rows", ex.unpack_rows, X, S)
    bad("dtype", ex.unpack_rows, Q, S, torch.float64)
    bad("scale", ex.unpack_rows, Q, S[:3])
    bad("scale", ex.unpack_rows, Q, S.view(torch.uint8))
    bad("scale", ex.unpack_rows, torch.zeros(4, 33).to(torch.float8_e4m3fn), S)
    bad("float32, bfloat16 or float16", ex.gated_silu, X.double())
    bad("x .* 2 F", ex.gated_silu, torch.zeros(4, 7))
    bad("x .* 2 F", ex.gated_silu, torch.zeros(4, 0))
    many = torch.empty(1 << 31, 2, device="meta")
    bad("2\\^31 rows", ex.pack_rows, many)
    bad("2\\^31 rows", ex.gated_silu, many)
    bad("2\\^31 rows", ex.unpack_rows, many.to(torch.float8_e4m3fn), many)


def test_embed_refusals():
    bad("float32, bfloat16 or float16", ex.embed, X.double(), I)
    bad("table", ex.embed, torch.zeros(8), I)
    bad("table", ex.embed, torch.zeros(0, 8), I)
    bad("table", ex.embed, torch.zeros(4, 0), I)
    bad("table", ex.embed, torch.zeros(1, 65537), I)
    bad("int32 or int64", ex.embed, X, I.float())
    bad("int32 or int64", ex.embed, X, I.to(torch.uint8))
    bad("a number", ex.embed, X, I, torch.ones(()))


def test_rows_by_expert_refusals():
    for f in (ex.expert_dispatch, ex.expert_return):
        bad("float32, bfloat16 or float16", f, X.double(), PLAN)
        bad("GroupPlan", f, X, I)
        bad("slots", f, torch.zeros(5, 8), PLAN)
        bad("columns", f, torch.zeros(4, 0), PLAN)
    bad("weight", ex.expert_return, X, PLAN, torch.ones(4))
    bad("weight", ex.expert_return, X, PLAN, torch.ones(4, 1).half())
    bad("residual", ex.expert_return, X, PLAN, residual=torch.zeros(4, 7))
    bad("residual", ex.expert_return, X, PLAN, residual=X.half())


def test_entry_points_refuse_bad_arguments():
    """The C entries: what they refuse before any launch, and the empty calls that launch nothing."""
    L = _lib.lib()
    ok = 1                                        # a non-null pointer that is never followed
    ln = lambda N=1, F=8, ld=8, dt=0, x=ok, y=ok, s=None, r=None, q=None, sc=None, bs=None, m=None, rs=None, eps=1e-6: \
        L.face_layer_norm_rows_fwd(x, ld, r, ld, N, F, dt, ok, None, eps, y, s, q, sc, bs, m, rs, None)
    assert ln(N=-1) == ln(F=0) == ln(ld=7) == ln(dt=3) == ln(x=None) == ln(y=None) == ln(s=ok) == ln(r=ok) == ln(eps=-1.0) == -1
    assert ln(q=ok) == ln(q=ok, sc=ok) == ln(q=ok, bs=ok) == ln(sc=ok) == ln(m=ok) == ln(y=None, q=ok, sc=ok, bs=ok) == -1
    assert ln(F=65537, ld=65537) == -2 and ln(N=0) == 0
    need = L.face_layer_norm_rows_bwd_work(5, 8)
    lb = lambda work=ok, n=need, s=ok, q=None, bs=None, m=ok, rs=ok, dw=ok, ld=8: L.face_layer_norm_rows_bwd(
        s, ld, q, bs, m, rs, ok, 8, None, 8, 5, 8, 0, ok, None, dw, None, work, n, None)
    assert need > 0 and lb(work=None) == lb(n=need - 1) == lb(s=None) == lb(m=None) == lb(rs=None) == lb(q=ok) == lb(ld=7) == -1
    assert lb(dw=None) == 0
    pk = lambda N=1, F=8, ld=8, dt=0, q=ok: L.face_pack_rows(ok, ld, N, F, dt, q, ok, None)
    assert pk(N=-1) == pk(F=0) == pk(ld=7) == pk(dt=3) == pk(q=None) == -1 and pk(N=0) == 0 and pk(N=1 << 31) == -2
    up = lambda N=1, F=40, ld=40, ls=2, dt=0, q=ok: L.face_unpack_rows(q, ld, ok, ls, N, F, dt, ok, None)
    assert up(N=-1) == up(F=0) == up(ld=39) == up(ls=1) == up(dt=3) == up(q=None) == -1 and up(N=0) == 0
    gf = lambda N=1, F=8, ld=16, q=None, s=None, y=ok: L.face_gated_silu_fwd(ok, ld, N, F, 0, y, q, s, None)
    assert gf(N=-1) == gf(F=0) == gf(ld=15) == gf(q=ok) == gf(s=ok) == gf(y=None) == -1 and gf(N=0) == 0
    gb = lambda x=ok, q=None, s=None, ld=8, N=1: L.face_gated_silu_bwd(x, 16, q, s, ok, ld, N, 8, 0, ok, None)
    assert gb(x=None) == gb(q=ok) == gb(x=None, q=ok) == gb(ld=7) == gb(N=-1) == -1 and gb(N=0) == 0
    ef = lambda N=1, V=3, F=8, ld=8, wide=0, dt=0, t=ok: L.face_embed_fwd(t, ld, ok, wide, N, V, F, dt, 1.0, ok, None, None)
    assert ef(N=-1) == ef(V=0) == ef(F=0) == ef(ld=7) == ef(wide=2) == ef(dt=3) == ef(t=None) == -1 and ef(N=0) == 0
    assert ef(N=1 << 31) == ef(V=(1 << 31) - 1) == -2
    need = L.face_embed_bwd_work(5000, 100, 8)
    eb = lambda N=5000, V=100, ld=8, n=need, work=ok, d=ok, key=ok: L.face_embed_bwd(key, ok, ld, N, V, 8, 0, 1.0, d, work, n, None)
    assert need > 0 and eb(N=-1) == eb(V=0) == eb(ld=7) == eb(n=need - 1) == eb(work=None) == eb(d=None) == eb(key=None) == -1
    assert L.face_embed_bwd_work(100, 100, 8) == 0
    dp = lambda N=4, k=2, G=2, F=8, ld=8, dt=0, x=ok: L.face_expert_dispatch(x, ld, k, ok, ok, None, N, G, F, dt, ok, None)
    assert dp(N=-1) == dp(k=0) == dp(G=0) == dp(F=0) == dp(ld=7) == dp(dt=3) == dp(x=None) == -1 and dp(N=0) == 0
    assert dp(N=1 << 30, k=2) == -2
    rf = lambda N=4, k=2, F=8, ld=8, p=ok, r=None, o=ok, G=2: L.face_expert_return_fwd(ok, ld, o, o, p, 0, ok, r, 7, N, k, G, F, 0, ok,
                                                                                     None)
    assert rf(N=-1) == rf(k=0) == rf(F=0) == rf(ld=7) == rf(p=None) == rf(r=ok) == rf(o=None) == rf(G=0) == -1 and rf(N=0) == 0
    rb = lambda dy=ok, dw=ok, y=ok, ld=8: L.face_expert_return_bwd(ok, ld, y, 8, ok, ok, ok, ok, 4, 2, 2, 8, 0, dy, dw, None)
    assert rb(y=None) == rb(ld=7) == -1 and rb(dy=None, dw=None) == 0
