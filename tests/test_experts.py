"""What the expert layer's operators refuse, before anything reaches a device: no GPU calls."""
import pytest
import torch

from face_amd import _lib
from face_amd import experts as ex


def bad(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


X = torch.zeros(4, 8)


def test_host_tensors_are_refused():
    plan = ex.GroupPlan(torch.tensor([0, 4], dtype=torch.int32), torch.arange(4, dtype=torch.int32), 4)
    q, s = torch.zeros(4, 8).to(torch.float8_e4m3fn), torch.ones(4)
    for f in (lambda: ex.rms_norm(X, torch.ones(8)), lambda: ex.rms_norm_q8(X, torch.ones(8)),
              lambda: ex.quantize_rows(X), lambda: ex.route(X, 2), lambda: ex.group_plan(torch.zeros(4, dtype=torch.int32), 2),
              lambda: ex.grouped_linear(X, torch.zeros(1, 3, 8), plan),
              lambda: ex.grouped_linear_q8(q, s, q[None, :3], s[None, :3], plan),
              lambda: ex.expert_combine(X, torch.ones(2, 2))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


def test_tangents_are_refused():
    """Forward mode: the kernels read values alone, so an operand with a tangent raises, whichever it is."""
    dual, level = torch.autograd.forward_ad.make_dual, torch.autograd.forward_ad.dual_level
    plan = ex.GroupPlan(torch.tensor([0, 4], dtype=torch.int32), torch.arange(4, dtype=torch.int32), 4)
    w, m, b, c = torch.ones(8), torch.zeros(1, 3, 8), torch.zeros(1, 3), torch.ones(2, 2)
    q, mq, s = X.to(torch.float8_e4m3fn), m.to(torch.float8_e4m3fn), torch.ones(4)
    with level():
        d = lambda t: dual(t, torch.ones_like(t))
        for f in (lambda: ex.rms_norm(d(X), w), lambda: ex.rms_norm(X, d(w)), lambda: ex.rms_norm(X, w, residual=d(X)),
                  lambda: ex.rms_norm_q8(d(X), w), lambda: ex.rms_norm_q8(X, w, residual=d(X)), lambda: ex.quantize_rows(d(X)),
                  lambda: ex.route(d(X), 2), lambda: ex.grouped_linear(d(X), m, plan),
                  lambda: ex.grouped_linear(X, d(m), plan), lambda: ex.grouped_linear(X, m, plan, bias=d(b)),
                  lambda: ex.grouped_linear_q8(q, d(s), mq, b, plan), lambda: ex.grouped_linear_q8(q, s, mq, d(b), plan),
                  lambda: ex.expert_combine(d(X), c), lambda: ex.expert_combine(X, d(c)),
                  lambda: ex.expert_combine(X, c, residual=d(X[:2]))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        with pytest.raises(RuntimeError, match="no CPU path"):       # others are checked as ever
            ex.rms_norm(X, w)


def test_norm_refusals():
    w = torch.ones(8)
    for f in (ex.rms_norm, ex.rms_norm_q8):
        bad("float32, bfloat16 or float16", f, X.double(), w.double())
        bad("x .* and w", f, X, torch.ones(7))
        bad("x .* and w", f, X, torch.ones(1, 8))
        bad("rows' type", f, X, w.bfloat16())
        bad("residual like x", f, X, w, residual=torch.zeros(3, 8))
        bad("residual like x", f, X, w, residual=X.half())
        bad("eps >= 0", f, X, w, -1.0)
        bad("eps >= 0", f, X, w, float("nan"))
        bad("columns", f, torch.zeros(4, 0), torch.ones(0))
        bad("columns", f, torch.zeros(1, 65537), torch.ones(65537))
    bad("x_op", ex.quantize_rows, X, "gelu")
    bad("float32, bfloat16 or float16", ex.quantize_rows, X.int())


def test_route_refusals():
    bad("logits", ex.route, torch.zeros(8), 1)
    bad("k <= min", ex.route, X, 0)
    bad("k <= min", ex.route, X, 9)
    bad("k <= min", ex.route, torch.zeros(2, 100), 17)
    bad("k <= min", ex.route, torch.zeros(2, 1025), 1)
    bad("group without allowed", ex.route, X, 1, group=torch.zeros(4, dtype=torch.int32))
    bad("allowed", ex.route, X, 1, allowed=torch.ones(1, 7, dtype=torch.bool))
    bad("allowed", ex.route, X, 1, allowed=torch.ones(1, 8))
    bad("allowed", ex.route, X, 1, allowed=torch.ones(0, 8, dtype=torch.bool))
    bad("needs group", ex.route, X, 1, allowed=torch.ones(2, 8, dtype=torch.bool))
    bad("group", ex.route, X, 1, allowed=torch.ones(2, 8, dtype=torch.bool), group=torch.zeros(4, dtype=torch.int64))
    bad("group", ex.route, X, 1, allowed=torch.ones(2, 8, dtype=torch.bool), group=torch.zeros(3, dtype=torch.int32))


def test_plan_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bad("expert", ex.group_plan, i(2, 2, 2), 3)
    bad("expert", ex.group_plan, i(2, 0), 3)
    bad("int32 or int64", ex.group_plan, torch.zeros(4), 3)
    bad("n_groups", ex.group_plan, i(4), 0)
    bad("n_groups", ex.group_plan, i(4), 1025)
    bad("int32 vector", ex.GroupPlan, i(2).long(), i(4), 4)
    bad("int32 vector", ex.GroupPlan, i(2), i(8)[::2], 4)
    bad("ptr", ex.GroupPlan, i(1), i(4), 4)
    bad("order", ex.GroupPlan, i(2), i(4), 4, 2)
    bad("rows >= 0", ex.GroupPlan, i(2), i(4), -1)
    bad("2\\^31", ex.GroupPlan, i(2), i(4), 1 << 30, 2)


def test_linear_refusals():
    plan = ex.GroupPlan(torch.zeros(4, dtype=torch.int32), torch.arange(8, dtype=torch.int32), 4, 2)
    w = torch.zeros(3, 5, 8)
    f = ex.grouped_linear
    bad("GroupPlan", f, X, w, None)
    bad("x_op", f, X, w, plan, x_op="relu")
    bad("x .* and w", f, X, w[:, :, :7], plan)
    bad("x .* and w", f, X, w[0], plan)
    bad("x .* and w", f, X[:, :0], w[:, :, :0], plan)
    bad("3 groups", f, X, w[:2], plan)
    bad("4 rows or 8 slots", f, torch.zeros(5, 8), w, plan)
    bad("rows' type", f, X, w.half(), plan)
    bad("bias", f, X, w, plan, bias=torch.zeros(3, 4))
    bad("bias", f, X, w, plan, bias=torch.zeros(3, 5).half())
    bad("float32, bfloat16 or float16", f, X.double(), w.double(), plan)
    q, wq, s = X.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn), torch.ones(4)
    g = ex.grouped_linear_q8
    bad("float8_e4m3fn", g, X, s, w, torch.ones(3, 5), plan)
    bad("x_scale", g, q, torch.ones(8), wq, torch.ones(3, 5), plan)
    bad("x_scale", g, q, s.half(), wq, torch.ones(3, 5), plan)
    bad("w_scale", g, q, s, wq, torch.ones(3), plan)
    bad("dtype", g, q, s, wq, torch.ones(3, 5), plan, dtype=torch.float64)
    bad("bias", g, q, s, wq, torch.ones(3, 5), plan, bias=torch.zeros(3, 5))


def test_combine_refusals():
    f = ex.expert_combine
    bad("y .* and weight", f, X, torch.ones(4, 2))
    bad("y .* and weight", f, X, torch.ones(4))
    bad("y .* and weight", f, X[:0], torch.ones(4, 0))
    bad("float32 weights", f, X, torch.ones(2, 2).half())
    bad("residual", f, X, torch.ones(2, 2), residual=torch.zeros(4, 8))
    bad("residual", f, X, torch.ones(2, 2), residual=torch.zeros(2, 8).half())


def test_entry_points_refuse_bad_arguments():
    """The C entries: what they refuse before any launch, and the empty calls that launch nothing."""
    L = _lib.lib()
    ok = 1                                        # a non-null pointer that is never followed
    norm = lambda N=1, F=8, ld=8, dt=0, x=ok, y=ok, q=None, s=None, r=None: L.face_rms_norm_fwd(
        x, ld, r, ld, N, F, dt, ok, 1e-6, y, s, q, None, None)
    assert norm(N=-1) == norm(F=0) == norm(ld=7) == norm(dt=3) == norm(x=None) == norm(y=None) == -1
    assert norm(q=ok) == norm(s=ok) == norm(r=ok) == norm(dt=-1) == -1
    assert norm(F=65537, ld=65537) == -2 and norm(N=0) == 0
    bwd = lambda work, n: L.face_rms_norm_bwd(ok, 8, ok, 8, None, 8, 5, 8, 0, ok, 1e-6, None, ok, work, n, None)
    need = L.face_rms_norm_bwd_work(5, 8)
    assert need > 0 and bwd(None, need) == -1 and bwd(ok, need - 1) == -1
    rt = lambda E=8, k=2, dt=0, a=None, g=None, ng=0, N=1, ld=None: L.face_route_fwd(
        ok, E if ld is None else ld, N, E, k, dt, a, g, ng, 1, None, None, None)
    assert rt(k=0) == rt(k=9) == rt(E=0) == rt(dt=5) == rt(g=ok) == rt(a=ok) == rt(a=ok, ng=2) == rt(ld=7) == rt() == -1
    assert rt(E=1025) == rt(E=64, k=17) == -2 and rt(N=0) == 0
    plan = lambda n=10, G=4, p=ok, w=None, nb=0: L.face_group_plan(ok, n, G, p, ok, w, nb, None)
    assert plan(n=-1) == plan(G=0) == plan(p=None) == plan(n=5000) == -1 and plan(G=1025) == plan(n=1 << 31) == -2
    lin = lambda n=5, k=8, dt=0, slots=4, G=3, xd=1, op=0, ldx=8, ldw=8, ldy=5, x=ok: L.face_grouped_linear(
        x, ldx, xd, op, ok, ldw, 40, None, 0, ok, ok, slots, G, n, k, dt, ok, ldy, None)
    assert lin(n=0) == lin(k=0) == lin(dt=3) == lin(slots=-1) == lin(G=0) == lin(xd=0) == lin(op=2) == lin(ldx=7) == -1
    assert lin(ldw=7) == lin(ldy=4) == lin(x=None) == -1 and lin(slots=0) == 0
    assert lin(slots=1 << 31) == lin(G=65536) == -2
    bwd = lambda slots=4, work=None, n=0, xd=1, dx=None, dw=None, db=None, w=ok, x=ok, ldy=5, op=0: L.face_grouped_linear_bwd(
        x, 8, xd, op, ok, ldy, w, 8, 40, ok, ok, slots, 3, 5, 8, 0, dx, dw, db, work, n, None)
    need = L.face_grouped_linear_bwd_work(5000, 5, 8, 0, 1, 1, 1, 0)
    assert need > 0 and bwd(5000, None, need, dw=ok) == -1 and bwd(5000, ok, need - 1, dw=ok) == -1
    assert L.face_grouped_linear_bwd_work(512, 5, 8, 0, 1, 1, 1, 1) == 0
    assert L.face_grouped_linear_bwd_work(512, 5, 8, 0, 2, 1, 0, 0) == 512 * 8 * 4
    assert bwd(dx=ok, xd=2) == bwd(dx=ok, xd=3) == bwd(db=ok) == bwd(dx=ok, w=None) == bwd(dw=ok, x=None) == -1
    assert bwd(dx=ok, x=None, op=1) == bwd(dx=ok, ldy=4) == bwd(dx=ok, op=2) == -1 and bwd() == 0
    cmb = lambda N=1, k=2, F=8, dt=0, ld=8, y=ok: L.face_expert_combine_fwd(y, ld, ok, None, 0, N, k, F, dt, ok, None)
    assert cmb(N=-1) == cmb(k=0) == cmb(F=0) == cmb(dt=3) == cmb(ld=7) == cmb(y=None) == -1 and cmb(N=0) == 0
