"""ad_distill_fwd / ad_distill_bwd against the formulas in 64 bits, and with the lists of ad_logprob_fwd."""
import ctypes as C

import numpy as np
import pytest

from arraydiff_cuda_b200 import abi
from tests import helpers as H
from tests import rows_ref as R

pytestmark = pytest.mark.gpu
NHWC, NCHW = abi.AD_NHWC, abi.AD_NCHW


def teacher(seed, x, k, rest, odd=True):
    """k classes and numbers per row: distinct classes where there are enough, then some that are no class or stand twice"""
    g = H.rng(seed)
    rows, Cc = x.shape
    cls = np.stack([g.choice(Cc, k, replace=k > Cc) for _ in range(rows)]).astype(np.uint32)
    t = g.normal(size=(rows, k)).astype(np.float32) * 2
    if odd and k > 2:
        cls[1::3, -1] = R.NO_CLASS
        cls[2::5, 1] = cls[2::5, 0]
        cls[3::7, 0] = Cc
        t[4::9, -2] = -np.inf
    if rest:   # numbers whose exponentials sum to less than 1
        share = g.uniform(0.3, 0.95, size=(rows, 1))
        t = (t - np.log(np.exp(t.astype(np.float64)).sum(1, keepdims=True)) + np.log(share)).astype(np.float32)
    return cls, t


def call(x, dtype, N, HW, layout, cls, t, way, scale=1.0, top_scale=1.0, rest=0, top_lse=None, pitch=0, gpitch=0, shift=0, gshift=0, dloss=None,
         accumulate=0, in_place=False, old=None, ask_loss=True):
    rows = N * HW
    d = R.Dev(x, N, HW, dtype, layout, pitch, shift, 1e4)
    dc, dt = R.dev_u32(cls), H.dev(t)
    dlse = H.dev(top_lse) if top_lse is not None else None
    a = R.distill_args(d, dtype, dc, dt, scale, top_scale, rest, dlse)
    loss = R.Out(rows, 1, "f")
    a.loss = loss.ptr() if ask_loss else None
    if way == "fwd":
        abi.check(abi.lib().ad_distill_fwd(C.byref(a), H.stream()))
        H.sync()
        assert d.guards_hold()
        return loss.get()
    g = d if in_place else R.Dev(old if old is not None else np.full(x.shape, 3.0, np.float32), N, HW, dtype, layout, gpitch, gshift, 5.0)
    dd = H.dev(dloss)
    a.dloss, a.dlogits, a.dlogits_pitch, a.accumulate = dd.data_ptr(), g.ptr(), g.pitch, accumulate
    abi.check(abi.lib().ad_distill_bwd(C.byref(a), H.stream()))
    H.sync()
    assert d.guards_hold() and g.guards_hold()
    return (loss.get() if ask_loss else None), g.rows()


def tolerances(x, t, scale, top_scale, planes):
    """Of log p (rows_ref.tol_log) and of log q: its sum of at most 128 exponentials and a few steps of its number"""
    big = np.where(np.isfinite(t), abs(t.astype(np.float64)), 0.0).max(1) * top_scale
    return R.tol_log(x, scale, planes) + R.EPS * 200 + 8 * R.EPS * big


def check_loss(got, loss, lmag, tol, k):
    # a term is q times a difference of logarithms: q is off by tol of itself, the difference by 2 tol; k terms are added
    weight = np.where(np.isfinite(lmag), lmag, 0.0)
    R.check_close(got, loss, (weight * (1 + R.EPS * (k + 8)) + 2) * 3 * tol + R.EPS * (k + 8) * weight, "loss")


def check_grad(got, grad, gmag, dloss, tol, dtype, old=None):
    d = dloss.astype(np.float64)[:, None]
    want, bound = grad * d, gmag * abs(d) * (3 * tol[:, None] + 16 * R.EPS)
    if old is not None:
        want = want + old
        bound = bound + R.EPS * abs(want)
    R.check_close(got, want, bound + R.half_step(dtype) * abs(np.nan_to_num(want)) + 1e-37, "dlogits")


SHAPES = [(1, 1, 1), (1, 2, 1), (300, 3, 2), (513, 19, 4), (40, 32, 7), (37, 33, 33), (65, 64, 9), (29, 65, 128), (33, 150, 5), (21, 256, 64), (18, 257, 3),
          (17, 1000, 10), (3, 2047, 20), (6, 4097, 100), (2, 8200, 128), (1, 32768, 16), (3, 50001, 20), (1, 131075, 64), (149, 10007, 8)]


@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,k", SHAPES)
def test_rows(rows, Cc, k, dtype, rest):
    x = R.logits(rows + Cc, rows, Cc, dtype)
    g = H.rng(Cc + k)
    dloss = g.uniform(-1, 2, size=rows).astype(np.float32)
    old = R.rounded(H.normal(6, x.shape), dtype)
    P = (Cc + 63) // 64 * 64
    for i, (scale, top_scale, with_lse, pitch, gpitch, shift, gshift, acc) in enumerate((
            (1.0, 1.0, False, 0, 0, 0, 0, 0), (0.5, 0.5, True, P, P, 0, 0, 1), (1.3, 1.0, False, Cc + 3, Cc + 9, 1, 2, 0), (1.0, 2.0, True, 0, P, 0, 1, 1))):
        cls, t = teacher(100 + i, x, k, rest)
        lse = None
        if rest and with_lse:
            lse = g.normal(size=rows).astype(np.float32)
            t = ((t + lse[:, None]) / top_scale).astype(np.float32)
        if rest and not with_lse:
            t = (t / top_scale).astype(np.float32)
        loss, lmag, grad, gmag = R.distill(x, scale, cls, t, top_scale, rest, lse)
        tol = tolerances(x, t, scale, top_scale, Cc <= 64)
        args = dict(scale=scale, top_scale=top_scale, rest=rest, top_lse=lse, pitch=pitch, shift=shift)
        check_loss(call(x, dtype, rows, 1, NHWC, cls, t, "fwd", **args), loss, lmag, tol, k)
        got_loss, got = call(x, dtype, rows, 1, NHWC, cls, t, "bwd", dloss=dloss, gpitch=gpitch, gshift=gshift, accumulate=acc, old=old, ask_loss=i != 1, **args)
        if got_loss is not None:
            check_loss(got_loss, loss, lmag, tol, k)
        check_grad(got, grad, gmag, dloss, tol, dtype, old if acc else None)


@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,HW,Cc,k,pitch,gpitch", [(1, 1, 19, 3, 4, 3), (3, 1, 40, 2, 1, 1), (2, 7, 5, 5, 0, 0), (2, 70, 19, 4, 75, 0), (1, 257, 33, 2, 0, 260),
                                                    (2, 64, 150, 8, 64, 64), (1, 33, 1100, 40, 40, 33)])
def test_planes(N, HW, Cc, k, pitch, gpitch, dtype, rest):
    x = R.logits(HW + Cc, N * HW, Cc, dtype)
    cls, t = teacher(3, x, k, rest)
    dloss = H.uniform(4, (N * HW,), 0.0, 1.0)
    old = R.rounded(H.normal(6, x.shape), dtype)
    loss, lmag, grad, gmag = R.distill(x, 0.8, cls, t, 1.0, rest)
    tol = tolerances(x, t, 0.8, 1.0, True)
    check_loss(call(x, dtype, N, HW, NCHW, cls, t, "fwd", scale=0.8, rest=rest, pitch=pitch), loss, lmag, tol, k)
    for acc in (0, 1):
        got_loss, got = call(x, dtype, N, HW, NCHW, cls, t, "bwd", scale=0.8, rest=rest, pitch=pitch, gpitch=gpitch, dloss=dloss, accumulate=acc, old=old)
        check_loss(got_loss, loss, lmag, tol, k)
        check_grad(got, grad, gmag, dloss, tol, dtype, old if acc else None)


@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Cc", [1, 2, 19, 64, 100, 257, 1000, 5000, 40001])
def test_special_rows(Cc, dtype, rest):
    x = R.special_rows(Cc, Cc, dtype)
    k = min(Cc, 9)
    cls, t = teacher(7, x, k, rest)
    dloss = H.uniform(8, (16,), 0.5, 1.0)
    loss, lmag, grad, gmag = R.distill(x, 1.0, cls, t, 1.0, rest)
    tol = tolerances(x, t, 1.0, 1.0, True)
    for layout, N, HW in ((NHWC, 16, 1), (NHWC, 4, 4), (NCHW, 2, 8)):
        check_loss(call(x, dtype, N, HW, layout, cls, t, "fwd", rest=rest), loss, lmag, tol, k)
        got_loss, got = call(x, dtype, N, HW, layout, cls, t, "bwd", rest=rest, dloss=dloss)
        check_loss(got_loss, loss, lmag, tol, k)
        check_grad(got, grad, gmag, dloss, tol, dtype)


@pytest.mark.parametrize("layout", [NHWC, NCHW])
@pytest.mark.parametrize("Cc", [6, 70, 3000])
def test_lists_at_their_ends(Cc, layout):
    """Empty lists, lists of every class, weights of nothing and of everything, classes that the student masks, and a student
    far surer than its teacher (the classes outside underflow against the row's maximum)"""
    k = min(Cc, 6)
    x = R.logits(9, 8, Cc, "f32", 1.0)
    cls = np.stack([H.rng(20 + r).permutation(Cc)[:k] for r in range(8)]).astype(np.uint32)
    t = np.log(np.full((8, k), 0.9 / k)).astype(np.float32)
    cls[0] = R.NO_CLASS                                     # no entry at all
    t[1] = -np.inf                                          # entries without weight
    t[2] = np.log(1.5 / k)                                  # more than everything: nothing is left for the others
    x[3, cls[3, 0]] = -np.inf                               # masked by the student alone
    x[4, cls[4, 1]] = -np.inf                               # masked by both
    t[4, 1] = -np.inf
    x[5, cls[5]] += 300                                     # the others are 2^-400 of the row
    x[6] = -np.inf
    x[6, cls[6]] = 1.0                                      # the student allows the list alone
    cls[7] = cls[7, 0]                                      # one class, k times
    dloss = H.uniform(8, (8,), 0.5, 1.0)
    N, HW = (8, 1) if layout == NHWC else (2, 4)
    for rest in (0, 1):
        loss, lmag, grad, gmag = R.distill(x, 1.0, cls, t, 1.0, rest)
        tol = tolerances(x, t, 1.0, 1.0, True)
        check_loss(call(x, "f32", N, HW, layout, cls, t, "fwd", rest=rest), loss, lmag, tol, k)
        got_loss, got = call(x, "f32", N, HW, layout, cls, t, "bwd", rest=rest, dloss=dloss)
        check_loss(got_loss, loss, lmag, tol, k)
        check_grad(got, grad, gmag, dloss, tol, "f32")


@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,layout", [(50, 19, NHWC), (50, 19, NCHW), (10, 150, NCHW), (9, 150, NHWC), (7, 1001, NHWC), (2, 40003, NHWC), (600, 9000, NHWC)])
def test_gradient_over_the_logits(rows, Cc, layout, dtype, rest):
    x = R.logits(11, rows, Cc, dtype)
    cls, t = teacher(12, x, 6, rest)
    dloss = H.uniform(13, (rows,), 0.0, 1.0)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    one = call(x, dtype, N, HW, layout, cls, t, "bwd", rest=rest, dloss=dloss)
    two = call(x, dtype, N, HW, layout, cls, t, "bwd", rest=rest, dloss=dloss, in_place=True)
    for a, b in zip(one, two):
        np.testing.assert_array_equal(a, b)
    loss, lmag, grad, gmag = R.distill(x, 1.0, cls, t, 1.0, rest)
    check_grad(two[1], grad, gmag, dloss, tolerances(x, t, 1.0, 1.0, True), dtype)


@pytest.mark.parametrize("rest", [0, 1])
def test_gradient_against_differences(rest):
    """Central differences of the loss in 64 bits, h = 1e-4"""
    Cc = 90
    x = R.logits(21, 3, Cc, "f32", 1.0)
    cls, t = teacher(22, x, 5, rest, odd=False)
    _, got = call(x, "f32", 3, 1, NHWC, cls, t, "bwd", scale=1.4, rest=rest, dloss=np.ones(3, np.float32))
    h = 1e-4
    for c in {0, 1, int(cls[0, 0]), int(cls[1, 1]), int(cls[2, 2]), Cc - 1}:
        up, down = x.astype(np.float64), x.astype(np.float64)
        up[:, c] += h
        down[:, c] -= h
        diff = (R.distill(up, 1.4, cls, t, 1.0, rest)[0] - R.distill(down, 1.4, cls, t, 1.0, rest)[0]) / (2 * h)
        assert (abs(got[:, c] - diff) <= 4 * 1.4 ** 3 * h * h + 1e-11 / h + 8 * R.tol_log(x, 1.4, False)).all()


@pytest.mark.parametrize("rows,Cc,layout", [(300, 19, NHWC), (300, 19, NCHW), (40, 1000, NHWC), (5, 40000, NHWC)])
def test_teacher_to_student(rows, Cc, layout):
    """The teacher's lists straight into the student's loss: a student that equals its teacher loses nothing and has no gradient,
    by log probabilities, by logits with their log-sum-exp, and under a temperature"""
    import torch
    L = abi.lib()
    k = min(8, Cc)
    N, HW = (2, rows // 2) if layout == NCHW else (rows, 1)
    x = R.logits(51, N * HW, Cc, "bf16", 2.0)
    d = R.Dev(x, N, HW, "bf16", layout, 0, 0, 0.0)
    n = N * HW
    lse, tl, tc = torch.empty(n, device="cuda"), torch.empty((n, k), device="cuda"), torch.empty((n, k), dtype=torch.int32, device="cuda")
    a = R.logprob_args(d, "bf16", 0.5)
    a.lse, a.top, a.top_class, a.top_logp = lse.data_ptr(), k, tc.data_ptr(), tl.data_ptr()
    abi.check(L.ad_logprob_fwd(C.byref(a), H.stream()))
    raw = ((tl + lse[:, None]) / 0.5).contiguous()
    one = torch.ones(n, device="cuda")
    for t, ts, rest, tlse in ((tl, 1.0, 1, None), (raw, 0.5, 1, lse), (tl, 1.0, 0, None), (raw, 0.5, 0, None)):
        loss, dx = torch.empty(n, device="cuda"), torch.full_like(d.flat, 9.0)
        b = R.distill_args(d, "bf16", tc, t, 0.5, ts, rest, tlse)
        b.loss, b.dloss, b.dlogits = loss.data_ptr(), one.data_ptr(), dx.data_ptr() + d.start * 2
        b.dlogits_pitch = d.pitch
        abi.check(L.ad_distill_bwd(C.byref(b), H.stream()))
        H.sync()
        g = dx[d.start:d.start + d.n].float()
        if rest:
            tol = float(tolerances(x, t.cpu().numpy(), 0.5, ts, True).max()) * 8
            assert float(loss.abs().max()) < 20 * tol and float(g.abs().max()) < tol
        else:   # the list renormalised: the student is told to leave the other classes
            p = torch.exp(tl).sum(1)
            assert float((loss + torch.log(p)).abs().max()) < 1e-4
            assert float(g.sum().abs()) < 1e-2 * n


def test_training_step():
    """A student's layer trained on a teacher's lists through the C ABI: linear, loss and gradient, linear's gradients; against
    the same step in 64 bits"""
    import torch
    L = abi.lib()
    B, F, Cc, k = 24, 40, 130, 6
    x, w, bias = H.normal(61, (B, F)), H.normal(62, (Cc, F), 0.2), H.normal(63, (Cc,), 0.1)
    wt = H.normal(64, (Cc, F), 0.3)
    dx_, dw_, db_, dwt = (H.dev(v) for v in (x, w, bias, wt))
    st = H.stream()
    zt, zs = torch.empty((B, Cc), device="cuda"), torch.empty((B, Cc), device="cuda")
    abi.check(L.ad_linear_fwd(abi.AD_F32, B, F, Cc, H.ptr(dx_), H.ptr(dwt), H.ptr(db_), H.ptr(zt), st))
    tl, tc = torch.empty((B, k), device="cuda"), torch.empty((B, k), dtype=torch.int32, device="cuda")
    a = abi.LogprobArgs(abi.AD_F32, NHWC, B, Cc, 1, 1.0, zt.data_ptr())
    a.top, a.top_class, a.top_logp = k, tc.data_ptr(), tl.data_ptr()
    abi.check(L.ad_logprob_fwd(C.byref(a), st))
    abi.check(L.ad_linear_fwd(abi.AD_F32, B, F, Cc, H.ptr(dx_), H.ptr(dw_), H.ptr(db_), H.ptr(zs), st))
    loss, dloss, dz = torch.empty(B, device="cuda"), torch.full((B,), 1.0 / B, device="cuda"), torch.empty((B, Cc), device="cuda")
    b = abi.DistillArgs(abi.AD_F32, NHWC, B, Cc, 1, 1.0, zs.data_ptr(), 0, k, 1, tc.data_ptr(), tl.data_ptr(), None, 1.0)
    b.loss, b.dloss, b.dlogits = loss.data_ptr(), dloss.data_ptr(), dz.data_ptr()
    abi.check(L.ad_distill_bwd(C.byref(b), st))
    gw, gb, gx = torch.empty((Cc, F), device="cuda"), torch.empty(Cc, device="cuda"), torch.empty((B, F), device="cuda")
    abi.check(L.ad_linear_bwd(abi.AD_F32, B, F, Cc, H.ptr(dx_), H.ptr(dw_), H.ptr(dz), H.ptr(gx), H.ptr(gw), H.ptr(gb), 0, 0, st))
    H.sync()
    X, W, Bv, WT = (torch.from_numpy(v).double() for v in (x, w, bias, wt))
    W.requires_grad_(), Bv.requires_grad_()
    with torch.no_grad():
        lt, idx = torch.log_softmax(X @ WT.T + Bv, 1).topk(k, 1)
    assert (idx.numpy() == tc.cpu().numpy()).all()
    ls = torch.log_softmax(X @ W.T + Bv, 1)
    rest = 1 - lt.exp().sum(1)
    keep = torch.ones(B, Cc, dtype=torch.bool).scatter(1, idx, False)
    ref = (lt.exp() * (lt - ls.gather(1, idx))).sum(1) + rest * (rest.log() - ls.masked_fill(~keep, -np.inf).logsumexp(1))
    (ref.sum() / B).backward()
    # 40-term products of unit numbers in fp32 (40 half steps of about 3), carried into weights of at most 1
    np.testing.assert_allclose(H.host(loss), ref.detach().numpy(), atol=2e-5)
    np.testing.assert_allclose(H.host(gw), W.grad.numpy(), atol=2e-5)
    np.testing.assert_allclose(H.host(gb), Bv.grad.numpy(), atol=2e-5)


@pytest.mark.parametrize("rows,Cc,layout", [(2000, 19, NHWC), (2000, 19, NCHW), (600, 300, NHWC), (5, 60000, NHWC)])
def test_same_bits_captured_and_on_two_streams(rows, Cc, layout):
    import torch
    k = 5
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    xs = [R.Dev(R.logits(s, rows, Cc, "bf16"), N, HW, "bf16", layout, 0, 0, 0.0) for s in (41, 42)]
    cls, t = teacher(43, np.zeros((rows, Cc), np.float32), k, 1)
    dc, dt, one = R.dev_u32(cls), H.dev(t), torch.ones(rows, device="cuda")

    def make(x):
        loss, g = torch.empty(rows, device="cuda"), torch.zeros_like(x.flat)
        a = R.distill_args(x, "bf16", dc, dt, 1.0, 1.0, 1)
        a.loss, a.dloss, a.dlogits, a.dlogits_pitch = loss.data_ptr(), one.data_ptr(), g.data_ptr() + x.start * 2, x.pitch
        return a, loss, g

    want = []
    for x in xs:
        a, loss, g = make(x)
        abi.check(abi.lib().ad_distill_bwd(C.byref(a), H.stream()))
        H.sync()
        want.append((loss, g))
    jobs, streams = [make(x) for x in xs], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, job in zip(streams, jobs):
            abi.check(abi.lib().ad_distill_bwd(C.byref(job[0]), C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    for job, w in zip(jobs, want):
        assert torch.equal(job[1], w[0]) and torch.equal(job[2], w[1])
    buf = R.Dev(xs[0].rows(), N, HW, "bf16", layout, 0, 0, 0.0)
    a, loss, g = make(buf)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        abi.check(abi.lib().ad_distill_bwd(C.byref(a), H.stream()))
    for x, w in ((xs[1], want[1]), (xs[0], want[0])):
        buf.flat.copy_(x.flat)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, w[0]) and torch.equal(g, w[1])


# Forms that only many rows reach, as for the log probabilities, and lists of masks that no shared memory holds
MANY = [(1200, 4100, "bf16"), (1200, 4099, "f32"), (470, 5003, "f32"), (460, 16391, "bf16"), (450, 33001, "bf16"), (230, 40003, "f32"), (112, 70001, "f32"),
        (56, 140005, "f32"), (57, 300007, "bf16")]


@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("rows,Cc,dtype", MANY)
def test_special_rows_among_many(rows, Cc, dtype, rest):
    x = R.logits(77, rows, Cc, "bf16")
    at = np.linspace(0, rows - 1, 16).astype(int)
    x[at] = R.special_rows(Cc, Cc, dtype)
    some = np.unique(np.concatenate([at, H.rng(3).integers(0, rows, 30)]))
    old = R.rounded(H.normal(6, x.shape), dtype)
    dloss = H.uniform(8, (rows,), 0.5, 1.0)
    for k, kw in ((9, dict()), (128, dict(in_place=True)), (40, dict(accumulate=1, old=old, gpitch=Cc + 7, gshift=1)),
                  (3, dict(accumulate=1, old=old, pitch=(Cc + 63) // 64 * 64, gpitch=(Cc + 63) // 64 * 64))):
        g = H.rng(k)
        cls = (g.integers(0, Cc, (rows, 1)) + np.arange(k) * (Cc // (k + 1))).astype(np.int64) % Cc
        cls[5::7, 0] = cls[5::7, -1]
        cls[:, 1] = np.where(g.random(rows) < 0.3, Cc - 1, cls[:, 1])   # among the last elements
        cls[3::5, 2] = 0
        cls = cls.astype(np.uint32)
        cls[2::9, 0] = R.NO_CLASS
        t = g.normal(size=(rows, k)).astype(np.float32)
        if rest:
            t = (t - np.log(np.exp(t.astype(np.float64)).sum(1, keepdims=True)) + np.log(0.7)).astype(np.float32)
        loss, lmag, grad, gmag = R.distill(x[some], 1.0, cls[some], t[some], 1.0, rest)
        tol = tolerances(x[some], t[some], 1.0, 1.0, False)
        check_loss(call(x, dtype, rows, 1, NHWC, cls, t, "fwd", rest=rest)[some], loss, lmag, tol, k)
        got_loss, got = call(x, dtype, rows, 1, NHWC, cls, t, "bwd", rest=rest, dloss=dloss, **kw)
        check_loss(got_loss[some], loss, lmag, tol, k)
        check_grad(got[some], grad, gmag, dloss[some], tol, dtype, old[some] if "old" in kw else None)


@pytest.mark.parametrize("rows,Cc,dtype", [(2, 300001, "f32"), (2, 1_000_003, "bf16"), (3, 4_100_003, "f32"), (450, 600_001, "bf16")])
def test_very_many_classes(rows, Cc, dtype):
    k = 12
    x = R.logits(5, rows, Cc, dtype)
    cls, t = teacher(6, x, k, 1)
    cls[0, 1] = Cc - 1
    dloss = H.uniform(8, (rows,), 0.5, 1.0)
    some = np.arange(min(rows, 4))
    loss, lmag, grad, gmag = R.distill(x[some], 1.0, cls[some], t[some], 1.0, 1)
    tol = tolerances(x[some], t[some], 1.0, 1.0, False)
    check_loss(call(x, dtype, rows, 1, NHWC, cls, t, "fwd", rest=1)[some], loss, lmag, tol, k)
    got_loss, got = call(x, dtype, rows, 1, NHWC, cls, t, "bwd", rest=1, dloss=dloss)
    check_loss(got_loss[some], loss, lmag, tol, k)
    check_grad(got[some], grad, gmag, dloss[some], tol, dtype)


@pytest.mark.parametrize("Cc,pitch,gpitch", [(3, 2 ** 30 - 1, 0), (2, 2 ** 30 + 3, 0), (2, 0, 2 ** 30 + 3)])
def test_planes_four_gigabytes_apart(Cc, pitch, gpitch):
    """Class strides in bytes on either side of 2^32, of the logits and of the gradient"""
    import torch
    x = R.logits(61, 5, Cc, "f32")
    cls, t = teacher(62, x, 2, 0, odd=False)
    loss, lmag, grad, gmag = R.distill(x, 0.8, cls, t, 1.0, 0)
    tol = tolerances(x, t, 0.8, 1.0, True)
    dloss = np.linspace(0.5, 2, 5).astype(np.float32)
    try:
        got_loss, got = call(x, "f32", 1, 5, NCHW, cls, t, "bwd", scale=0.8, pitch=pitch, gpitch=gpitch, dloss=dloss)
        check_loss(got_loss, loss, lmag, tol, 2)
        check_grad(got, grad, gmag, dloss, tol, "f32")
    finally:
        torch.cuda.empty_cache()
