"""ad_logprob_fwd / ad_logprob_bwd against the formulas in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from arraydiff_cuda_b200 import abi
from tests import helpers as H
from tests import rows_ref as R

pytestmark = pytest.mark.gpu
NHWC, NCHW = abi.AD_NHWC, abi.AD_NCHW


def labels(seed, x):
    """Random classes, the row's largest, and some that are no class"""
    g = H.rng(seed)
    rows, Cc = x.shape
    lab = g.integers(0, Cc, rows).astype(np.uint32)
    best = np.where(np.isnan(x), -np.inf, x).argmax(1).astype(np.uint32)
    lab = np.where(g.random(rows) < 0.4, best, lab)
    none = g.random(rows) < 0.15
    return np.where(none, g.choice(np.array([Cc, 255 if Cc <= 255 else Cc + 7, R.NO_CLASS], np.uint32), rows), lab).astype(np.uint32)


def fwd(x, lab, dtype, N, HW, layout, k, scale=1.0, pitch=0, shift=0, want=("lse", "entropy", "logp", "rank", "top")):
    rows = N * HW
    d = R.Dev(x, N, HW, dtype, layout, pitch, shift, 1e4)
    dl = R.dev_u32(lab)
    a = R.logprob_args(d, dtype, scale)
    a.label = dl.data_ptr()
    outs = {n: R.Out(rows, 1, "i" if n == "rank" else "f") for n in ("lse", "entropy", "logp", "rank")}
    for n, o in outs.items():
        if n in want:
            setattr(a, n, o.ptr())
    tc, tl = R.Out(rows, max(k, 1), "i"), R.Out(rows, max(k, 1), "f")
    if "top" in want:
        a.top, a.top_class, a.top_logp = k, tc.ptr(), tl.ptr()
    abi.check(abi.lib().ad_logprob_fwd(C.byref(a), H.stream()))
    H.sync()
    assert d.guards_hold()
    got = {n: outs[n].get() for n in outs if n in want}
    if "top" in want and k:
        got["top_class"], got["top_logp"] = tc.get().reshape(rows, k), tl.get().reshape(rows, k)
    return got


def check_fwd(x, lab, got, scale, k, planes):
    want = R.logprob(x, scale, lab, k)
    tol = R.tol_log(x, scale, planes)
    for n in ("rank", "top_class"):
        if n in got:
            np.testing.assert_array_equal(got[n], want[n], err_msg=n)
    for n in ("lse", "logp"):
        if n in got:
            R.check_close(got[n], want[n], tol + 2 * R.EPS * abs(np.nan_to_num(want[n], posinf=0, neginf=0)), n)
    if "entropy" in got:
        # log S and the weighted mean of u, which is off by the sums' error on top
        R.check_close(got["entropy"], want["entropy"], tol * (2 + abs(np.nan_to_num(want["entropy"]))), "entropy")
    if "top_logp" in got:
        w = want["top_logp"]
        R.check_close(got["top_logp"], w, tol[:, None] + 2 * R.EPS * abs(np.nan_to_num(w, posinf=0, neginf=0)), "top_logp")


def bwd(x, lab, dtype, N, HW, layout, d3, scale=1.0, pitch=0, gpitch=0, shift=0, gshift=0, accumulate=0, in_place=False, old=None, outs=True):
    rows = N * HW
    d = R.Dev(x, N, HW, dtype, layout, pitch, shift, 1e4)
    g = d if in_place else R.Dev(old if old is not None else np.full(x.shape, 3.0, np.float32), N, HW, dtype, layout, gpitch, gshift, 5.0)
    dl = R.dev_u32(lab)
    a = R.logprob_args(d, dtype, scale)
    a.label = dl.data_ptr()
    keep = [None if v is None else H.dev(v.astype(np.float32)) for v in d3]
    a.dlse, a.dentropy, a.dlogp = (v.data_ptr() if v is not None else None for v in keep)
    a.dlogits, a.dlogits_pitch, a.accumulate = g.ptr(), g.pitch, accumulate
    o = {n: R.Out(rows, 1, "f") for n in ("lse", "entropy", "logp")}
    if outs:
        for n, v in o.items():
            setattr(a, n, v.ptr())
    abi.check(abi.lib().ad_logprob_bwd(C.byref(a), H.stream()))
    H.sync()
    assert d.guards_hold() and g.guards_hold()
    return g.rows(), ({n: v.get() for n, v in o.items()} if outs else {})


def check_bwd(x, lab, got, d3, dtype, scale, planes, old=None):
    z = [np.zeros(len(x)) if v is None else v.astype(np.float32).astype(np.float64) for v in d3]
    want, mag = R.logprob_grad(x, scale, lab, *z)
    tol = mag * (2 * R.tol_log(x, scale, planes)[:, None] + 16 * R.EPS)
    if old is not None:
        want = want + old
        tol = tol + R.EPS * abs(want)
    R.check_close(got, want, tol + R.half_step(dtype) * abs(np.nan_to_num(want)) + 1e-37, "dlogits")


# few classes, a warp's, a block's; ragged; one and many rows
SHAPES = [(1, 1), (1, 2), (300, 3), (513, 19), (40, 32), (37, 33), (65, 64), (29, 65), (33, 150), (9, 255), (21, 256), (18, 257), (17, 1000), (5, 1024),
          (3, 2047), (6, 4097), (2, 8200), (1, 32768), (3, 50001), (1, 131075), (149, 10007)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc", SHAPES)
def test_forward_of_rows(rows, Cc, dtype):
    x = R.logits(rows + Cc, rows, Cc, dtype)
    lab = labels(Cc, x)
    for k, scale, pitch, shift in ((1, 1.0, 0, 0), (5, 0.5, Cc + 5, 3), (20, 1.7, (Cc + 63) // 64 * 64, 0), (128, 1.0, 0, 1)):
        got = fwd(x, lab, dtype, rows, 1, NHWC, k, scale, pitch, shift)
        check_fwd(x, lab, got, scale, k, Cc <= 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Cc", [1, 2, 19, 31, 64, 100, 257, 1000, 5000, 40001])
def test_forward_of_special_rows(Cc, dtype):
    x = R.special_rows(Cc, Cc, dtype)
    lab = labels(Cc + 1, x)
    for k in (3, 40):
        for N, HW in ((16, 1), (2, 8)):
            check_fwd(x, lab, fwd(x, lab, dtype, N, HW, NHWC, k), 1.0, k, Cc <= 64)
        check_fwd(x, lab, fwd(x, lab, dtype, 2, 8, NCHW, k), 1.0, k, True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,HW,Cc,pitch", [(1, 1, 19, 0), (1, 1, 19, 4), (3, 1, 40, 1), (2, 7, 5, 0), (2, 70, 19, 75), (1, 257, 33, 0), (2, 64, 150, 64), (1, 33, 1100, 40)])
def test_forward_of_planes(N, HW, Cc, pitch, dtype):
    x = R.logits(HW + Cc, N * HW, Cc, dtype)
    lab = labels(Cc, x)
    for k in (1, 4, 12):
        check_fwd(x, lab, fwd(x, lab, dtype, N, HW, NCHW, k, 1.3, pitch, 1), 1.3, k, True)


@pytest.mark.parametrize("Cc,layout", [(19, NHWC), (19, NCHW), (500, NHWC), (500, NCHW), (9000, NHWC)])
def test_results_one_at_a_time(Cc, layout):
    """What is not asked for is not written, and does not change the rest"""
    x = R.logits(7, 24, Cc, "bf16")
    lab = labels(8, x)
    full = fwd(x, lab, "bf16", 4, 6, layout, 6)
    check_fwd(x, lab, full, 1.0, 6, True)
    for n in ("lse", "entropy", "logp", "rank", "top"):
        got = fwd(x, lab, "bf16", 4, 6, layout, 6, want=(n,))
        for m in got:
            np.testing.assert_array_equal(got[m], full[m])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Cc", [700, 4096, 33000])
def test_top_where_the_large_classes_lie_together(Cc, dtype):
    """All of the largest in one stretch, every 8th, every 256th, every 2048th class: lists longer than a thread's share"""
    x = R.logits(3, 12, Cc, dtype, 0.5)
    for i, step in enumerate((1, 4, 8, 256, 1024, 2048)):
        at = np.arange(0, Cc, step)[:200]
        x[i, at] += 20
        x[i + 6, at] = 7.0
    x = R.rounded(x, dtype)
    lab = labels(4, x)
    for k in (7, 64, 128):
        check_fwd(x, lab, fwd(x, lab, dtype, 12, 1, NHWC, k), 1.0, k, False)


def factors(seed, rows):
    g = H.rng(seed)
    return [g.normal(size=rows).astype(np.float32) for _ in range(3)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc", SHAPES)
def test_gradient_of_rows(rows, Cc, dtype):
    x = R.logits(rows + Cc + 1, rows, Cc, dtype)
    lab = labels(Cc, x)
    dz, de, dl = factors(5, rows)
    old = R.rounded(H.normal(6, x.shape), dtype)
    P = (Cc + 63) // 64 * 64
    for d3, scale, pitch, gpitch, shift, gshift, acc in (((dz, de, dl), 1.0, 0, 0, 0, 0, 0), ((None, None, dl), 0.5, P, P, 0, 0, 1), ((None, de, None), 1.3, Cc + 3, Cc + 9, 1, 2, 0),
                                                         ((dz, None, dl), 1.0, 0, 0, 3, 3, 1), ((None, de, dl), 1.0, 0, P, 0, 1, 1)):
        got, outs = bwd(x, lab, dtype, rows, 1, NHWC, d3, scale, pitch, gpitch, shift, gshift, acc, old=old)
        check_bwd(x, lab, got, d3, dtype, scale, Cc <= 64, old if acc else None)
        check_fwd(x, lab, outs, scale, 0, Cc <= 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Cc", [1, 2, 19, 31, 64, 100, 257, 1000, 5000, 40001])
def test_gradient_of_special_rows(Cc, dtype):
    x = R.special_rows(Cc, Cc, dtype)
    lab = labels(Cc + 1, x)
    d3 = factors(9, 16)
    for layout, N, HW in ((NHWC, 16, 1), (NHWC, 4, 4), (NCHW, 2, 8)):
        got, _ = bwd(x, lab, dtype, N, HW, layout, d3)
        check_bwd(x, lab, got, d3, dtype, 1.0, True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,HW,Cc,pitch,gpitch", [(1, 1, 19, 4, 3), (3, 1, 40, 1, 1), (2, 7, 5, 0, 0), (2, 70, 19, 75, 0), (1, 257, 33, 0, 260), (2, 64, 150, 64, 64), (1, 33, 1100, 40, 33)])
def test_gradient_of_planes(N, HW, Cc, pitch, gpitch, dtype):
    x = R.logits(HW + Cc, N * HW, Cc, dtype)
    lab = labels(Cc, x)
    d3 = factors(10, N * HW)
    old = R.rounded(H.normal(6, x.shape), dtype)
    for acc in (0, 1):
        got, outs = bwd(x, lab, dtype, N, HW, NCHW, d3, 0.7, pitch, gpitch, 1, 0, acc, old=old)
        check_bwd(x, lab, got, d3, dtype, 0.7, True, old if acc else None)
        check_fwd(x, lab, outs, 0.7, 0, True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,layout", [(50, 19, NHWC), (50, 19, NCHW), (10, 150, NCHW), (9, 150, NHWC), (7, 1001, NHWC), (2, 40003, NHWC), (600, 9000, NHWC)])
def test_gradient_over_the_logits(rows, Cc, layout, dtype):
    x = R.logits(11, rows, Cc, dtype)
    lab = labels(12, x)
    d3 = factors(13, rows)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    got, outs = bwd(x, lab, dtype, N, HW, layout, d3, in_place=True)
    check_bwd(x, lab, got, d3, dtype, 1.0, True)
    check_fwd(x, lab, outs, 1.0, 0, True)
    apart, _ = bwd(x, lab, dtype, N, HW, layout, d3)
    np.testing.assert_array_equal(apart, got)


@pytest.mark.parametrize("Cc", [7, 90, 2100])
def test_gradient_against_differences(Cc):
    """Central differences of the forward results in 64 bits, h = 1e-4: off by h^2 times the third derivative (< 4) and by the
    64-bit rounding over h"""
    x = R.logits(21, 3, Cc, "f32", 1.0).astype(np.float64)
    lab = np.array([0, Cc // 2, Cc - 1], np.uint32)
    dz, de, dl = factors(22, 3)
    got, _ = bwd(x.astype(np.float32), lab, "f32", 3, 1, NHWC, (dz, de, dl), 1.4)

    def value(y):
        w = R.logprob(y, 1.4, lab, 0)
        return dz * w["lse"] + de * w["entropy"] + dl * w["logp"]

    h = 1e-4
    for c in {0, 1, Cc // 2, Cc - 1}:
        up, down = x.copy(), x.copy()
        up[:, c] += h
        down[:, c] -= h
        diff = (value(up) - value(down)) / (2 * h)
        weight = 1 + abs(dz) + abs(de) * (1 + np.log(Cc)) + abs(dl)
        assert (abs(got[:, c] - diff) <= weight * (4 * 1.4 ** 3 * h * h + 1e-11 / h + R.tol_log(x, 1.4, False) * 4)).all()


def test_far_offsets():
    """Rows behind 2^31 elements, of few classes and of many"""
    import torch
    for Cc, rows in ((131072, 16500), (16, 140_000_000)):
        x = torch.zeros((rows, Cc), dtype=torch.bfloat16, device="cuda")
        last = R.logits(31, 4, Cc, "bf16")
        x[-4:] = torch.from_numpy(last).cuda()
        lab = torch.full((rows,), 3, dtype=torch.int32, device="cuda")
        lse = torch.empty(rows, device="cuda")
        top = torch.empty((rows, 2), dtype=torch.int32, device="cuda")
        a = abi.LogprobArgs(abi.AD_BF16, NHWC, rows, Cc, 1, 1.0, x.data_ptr(), 0, lab.data_ptr(), lse.data_ptr())
        a.top, a.top_class = 2, top.data_ptr()
        abi.check(abi.lib().ad_logprob_fwd(C.byref(a), H.stream()))
        d = torch.ones(rows, device="cuda")
        a.dlogp, a.dlogits = d.data_ptr(), x.data_ptr()
        want = R.logprob(last, 1.0, np.full(4, 3, np.uint32), 2)
        np.testing.assert_array_equal(top[-4:].cpu().numpy(), want["top_class"].view(np.int32))
        R.check_close(lse[-4:].cpu().numpy(), want["lse"], R.tol_log(last, 1.0, Cc <= 64), "lse")
        assert abs(float(lse[0]) - np.log(Cc)) < 1e-5 and top[0].tolist() == [0, 1]
        abi.check(abi.lib().ad_logprob_bwd(C.byref(a), H.stream()))
        H.sync()
        check_bwd(last, np.full(4, 3, np.uint32), x[-4:].float().cpu().numpy(), (None, None, np.ones(4)), "bf16", 1.0, Cc <= 64)
        del x, lab, lse, top, d
        torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,Cc", [(2000, 19), (600, 300), (5, 60000), (700, 20000)])
def test_same_bits_on_streams_and_in_graphs(rows, Cc):
    """Two streams at once, a captured call replayed on new inputs, and the same call again give the same bits"""
    import torch
    x1, x2 = R.logits(41, rows, Cc, "bf16"), R.logits(42, rows, Cc, "bf16")
    lab = labels(43, x1)
    one, two = fwd(x1, lab, "bf16", rows, 1, NHWC, 5), fwd(x2, lab, "bf16", rows, 1, NHWC, 5)
    xs = [torch.from_numpy(v).cuda().bfloat16() for v in (x1, x2)]
    dl = R.dev_u32(lab)

    def make(x):
        o = dict(lse=torch.empty(rows, device="cuda"), top_logp=torch.empty((rows, 5), device="cuda"), top_class=torch.empty((rows, 5), dtype=torch.int32, device="cuda"))
        a = abi.LogprobArgs(abi.AD_BF16, NHWC, rows, Cc, 1, 1.0, x.data_ptr(), 0, dl.data_ptr(), o["lse"].data_ptr())
        a.top, a.top_class, a.top_logp = 5, o["top_class"].data_ptr(), o["top_logp"].data_ptr()
        return a, o

    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs = [make(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (a, _o) in zip(streams, jobs):
            abi.check(abi.lib().ad_logprob_fwd(C.byref(a), C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    for (_, o), want in zip(jobs, (one, two)):
        for n in o:
            np.testing.assert_array_equal(o[n].cpu().numpy().view(np.uint32), want[n].view(np.uint32))
    buf = xs[0].clone()
    a, o = make(buf)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        abi.check(abi.lib().ad_logprob_fwd(C.byref(a), H.stream()))
    for x, want in ((xs[1], two), (xs[0], one)):
        buf.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        for n in o:
            np.testing.assert_array_equal(o[n].cpu().numpy().view(np.uint32), want[n].view(np.uint32))


# Forms that only many rows reach: a warp per row of up to tens of KB, blocks that stay (from 444 rows on) with rows that
# are kept or copied twice, and clusters that share a row (rows of more than 135, 270 and 540 KB)
MANY = [(1200, 4100, "bf16"), (1200, 4099, "f32"), (470, 5003, "f32"), (460, 16391, "bf16"), (450, 33001, "bf16"), (230, 40003, "f32"), (112, 70001, "f32"),
        (56, 140005, "f32"), (57, 300007, "bf16")]


def spread(x, rows):
    """Special rows among ordinary ones, at odd places"""
    out = R.logits(77, rows, x.shape[1], "bf16")
    at = np.linspace(0, rows - 1, len(x)).astype(int)
    out[at] = x
    return out, at


@pytest.mark.parametrize("rows,Cc,dtype", MANY)
def test_special_rows_among_many(rows, Cc, dtype):
    x, at = spread(R.special_rows(Cc, Cc, dtype), rows)
    lab = labels(Cc + 1, x)
    some = np.unique(np.concatenate([at, H.rng(3).integers(0, rows, 30)]))
    for k, shift in ((9, 3), (100, 0)):
        got = fwd(x, lab, dtype, rows, 1, NHWC, k, shift=shift)
        check_fwd(x[some], lab[some], {n: v[some] for n, v in got.items()}, 1.0, k, False)
    old = R.rounded(H.normal(6, x.shape), dtype)
    d3 = factors(9, rows)
    for kw in (dict(), dict(in_place=True), dict(accumulate=1, old=old, gpitch=Cc + 7, gshift=1), dict(accumulate=1, old=old, pitch=(Cc + 63) // 64 * 64, gpitch=(Cc + 63) // 64 * 64)):
        for f3 in (d3, (None, None, d3[2])):
            got, outs = bwd(x, lab, dtype, rows, 1, NHWC, f3, **kw)
            sub = [None if v is None else v[some] for v in f3]
            check_bwd(x[some], lab[some], got[some], sub, dtype, 1.0, False, old[some] if "old" in kw else None)
            check_fwd(x[some], lab[some], {n: v[some] for n, v in outs.items()}, 1.0, 0, False)


@pytest.mark.parametrize("rows,Cc,dtype", [(1200, 3500, "f32"), (480, 33000, "bf16"), (480, 9000, "f32"), (444, 140000, "bf16")])
def test_top_of_many_rows_where_the_large_classes_lie_together(rows, Cc, dtype):
    """As above, by the blocks that stay: stretches and combs of large and of equal classes, rows of one value"""
    x = R.logits(3, rows, Cc, dtype, 0.5)
    steps = (1, 4, 8, 256, 1024, 2048, 8192)
    for i, step in enumerate(steps):
        c = np.arange(i, Cc, step)[:300]
        x[i, c] += 20
        x[rows - 1 - i, c] = 7.0
    x[20] = 1.0
    x[21, : Cc // 2] = -np.inf
    x[22] = -np.inf
    x[22, Cc - 3:] = 0.0
    x = R.rounded(x, dtype)
    lab = labels(4, x)
    some = np.concatenate([np.arange(25), np.arange(rows - 8, rows)])
    for k in (1, 12, 128):
        got = fwd(x, lab, dtype, rows, 1, NHWC, k, shift=2)
        check_fwd(x[some], lab[some], {n: v[some] for n, v in got.items()}, 1.0, k, False)


def test_masked_rows_keep_their_exact_values():
    """What is masked by -1e9, by the type's lowest value or by -inf does not touch the rest of a row, and a row of the lowest
    value alone is uniform"""
    for dtype in ("f32", "bf16"):
        for rows, Cc in ((40, 19), (40, 50), (40, 300), (40, 5000), (480, 9000)):
            x = R.logits(5, rows, Cc, dtype)
            keep = np.zeros(Cc, bool)
            keep[H.rng(Cc).permutation(Cc)[:max(2, Cc // 3)]] = True
            want = R.logprob(np.where(keep, x, -np.inf), 1.0, np.zeros(rows, np.uint32), 0)
            for mask in (-np.inf, -1e9, -1e30, R.LOWEST[dtype]):
                y = R.rounded(np.where(keep, x, mask), dtype)
                got = fwd(y, np.zeros(rows, np.uint32), dtype, rows, 1, NHWC, 0, want=("lse", "entropy"))
                tol = R.tol_log(x, 1.0, Cc <= 64)
                R.check_close(got["lse"], want["lse"], tol + 2 * R.EPS * abs(want["lse"]), "lse")
                R.check_close(got["entropy"], want["entropy"], tol * (2 + abs(want["entropy"])), "entropy")
            low = np.full((rows, Cc), R.LOWEST[dtype], np.float32)
            got = fwd(low, np.zeros(rows, np.uint32), dtype, rows, 1, NHWC, 0, want=("entropy", "logp"))
            np.testing.assert_allclose(got["entropy"], np.log(Cc), rtol=1e-5)
            np.testing.assert_allclose(got["logp"], -np.log(Cc), rtol=1e-5)


def test_gradients_captured_with_clusters_and_on_two_streams():
    """Rows that clusters share, replayed from a graph and on two streams at once, give the bits of a call by itself"""
    import torch
    rows, Cc = 230, 40004
    xs = [torch.from_numpy(R.logits(s, rows, Cc, "f32")).cuda() for s in (1, 2)]
    lab = torch.randint(0, Cc, (rows,), device="cuda", dtype=torch.int32)
    one = torch.randn(rows, device="cuda")

    def make(x):
        g, lse = torch.empty_like(x), torch.empty(rows, device="cuda")
        a = abi.LogprobArgs(abi.AD_F32, NHWC, rows, Cc, 1, 1.0, x.data_ptr(), 0, lab.data_ptr(), lse.data_ptr())
        a.dlogp = a.dentropy = one.data_ptr()
        a.dlogits = g.data_ptr()
        return a, g, lse

    want = []
    for x in xs:
        a, g, lse = make(x)
        abi.check(abi.lib().ad_logprob_bwd(C.byref(a), H.stream()))
        H.sync()
        want.append((g, lse))
    jobs, streams = [make(x) for x in xs], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, j in zip(streams, jobs):
            abi.check(abi.lib().ad_logprob_bwd(C.byref(j[0]), C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    for j, w in zip(jobs, want):
        assert torch.equal(j[1], w[0]) and torch.equal(j[2], w[1])
    buf = xs[0].clone()
    a, g, lse = make(buf)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        abi.check(abi.lib().ad_logprob_bwd(C.byref(a), H.stream()))
    for x, w in ((xs[1], want[1]), (xs[0], want[0])):
        buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, w[0]) and torch.equal(lse, w[1])


@pytest.mark.parametrize("rows,Cc,dtype,V", [(448, 140000, "bf16", 8), (446, 140000, "f32", 4), (3, 140000, "bf16", 8), (1200, 16000, "bf16", 8)])
def test_top_of_rows_whose_large_classes_share_a_thread(rows, Cc, dtype, V):
    """Hundreds of large classes, different and equal, in the vectors that one thread or lane takes"""
    x = R.logits(3, rows, Cc, dtype, 0.5)
    mine = (np.arange(Cc) // V) % 256
    g = H.rng(9)
    for i in range(min(rows, 3)):
        at = np.flatnonzero((mine == 5) | (mine == 77 + i))
        x[i, at] = 30 + g.normal(size=len(at)) * (3.0 if i < 2 else 0.0)   # the third: all alike
    x = R.rounded(x, dtype)
    lab = labels(4, x)
    some = np.arange(min(rows, 6))
    for k in (1, 5, 12, 33):
        got = fwd(x, lab, dtype, rows, 1, NHWC, k)
        check_fwd(x[some], lab[some], {n: v[some] for n, v in got.items()}, 1.0, k, False)


@pytest.mark.parametrize("Cc,pitch,gpitch", [(3, 2 ** 30 - 1, 0), (2, 2 ** 30 + 3, 0), (2, 0, 2 ** 30 + 3)])
def test_planes_four_gigabytes_apart(Cc, pitch, gpitch):
    """Class strides in bytes on either side of 2^32, of the logits and of the gradient"""
    import torch
    x = R.logits(51, 5, Cc, "f32")
    lab = np.array([0, 1, Cc - 1, R.NO_CLASS, 1], np.uint32)
    d3 = factors(52, 5)
    try:
        if pitch:
            check_fwd(x, lab, fwd(x, lab, "f32", 1, 5, NCHW, 2, 0.9, pitch), 0.9, 2, True)
            torch.cuda.empty_cache()
        got, _ = bwd(x, lab, "f32", 1, 5, NCHW, d3, 0.9, pitch, gpitch)
        check_bwd(x, lab, got, d3, "f32", 0.9, True)
    finally:
        torch.cuda.empty_cache()
