"""Log probabilities and distillation of rows with masks and special values against 64 bits, with tolerances made from what a
result is put together from: a masked number widens none of them.  Masks that leave nothing of a class give the same bits."""
import numpy as np
import pytest

from arraydiff_cuda_b200 import abi
from tests import helpers as H
from tests import rows_ref as R
from tests import test_gpu_distill as D
from tests.test_gpu_logprob import bwd, fwd
from tests.test_gpu_masked_rows import FORMS, NCHW, NHWC, bounds, chain, entropy_bound, masked

pytestmark = pytest.mark.gpu
EPS = R.EPS
LOST = 2.0 ** -125             # exponentials below 2^-126 are 0


def gradient_bound(want, mag, p, off, n, scale, d3, Hs, dtype):
    """mag: p's and the terms' magnitudes (rows_ref.logprob_grad).  p is off by `off` of itself, the entropy by entropy_bound"""
    dz, de, dl = (abs(v.astype(np.float64))[:, None] for v in d3)
    tol = mag * (2 * off + 16 * EPS) + scale * (de * p * 32 * (n + 4) * EPS + LOST * (dz + dl + de * (200 + Hs[:, None])))
    return tol + R.half_step(dtype) * abs(np.nan_to_num(want))


def listed(seed, x, keep, rest):
    """Lists of up to three of the classes that stay, not all of them, and one masked class without weight; row 2: no entry"""
    g = H.rng(seed)
    rows, Cc = x.shape
    cls = np.full((rows, 4), R.NO_CLASS, np.uint32)
    t = (g.normal(size=(rows, 4)) - 2.5).astype(np.float32)
    for r in range(rows):
        c = np.flatnonzero(keep[r])
        c = g.permutation(c)[:min(3, len(c) - 1)]
        cls[r, :len(c)] = c
        gone = np.flatnonzero(~keep[r])
        if len(gone):
            cls[r, 3], t[r, 3] = gone[0], -np.inf
    if rest:
        with np.errstate(divide="ignore"):
            t = (t - np.log(np.exp(t.astype(np.float64)).sum(1, keepdims=True)) + np.log(0.8)).astype(np.float32)
    return cls, t


def list_bound(n, t):
    big = np.where(np.isfinite(t), abs(t.astype(np.float64)), 0.0).max(1)
    return EPS * (n + 300) + 8 * EPS * big


def distill_check(got_loss, got, loss, lmag, grad, gmag, dloss, tol, k, dtype):
    """A probability is off by three steps of an argument of at most 104 (what is beyond is lost) and by the sums"""
    D.check_loss(got_loss, loss, lmag, tol, k)
    d = abs(dloss.astype(np.float64))[:, None]
    want = grad * dloss.astype(np.float64)[:, None]
    bound = gmag * d * (3 * tol[:, None] + 6 * 104 * EPS + 16 * EPS) + 4 * LOST * d
    R.check_close(got, want, bound + R.half_step(dtype) * abs(np.nan_to_num(want)), "dlogits")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,layout", FORMS)
def test_log_probabilities_of_masked_rows(rows, Cc, layout, dtype):
    scale, k = 1.3, 2
    x, keep = masked(Cc + 1, rows, Cc, dtype, 1.0)
    g = H.rng(4)
    lab = np.array([g.choice(np.flatnonzero(keep[r])) for r in range(rows)], np.uint32)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    gone = np.where(keep, x, -np.inf)
    n = chain(Cc, layout)
    off = bounds(x, keep, scale, n)
    want = R.logprob(gone, scale, lab, k)
    m = abs(gone.max(1).astype(np.float64)) * scale
    d3 = [g.normal(size=rows).astype(np.float32) for _ in range(3)]
    dwant, mag = R.logprob_grad(gone, scale, lab, *d3)
    _, _, p, _ = R.softmax_rows(gone.astype(np.float64) * scale)
    first = None
    for mask in (-np.inf, R.LOWEST[dtype], -1e30, -1e9):
        y = R.rounded(np.where(keep, x, mask), dtype)
        got = fwd(y, lab, dtype, N, HW, layout, k, scale)
        at = np.arange(rows)
        np.testing.assert_array_equal(got["rank"], want["rank"])
        np.testing.assert_array_equal(got["top_class"][at != 2], want["top_class"][at != 2])   # row 2 has one class
        R.check_close(got["lse"], want["lse"], EPS * (n + 100) + 3 * EPS * (m + abs(want["lse"])), "lse")
        R.check_close(got["logp"], want["logp"], off[at, lab] + 2 * EPS * abs(want["logp"]), "logp")
        R.check_close(got["top_logp"][:, 0], want["top_logp"][:, 0], off.min(1) + 2 * EPS * abs(want["top_logp"][:, 0]), "top_logp")
        R.check_close(got["entropy"], want["entropy"], entropy_bound(n, want["entropy"]), "entropy")
        grad, outs = bwd(y, lab, dtype, N, HW, layout, d3, scale)
        R.check_close(grad, dwant, gradient_bound(dwant, mag, p, off, n, scale, d3, want["entropy"], dtype), "dlogits")
        assert (grad[~keep] == 0).all()
        every = [got["lse"], got["entropy"], got["logp"], got["top_logp"][:, 0], grad, outs["lse"], outs["entropy"], outs["logp"]]
        first = first or every
        for a, b in zip(every, first):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,layout", FORMS)
def test_distillation_of_masked_rows(rows, Cc, layout, dtype, rest):
    x, keep = masked(Cc + 2, rows, Cc, dtype, 1.0)
    cls, t = listed(Cc, x, keep, rest)
    dloss = H.uniform(5, (rows,), 0.5, 1.5)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    loss, lmag, grad, gmag = R.distill(np.where(keep, x, -np.inf), 0.8, cls, t, 1.0, rest)
    tol = list_bound(chain(Cc, layout), t)
    first = None
    for mask in (-np.inf, R.LOWEST[dtype], -1e30, -1e9):
        y = R.rounded(np.where(keep, x, mask), dtype)
        alone = D.call(y, dtype, N, HW, layout, cls, t, "fwd", scale=0.8, rest=rest)
        got_loss, got = D.call(y, dtype, N, HW, layout, cls, t, "bwd", scale=0.8, rest=rest, dloss=dloss)
        D.check_loss(alone, loss, lmag, tol, 4)
        distill_check(got_loss, got, loss, lmag, grad, gmag, dloss, tol, 4, dtype)
        assert (got[~keep] == 0).all()
        first = first or [alone, got_loss, got]
        for a, b in zip([alone, got_loss, got], first):
            np.testing.assert_array_equal(a, b)


def from_maximum(x):
    """The same softmax from logits of at most 0: next to a log-sum-exp of -3e38 the logarithm of a share is lost in 64 bits, too"""
    with np.errstate(all="ignore"):
        y = x.astype(np.float64)
        m = np.where(np.isnan(y), -np.inf, y).max(1, keepdims=True)
        return y - np.where(np.isneginf(m), 0.0, m)


def special_bounds(x, n):
    """Of rows that may be done by plain loops, whose sums are longer: far as in `bounds`, for what has any probability"""
    with np.errstate(all="ignore"):
        y = x.astype(np.float64)
        m = np.where(np.isnan(y), -np.inf, y).max(1, keepdims=True)
        far = np.where(np.isfinite(y) & np.isfinite(m), m - y, 0.0)
    return EPS * (n + 100) + 3 * EPS * far


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Cc,layout", [(2, NHWC), (19, NHWC), (19, NCHW), (64, NHWC), (150, NCHW), (257, NHWC), (1000, NHWC), (40001, NHWC)])
def test_special_rows(Cc, layout, dtype):
    x = R.special_rows(Cc, Cc, dtype)
    g = H.rng(Cc)
    lab = g.integers(0, Cc, 16).astype(np.uint32)
    n = Cc + 16 if layout == NCHW or Cc <= 64 else 40 + Cc / 32
    off = special_bounds(x, n)
    d3 = [g.normal(size=16).astype(np.float32) for _ in range(3)]
    N, HW = (2, 8) if layout == NCHW else (16, 1)
    want = R.logprob(x, 1.0, lab, 1)
    got = fwd(x, lab, dtype, N, HW, layout, 1)
    with np.errstate(all="ignore"):
        m = np.nan_to_num(abs(np.where(np.isnan(x), -np.inf, x).max(1).astype(np.float64)), posinf=0.0)
    fin = {k: abs(np.nan_to_num(v, posinf=0.0, neginf=0.0)) for k, v in want.items()}
    R.check_close(got["lse"], want["lse"], EPS * (n + 100) + 3 * EPS * (m + fin["lse"]), "lse")
    R.check_close(got["logp"], want["logp"], off[np.arange(16), lab] + 2 * EPS * fin["logp"], "logp")
    R.check_close(got["entropy"], want["entropy"], entropy_bound(n, fin["entropy"]), "entropy")
    grad, outs = bwd(x, lab, dtype, N, HW, layout, d3)
    dwant, mag = R.logprob_grad(x, 1.0, lab, *d3)
    _, _, p, _ = R.softmax_rows(x)
    R.check_close(grad, dwant, gradient_bound(dwant, np.nan_to_num(mag), np.nan_to_num(p), off, n, 1.0, d3, fin["entropy"], dtype), "dlogits")
    for name in outs:
        np.testing.assert_array_equal(np.isnan(outs[name]), np.isnan(got[name]))
    R.check_close(outs["entropy"], want["entropy"], entropy_bound(n, fin["entropy"]), "entropy")
    for rest in (0, 1):
        k = min(Cc, 7)
        cls, t = D.teacher(7, x, k, rest)
        dloss = H.uniform(8, (16,), 0.5, 1.0)
        loss, lmag, dgrad, gmag = R.distill(from_maximum(x), 1.0, cls, t, 1.0, rest)
        got_loss, dgot = D.call(x, dtype, N, HW, layout, cls, t, "bwd", rest=rest, dloss=dloss)
        distill_check(got_loss, dgot, loss, lmag, dgrad, np.nan_to_num(gmag), dloss, list_bound(n, t), k, dtype)


@pytest.mark.parametrize("rows,Cc,layout", FORMS)
def test_entropy_of_nearly_certain_rows(rows, Cc, layout):
    """One class 2 to 30 above the others, at the row's start, in its middle or at its end: references that follow the maximum from
    behind, and entropies far smaller than the sums that they come from"""
    g = H.rng(Cc)
    x = H.normal(6, (rows, Cc), 1.0)
    ahead = np.linspace(2, 30, rows)
    at = np.array([(0, Cc // 2, Cc - 1)[r % 3] for r in range(rows)])
    x[np.arange(rows), at] = (x.max(1) + ahead).astype(np.float32)
    lab = np.full(rows, R.NO_CLASS, np.uint32)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    n = chain(Cc, layout)
    want = R.logprob(x, 1.0, lab, 0)
    got = fwd(x, lab, "f32", N, HW, layout, 0, want=("lse", "entropy"))
    R.check_close(got["entropy"], want["entropy"], entropy_bound(n, want["entropy"]), "entropy")
    R.check_close(got["lse"], want["lse"], EPS * (n + 100) + 3 * EPS * (abs(x.max(1)) + abs(want["lse"])), "lse")
    d3 = [g.normal(size=rows).astype(np.float32) for _ in range(3)]
    dwant, mag = R.logprob_grad(x, 1.0, lab, *d3)
    _, _, p, _ = R.softmax_rows(x)
    got, _ = bwd(x, lab, "f32", N, HW, layout, d3)
    R.check_close(got, dwant, gradient_bound(dwant, mag, p, bounds(x, np.ones(x.shape, bool), 1.0, n), n, 1.0, d3, want["entropy"], "f32"), "dlogits")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,layout", FORMS + [(300, 31, NHWC), (300, 32, NCHW), (1200, 5000, NHWC)])
def test_signs_of_nearly_certain_rows(rows, Cc, layout, dtype):
    """An entropy is not below 0 and a log probability not above it, whatever the rounding of the sums that they come from"""
    x = H.normal(7, (rows, Cc), 1.0)
    at = H.rng(Cc).integers(0, Cc, rows)
    x[np.arange(rows), at] = (x.max(1) + np.linspace(13, 40, rows)).astype(np.float32)
    one = np.arange(rows) % 4 == 3
    x[one] = np.where(np.arange(Cc) == at[one, None], x[one], -np.inf)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    for scale in (1.0, 0.83):
        got = fwd(R.rounded(x, dtype), at.astype(np.uint32), dtype, N, HW, layout, 2, scale)
        assert (got["entropy"] >= 0).all() and (got["logp"] <= 0).all() and (got["top_logp"] <= 0).all()
        _, outs = bwd(R.rounded(x, dtype), at.astype(np.uint32), dtype, N, HW, layout, (np.ones(rows), None, None), scale)
        assert (outs["entropy"] >= 0).all() and (outs["logp"] <= 0).all()
