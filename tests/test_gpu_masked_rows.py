"""Masked classes and large factors: what a mask of -inf, of -1e9 or of the type's lowest value leaves of a row, of its gradients and
of a distillation loss, with tolerances that the masked numbers have no part in."""
import numpy as np
import pytest

from arraydiff_cuda_b200 import abi
from tests import helpers as H
from tests import rows_ref as R
from tests.test_gpu_logprob import bwd

pytestmark = pytest.mark.gpu
NHWC, NCHW = abi.AD_NHWC, abi.AD_NCHW
EPS = R.EPS


def masked(seed, rows, Cc, dtype, scale):
    """Logits and which of them stay: two classes at least; one row is nearly certain of a class, one has a single class"""
    g = H.rng(seed)
    x = (H.normal(seed, (rows, Cc), 3.0) / scale).astype(np.float32)
    keep = g.random((rows, Cc)) < 0.6
    for r in range(rows):
        keep[r, g.choice(Cc, 2, replace=False)] = True
    some = g.integers(0, Cc, rows)
    x[1, some[1]] = 20 / scale
    keep[1, some[1]] = True
    keep[2] = False
    keep[2, some[2]] = True
    return R.rounded(x, dtype), keep


def chain(Cc, layout):
    """Additions one behind the other in a row's sums.  A thread adds a batch of at most 64 elements in four sums, and batches of
    512 elements a warp at least one behind the other, then 5 + 4 + 3 joins; a position's threads batches of eight."""
    return 16 + Cc / 8 if layout == NCHW or Cc <= 64 else 40 + Cc / 512


def bounds(x, keep, scale, n):
    """Per row and class, in units of p: how far log p may be off.  Sums (n additions, half a step each), exponentials (2^-22, and
    half a step of an argument whose weighted mean is below 32, twice: 100 with the last steps), and the steps of (x - max)
    scale, which is rounded three times."""
    y = np.where(keep, x.astype(np.float64), np.nan)
    far = np.nan_to_num((np.nanmax(y, 1, keepdims=True) - y) * scale)
    return EPS * (n + 100) + 3 * EPS * far


def entropy_bound(n, Hs):
    """log S and the weighted mean of u by the sums' error; the additions of E, whose terms stand against a reference that may
    be 16 (in units of log 2) behind the maximum"""
    return EPS * ((n + 100) * (2 + Hs) + (n + 4) * 16)


FORMS = [(7, 19, NHWC), (8, 19, NCHW), (9, 50, NHWC), (8, 150, NCHW), (9, 150, NHWC), (6, 1000, NHWC), (5, 5000, NHWC), (3, 50001, NHWC), (450, 33001, NHWC)]


@pytest.mark.parametrize("scale,factor", [(1e12, 1.0), (1.0, 1e11), (1.0, 1e33), (1e30, 1e3), (1.0, 1e37)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,Cc,layout", FORMS)
def test_gradient_of_the_entropy_with_large_factors(rows, Cc, layout, dtype, scale, factor):
    """Masked classes have a gradient of zero whatever the factor, as long as the others' are finite.  What underflows (p below
    2^-126) is lost: 2^-125 of the factor and a logarithm of at most 200."""
    x, keep = masked(Cc, rows, Cc, dtype, scale)
    lab = np.full(rows, R.NO_CLASS, np.uint32)
    de = (H.uniform(2, (rows,), 0.5, 1.0) * factor).astype(np.float32)
    N, HW = (1, rows) if layout == NCHW else (rows, 1)
    gone = np.where(keep, x, -np.inf)
    zero = np.zeros(rows)
    want, mag = R.logprob_grad(gone, scale, lab, zero, de, zero)
    n = chain(Cc, layout)
    _, _, p, _ = R.softmax_rows(gone.astype(np.float64) * scale)
    off = bounds(x, keep, scale, n)
    tol = mag * (2 * off + 16 * EPS) + scale * abs(de[:, None].astype(np.float64)) * (p * 32 * (n + 4) * EPS + 2.0 ** -125 * 200)
    first = None
    for mask in (-np.inf, R.LOWEST[dtype], -1e9):
        got, _ = bwd(R.rounded(np.where(keep, x, mask), dtype), lab, dtype, N, HW, layout, (None, de, None), scale, outs=False)
        assert (got[~keep] == 0).all()
        R.check_close(got, want, tol + R.half_step(dtype) * abs(want), "dlogits")
        if first is None:
            first = got
        np.testing.assert_array_equal(got, first)
