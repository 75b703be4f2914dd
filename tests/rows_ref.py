"""Rows of logits for the tests of the log-probability and distillation operators: the formulas in 64 bits, rows with
special values, tolerances, and calls through the C ABI with guarded buffers."""
import ctypes as C

import numpy as np

from arraydiff_cuda_b200 import abi
from tests import helpers as H

NO_CLASS = 0xFFFFFFFF
EPS = 2.0 ** -24                                   # half a step of fp32, relative


# ---------------------------------------------------------------- formulas
def softmax_rows(z):
    """lse, log p, p and which rows have any weight, of z [rows][C] in float64; NaN rows stay NaN"""
    z = np.asarray(z, np.float64)
    with np.errstate(all="ignore"):
        m = np.where(np.isnan(z), -np.inf, z).max(1, keepdims=True)
        m = np.where(np.isneginf(m), 0.0, m)
        S = np.exp(z - m).sum(1, keepdims=True)
        some = ~(S == 0)
        logS = np.log(S)
        lse = (m + logS)[:, 0]
        logp = (z - m) - logS
        logp = np.where(some, logp, -np.inf)
        p = np.where(some, np.exp(logp), 0.0)
    return lse, logp, p, some[:, 0]


def order(x):
    """Classes of a row by (value descending, class ascending), NaN left out"""
    x = np.asarray(x, np.float64)
    c = np.flatnonzero(~np.isnan(x))
    return c[np.lexsort((c, -x[c]))]


def logprob(x, scale, label, k):
    x = np.asarray(x, np.float64)
    rows, Cc = x.shape
    lse, logs, p, some = softmax_rows(x * scale)
    with np.errstate(all="ignore"):
        H_ = -np.where(p > 0, p * logs, np.where(np.isnan(p), np.nan, 0.0)).sum(1)
    H_ = np.where(some, H_, 0.0)
    logp, rank = np.zeros(rows), np.full(rows, NO_CLASS, np.uint32)
    top_class, top_logp = np.full((rows, k), NO_CLASS, np.uint32), np.full((rows, k), -np.inf)
    cls = np.arange(Cc)
    for r in range(rows):
        l = int(label[r])
        if l < Cc:
            logp[r] = logs[r, l]
            rank[r] = int(((x[r] > x[r, l]) | ((x[r] == x[r, l]) & (cls < l))).sum())
        o = order(x[r])[:k]
        top_class[r, :len(o)] = o
        top_logp[r, :len(o)] = logs[r, o]
    return dict(lse=lse, entropy=H_, logp=logp, rank=rank, top_class=top_class, top_logp=top_logp)


def logprob_grad(x, scale, label, dlse, dent, dlogp):
    """The gradient and, for its tolerance, the sum of its terms' magnitudes"""
    x = np.asarray(x, np.float64)
    rows, Cc = x.shape
    _, logs, p, some = softmax_rows(x * scale)
    with np.errstate(all="ignore"):
        plog = np.where(p > 0, p * logs, np.where(np.isnan(p), np.nan, 0.0))
    H_ = np.where(some, -plog.sum(1), 0.0)[:, None]
    hot = np.zeros((rows, Cc))
    known = (label < Cc) & some
    hot[np.flatnonzero(known), label[known].astype(np.int64)] = 1.0
    dl = np.where(known, dlogp, 0.0)[:, None]
    dz, de = dlse[:, None], dent[:, None]
    d = scale * (p * (dz - dl) - de * (plog + p * H_) + dl * hot)
    # by tol, a row's error of log p: p is off by tol of itself, log p by tol, H by tol (2 + H) (its check): the entropy's term
    # p (log p + H) by tol (|p log p| + p H) + p (tol + tol (2 + H)), which is not 0 where log p + H is
    mag = scale * (p * (abs(dz) + abs(dl)) + abs(de) * (abs(plog) + p * (3 + 2 * H_)) + abs(dl) * hot)
    return d, mag


def distill(x, scale, cls, t, top_scale, rest, top_lse=None):
    """loss, the magnitude of its terms, d loss / d logits and the magnitude of its terms"""
    x = np.asarray(x, np.float64)
    rows, Cc = x.shape
    _, logs, p, some = softmax_rows(x * scale)
    loss, lmag, grad, gmag = np.zeros(rows), np.zeros(rows), np.zeros((rows, Cc)), np.zeros((rows, Cc))
    with np.errstate(all="ignore"):
        for r in range(rows):
            if not some[r]:
                continue
            ok = cls[r] < Cc
            c, a = cls[r][ok].astype(np.int64), t[r][ok].astype(np.float64) * top_scale
            if rest:
                a = a - (0.0 if top_lse is None else float(top_lse[r]))
            else:
                lse_t = softmax_rows(a[None])[0][0] if len(a) else 0.0
                a = a - (lse_t if np.isfinite(lse_t) else 0.0)
            q = np.exp(a)
            terms = np.where(q > 0, q * (a - logs[r, c]), 0.0)
            full = np.zeros(Cc)
            np.add.at(full, c, q)
            inside = np.zeros(Cc, bool)
            inside[c] = True
            Q, qr = q.sum(), 0.0
            lmag[r] = np.where(q > 0, q * (abs(a) + abs(logs[r, c])), 0.0).sum()
            L = terms.sum()
            away = np.zeros(Cc)
            if rest and (x[r][~inside] > -np.inf).any() and Q < 1:
                z = x[r] * scale
                zo = np.where(inside, -np.inf, z)
                lse_o = softmax_rows(zo[None])[0][0]
                lse = softmax_rows(z[None])[0][0]
                qr = 1.0 - Q
                L += qr * (np.log(qr) - (lse_o - lse))
                lmag[r] += qr * (abs(np.log(qr)) + abs(lse_o - lse)) + (abs(np.log(qr)) + abs(lse_o - lse) + 1)
                away = np.where(inside, 0.0, qr * np.exp(zo - lse_o))
            if np.isnan(p[r]).any():
                loss[r], grad[r] = np.nan, np.nan
                continue
            loss[r] = L
            grad[r] = scale * (p[r] * (Q + qr) - full - away)
            gmag[r] = scale * (p[r] * (Q + qr) + full + away) + (scale * np.where(inside, p[r], away / max(qr, 1e-300) + p[r]) if rest else 0.0)
    return loss, lmag, grad, gmag


# ---------------------------------------------------------------- tolerances
def tol_log(x, scale, planes):
    """How far log p, lse and an entropy may be off, per row.  A thread adds C / 32 + 32 terms in a row (a thread per position:
    C), each addition is off by half a step; an exponential by 2^-22 and by half a step of its argument, whose weighted mean
    is below 32, twice; then a few steps of the largest z that a result is put together from."""
    x = np.asarray(x, np.float64)
    chain = x.shape[1] if planes else x.shape[1] / 32 + 32
    big = np.where(np.isfinite(x), abs(x), 0.0).max(1) * scale
    return EPS * (chain + 4 + 64 + 32) + 4 * EPS * big


def half_step(dtype):
    return 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24


def check_close(got, want, tol, what):
    """Non-finite values alike, finite ones within tol"""
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(tol, np.shape(want))
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)], err_msg=what)
    off = abs(got[fine] - want[fine]) - tol[fine]
    assert not off.size or off.max() <= 0, (what, float(abs(got[fine] - want[fine]).max()), float(off.max()))


# ---------------------------------------------------------------- inputs
def rounded(x, dtype):
    """x as the type holds it, in float32"""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32))
    return (t.bfloat16().float() if dtype == "bf16" else t).numpy()


def logits(seed, rows, Cc, dtype, std=3.0):
    return rounded(H.normal(seed, (rows, Cc), std), dtype)


LOWEST = {"bf16": -3.3895313892515355e38, "f32": -3.4028234663852886e38}


def special_rows(seed, Cc, dtype):
    """One row of each kind where a softmax goes wrong"""
    g = H.rng(seed)
    base = logits(seed, 16, Cc, dtype)
    low = LOWEST[dtype]
    base[0] = -np.inf                                        # nothing
    base[1] = low                                            # all masked by the lowest value: uniform
    base[2, g.random(Cc) < 0.7] = low                        # some masked so
    base[3, g.random(Cc) < 0.9] = -np.inf
    base[4] = -np.inf
    base[4, Cc // 2] = 1.25                                  # one class
    base[5] = 0.5                                            # ties
    base[6] = np.where(g.random(Cc) < 0.5, 0.0, -0.0)
    base[7, Cc - 1] = np.nan
    base[8, Cc // 3] = np.inf
    base[9] = rounded(base[9] * 1e36, dtype)                 # far apart
    base[10] = low
    base[10, : Cc // 2 + 1] = -np.inf
    base[11] = rounded(base[11] + 2.0e4, dtype)              # large and alike
    base[12] = np.sort(base[12])
    base[13] = np.sort(base[13])[::-1]
    base[14] = (g.random(Cc) < 0.5).astype(np.float32)       # two values
    base[15] = np.nan
    return base


# ---------------------------------------------------------------- device buffers
class Dev:
    """[N][HW][C] or [N][C][HW] on the device with a pitch, `shift` elements behind a 256-byte boundary and guards of 64
    elements around; what does not belong to the rows holds `fill`"""

    def __init__(self, rows, N, HW, dtype, layout, pitch, shift, fill):
        import torch
        R, Cc = rows.shape
        assert R == N * HW
        T = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.N, self.HW, self.C, self.layout = N, HW, Cc, layout
        inner, outer = (Cc, R) if layout == abi.AD_NHWC else (HW, N * Cc)
        self.pitch, self.inner, self.outer = pitch or inner, inner, outer
        self.n = self.pitch * outer
        self.flat = torch.full((self.n + 128 + shift,), fill, dtype=T, device="cuda")
        self.start = 64 + shift
        self.put(rows)
        self.before = self.flat.clone()

    def body(self):
        return self.flat[self.start:self.start + self.n].view(self.outer, self.pitch)[:, :self.inner]

    def put(self, rows):
        import torch
        t = torch.from_numpy(np.ascontiguousarray(rows, np.float32)).cuda()
        if self.layout == abi.AD_NCHW:
            t = t.view(self.N, self.HW, self.C).transpose(1, 2).reshape(self.outer, self.inner)
        self.body().copy_(t)

    def rows(self):
        b = self.body().float()
        if self.layout == abi.AD_NCHW:
            b = b.reshape(self.N, self.C, self.HW).transpose(1, 2).reshape(self.N * self.HW, self.C)
        return b.cpu().numpy()

    def ptr(self):
        return self.flat.data_ptr() + self.start * self.flat.element_size()

    def guards_hold(self):
        import torch
        a, b = self.flat.clone(), self.before.clone()
        for t in (a, b):
            t[self.start:self.start + self.n].view(self.outer, self.pitch)[:, :self.inner] = 0
        it = torch.int16 if a.element_size() == 2 else torch.int32
        return bool((a.view(it) == b.view(it)).all())


class Out:
    """A result by rows, with two guarded rows behind it"""

    def __init__(self, rows, width, kind):
        import torch
        self.t = torch.full((rows + 2, width), 77, dtype=torch.int32 if kind == "i" else torch.float32, device="cuda")
        self.rows, self.kind = rows, kind

    def ptr(self):
        return self.t.data_ptr()

    def get(self):
        a = self.t.cpu().numpy()
        assert (a[self.rows:] == 77).all()
        a = a[:self.rows]
        a = a.view(np.uint32) if self.kind == "i" else a
        return a[:, 0] if a.shape[1] == 1 else a


def dtype_of(dtype):
    return abi.AD_BF16 if dtype == "bf16" else abi.AD_F32


def logprob_args(x, dtype, scale=1.0):
    a = abi.LogprobArgs()
    a.dtype, a.layout, a.N, a.C, a.HW, a.scale = dtype_of(dtype), x.layout, x.N, x.C, x.HW, scale
    a.logits, a.pitch = x.ptr(), x.pitch
    return a


def distill_args(x, dtype, cls, t, scale=1.0, top_scale=1.0, rest=0, top_lse=None):
    a = abi.DistillArgs()
    a.dtype, a.layout, a.N, a.C, a.HW, a.scale = dtype_of(dtype), x.layout, x.N, x.C, x.HW, scale
    a.logits, a.pitch = x.ptr(), x.pitch
    a.top, a.rest, a.top_class, a.top_logit, a.top_scale = cls.shape[1], rest, cls.data_ptr(), t.data_ptr(), top_scale
    a.top_lse = top_lse.data_ptr() if top_lse is not None else None
    return a


def dev_u32(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.uint32).view(np.int32)).cuda()
