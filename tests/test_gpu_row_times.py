"""Calls whose rows leave the common way stay within a few times the ordinary call: ratios that are far from what is measured."""
import ctypes as C

import numpy as np
import pytest

from arraydiff_cuda_b200 import abi
from tests import helpers as H
from tests import rows_ref as R

pytestmark = pytest.mark.gpu


def least(call):
    """The shortest of a few runs, in ms"""
    import torch
    times = []
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times[1:])


def test_distillation_whose_mask_no_block_holds():
    """Lists with the rest on rows of fp32 classes on either side of what one block's mask holds (491 504): forward and backward,
    and the numbers of a few rows"""
    import torch
    rows, k, last = 230, 5, 4
    times = {}
    for Cc in (480_001, 500_003):
        x = torch.randn((rows, Cc), device="cuda")
        at = torch.randint(0, Cc, (rows, 1), device="cuda")
        cls = ((at + torch.arange(k, device="cuda") * 99_991) % Cc).int()
        cls[0, 0], cls[1, 1] = Cc - 1, 0
        t = (torch.randn((rows, k), device="cuda") - 3).contiguous()
        loss, one, g = torch.empty(rows, device="cuda"), torch.ones(rows, device="cuda"), torch.empty_like(x)
        a = abi.DistillArgs(abi.AD_F32, abi.AD_NHWC, rows, Cc, 1, 1.0, x.data_ptr(), 0, k, 1, cls.data_ptr(), t.data_ptr(), None, 1.0)
        a.loss, a.dloss, a.dlogits = loss.data_ptr(), one.data_ptr(), g.data_ptr()
        times[Cc] = [least(lambda: abi.check(f(C.byref(a), H.stream()))) for f in (abi.lib().ad_distill_fwd, abi.lib().ad_distill_bwd)]
        xs, cs, ts = (v[:last].cpu().numpy() for v in (x, cls.view(torch.int32), t))
        want, lmag, grad, gmag = R.distill(xs, 1.0, cs.view(np.uint32), ts, 1.0, 1)
        tol = R.EPS * (Cc / 512 + 400)   # additions one behind the other, exponentials, the list's
        R.check_close(loss[:last].cpu().numpy(), want, (lmag + 2) * 3 * tol, "loss")
        R.check_close(g[:last].cpu().numpy(), grad, gmag * (3 * tol + 16 * R.EPS) + 1e-37, "dlogits")
        del x, g
        torch.cuda.empty_cache()
    for few, many in zip(*times.values()):
        assert many < 6 * few, times
