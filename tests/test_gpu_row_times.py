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


@pytest.mark.parametrize("rows", [8, 2001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_padded_row_among_others(rows, dtype):
    """One row of the type's lowest value, of a batch with long lists: its sums are done again, its list and its rank are not"""
    import torch
    Cc, k, at = 50_001, 128, rows // 2
    T = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = torch.randn((rows, Cc), device="cuda").mul_(2.5).to(T)
    lab = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    lse, ent, logp = (torch.empty(rows, device="cuda") for _ in range(3))
    rank, cls = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty((rows, k), dtype=torch.int32, device="cuda")
    top = torch.empty((rows, k), device="cuda")
    a = abi.LogprobArgs(R.dtype_of(dtype), abi.AD_NHWC, rows, Cc, 1, 1.0, x.data_ptr(), 0, lab.data_ptr(), lse.data_ptr(), ent.data_ptr(), logp.data_ptr(), rank.data_ptr(), k)
    a.top_class, a.top_logp = cls.data_ptr(), top.data_ptr()
    call = lambda: abi.check(abi.lib().ad_logprob_fwd(C.byref(a), H.stream()))
    ordinary = least(call)
    x[at] = torch.finfo(T).min
    padded = least(call)
    assert rank[at].item() == 77 and (cls[at] == torch.arange(k, device="cuda")).all()
    np.testing.assert_allclose([ent[at].item(), -logp[at].item()] + (-top[at]).tolist(), np.log(Cc), rtol=1e-6)
    x[at, 40_000], x[at, 77] = -1e9, -1e30               # some above the others
    call()
    H.sync()
    assert rank[at].item() == 1 and cls[at, :3].tolist() == [40_000, 77, 0] and ent[at].item() == 0 and top[at, 0].item() == 0
    assert padded < 6 * ordinary, (ordinary, padded)
