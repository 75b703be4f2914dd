"""What ad_logprob_* and ad_distill_* refuse, before anything is launched: needs no GPU (the pointers are never followed)."""
import ctypes as C

import pytest

from arraydiff_cuda_b200 import abi

X, G = 0x100000, 0x900000        # addresses that nothing reads


def logprob(**over):
    a = abi.LogprobArgs()
    a.dtype, a.layout, a.N, a.C, a.HW, a.scale = abi.AD_BF16, abi.AD_NHWC, 4, 100, 1, 1.0
    a.logits, a.label, a.lse, a.logp = X, 0x2000, 0x3000, 0x4000
    a.dlogp, a.dlogits = 0x5000, G
    for k, v in over.items():
        setattr(a, k, v)
    return a


def distill(**over):
    a = abi.DistillArgs()
    a.dtype, a.layout, a.N, a.C, a.HW, a.scale = abi.AD_BF16, abi.AD_NHWC, 4, 100, 1, 1.0
    a.logits, a.top, a.top_class, a.top_logit, a.top_scale = X, 5, 0x2000, 0x3000, 1.0
    a.loss, a.dloss, a.dlogits = 0x4000, 0x5000, G
    for k, v in over.items():
        setattr(a, k, v)
    return a


BOTH = [
    (dict(dtype=1), abi.AD_ERR_UNSUPPORTED), (dict(layout=2), abi.AD_ERR_UNSUPPORTED),
    (dict(C=0), abi.AD_ERR_BAD_ARG), (dict(C=(1 << 30) + 1), abi.AD_ERR_LIMIT),
    (dict(pitch=-1), abi.AD_ERR_BAD_ARG), (dict(pitch=99), abi.AD_ERR_BAD_ARG), (dict(layout=abi.AD_NCHW, HW=9, pitch=8), abi.AD_ERR_BAD_ARG),
    (dict(logits=None), abi.AD_ERR_BAD_ARG), (dict(logits=X + 1), abi.AD_ERR_ALIGN), (dict(dtype=abi.AD_F32, logits=X + 2), abi.AD_ERR_ALIGN),
    (dict(scale=0.0), abi.AD_ERR_BAD_ARG), (dict(scale=-1.0), abi.AD_ERR_BAD_ARG), (dict(scale=float("nan")), abi.AD_ERR_BAD_ARG), (dict(scale=float("inf")), abi.AD_ERR_BAD_ARG),
]
GRADIENT = [
    (dict(dlogits=None), abi.AD_ERR_BAD_ARG), (dict(dlogits=G + 1), abi.AD_ERR_ALIGN), (dict(dlogits_pitch=99), abi.AD_ERR_BAD_ARG), (dict(dlogits_pitch=-5), abi.AD_ERR_BAD_ARG),
    (dict(dlogits=X, accumulate=1), abi.AD_ERR_BAD_ARG), (dict(dlogits=X, dlogits_pitch=128), abi.AD_ERR_BAD_ARG), (dict(dlogits=X + 16), abi.AD_ERR_BAD_ARG),
    (dict(dlogits=X - 100, pitch=128), abi.AD_ERR_BAD_ARG), (dict(dlogits=X + 2 * 399), abi.AD_ERR_BAD_ARG),
]


def status(name, a):
    lib = abi.lib()
    before = lib.ad_launch_count()
    rc = getattr(lib, name)(C.byref(a) if a is not None else None, None)
    assert lib.ad_launch_count() == before
    return rc


@pytest.mark.parametrize("over,want", BOTH)
def test_both_ways(over, want):
    for name, make in (("ad_logprob_fwd", logprob), ("ad_logprob_bwd", logprob), ("ad_distill_fwd", distill), ("ad_distill_bwd", distill)):
        assert status(name, make(**over)) == want, name


@pytest.mark.parametrize("over,want", GRADIENT)
def test_gradients(over, want):
    assert status("ad_logprob_bwd", logprob(**over)) == want
    assert status("ad_distill_bwd", distill(**over)) == want


@pytest.mark.parametrize("over,want", [
    (dict(label=None), abi.AD_ERR_BAD_ARG), (dict(logp=None, label=None, rank=0x6000), abi.AD_ERR_BAD_ARG), (dict(top=129, top_class=0x6000), abi.AD_ERR_LIMIT),
    (dict(top=3), abi.AD_ERR_BAD_ARG), (dict(lse=None, logp=None), abi.AD_ERR_BAD_ARG)])
def test_logprob_forward(over, want):
    assert status("ad_logprob_fwd", logprob(**over)) == want


@pytest.mark.parametrize("over,want", [(dict(dlogp=None), abi.AD_ERR_BAD_ARG), (dict(label=None, logp=None), abi.AD_ERR_BAD_ARG)])
def test_logprob_gradient(over, want):
    assert status("ad_logprob_bwd", logprob(**over)) == want


@pytest.mark.parametrize("over,want", [
    (dict(top=0), abi.AD_ERR_BAD_ARG), (dict(top=129), abi.AD_ERR_LIMIT), (dict(top_class=None), abi.AD_ERR_BAD_ARG), (dict(top_logit=None), abi.AD_ERR_BAD_ARG),
    (dict(top_scale=0.0), abi.AD_ERR_BAD_ARG), (dict(top_scale=float("nan")), abi.AD_ERR_BAD_ARG)])
def test_distill(over, want):
    assert status("ad_distill_fwd", distill(**over)) == want
    assert status("ad_distill_bwd", distill(**over)) == want


@pytest.mark.parametrize("name", ["label", "lse", "entropy", "logp", "rank", "top_class", "top_logp"])
def test_logprob_words(name):
    assert status("ad_logprob_fwd", logprob(**{"top": 2, "top_class": 0x6000, name: 0x7002})) == abi.AD_ERR_ALIGN


@pytest.mark.parametrize("name", ["label", "lse", "entropy", "logp", "dlse", "dentropy", "dlogp"])
def test_logprob_gradient_words(name):
    assert status("ad_logprob_bwd", logprob(**{name: 0x7001})) == abi.AD_ERR_ALIGN


@pytest.mark.parametrize("name", ["top_class", "top_logit", "top_lse", "loss", "dloss"])
def test_distill_words(name):
    assert status("ad_distill_bwd", distill(**{name: 0x7003})) == abi.AD_ERR_ALIGN


def test_distill_pointers():
    assert status("ad_distill_fwd", distill(loss=None)) == abi.AD_ERR_BAD_ARG
    assert status("ad_distill_bwd", distill(dloss=None)) == abi.AD_ERR_BAD_ARG


def test_nothing_to_do():
    for over in (dict(N=0), dict(HW=0), dict(HW=0, layout=abi.AD_NCHW)):
        for name, make in (("ad_logprob_fwd", logprob), ("ad_logprob_bwd", logprob), ("ad_distill_fwd", distill), ("ad_distill_bwd", distill)):
            assert status(name, make(logits=None, **over)) == abi.AD_OK
    for name in ("ad_logprob_fwd", "ad_logprob_bwd", "ad_distill_fwd", "ad_distill_bwd"):
        assert status(name, None) == abi.AD_ERR_BAD_ARG
