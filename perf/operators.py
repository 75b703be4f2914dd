"""Timed calls of the row-wise classification operators: log probabilities of given classes with entropy, rank and top
alternatives (`logprob`), and distillation from a teacher's top classes (`distill`), each in both directions.

A row is one position of a classifier's output: logits [N][HW][C] (NHWC; HW = 1 for a plain [rows][classes] matrix, whose
rows may lie `pitch` elements apart) or [N][C][HW] (NCHW).

`own` false: the formulas in elementary torch operations and 32 bits; true: the C ABI, as a Python program calls it.
"""
import ctypes as C
import math

import torch

own = False


def listed():
    return [
        # One row of a large vocabulary: the call after each generated token, latency alone.
        dict(name="lp_fwd_1x32768_bf16_k5", op="logprob", way="fwd", dtype="bf16", layout="nhwc", N=1, C=32768, HW=1, pitch=0, k=5, rest=0, masked=False, scale=1.0),
        # A batch of rows with twenty alternatives each, under a temperature.
        dict(name="lp_fwd_64x131072_bf16_k20", op="logprob", way="fwd", dtype="bf16", layout="nhwc", N=64, C=131072, HW=1, pitch=0, k=20, rest=0, masked=False, scale=1.25),
        # Scoring whole texts: thousands of rows, an odd class count, so that every row starts at another alignment.
        dict(name="lp_fwd_4001x50001_bf16_k8", op="logprob", way="fwd", dtype="bf16", layout="nhwc", N=4001, C=50001, HW=1, pitch=0, k=8, rest=0, masked=True, scale=1.0),
        # Validation of a 1000-class classifier, 256 images: top-5 and the label's rank, in the default arithmetic of the tools.
        dict(name="lp_fwd_256x1000_f32_k5", op="logprob", way="fwd", dtype="f32", layout="nhwc", N=256, C=1000, HW=1, pitch=0, k=5, rest=0, masked=False, scale=1.0),
        # Confidence maps of the dense-prediction head: 19 classes at each pixel of two 1024 x 2048 images.
        dict(name="lp_fwd_2x19x1024x2048_bf16_k3", op="logprob", way="fwd", dtype="bf16", layout="nhwc", N=2, C=19, HW=2097152, pitch=0, k=3, rest=0, masked=False, scale=1.0),
        # A training step on log probabilities with an entropy bonus, rows of a padded vocabulary.
        dict(name="lp_bwd_4096x32000_bf16", op="logprob", way="bwd", dtype="bf16", layout="nhwc", N=4096, C=32000, HW=1, pitch=32064, k=0, rest=0, masked=False, scale=1.0),
        # The same on the planes of a fp32 map of 150 classes.
        dict(name="lp_bwd_2x150x256x255_f32_nchw", op="logprob", way="bwd", dtype="f32", layout="nchw", N=2, C=150, HW=65280, pitch=0, k=0, rest=0, masked=False, scale=1.0),
        # A student's training step on stored top classes with the remaining probability as one more class.
        dict(name="ds_bwd_4096x65536_bf16_k64", op="distill", way="bwd", dtype="bf16", layout="nhwc", N=4096, C=65536, HW=1, pitch=0, k=64, rest=1, masked=False, scale=1.0),
        # fp32 logits of an odd class count, the list renormalised, temperature 2.
        dict(name="ds_bwd_1001x50001_f32_k20", op="distill", way="bwd", dtype="f32", layout="nhwc", N=1001, C=50001, HW=1, pitch=0, k=20, rest=0, masked=True, scale=0.5),
        # A segmentation student: four classes of the teacher at each pixel.
        dict(name="ds_bwd_1x19x1024x2048_bf16_k4", op="distill", way="bwd", dtype="bf16", layout="nhwc", N=1, C=19, HW=2097152, pitch=0, k=4, rest=0, masked=False, scale=1.0),
        # A small batch of a 1000-class student: the smallest training call.
        dict(name="ds_bwd_64x1000_f32_k10", op="distill", way="bwd", dtype="f32", layout="nhwc", N=64, C=1000, HW=1, pitch=0, k=10, rest=1, masked=False, scale=0.5),
        # Validation of a student, the loss alone.
        dict(name="ds_fwd_2048x32000_bf16_k16", op="distill", way="fwd", dtype="bf16", layout="nhwc", N=2048, C=32000, HW=1, pitch=0, k=16, rest=1, masked=False, scale=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, way, dtype = rng.choice(["logprob", "distill"]), rng.choice(["fwd", "bwd"]), rng.choice(["bf16", "bf16", "f32"])
    if rng.random() < 0.3:   # a map
        classes = _log(rng, 2, 200)
        layout, N = rng.choice(["nhwc", "nchw"]), rng.choice([1, 2, 3])
        HW, pitch = _log(rng, 7, 30_000_000 // (classes * N)), 0
    else:
        classes = _log(rng, 10, 150_000)
        layout, HW = "nhwc", 1
        N = _log(rng, 1, min(8192, 100_000_000 // classes))
        pitch = rng.choice([0, 0, (classes + 63) // 64 * 64])
    k = 0 if op == "logprob" and way == "bwd" else min(classes, _log(rng, 1, 100))
    return dict(op=op, way=way, dtype=dtype, layout=layout, N=N, C=classes, HW=HW, pitch=pitch, k=k,
                rest=rng.choice([0, 1]) if op == "distill" else 0, masked=rng.random() < 0.3, scale=rng.choice([1.0, 1.0, 0.5, 1.3]))


def _classes(rows, classes, k, g):
    """k distinct classes per row"""
    start = torch.randint(0, classes, (rows, 1), generator=g, device="cuda")
    step = 1 + (torch.rand((rows, 1), generator=g, device="cuda") * (classes // max(k, 1))).long().clamp_(max=max(0, classes // max(k, 1) - 1))
    return (start + step * torch.arange(k, device="cuda")) % classes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, classes, k = case["N"] * case["HW"], case["C"], case["k"]
    T = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    pitch = case["pitch"] or classes

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # A few classes stand out of the others; the last ones of a padded vocabulary, and random ones of some rows, are masked.
    few = max(1, min(classes, k or 4))
    liked = _classes(rows, classes, few, g)
    x = normal(rows, classes).mul_(1.5 if classes < 200 else 2.5)
    if case["masked"]:
        x[:, classes - classes // 32:] = -math.inf
        x[::3].masked_fill_(torch.rand(x[::3].shape, generator=g, device="cuda") < 0.5, -math.inf)
    x.scatter_(1, liked, normal(rows, few).add_(2 + math.log(classes) / 1.5 - 2.0 * torch.arange(few, device="cuda") / few))
    if case["masked"] and rows >= 4:
        x[rows // 2] = -math.inf
    s = {"case": case, "rows": rows}
    if case["layout"] == "nchw":
        s["x"] = x.view(case["N"], case["HW"], classes).transpose(1, 2).contiguous().to(T)
    else:
        s["x"] = torch.full((rows, pitch), 1e4, dtype=T, device="cuda") if pitch != classes else torch.empty((rows, classes), dtype=T, device="cuda")
        s["x"][:, :classes] = x
    del x
    rand = torch.rand(rows, generator=g, device="cuda")
    if case["op"] == "logprob":
        label = torch.where(rand < 0.7, liked[:, 0], torch.randint(0, classes, (rows,), generator=g, device="cuda"))
        s["label"] = torch.where(rand > 0.97, -1, label).int()   # -1: no class
        s["dlogp"], s["dentropy"] = normal(rows) / rows, normal(rows) * (0.1 / rows)
        s["logp"], s["entropy"], s["lse"] = (torch.empty(rows, device="cuda") for _ in range(3))
        s["rank"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["top_logp"] = torch.empty((rows, k), device="cuda")
        s["top_out"] = torch.empty((rows, k), dtype=torch.int32, device="cuda")
    else:
        s["top_class"] = liked.int()
        t = (normal(rows, k) - 3.0 * torch.arange(k, device="cuda") / k).sort(1, descending=True).values
        if case["rest"]:         # log probabilities of a list that holds 60 to 99.9 % of the weight
            t = t - t.logsumexp(1, keepdim=True) + torch.log(0.6 + 0.399 * rand)[:, None]
        s["top_logit"] = t.contiguous()
        s["dloss"] = torch.rand(rows, generator=g, device="cuda") / rows
        s["loss"] = torch.empty(rows, device="cuda")
    if case["way"] == "bwd":
        s["dx"] = torch.zeros_like(s["x"])
    return s


# ---------------------------------------------------------------- the plain form
def _rows(s):
    c = s["case"]
    x = s["x"].transpose(1, 2).reshape(s["rows"], c["C"]) if c["layout"] == "nchw" else s["x"][:, :c["C"]]
    return x.float()


def _put(s, d):
    """A gradient [rows][classes] in the layout of the logits; what lies between rows is nobody's and stays zero"""
    c, T = s["case"], s["x"].dtype
    if c["layout"] == "nchw":
        return d.view(c["N"], c["HW"], c["C"]).transpose(1, 2).to(T).contiguous()
    out = torch.zeros_like(s["x"])
    out[:, :c["C"]] = d
    return out


def _stats(x, scale):
    """z, exp(z - max), its sum, log-sum-exp; a row of -inf has the sum 0"""
    z = x * scale
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(z - m)
    return z, m, e, e.sum(1, keepdim=True)


def _entropy(z, m, e, S):
    some = S > 0
    part = torch.where(e > 0, e * (z - m), 0.0).sum(1, keepdim=True)
    return torch.where(some, torch.log(S) - part / S, 0.0)


def _logprob(s):
    c = s["case"]
    x = _rows(s)
    z, m, e, S = _stats(x, c["scale"])
    some, lse, H = S > 0, m + torch.log(S), _entropy(z, m, e, S)
    label = s["label"].long()[:, None]
    known = label >= 0
    at = label.clamp(min=0)
    xl, zl = x.gather(1, at), z.gather(1, at)
    logp = torch.where(known, torch.where(some, (zl - m) - torch.log(S), -math.inf), 0.0)
    if c["way"] == "bwd":
        p = torch.where(some, e / S, 0.0)
        logs = torch.where(p > 0, (z - m) - torch.log(S), 0.0)
        dl = torch.where(known & some, s["dlogp"][:, None], 0.0)
        d = p * (-dl - s["dentropy"][:, None] * (logs + H))
        d = d.scatter_add(1, at, dl) * c["scale"]
        return {"dlogits": _put(s, d), "lse": lse[:, 0], "entropy": H[:, 0], "logp": logp[:, 0]}
    cls = torch.arange(c["C"], device="cuda")
    rank = torch.where(known, ((x > xl) | ((x == xl) & (cls < at))).sum(1, keepdim=True), -1).int()
    bits = (x + 0.0).view(torch.int32)                      # order by value, then by the lower class
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order.mul_(1 << 32).add_(c["C"] - 1 - cls).topk(c["k"], dim=1).values
    top = c["C"] - 1 - (key & 0xFFFFFFFF)
    top_logp = torch.where(some, (z.gather(1, top) - m) - torch.log(S), -math.inf)
    return {"lse": lse[:, 0], "entropy": H[:, 0], "logp": logp[:, 0], "rank": rank[:, 0], "top_class": top.int(), "top_logp": top_logp}


def _distill(s):
    c = s["case"]
    z, m, e, S = _stats(_rows(s), c["scale"])
    some, at = S > 0, s["top_class"].long()
    a = s["top_logit"] * (1.0 if c["rest"] else c["scale"])
    if not c["rest"]:
        a = a - a.amax(1, keepdim=True)
        a = a - torch.log(torch.exp(a).sum(1, keepdim=True))
    q = torch.exp(a)
    loss = (q * (a - ((z.gather(1, at) - m) - torch.log(S)))).sum(1, keepdim=True)
    Q, qr, Sr = q.sum(1, keepdim=True), 0.0, 1.0
    if c["rest"]:
        outside = e.scatter(1, at, 0.0)
        Sr = outside.sum(1, keepdim=True)
        qr = torch.where(Sr > 0, (1.0 - Q).clamp(min=0.0), 0.0)
        loss = loss + torch.where(qr > 0, qr * (torch.log(qr) - torch.log(Sr) + torch.log(S)), 0.0)
        Q = Q + qr
    loss = torch.where(some, loss, 0.0)
    if c["way"] == "fwd":
        return {"loss": loss[:, 0]}
    d = torch.where(some, e / S, 0.0) * Q
    if c["rest"]:
        d = d - torch.where(qr > 0, outside * (qr / Sr), 0.0)
    d = d.scatter_add(1, at, torch.where(some, -q, 0.0)) * (s["dloss"][:, None] * c["scale"])
    return {"dlogits": _put(s, d), "loss": loss[:, 0]}


# ---------------------------------------------------------------- the framework's calls
def _p(t):
    return t.data_ptr() if t is not None else None


def _logprob_own(s):
    from arraydiff_cuda_b200 import abi
    c, L = s["case"], abi.lib()
    a = abi.LogprobArgs(abi.AD_BF16 if c["dtype"] == "bf16" else abi.AD_F32, abi.AD_NCHW if c["layout"] == "nchw" else abi.AD_NHWC, c["N"], c["C"], c["HW"],
                        c["scale"], _p(s["x"]), c["pitch"], _p(s["label"]), _p(s["lse"]), _p(s["entropy"]), _p(s["logp"]))
    st = torch.cuda.current_stream().cuda_stream
    if c["way"] == "bwd":
        a.dentropy, a.dlogp, a.dlogits, a.dlogits_pitch = _p(s["dentropy"]), _p(s["dlogp"]), _p(s["dx"]), c["pitch"]
        abi.check(L.ad_logprob_bwd(C.byref(a), st), "ad_logprob_bwd")
        return {"dlogits": s["dx"], "lse": s["lse"], "entropy": s["entropy"], "logp": s["logp"]}
    a.rank, a.top, a.top_class, a.top_logp = _p(s["rank"]), c["k"], _p(s["top_out"]), _p(s["top_logp"])
    abi.check(L.ad_logprob_fwd(C.byref(a), st), "ad_logprob_fwd")
    return {"lse": s["lse"], "entropy": s["entropy"], "logp": s["logp"], "rank": s["rank"], "top_class": s["top_out"], "top_logp": s["top_logp"]}


def _distill_own(s):
    from arraydiff_cuda_b200 import abi
    c, L = s["case"], abi.lib()
    a = abi.DistillArgs(abi.AD_BF16 if c["dtype"] == "bf16" else abi.AD_F32, abi.AD_NCHW if c["layout"] == "nchw" else abi.AD_NHWC, c["N"], c["C"], c["HW"],
                        c["scale"], _p(s["x"]), c["pitch"], c["k"], c["rest"], _p(s["top_class"]), _p(s["top_logit"]), None,
                        1.0 if c["rest"] else c["scale"])
    a.loss = _p(s["loss"])
    st = torch.cuda.current_stream().cuda_stream
    if c["way"] == "fwd":
        abi.check(L.ad_distill_fwd(C.byref(a), st), "ad_distill_fwd")
        return {"loss": s["loss"]}
    a.dloss, a.dlogits, a.dlogits_pitch = _p(s["dloss"]), _p(s["dx"]), c["pitch"]
    abi.check(L.ad_distill_bwd(C.byref(a), st), "ad_distill_bwd")
    return {"dlogits": s["dx"], "loss": s["loss"]}


def run(state):
    if state["case"]["op"] == "logprob":
        return _logprob_own(state) if own else _logprob(state)
    return _distill_own(state) if own else _distill(state)


# ---------------------------------------------------------------- work and the definition in 64 bits
def work(case):
    rows, e, k = case["N"] * case["HW"], 2 if case["dtype"] == "bf16" else 4, case["k"]
    row = case["C"] * e * (2 if case["way"] == "bwd" else 1)
    if case["op"] == "logprob":
        row += 4 + 12 + (8 if case["way"] == "bwd" else 4 + 8 * k)
    else:
        row += 8 * k + 4 + (4 if case["way"] == "bwd" else 0)
    return {"bytes": rows * row, "flops": rows * case["C"] * (10 if case["way"] == "bwd" else 6)}


def exact(case, seed):
    s = prepare(case, seed)
    classes, rows = case["C"], s["rows"]
    nchw = case["layout"] == "nchw"
    x = s["x"].transpose(1, 2).reshape(rows, classes) if nchw else s["x"][:, :classes]
    names = {("logprob", "fwd"): ("lse", "entropy", "logp", "top_logp"), ("logprob", "bwd"): ("lse", "entropy", "logp", "dlogits"),
             ("distill", "fwd"): ("loss",), ("distill", "bwd"): ("loss", "dlogits")}[case["op"], case["way"]]
    out = {n: [] for n in names}
    part = max(1, 60_000_000 // classes)
    for lo in range(0, rows, part):
        z = x[lo:lo + part].double() * case["scale"]
        n = z.shape[0]
        empty = (z == -math.inf).all(1)
        lse = torch.logsumexp(z, 1)
        logs = (z - torch.where(empty, 0.0, lse)[:, None])          # log softmax; -inf throughout an empty row
        p = logs.exp()
        if case["op"] == "logprob":
            H = -torch.special.xlogy(p, p).sum(1)
            label = s["label"][lo:lo + part].long()
            known = label >= 0
            hot = torch.zeros_like(z)
            hot[torch.arange(n, device="cuda")[known], label[known]] = 1.0
            out["lse"].append(lse)
            out["entropy"].append(H)
            out["logp"].append(torch.where(known, logs[torch.arange(n, device="cuda"), label.clamp(min=0)], 0.0))
            if case["way"] == "fwd":
                out["top_logp"].append(logs.sort(1, descending=True).values[:, :case["k"]])
            else:
                dl, dh = s["dlogp"][lo:lo + part].double()[:, None], s["dentropy"][lo:lo + part].double()[:, None]
                by_label = torch.where(known[:, None], hot - p, 0.0) * dl
                d = by_label - dh * (torch.special.xlogy(p, p) + p * H[:, None])
        else:
            at = s["top_class"][lo:lo + part].long()
            t = s["top_logit"][lo:lo + part].double()
            q = t.exp() if case["rest"] else torch.softmax(t * case["scale"], 1)
            full = torch.zeros_like(z).scatter_add_(1, at, q)
            kept = torch.zeros_like(z, dtype=torch.bool).scatter_(1, at, True)
            want = torch.special.xlogy(q, q).sum(1) - torch.where(q > 0, q * logs.gather(1, at), 0.0).sum(1)
            d = p * q.sum(1, keepdim=True) - full
            if case["rest"]:
                pr = torch.where(kept, 0.0, p).sum(1)
                qr = torch.where(pr > 0, (1.0 - q.sum(1)).clamp(min=0.0), 0.0)
                safe = torch.where(pr > 0, pr, 1.0)
                want = want + torch.special.xlogy(qr, qr) - qr * safe.log()
                d = d + p * qr[:, None] - torch.where(kept, 0.0, p) * (qr / safe)[:, None]
            d = d * s["dloss"][lo:lo + part].double()[:, None]
            out["loss"].append(torch.where(empty, 0.0, want))
        if case["way"] == "bwd":
            out["dlogits"].append(torch.where(empty[:, None], 0.0, d) * case["scale"])
    r = {n: torch.cat(v) for n, v in out.items()}
    if "dlogits" in r:
        d = r["dlogits"]
        if nchw:
            r["dlogits"] = d.view(case["N"], case["HW"], classes).transpose(1, 2).contiguous()
        else:
            r["dlogits"] = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
            r["dlogits"][:, :classes] = d
    if case["op"] == "logprob" and case["way"] == "fwd":
        r["rank"] = r["top_class"] = None
    return r
