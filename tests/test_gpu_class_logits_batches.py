"""Class-logit operators on whole batches: every row against the same operators in torch, in 64 bits on the
device.  Tolerances as in test_gpu_class_logits.py, with a reach of at most 40."""
import numpy as np
import pytest

import catboost_rs_b200 as cb
from tests import test_gpu_class_logits as base

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def rows(n, V, dtype, layout, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    a = torch.randn((n, V), generator=gen, device="cuda", dtype=torch.float64) * 2.0
    t = a.to(base.DTYPES[dtype])
    if layout == "rows":
        return t
    if layout == "dims":
        return t.t().contiguous().t()
    big = torch.full((n, V + 3), float("nan"), dtype=t.dtype, device="cuda")
    big[:, 1:V + 1] = t
    return big[:, 1:V + 1]


# (up to 512 classes and above, few rows and many, one block a row and clusters of 2 to 16)
BATCHES = [(30011, 3, "f32", "dims"), (30011, 10, "f64", "dims"), (30011, 16, "f64", "rows"), (20003, 17, "f32", "rows"),
           (20003, 33, "bf16", "offset"), (20003, 100, "f32", "rows"), (20003, 128, "f16", "offset"),
           (9999, 129, "f32", "rows"), (9999, 300, "bf16", "rows"), (9999, 512, "f32", "offset"), (5003, 513, "f32", "rows"),
           (5003, 1000, "bf16", "offset"), (5003, 1024, "f64", "rows"), (5003, 1025, "f16", "rows"),
           (2011, 4099, "f32", "offset"), (1009, 20001, "bf16", "rows"), (601, 40003, "f16", "offset"),
           (301, 70001, "f32", "rows"), (101, 262144, "bf16", "rows"), (51, 262143, "f32", "offset")]


@pytest.mark.parametrize("n,V,dtype,layout", BATCHES)
def test_every_row(n, V, dtype, layout):
    T, u = 1.5, base.unit(dtype)
    x, y = rows(n, V, dtype, layout, V), rows(n, V, dtype, "rows", V + 1)
    for k in sorted({1, min(V, 8), min(V, 40)}):
        top = cb.top_logits(y, k, temperature=T)
        value, order = torch.sort(y.double(), dim=1, descending=True, stable=True)
        assert torch.equal(top.index.long(), order[:, :k]) and torch.equal(top.value.double(), value[:, :k])
        rest = torch.logsumexp(value[:, k:] / T, dim=1)
        if k < V:
            assert ((top.tail.double() - rest).abs() <= u * (124 + 3 * rest.abs())).all()
        del value, order, rest
    wide = torch.float64 if dtype == "f64" else torch.float32
    gen = torch.Generator("cuda").manual_seed(V)
    w = torch.rand((n,), generator=gen, device="cuda", dtype=wide) + 0.5
    d = cb.distill_derivatives(x, top, weight=w, temperature=T)
    tail = top.tail.double()
    log_q = torch.log_softmax(torch.cat([top.value.double() / T, tail[:, None]], 1), 1)
    q, at, p = log_q.exp(), top.index.long(), torch.softmax(x.double() / T, 1)
    share = p.gather(1, at)
    others = p.scatter(1, at, 0.0)
    mass = others.sum(1, keepdim=True)
    loss = (q[:, :-1] * (log_q[:, :-1] - share.log())).sum(1)
    if k < V:
        loss += q[:, -1] * (log_q[:, -1] - mass[:, 0].log())
        target = others * (q[:, -1:] / mass)
    else:
        target = torch.zeros_like(p)
    target.scatter_(1, at, q[:, :-1])
    rel = 2 * u * 124
    loss = loss * w.double() * T * T
    # (scaled logits and the tail are below 40)
    bound = w.double() * T * T * (2 * rel + 6 * u * 40) + 4 * u * loss.abs()
    assert ((d.loss.double() - loss).abs() <= bound).all()
    assert torch.equal(cb.distill_loss(x, top, weight=w, temperature=T), d.loss)
    wt = (w.double() * T)[:, None]
    small = float(torch.finfo(x.dtype).smallest_normal) * float(torch.finfo(x.dtype).eps)
    off = d.der1.double() - wt * (target - p)
    off = off.abs_() - (wt * (p + target) * (2 * rel) + (wt * (target - p)).abs() * base.rounding(dtype) + small)
    assert off.max() <= 0
    del p, others, target, off
    # draws: numbers that lie 1e-9 and more from a border of the mass
    e = ((x.double() - x.double().max(1, keepdim=True).values) / T).exp()
    for kw in (dict(), dict(top_k=min(V, 7)), dict(min_p=0.05), dict(top_k=max(1, V // 3))):
        kept = e
        if "top_k" in kw:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :kw["top_k"]]
            kept = torch.zeros_like(e).scatter_(1, order, e.gather(1, order))
        if "min_p" in kw:
            kept = torch.where(e >= kw["min_p"], e, torch.zeros_like(e))
        upto = kept.cumsum(1)
        upto /= upto[:, -1:].clone()
        r = torch.rand((n, 1), generator=gen, device="cuda", dtype=torch.float64)
        clear = ((upto - r).abs().min(1).values > 1e-9) & ~((e / kw.get("min_p", 1.0) - 1.0).abs() < 1e-9).where(
            torch.tensor("min_p" in kw, device="cuda"), torch.zeros((), dtype=torch.bool, device="cuda")).any(1)
        want = torch.searchsorted(upto, r, right=True)[:, 0]
        got = cb.sample_classes(x, r[:, 0].contiguous(), temperature=T, **kw).long()
        assert torch.equal(got[clear], want[clear]) and clear.double().mean() > 0.9, kw
