"""Views that torch negates when they are read: their memory holds the other sign."""
import pytest

import catboost_rs_b200 as cb

torch = pytest.importorskip("torch")


def negated(*shape, device="cpu"):
    v = torch.randn(shape, dtype=torch.complex64, device=device).conj().imag
    assert v.is_neg()
    return v


def test_negated_logits_are_refused():
    t = cb.TopLogits(torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 1)))
    for call in (lambda x: cb.top_logits(x, 2), lambda x: cb.distill_loss(x, t), lambda x: cb.distill_derivatives(x, t),
                 lambda x: cb.sample_classes(x, torch.zeros(4))):
        with pytest.raises(cb.CbGpuError, match="negated"):
            call(negated(4, 9))


@pytest.mark.gpu
def test_negated_operands_are_refused():
    x, u = torch.randn((4, 9), device="cuda"), torch.zeros((4,), device="cuda")
    top = cb.top_logits(x, 2)
    one, two = negated(4, device="cuda"), negated(4, 9, device="cuda")
    for call in (lambda: cb.distill_loss(x, cb.TopLogits(top.index, two[:, :2])),
                 lambda: cb.distill_loss(x, cb.TopLogits(top.index, top.value, one)),
                 lambda: cb.distill_loss(x, top, weight=one), lambda: cb.distill_derivatives(x, top, out=two),
                 lambda: cb.sample_classes(x, one), lambda: cb.sample_classes(x, u, temperature=one),
                 lambda: cb.sample_classes(x, u, top_p=one), lambda: cb.sample_classes(x, u, min_p=one)):
        with pytest.raises(cb.CbGpuError, match="negated"):
            call()
    # resolved, they are taken
    assert torch.equal(cb.top_logits(two.resolve_neg(), 3).value, torch.topk(two, 3, dim=1).values)
