"""Class-logit operators without a GPU: what the entry points and the Python layer refuse, and the
64-bit forms the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import catboost_rs_b200 as cb
from catboost_rs_b200 import _lib
from tests import logits_reference as ref

INVALID = 2
SOME = 1 << 20  # a non-NULL pointer that no refused call reads


def logits(**kw):
    d = dict(data=SOME, dtype=_lib.F32, n_classes=10, n=4, row_stride=10, class_stride=1)
    d.update(kw)
    return _lib.Logits(**d)


def teacher(**kw):
    d = dict(index=SOME << 1, value=SOME << 2, tail=None, index_bytes=4, value_dtype=_lib.F32, k=3)
    d.update(kw)
    return _lib.Teacher(**d)


def sampling(**kw):
    d = dict(uniform=SOME, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, uniform_dtype=_lib.F32)
    d.update(kw)
    return _lib.Sampling(**d)


def refused(rc, text):
    assert rc == INVALID
    assert text in _lib.last_error(), _lib.last_error()


BAD_LOGITS = [(dict(dtype=4), "dtype 4"), (dict(n_classes=0), "n_classes = 0"), (dict(n_classes=262145), "262145"),
              (dict(n=-1), "n = -1"), (dict(n=1 << 31), "2147483648"), (dict(row_stride=-10), "negative"),
              (dict(class_stride=-1), "negative"), (dict(data=None), "NULL"), (dict(data=SOME + 2), "aligned")]


@pytest.mark.parametrize("change,text", BAD_LOGITS)
def test_bad_logits_are_refused(change, text):
    L, x = _lib.load(), logits(**change)
    refused(L.cbgpu_top_logits(C.byref(x), 1, 1.0, SOME, SOME, None, None), text)
    refused(L.cbgpu_distill(C.byref(x), C.byref(teacher()), None, 1.0, SOME, None, 0, 0, None), text)
    refused(L.cbgpu_sample_classes(C.byref(x), C.byref(sampling()), SOME, None), text)


def test_null_arguments_are_refused():
    L, x = _lib.load(), logits()
    refused(L.cbgpu_top_logits(None, 1, 1.0, SOME, SOME, None, None), "NULL")
    refused(L.cbgpu_top_logits(C.byref(x), 1, 1.0, None, SOME, None, None), "NULL")
    refused(L.cbgpu_distill(C.byref(x), None, None, 1.0, SOME, None, 0, 0, None), "NULL")
    refused(L.cbgpu_distill(C.byref(x), C.byref(teacher()), None, 1.0, None, None, 0, 0, None), "NULL")
    refused(L.cbgpu_distill(C.byref(x), C.byref(teacher(index=None)), None, 1.0, SOME, None, 0, 0, None), "NULL")
    refused(L.cbgpu_sample_classes(C.byref(x), None, SOME, None), "NULL")
    refused(L.cbgpu_sample_classes(C.byref(x), C.byref(sampling(uniform=None)), SOME, None), "NULL")


@pytest.mark.parametrize("k", [-1, 0, 11, 257])
def test_bad_k_is_refused(k):
    L, x = _lib.load(), logits()
    refused(L.cbgpu_top_logits(C.byref(x), k, 1.0, SOME, SOME, None, None), f"k = {k}")
    if k != 11:  # a teacher may know more classes than the student has
        refused(L.cbgpu_distill(C.byref(x), C.byref(teacher(k=k)), None, 1.0, SOME, None, 0, 0, None), f"k = {k}")


@pytest.mark.parametrize("t", [0.0, -1.0, float("nan"), float("inf"), 1e-7, 1e7])
def test_bad_temperature_is_refused(t):
    L, x = _lib.load(), logits()
    refused(L.cbgpu_top_logits(C.byref(x), 1, t, SOME, SOME, None, None), "temperature")
    refused(L.cbgpu_distill(C.byref(x), C.byref(teacher()), None, t, SOME, None, 0, 0, None), "temperature")
    if t != 0.0:
        refused(L.cbgpu_sample_classes(C.byref(x), C.byref(sampling(temperature=t)), SOME, None), "temperature")


@pytest.mark.parametrize("change,text", [
    (dict(top_p=1.5), "top_p"), (dict(top_p=float("nan")), "top_p"), (dict(min_p=-0.1), "min_p"),
    (dict(min_p=1.1), "min_p"), (dict(top_k=-1), "top_k"), (dict(uniform_dtype=_lib.BF16), "uniform")])
def test_bad_sampling_settings_are_refused(change, text):
    L, x = _lib.load(), logits()
    refused(L.cbgpu_sample_classes(C.byref(x), C.byref(sampling(**change)), SOME, None), text)


@pytest.mark.parametrize("der1,rs,cs,text", [
    (SOME + 4, 10, 1, "overlaps the logits"),      # shifted by one element
    (SOME, 1, 4, "overlaps the logits"),           # the same memory, another layout
    (SOME + 64, 0, 1, "share memory"), (SOME + 4096, 9, 1, "share memory"), (SOME + 4096, 1, 3, "share memory"),
    (SOME + 4096, -10, 1, "negative"), ((SOME << 1) - 4, 10, 1, "overlaps the teacher"),
    ((SOME << 2) + 8, 10, 1, "overlaps the teacher"), (SOME + 4098, 10, 1, "aligned")])
def test_bad_der1_is_refused(der1, rs, cs, text):
    L, x = _lib.load(), logits()
    refused(L.cbgpu_distill(C.byref(x), C.byref(teacher()), None, 1.0, SOME << 3, der1, rs, cs, None), text)


@pytest.mark.parametrize("change,text", [(dict(index_bytes=2), "index_bytes"), (dict(value_dtype=7), "value_dtype")])
def test_bad_teacher_is_refused(change, text):
    L, x = _lib.load(), logits()
    refused(L.cbgpu_distill(C.byref(x), C.byref(teacher(**change)), None, 1.0, SOME, None, 0, 0, None), text)


def test_unaligned_arrays_are_refused():
    L, x, odd = _lib.load(), logits(), SOME + 4098
    far = SOME << 4
    for v, i, t in ((odd, far, None), (far, odd, None), (far, far, odd)):
        refused(L.cbgpu_top_logits(C.byref(x), 1, 1.0, v, i, t, None), "aligned")
    for t, w, loss in ((teacher(index=odd), None, far), (teacher(value=odd), None, far), (teacher(tail=odd), None, far),
                       (teacher(index=far + 4, index_bytes=8), None, far), (teacher(), odd, far), (teacher(), None, odd)):
        refused(L.cbgpu_distill(C.byref(x), C.byref(t), w, 1.0, loss, None, 0, 0, None), "aligned")
    for name in ("uniform", "temperature_rows", "top_p_rows", "min_p_rows", "top_k_rows"):
        refused(L.cbgpu_sample_classes(C.byref(x), C.byref(sampling(**{name: odd})), far, None), "aligned")
    refused(L.cbgpu_sample_classes(C.byref(x), C.byref(sampling()), odd, None), "aligned")


def test_no_rows_is_no_work():
    # needs no device: nothing is launched
    L, x = _lib.load(), logits(n=0, data=None)
    assert L.cbgpu_top_logits(C.byref(x), 1, 1.0, None, None, None, None) == 0
    assert L.cbgpu_distill(C.byref(x), C.byref(teacher()), None, 1.0, None, None, 0, 0, None) == 0
    assert L.cbgpu_sample_classes(C.byref(x), C.byref(sampling(uniform=None)), None, None) == 0


def test_python_layer_refuses():
    torch = pytest.importorskip("torch")
    x = torch.zeros((2, 4))
    t = cb.TopLogits(torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)))
    for call in (lambda v: cb.top_logits(v, 1), lambda v: cb.distill_loss(v, t),
                 lambda v: cb.distill_derivatives(v, t), lambda v: cb.sample_classes(v, torch.zeros(2))):
        for v, text in ((np.zeros((2, 4)), "torch tensor"), (x[0], "classes"), (x.int(), "float64"),
                        (x, "CUDA"), (torch.zeros((2, 0)), "0 classes")):
            with pytest.raises(cb.CbGpuError, match=text):
                call(v)


def test_struct_layouts_match_the_header():
    import os
    import re
    hdr = open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "include", "cbgpu.h")).read()
    for cls, name in ((_lib.Logits, "cbgpu_logits"), (_lib.Teacher, "cbgpu_teacher"), (_lib.Sampling, "cbgpu_sampling")):
        end = hdr.index("} " + name + ";")
        body = re.sub(r"/\*.*?\*/", "", hdr[hdr.rindex("typedef struct {", 0, end):end], flags=re.S)
        assert re.findall(r"\b(\w+);", body) == [f for f, _ in cls._fields_]
    ids = dict(re.findall(r"CBGPU_(F64|F32|F16|BF16) = (\d)", hdr))
    assert {k: int(v) for k, v in ids.items()} == dict(F64=_lib.F64, F32=_lib.F32, F16=_lib.F16, BF16=_lib.BF16)


# ---- the 64-bit forms themselves ---------------------------------------------

@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("tail", [-np.inf, 0.3])
def test_reference_der1_is_minus_the_gradient_by_differences(seed, tail):
    rs = np.random.RandomState(seed)
    V, T, w, h = 9, 1.7, 0.6, 1e-5
    a = rs.randn(V) * 2
    index, value = np.array([4, 1, -1, 4, 7]), rs.randn(5)
    loss, der1, _, _ = ref.distill(a, index, value, tail, w, T)
    assert loss > 0
    for i in range(V):
        up, dn = a.copy(), a.copy()
        up[i] += h
        dn[i] -= h
        num = (ref.distill(up, index, value, tail, w, T)[0] - ref.distill(dn, index, value, tail, w, T)[0]) / (2 * h)
        assert abs(der1[i] + num) < 1e-8  # O(h^2) and 1e-16 / h


def test_reference_is_zero_at_the_teacher():
    rs = np.random.RandomState(5)
    a = rs.randn(20)
    index, value, rest = ref.top(a, 6, 1.3)
    loss, der1, _, _ = ref.distill(a, index, value, rest, 1.0, 1.3)
    assert abs(loss) < 1e-14 and np.abs(der1).max() < 1e-15


def test_reference_sampling_frequencies():
    row = np.array([1.0, 3.0, 2.0, 3.0, -np.inf])
    us = (np.arange(10000) + 0.5) / 10000
    got = np.bincount([ref.sample(row, u, 1.0, 3, 1.0, 0.0) for u in us], minlength=5) / 10000
    e = np.array([0, 1, np.exp(-1), 1, 0])
    assert np.abs(got - e / e.sum()).max() <= 2e-4
    assert {ref.sample(row, u, 1.0, 0, 0.2, 0.0) for u in us} == {1}      # the lower index of the tie
    assert {ref.sample(row, u, 1.0, 0, 1.0, 0.5) for u in us} == {1, 3}
    assert {ref.sample(row, u, 0.0, 0, 1.0, 0.0) for u in us} == {1}


def test_torch_can_be_imported_after_the_library():
    import subprocess
    import sys
    pytest.importorskip("torch")
    code = "import catboost_rs_b200 as cb; cb.load_library(); import torch"
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_set_teacher_rejects_a_null_session_on_the_host():
    refused(_lib.load().cbgpu_multi_set_teacher(None, None, None, None, 1, 1.0), "no session")
