"""MultiClass sessions on a teacher: replaced teachers, and what a call that fails leaves behind."""
import numpy as np
import pytest

import catboost_rs_b200 as cb
from tests.test_gpu_class_logits import columns

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def session(X, borders, K):
    rt = cb.B200MultiRuntime()
    assert rt.begin_device_training_raw("MultiClass", 3, True, 1, "Cosine", [c.copy() for c in X.T], borders, None,
                                        len(X), X.shape[1], 33, 0.1, 3.0, cb.DeviceTrainConfig(), approx_dim=K)
    return rt


def grow(rt, K, target=None):
    t = rt.grow_tree_on_device(None, target, [], family=("MultiOutput", None, K), leaf_of_bytes=0, resident_approx=True)
    return t.splits, np.array(t.leaf_values)


def all_device_memory_but(room):
    torch.cuda.empty_cache()
    while True:
        free = torch.cuda.mem_get_info()[0]
        try:
            return torch.empty((free - room,), dtype=torch.uint8, device="cuda")
        except torch.OutOfMemoryError:
            room += 64 << 20


def test_a_teacher_that_finds_no_memory_leaves_the_one_before():
    n, K, T = 300000, 4, 2.0
    X, borders, rs = columns(n, 3, 5)
    z = rs.standard_normal((n, K))
    index = np.tile(np.arange(K, dtype=np.int32), (n, 1))
    rt = session(X, borders, K)
    assert rt.set_teacher(index, z, None, T)
    want = grow(rt, K)
    rt.end_device_training()

    rt = session(X, borders, K)
    assert rt.set_teacher(index, z, None, T)
    large = np.full((n, 256), -1, dtype=np.int32), np.zeros((n, 256))  # 0.9 GB
    held = all_device_memory_but(256 << 20)
    with pytest.raises(cb.CbGpuError, match="cudaMalloc"):
        rt.set_teacher(*large, None, 1.0)
    del held
    torch.cuda.empty_cache()
    got = grow(rt, K)
    rt.end_device_training()
    assert got[0] == want[0] and np.array_equal(got[1], want[1])


def test_a_replaced_teacher_counts():
    n, K = 5000, 4
    X, borders, rs = columns(n, 3, 6)
    index = np.tile(np.arange(K, dtype=np.int32), (n, 1))
    z, tail = rs.standard_normal((n, K)), rs.standard_normal(n)
    want = []
    for first in (False, True):
        rt = session(X, borders, K)
        if first:
            assert rt.set_teacher(index, -z, tail, 3.0)
            with pytest.raises(cb.CbGpuError):
                rt.set_teacher(index + K, z)
        assert rt.set_teacher(index[:, :2], z[:, :2], tail, 1.5)
        want.append(grow(rt, K))
        rt.end_device_training()
    assert want[0][0] == want[1][0] and np.array_equal(want[0][1], want[1][1])


@pytest.mark.parametrize("V", [10, 100, 700])
def test_an_error_of_another_call_is_not_a_launchs(V):
    x, u = torch.randn((8, V), device="cuda"), torch.full((8,), 0.5, device="cuda")
    few = torch.randn((10000, 100), device="cuda")
    top = cb.top_logits(x, 3)
    calls = [lambda: cb.top_logits(x, 3), lambda: cb.top_logits(few, 8), lambda: cb.distill_derivatives(x, top),
             lambda: cb.sample_classes(x, u)]
    for call in calls:
        call()
    n = 60 << 20  # a prediction that needs 720 MB of device memory
    model = (np.zeros(1, np.uint32), np.zeros(1), np.array([0, 1], np.uint32), np.zeros(2), np.array([0, 2], np.uint32))
    held = all_device_memory_but(256 << 20)
    for call in calls:
        with pytest.raises(cb.CbGpuError, match="out of memory"):
            cb.apply_oblivious(np.zeros((1, n), np.float32), model)
        call()
    del held
    torch.cuda.empty_cache()


def test_a_call_that_fails_leaves_no_error_for_the_next():
    n, K = 2000, 3
    X, borders, rs = columns(n, 3, 7)
    y = rs.randint(0, K, n)
    model = (np.zeros(1, np.uint32), np.zeros(1), np.array([0, 1], np.uint32), np.zeros(2), np.array([0, 2], np.uint32))
    scalar = cb.FitParams(loss="RMSE", depth=3, iterations=2, bootstrap_type="No", random_seed=1)
    cols = [c.copy() for c in X.T]

    def multi():
        rt = session(X, borders, K)
        grow(rt, K, y)
        rt.end_device_training()

    for call in (lambda: cb.fit(cols, borders, X[:, 0].astype(np.float64), scalar), multi,
                 lambda: cb.select_borders([cols[0]], 16), lambda: cb.apply_oblivious(np.zeros((1, 64), np.float32), model)):
        call()
        held = all_device_memory_but(512 << 20)
        with pytest.raises(cb.CbGpuError, match="out of memory"):
            cb.apply_oblivious(np.zeros((1, 120 << 20), np.float32), model)
        call()
        del held
        torch.cuda.empty_cache()
