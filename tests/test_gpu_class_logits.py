"""Class-logit operators on the device against their plain 64-bit forms (logits_reference.py).

Tolerances.  u is the unit roundoff of the arithmetic (2^-24 for 16- and 32-bit
logits, 2^-53 for f64).  An exponential's argument (a - m) / T passes two
rounded operations and a scale rounded once, so it is off by at most 3u times
its size; with `reach` the largest such size that matters (beyond it the
probability is below u) an exponential is off by 3u reach plus 2 ulp = 4u of its
own, a probability (two of them) by 2 (3u reach + 4u) of itself.  Outputs add
half a step of their type.  The logarithm of a sum is off by one such relative
error, absolutely; a loss holds two of them and 3u of the scaled logits it
subtracts.
"""
import numpy as np
import pytest

import catboost_rs_b200 as cb
from tests import logits_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def unit(dtype):
    return 2.0 ** -53 if dtype == "f64" else 2.0 ** -24


def rounding(dtype):
    return torch.finfo(DTYPES[dtype]).eps / 2


def host(x):
    return x.detach().to("cpu").double().numpy()


def make(n, V, dtype, layout, seed, masked=0.0, spread=2.5):
    """Device logits with the layout asked for; ties are frequent in 16 bits."""
    rs = np.random.RandomState(seed)
    a = rs.standard_normal((n, V)) * spread
    if V > 50:
        a[np.arange(n)[:, None], rs.randint(0, V, (n, 4))] += rs.uniform(3, 9, (n, 4))
    if masked:
        a[rs.uniform(size=(n, V)) < masked] = -np.inf
    return put(a, dtype, layout)


def put(a, dtype, layout="rows"):
    n, V = a.shape
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DTYPES[dtype]).cuda()
    if layout == "rows":
        return t
    if layout == "dims":
        return t.t().contiguous().t()
    if layout == "offset":  # rows that start at no particular alignment, with room behind them
        big = torch.full((n, V + 3), float("nan"), dtype=t.dtype, device="cuda")
        big[:, 1:V + 1] = t
        return big[:, 1:V + 1]
    if layout == "strided":
        big = torch.full((2 * n, 3 * V), float("nan"), dtype=t.dtype, device="cuda")
        big[::2, ::3] = t
        return big[::2, ::3]
    raise ValueError(layout)


SHAPES = [(1, 1), (5, 2), (300, 7), (70, 12), (33, 13), (40, 100), (9, 128), (21, 129), (10, 1000), (3, 1024),
          (4, 1025), (3, 2048), (2, 4099), (2, 33000), (1, 131071), (1, 262144)]
LAYOUTS = ["rows", "dims", "offset", "strided"]


def grid(shapes=SHAPES):
    """Every shape with every type; the layout and the mask go round."""
    out = []
    for s, (n, V) in enumerate(shapes):
        for d, dtype in enumerate(DTYPES):
            out.append((n, V, dtype, LAYOUTS[(s + d) % 4], [0.0, 0.3][(s + d // 2) % 2]))
    return out


# ---- top_logits ------------------------------------------------------------------

def check_top(x, k, temperature, dtype):
    got = cb.top_logits(x, k, temperature=temperature)
    a = host(x)
    u = unit(dtype)
    idx, val, tail = got.index.cpu().numpy(), host(got.value), host(got.tail)
    assert got.index.dtype == torch.int32 and got.value.dtype == x.dtype
    for r in range(a.shape[0]):
        wi, wv, wt = ref.top(a[r], k, temperature)
        assert (idx[r] == wi).all(), (r, idx[r], wi)
        assert np.array_equal(val[r], wv, equal_nan=True)
        if np.isfinite(wt):
            rest = np.delete(a[r], wi) / temperature
            reach = min(np.max(rest) - np.min(rest[np.isfinite(rest)]), 40.0)
            assert abs(tail[r] - wt) <= u * (3 * reach + 4) + 3 * u * abs(wt), (r, tail[r], wt)
        else:
            assert np.array_equal(tail[r], wt, equal_nan=True), (r, tail[r], wt)


@pytest.mark.parametrize("n,V,dtype,layout,masked", grid())
def test_top_logits(n, V, dtype, layout, masked):
    x = make(n, V, dtype, layout, V + n, masked)
    for k in sorted({1, min(V, 5), min(V, 64), min(V, 256)}):
        check_top(x, k, 0.7, dtype)


@pytest.mark.parametrize("V", [5, 60, 700, 5000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_top_logits_ties_masks_and_nan(V, dtype):
    rows = [np.zeros(V), np.full(V, -np.inf), np.where(np.arange(V) % 2, -0.0, 0.0),
            np.where(np.arange(V) % 3, 1.0, -np.inf), np.full(V, np.nan), np.arange(V) % 4 * 1.0]
    one = np.linspace(3, -3, V)
    one[V // 2] = np.nan
    low = np.full(V, float(torch.finfo(DTYPES[dtype]).min))
    low[V - 1] = 1.0
    rows += [one, low, np.sort(np.arange(V) * 0.125)[::-1].copy()]
    x = put(np.array(rows), dtype)
    for k in {1, 3, min(V, 200)}:
        check_top(x, k, 1.0, dtype)
    got = cb.top_logits(x, 2, tail=False)
    assert got.tail is None


@pytest.mark.parametrize("n,V", [(6, 14), (6, 100), (6, 400), (6, 700), (6, 5000), (40000, 14), (40000, 100)])
@pytest.mark.parametrize("dtype", ["f64", "f32"])
def test_tails_far_below_and_infinite(V, dtype, n):
    # the rest lies 300 (e^-300 is below any f32) to 30000 under the first k; with infinite logits the first
    # k may be those alone, or leave one to the rest
    rs = np.random.RandomState(V)
    a = rs.standard_normal((6, V))
    at = rs.permutation(V)[:7]
    for r, lift in enumerate((300.0, 3000.0, 30000.0, np.inf, -np.inf, 60.0)):
        a[r, at] += lift if lift > 0 else 0.0
        if lift < 0:
            a[r, np.delete(np.arange(V), at)] = -np.inf
    x = put(np.tile(a, (-(-n // 6), 1))[:n], dtype)
    same = torch.arange(n, device="cuda") % 6
    for k in (7, 8):
        check_top(x[:6].contiguous(), k, 1.0, dtype)
        few, many = cb.top_logits(x[:6].contiguous(), k), cb.top_logits(x, k)
        assert torch.equal(many.index, few.index[same]) and torch.equal(many.value, few.value[same])
        fine, u = torch.isfinite(few.tail), unit(dtype)
        assert torch.equal(torch.isfinite(many.tail), fine[same])
        # each within u (3 reach + 4) + 3 u |tail| of the 64-bit value, reach at most 40
        bound = 2 * u * (124 + 3 * few.tail[fine].abs())
        assert ((many.tail[:6] - few.tail)[fine].abs() <= bound).all()
    tail = cb.top_logits(x, 5).tail  # of row 3 two infinite ones are left
    assert torch.isnan(tail[3]) and not torch.isnan(tail[:3]).any()


@pytest.mark.parametrize("V", [9, 300, 6000])
def test_rows_and_classes_that_share_memory(V):
    # strides of 0 are allowed for what is read
    one = make(1, V, "f32", "rows", 3)
    t, u = make_teacher(1, V, 4, "f32", 5, True), torch.full((50,), 0.4, device="cuda")
    many = cb.TopLogits(*(v.repeat_interleave(50, 0) for v in (t.index, t.value, t.tail)))
    x = one.expand(50, V)
    out = torch.empty((50, V), device="cuda")
    d = cb.distill_derivatives(x, many, out=out)
    for got, want in ((d.der1, cb.distill_derivatives(one.repeat(50, 1), many).der1),
                      (cb.top_logits(x, 3).tail, cb.top_logits(one.repeat(50, 1), 3).tail),
                      (cb.sample_classes(x, u, top_p=0.8), cb.sample_classes(one.repeat(50, 1), u, top_p=0.8))):
        assert torch.equal(got, want)
    same = one[:, :1].expand(50, V)  # every class one number
    top = cb.top_logits(same, 3)
    assert (top.index == torch.arange(3, device="cuda")).all() and (top.value == one[0, 0]).all()
    assert (cb.sample_classes(same, u) == int(np.float32(0.4) * np.float64(V))).all()
    with pytest.raises(cb.CbGpuError):
        cb.distill_derivatives(x, many, out=x)


def test_calls_that_overlap_on_streams():
    # nothing is shared between calls: as many at a time as the streams allow
    sets = [batch(V, dtype, n) for V, dtype, n in
            ((10, "f64", 4000), (100, "f32", 4000), (1000, "bf16", 900), (40000, "bf16", 60), (131071, "f32", 4))]

    def call(x, t, u):
        d = cb.distill_derivatives(x, t, temperature=1.5)
        top = cb.top_logits(x, 7)
        return d.loss, d.der1, top.value, top.index, top.tail, cb.sample_classes(x, u, top_p=0.9), \
            cb.sample_classes(x, u, top_k=6)

    want = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for turn in range(4):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(call(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % len(sets)]))


# ---- distillation -------------------------------------------------------------------

def check_distill(x, teacher, weight, temperature, dtype, out=None, lost=0.0):
    u, V = unit(dtype), x.shape[1]
    a = host(x)
    loss_only = host(cb.distill_loss(x, teacher, weight=weight, temperature=temperature))
    got = cb.distill_derivatives(x, teacher, weight=weight, temperature=temperature, out=out)
    assert got.der1.dtype == x.dtype and got.der1.shape == x.shape
    loss, der1 = host(got.loss), host(got.der1)
    idx, val = teacher.index.cpu().numpy(), host(teacher.value)
    tail = np.full(len(a), -np.inf) if teacher.tail is None else host(teacher.tail)
    w = np.ones(len(a)) if weight is None else host(weight)
    small = float(torch.finfo(x.dtype).smallest_normal) * float(torch.finfo(x.dtype).eps)
    for r in range(len(a)):
        wl, wd, p, q = ref.distill(a[r], idx[r], val[r], tail[r], w[r], temperature)
        scaled = np.concatenate([a[r], val[r], [0.0]]) / temperature
        scaled = np.concatenate([scaled[np.isfinite(scaled)], tail[r:r + 1][np.isfinite(tail[r:r + 1])]])
        size = np.abs(scaled).max()
        reach = min(scaled.max() - scaled.min(), 40.0)
        rel = 2 * u * (3 * reach + 4)
        wt2 = abs(w[r]) * temperature * temperature
        for g in (loss[r], loss_only[r]):
            if np.isfinite(wl):
                assert abs(g - wl) <= wt2 * (2 * rel + 6 * u * size) + 4 * u * abs(wl), (r, g, wl)
            else:
                assert np.array_equal(g, wl, equal_nan=True), (r, g, wl)
        if np.isnan(wd).any():
            assert np.isnan(der1[r]).all()
            continue
        bound = abs(w[r]) * temperature * rel * 2 * (p + q) + rounding(dtype) * np.abs(wd) + small + abs(w[r]) * temperature * lost
        off = np.abs(der1[r] - wd) - bound
        assert off.max() <= 0, (r, int(off.argmax()), der1[r][off.argmax()], wd[off.argmax()])
    return got


def make_teacher(n, V, k, dtype, seed, tail, masked=0.0, int64=False, temperature=1.0):
    z = make(n, V, dtype, "rows", seed, masked)
    t = cb.top_logits(z, min(k, V), temperature=temperature)
    index = t.index.long() if int64 else t.index
    return cb.TopLogits(index, t.value, t.tail if tail else None)


@pytest.mark.parametrize("n,V,dtype,layout,masked", grid())
def test_distill(n, V, dtype, layout, masked):
    # a class that only the student masks gives +inf: the masks are the teacher's, and half of
    # the shapes have them
    x = make(n, V, dtype, layout, V + n, 0.0)
    wide = torch.float64 if dtype == "f64" else torch.float32
    weight = torch.rand((n,), dtype=wide, device="cuda", generator=torch.Generator("cuda").manual_seed(V)) + 0.5
    for k, tail, w, temperature in ((1, True, None, 1.0), (16, False, weight, 2.0), (256, True, weight, 0.7)):
        check_distill(x, make_teacher(n, V, k, dtype, V + 7, tail, masked, k == 16, temperature), w, temperature,
                      dtype)


@pytest.mark.parametrize("V", [6, 60, 900, 6000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_distill_edges(V, dtype):
    wide = torch.float64 if dtype == "f64" else torch.float32
    rs = np.random.RandomState(V)
    ninf, nan, inf = -np.inf, np.nan, np.inf
    rows, idx, val, tail, w = [], [], [], [], []

    def add(row, i, z, t=ninf, weight=1.0):
        i = list(i) + [-1] * (5 - len(i))
        z = list(z) + [0.0] * (5 - len(z))
        rows.append(row), idx.append(i), val.append(z), tail.append(t), w.append(weight)

    plain = rs.randn(V)
    add(plain, [0, 1], [1, 2])                                    # entries missing
    add(plain, [], [])                                            # no entry at all
    add(plain, [], [], 0.5)                                       # the others only: loss 0
    add(plain, [3, 3, 3], [1, 7, nan], 0.2)                       # the same index: the first counts
    add(plain, [1, V, -5, V + 100, 2], [1, 9, 9, 9, 2], 0.1)      # indices outside
    add(np.full(V, ninf), [1], [1.0], 0.1)                        # every class masked
    add(np.full(V, nan), [1], [1.0], 0.1, 0.0)                    # weight 0: not read
    add(np.full(V, nan), [1], [1.0], 0.1)
    add(np.where(np.arange(V) == 2, nan, plain), [1], [1.0])
    add(np.where(np.arange(V) == 2, inf, plain), [1], [1.0])
    add(np.where(np.arange(V) == 2, ninf, plain), [1, 2], [1.0, 1.0])   # the student masks an entry: +inf
    add(np.where(np.arange(V) == 2, ninf, plain), [1, 2], [1.0, ninf])  # both do
    add(np.where(np.arange(V) == 0, 1.0, ninf), [0], [1.0], 0.3)  # the student masks all others: +inf
    add(np.where(np.arange(V) == 0, 1.0, ninf), [0], [1.0])       # both do: loss 0
    add(plain, [1], [nan])
    add(plain, [1], [1.0], nan)
    add(plain, [1], [inf])
    add(plain, [0, 1, 2], [ninf, ninf, ninf])                     # entries of no weight
    add(np.full(V, float(torch.finfo(DTYPES[dtype]).min)), [0, 4], [1.0, 2.0], 0.5)  # masked by the lowest value
    add(np.zeros(V), [4, 0], [0.0, 0.0], 0.5, -2.0)
    for layout in ("rows", "dims"):
        x = put(np.array(rows), dtype, layout)
        t = cb.TopLogits(torch.tensor(idx, dtype=torch.int32, device="cuda"),
                         torch.tensor(val, dtype=DTYPES[dtype], device="cuda"),
                         torch.tensor(tail, dtype=wide, device="cuda"))
        check_distill(x, t, torch.tensor(w, dtype=wide, device="cuda"), 1.0, dtype)


@pytest.mark.parametrize("V", [9, 14, 60, 400, 900, 6000, 40000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_distill_others_far_below(V, dtype):
    # the student's other classes lie so far below the teacher's that their exponentials beside them are 0 or
    # nearly so, all of them or those of a part of the row; the teacher's others weigh something
    rs = np.random.RandomState(V)
    a = rs.standard_normal((8, V))
    at = np.stack([rs.permutation(V)[:5] for _ in a])
    for r, lift in enumerate((40.0, 60.0, 85.0, 100.0, 300.0, 1000.0, 20000.0, 100.0)):
        a[r, at[r]] += lift
    a[7, np.delete(np.arange(V), at[7])] -= np.linspace(0, 400, V - 5)
    a[6, V // 2] = -np.inf  # (an entry for some V: a loss of +inf)
    wide = torch.float64 if dtype == "f64" else torch.float32
    t = cb.TopLogits(torch.tensor(at, dtype=torch.int32, device="cuda"),
                     torch.tensor(rs.standard_normal((8, 5)), dtype=DTYPES[dtype], device="cuda"),
                     torch.tensor(rs.uniform(-1, 2, 8), dtype=wide, device="cuda"))
    # in f32 an exponential below 2^-126 of its unit is 0.  The others' sum s is at least 1e-20 in that unit (or
    # the unit is their largest, and s >= 1), so Q e / s and e / (s and the rest) lose at most 2^-126 1e20 each
    lost = 0.0 if dtype == "f64" else 2 * 2.0 ** -126 * 1e20
    for layout in ("rows", "dims"):
        x = put(a, dtype, layout)
        got = check_distill(x, t, None, 1.0, dtype, lost=lost)
        assert torch.isfinite(got.loss[:6]).all() and (got.der1.double().max(1).values > 0).all()
        check_distill(x, t, None, 1.0, dtype, out=x, lost=lost)


@pytest.mark.parametrize("V", [10, 100, 1000, 5000])
@pytest.mark.parametrize("dtype", ["f64", "bf16"])
def test_distill_out(V, dtype):
    n = 37
    x = make(n, V, dtype, "rows", 3)
    t = make_teacher(n, V, 8, dtype, 4, True)
    want = check_distill(x, t, None, 1.0, dtype).der1
    # a strided view: what lies between and behind its rows stays
    big = torch.full((n + 2, 2 * V + 5), 7.0, dtype=x.dtype, device="cuda")
    view = big[1:n + 1, 2:2 + 2 * V:2]
    got = cb.distill_derivatives(x, t, out=view)
    assert got.der1.data_ptr() == view.data_ptr() and torch.equal(view, want)
    view.fill_(7.0)
    assert (big == 7.0).all()
    dims = torch.empty((V, n), dtype=x.dtype, device="cuda").t()
    assert torch.equal(cb.distill_derivatives(x, t, out=dims).der1, want)
    # in place: the same bits as beside; in another layout a row is summed in another grouping, so
    # there the derived bounds of check_distill hold
    y = x.clone()
    assert torch.equal(cb.distill_derivatives(y, t, out=y).der1, want) and torch.equal(y, want)
    for layout in LAYOUTS:
        y = put(host(x), dtype, layout)
        beside = check_distill(y, t, None, 1.0, dtype).der1
        check_distill(y, t, None, 1.0, dtype, out=y)
        assert torch.equal(y, beside)
    # rows that share memory can be read
    one = x[:1].expand(n, V)
    check_distill(one, t, None, 1.0, dtype)


def test_distill_teacher_types_mix():
    x = make(6, 50, "bf16", "rows", 1)
    for vd in DTYPES.values():
        t = cb.TopLogits(torch.arange(18, device="cuda").view(6, 3), torch.randn((6, 3), device="cuda").to(vd))
        check_distill(x, t, None, 1.0, "bf16")
        wide = cb.TopLogits(t.index[:, ::2], t.value[:, ::2], torch.zeros((12,), device="cuda")[::2])
        check_distill(x, wide, None, 1.0, "bf16")  # operands that are not contiguous


def test_der1_is_minus_the_gradient_by_differences():
    n, V, k, h = 3, 1500, 9, 1e-4
    for V in (11, 1500):
        x = make(n, V, "f64", "rows", 8)
        t = make_teacher(n, V, k, "f64", 9, True)
        der1 = host(cb.distill_derivatives(x, t, temperature=1.5).der1)
        probe = list(range(4)) + [int(i) for i in t.index[0, :4]] + [V - 1]
        for i in probe:
            up, dn = x.clone(), x.clone()
            up[:, i] += h
            dn[:, i] -= h
            num = host(cb.distill_loss(up, t, temperature=1.5) - cb.distill_loss(dn, t, temperature=1.5)) / (2 * h)
            assert np.abs(der1[:, i] + num).max() < 1e-7  # third derivative h^2 / 6 < 1e-8; 1e-15 / h


# ---- sampling ----------------------------------------------------------------------

SETTINGS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.0), dict(top_p=0.3), dict(top_p=0.9),
            dict(min_p=0.1), dict(min_p=1.0), dict(top_k=300, top_p=0.95, min_p=0.01), dict(temperature=0.0),
            dict(temperature=0.3, top_p=0.8), dict(temperature=5.0, top_k=70, top_p=0.99)]


def check_sample(x, u, **kw):
    got = cb.sample_classes(x, u, **kw)
    assert got.dtype == torch.int32
    a, uh = host(x), host(u)
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    full.update(kw)
    full = {k: (host(v) if isinstance(v, torch.Tensor) else np.full(len(a), v)) for k, v in full.items()}
    want = [ref.sample(a[r], uh[r], full["temperature"][r], int(full["top_k"][r]), full["top_p"][r], full["min_p"][r])
            for r in range(len(a))]
    assert got.cpu().tolist() == [int(v) for v in want], kw


@pytest.mark.parametrize("n,V,dtype,layout,masked", grid())
def test_sample_classes(n, V, dtype, layout, masked):
    x = make(n, V, dtype, layout, V + n, masked)
    if V == 1:
        x = put(np.zeros((n, 1)), dtype)
    gen = torch.Generator("cuda").manual_seed(V)
    for i, kw in enumerate(SETTINGS if V < 30000 else SETTINGS[V % 2::3]):
        u = torch.rand((n,), generator=gen, device="cuda", dtype=torch.float64 if i % 2 else torch.float32)
        check_sample(x, u, **kw)


@pytest.mark.parametrize("V", [8, 90, 1000, 9000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_sample_edges(V, dtype):
    nan, inf = np.nan, np.inf
    flat = np.zeros(V)
    lone = np.full(V, -inf)
    lone[V // 3] = -7.0
    bad = np.random.RandomState(0).randn(V)
    bad[V - 1] = nan
    infs = np.random.RandomState(1).randn(V)
    infs[[1, V - 2]] = inf
    low = np.full(V, float(torch.finfo(DTYPES[dtype]).min))
    low[2] = 0.0
    steps = -(np.arange(V) % 5) * 1.0
    one = np.full(V, -30.0)
    one[V // 2] = 3.0
    x = put(np.array([flat, lone, bad, infs, low, steps, one, np.full(V, -inf), np.full(V, nan)]), dtype)
    n = x.shape[0]
    for u0 in (0.0, 0.37, 0.75, float(np.nextafter(np.float32(1), np.float32(0)))):
        u = torch.full((n,), u0, device="cuda")
        for kw in SETTINGS:
            check_sample(x, u, **kw)


def test_sample_per_row_settings_and_strange_numbers():
    n, V = 64, 300
    x = make(n, V, "f32", "rows", 5)
    u = torch.rand((n,), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    rs = np.random.RandomState(2)
    t = torch.from_numpy(rs.choice([0.0, 0.5, 1.0, 2.0, -1.0], n).astype(np.float32)).cuda()
    k = torch.from_numpy(rs.choice([-3, 0, 1, 7, 299, 300, 1000], n).astype(np.int32)).cuda()
    p = torch.from_numpy(rs.choice([0.0, 0.5, 0.95, 1.0, 2.0], n).astype(np.float32)).cuda()
    m = torch.from_numpy(rs.choice([-1.0, 0.0, 0.05, 1.0, 3.0], n).astype(np.float32)).cuda()
    check_sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    # numbers outside [0, 1) draw the first or the last class that stays
    out = cb.sample_classes(x[:3], torch.tensor([-1.0, float("nan"), 1.0], device="cuda"))
    assert out.cpu().tolist()[:2] == [0, 0] and 0 <= int(out[2]) < V
    nan = torch.full((n,), float("nan"), device="cuda")
    assert torch.equal(cb.sample_classes(x, u, top_p=nan, min_p=nan), cb.sample_classes(x, u))
    assert torch.equal(cb.sample_classes(x, u, temperature=nan), cb.sample_classes(x, u, temperature=0.0))


def test_sampling_frequencies_follow_the_softmax():
    # evenly spaced numbers: each class is drawn its share of them, to one draw at each border
    n, V = 20000, 23
    row = make(1, V, "f32", "rows", 11)
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n
    got = np.bincount(cb.sample_classes(row.expand(n, V), u).cpu().numpy(), minlength=V) / n
    p = torch.softmax(row.double(), 1)[0].cpu().numpy()
    assert np.abs(got - p).max() <= 1.5 / n


# ---- many rows -------------------------------------------------------------------------
# Rows of some hundred classes are worked on by a warp each where there are many of them, and wide rows
# by fewer blocks each: every operator on whole batches, compared on some of the rows.

MANY = [(1300, 129, "f32", "rows"), (1201, 300, "bf16", "offset"), (1185, 512, "f16", "rows"),
        (1190, 257, "f64", "dims"), (1250, 64, "f32", "strided"), (1250, 513, "bf16", "rows"),
        (1200, 700, "f32", "offset"), (1190, 1024, "f64", "rows"), (1184, 1023, "f16", "dims"),
        (200, 40007, "bf16", "rows"), (180, 33000, "f32", "offset"), (160, 20000, "f64", "rows")]


def some(n):
    return sorted({0, 1, n // 3, n // 2, n - 2, n - 1})


@pytest.mark.parametrize("n,V,dtype,layout", MANY)
def test_many_rows(n, V, dtype, layout):
    x = make(n, V, dtype, layout, V)
    wide = torch.float64 if dtype == "f64" else torch.float32
    at = torch.tensor(some(n), device="cuda")
    host_x = x.index_select(0, at)
    for k in (5, 40):
        top = cb.top_logits(x, k)
        for j, r in enumerate(some(n)):
            wi, wv, wt = ref.top(host(host_x[j:j + 1])[0], k, 1.0)
            assert (top.index[r].cpu().numpy() == wi).all() and (host(top.value[r]) == wv).all()
            assert abs(float(top.tail[r]) - wt) <= 130 * unit(dtype) + 3 * unit(dtype) * abs(wt)
    t = make_teacher(n, V, 24, dtype, V + 1, True)
    w = torch.linspace(0.5, 2.0, n, device="cuda", dtype=wide)
    d = cb.distill_derivatives(x, t, weight=w, temperature=1.5)
    for j, r in enumerate(some(n)):
        wl, wd, p, q = ref.distill(host(host_x[j:j + 1])[0], t.index[r].cpu().numpy(), host(t.value[r]), float(t.tail[r]),
                                   float(w[r]), 1.5)
        rel = 2 * unit(dtype) * (3 * 40 + 4)  # reach <= 40, as in check_distill
        assert abs(float(d.loss[r]) - wl) <= 2.25 * float(w[r]) * (2 * rel + 6 * unit(dtype) * 40) + 4 * unit(dtype) * wl
        small = float(torch.finfo(x.dtype).smallest_normal) * float(torch.finfo(x.dtype).eps)
        bound = float(w[r]) * 1.5 * rel * 2 * (p + q) + rounding(dtype) * np.abs(wd) + small
        assert (np.abs(host(d.der1[r]) - wd) <= bound).all()
    u = torch.rand((n,), generator=torch.Generator("cuda").manual_seed(V), device="cuda")
    for kw in (dict(), dict(top_k=7), dict(top_p=0.8), dict(top_k=100, top_p=0.9, min_p=0.01), dict(min_p=0.2),
               dict(top_k=300, top_p=0.97, temperature=2.0), dict(temperature=0.0)):
        got = cb.sample_classes(x, u, **kw)
        full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw)
        for j, r in enumerate(some(n)):
            assert int(got[r]) == ref.sample(host(host_x[j:j + 1])[0], float(u[r]), **full), (kw, r)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,layout", [(17, "rows"), (40, "rows"), (100, "offset"), (128, "rows"), (64, "dims")])
def test_top_logits_of_very_many_rows(V, layout, dtype):
    # enough rows for a thread a row; the rows that can go wrong are among them
    n = 148 * 256 + 5
    a = np.random.RandomState(V).standard_normal((n, V)) * 3
    a[0] = 0.0
    a[1] = -np.inf
    a[2, 3:] = -np.inf
    a[3, V // 2] = np.nan
    a[4] = np.where(np.arange(V) % 2, -0.0, 0.0)
    a[5] = np.arange(V) * 0.25
    a[6] = -np.arange(V) * 0.25
    a[7] = np.arange(V) // 4 % 3
    a[8, V - 1] = np.inf
    a[9] = np.nan
    a[10, :9] = 300.0  # the rest lies far below
    x = put(a, dtype, layout)
    some_rows = torch.arange(0, 40, device="cuda")
    h = host(x.index_select(0, some_rows))
    for k in (1, 3, 4, 8):
        got = cb.top_logits(x, k, temperature=0.8)
        for r in range(40):
            wi, wv, wt = ref.top(h[r], k, 0.8)
            assert (got.index[r].cpu().numpy() == wi).all(), (r, got.index[r], wi)
            assert np.array_equal(host(got.value[r]), wv, equal_nan=True)
            t = float(got.tail[r])
            if np.isfinite(wt):
                assert abs(t - wt) <= 130 * unit(dtype) + 3 * unit(dtype) * abs(wt), (r, t, wt)
            else:
                # +inf among the rest: the difference of infinities is a NaN
                assert np.array_equal(t, wt, equal_nan=True) or wt == np.inf, (r, t, wt)
        assert torch.equal(got.index, cb.top_logits(x, k).index)
        assert cb.top_logits(x, k, tail=False).tail is None


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [17, 33, 75, 90, 100, 127, 128])
def test_top_logits_of_many_rows_in_every_layout(V, dtype):
    # rows that start on 16, 8, 4 and 2 bytes, rows by the class and with gaps; every row against a stable sort
    n, u = 148 * 64 + 7, unit(dtype)
    a = np.random.RandomState(V).standard_normal((n, V)) * 3
    a[::3] = np.round(a[::3])  # ties, also across the k-th
    a[1::50, 5:] = -np.inf
    for layout in LAYOUTS:
        x = put(a, dtype, layout)
        wide = x.double()
        value, order = torch.sort(wide, dim=1, descending=True, stable=True)
        for k in (1, 2, 4, 7, 8):
            got = cb.top_logits(x, k, temperature=0.6)
            assert torch.equal(got.index.long(), order[:, :k])
            assert torch.equal(got.value.double(), value[:, :k])
            want = torch.logsumexp(value[:, k:] / 0.6, dim=1)
            fine = torch.isfinite(want)
            assert torch.equal(got.tail[~fine].double(), want[~fine])
            # u (3 reach + 4), reach at most 40, as in check_top
            assert ((got.tail.double() - want)[fine].abs() <= u * (124 + 3 * want[fine].abs())).all()


# ---- how they are called ---------------------------------------------------------------

def batch(V, dtype="bf16", n=130):
    x = make(n, V, dtype, "rows", 1)
    t = cb.top_logits(make(n, V, dtype, "rows", 2), 8)
    return x, t, torch.rand((n,), generator=torch.Generator("cuda").manual_seed(3), device="cuda")


@pytest.mark.parametrize("V", [10, 100, 1000, 40000])
def test_same_results_again_on_another_stream_and_in_a_graph(V):
    x, t, u = batch(V)

    def call():
        d = cb.distill_derivatives(x, t, temperature=2.0)
        top = cb.top_logits(x, 6)
        return d.loss, d.der1, top.index, top.value, top.tail, cb.sample_classes(x, u, top_p=0.9, top_k=40)

    want = [v.clone() for v in call()]
    assert all(torch.equal(a, b) for a, b in zip(call(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            held = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for v in held:
        v.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    # new inputs through the same graph
    x.copy_(x.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, [v.clone() for v in call()]))


@pytest.mark.parametrize("V", [100, 3000, 40000])
def test_the_same_bits_every_time(V):
    # f64 sums show an order that changes; rows with the largest classes side by side and spread
    x = make(64, V, "f64", "rows", 9)
    x[::2, :90] += 12.0
    t = cb.top_logits(x.flip(0).contiguous(), 33)
    first = None
    for _ in range(20):
        top = cb.top_logits(x, 40)
        d = cb.distill_derivatives(x, t)
        got = (top.tail, top.index, d.loss, d.der1)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_empty_batches_and_refusals():
    x = torch.empty((0, 9), device="cuda")
    assert cb.top_logits(x, 3).index.shape == (0, 3)
    t = cb.TopLogits(torch.empty((0, 3), dtype=torch.int32, device="cuda"), torch.empty((0, 3), device="cuda"))
    assert cb.distill_derivatives(x, t).der1.shape == (0, 9)
    assert cb.sample_classes(x, torch.empty((0,), device="cuda")).shape == (0,)
    x = torch.zeros((4, 9), device="cuda")
    t = cb.TopLogits(torch.zeros((4, 3), dtype=torch.int32, device="cuda"), torch.zeros((4, 3), device="cuda"))
    u = torch.zeros((4,), device="cuda")
    big = torch.zeros((8, 9), device="cuda")
    bad = [lambda: cb.top_logits(x, 10), lambda: cb.top_logits(x, 0), lambda: cb.top_logits(x, 1, temperature=0.0),
           lambda: cb.distill_loss(x, (t.index, t.value)), lambda: cb.distill_loss(x[:3], t),
           lambda: cb.distill_loss(x, cb.TopLogits(t.index.short(), t.value)),
           lambda: cb.distill_loss(x, cb.TopLogits(t.index, t.value.cpu())),
           lambda: cb.distill_loss(x, cb.TopLogits(t.index, t.value[:, :2])),
           lambda: cb.distill_loss(x, cb.TopLogits(t.index, t.value, u.double())),
           lambda: cb.distill_loss(x, t, weight=u.double()), lambda: cb.distill_loss(x, t, weight=u[:3]),
           lambda: cb.distill_derivatives(x, t, out=x.half()), lambda: cb.distill_derivatives(x, t, out=x[:3]),
           lambda: cb.distill_derivatives(x, t, out=x[:1].expand(4, 9)),
           lambda: cb.distill_derivatives(big[:4], t, out=big[1:5]),
           lambda: cb.sample_classes(x, u.half()), lambda: cb.sample_classes(x, u[:2]),
           lambda: cb.sample_classes(x, u.cpu()), lambda: cb.sample_classes(x, u, temperature=-1.0),
           lambda: cb.sample_classes(x, u, top_p=1.1), lambda: cb.sample_classes(x, u, min_p=float("nan")),
           lambda: cb.sample_classes(x, u, top_k=-1), lambda: cb.sample_classes(x, u, top_k=u),
           lambda: cb.top_logits(torch.zeros((2, 262145), device="cuda"), 1)]
    for call in bad:
        with pytest.raises(cb.CbGpuError):
            call()


def test_rows_behind_32_bit_offsets():
    # the last rows start beyond 2^32 elements
    n, V = 3, 2000
    store = torch.empty(((1 << 32) + 4096,), dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(store, (n, V), (1 << 31, 1))
    y = make(n, V, "bf16", "rows", 4)
    x.copy_(y)
    t = make_teacher(n, V, 8, "bf16", 5, True)
    u = torch.rand((n,), device="cuda")
    assert torch.equal(cb.distill_derivatives(x, t, out=x.clone()).der1, cb.distill_derivatives(y, t).der1)
    assert torch.equal(cb.top_logits(x, 9).index, cb.top_logits(y, 9).index)
    assert torch.equal(cb.sample_classes(x, u), cb.sample_classes(y, u))
    want = cb.distill_derivatives(y, t).der1
    assert torch.equal(cb.distill_derivatives(x, t, out=x).der1, want)


def test_from_a_teachers_rows_to_drawn_labels():
    """The operators as they are used together: a teacher's rows are reduced to their top logits, a
    student's rows follow der1 towards them, labels are drawn from the student."""
    n, V = 500, 3000
    teacher = make(n, V, "f32", "rows", 21, spread=1.0)
    top = cb.top_logits(teacher, 32)
    student = torch.zeros((n, V), device="cuda")
    buf = torch.empty_like(student)
    # at the teacher's own logits the loss is 0 and der1 vanishes, to rounding
    at = cb.distill_derivatives(teacher, top)
    assert float(at.loss.abs().max()) < 1e-5 and float(at.der1.abs().max()) < 1e-5
    for _ in range(3):
        before = student.clone()
        d = cb.distill_derivatives(student, top, out=buf)
        student += 5.0 * d.der1
        # the step is uphill in -loss: the loss' derivative along it is -|der1|^2 < 0
        eps = 1e-2
        moved = cb.distill_loss(before + eps * d.der1, top)
        assert bool((moved < d.loss).all())
    u = torch.rand((n,), generator=torch.Generator("cuda").manual_seed(5), device="cuda")
    labels = cb.sample_classes(student, u, top_k=8)
    best = cb.top_logits(student, 8).index
    assert bool((best == labels[:, None]).any(dim=1).all())


# ---- a booster trained on a teacher ------------------------------------------------------

def columns(n, F, seed):
    from oracle import oracle
    rs = np.random.RandomState(seed)
    X = rs.standard_normal((n, F)).astype(np.float32)
    return X, [oracle.select_borders(X[:, f], 32) for f in range(F)], rs


def fit(X, borders, K, **kw):
    fp = cb.FitParams(loss="MultiClass", depth=4, iterations=4, learning_rate=0.2, l2_leaf_reg=3.0,
                      boost_from_average=False, bootstrap_type=kw.pop("boot", "No"), random_seed=3)
    return cb.fit_multiclass([X[:, f].copy() for f in range(X.shape[1])], borders, kw.pop("y", None), K, fp,
                             staged=True, **kw)


def same_trees(a, b, scale=1.0):
    np.testing.assert_array_equal(a.split_feature, b.split_feature)
    np.testing.assert_array_equal(a.split_bin, b.split_bin)
    # sums of n values rounded to 2^-40 of their largest, and a Newton solve: the bar of the suite
    assert np.abs(a.leaf_values - scale * b.leaf_values).max() <= 1e-9 * scale
    assert np.abs(a.staged - scale * b.staged).max() <= 1e-9 * scale


@pytest.mark.parametrize("boot", ["No", "Bernoulli"])
def test_fit_on_a_teacher_that_is_sure_is_a_fit_on_labels(boot):
    n, F, K = 6000, 6, 5
    X, borders, rs = columns(n, F, 1)
    y = rs.randint(0, K, n)
    y[X[:, 0] > 0.3] = 2
    w = rs.uniform(0.5, 2.0, n)
    want = fit(X, borders, K, y=y, weights=w, boot=boot)
    top = cb.TopLogits(y[:, None].astype(np.int32), np.zeros((n, 1)))
    same_trees(fit(X, borders, K, teacher=top, weights=w, boot=boot), want)


def test_fit_on_a_teacher_is_a_weighted_fit_on_every_class():
    # soft targets q_c: the oracle's fit on every row once a class, weighted by q_c
    from oracle import oracle
    n, F, K = 3000, 5, 4
    X, borders, rs = columns(n, F, 2)
    z = 2.0 * np.nan_to_num(X[:, :K]) + 0.3 * rs.standard_normal((n, K))
    q = np.exp(z - z.max(1, keepdims=True))
    q /= q.sum(1, keepdims=True)
    top = cb.top_logits(torch.from_numpy(z).cuda(), K)
    got = fit(X, borders, K, teacher=top)
    bins = oracle.quantize(X.T.copy(), borders)
    # l2 is scaled by the mean weight: 1 / K over the expanded rows
    o = oracle.train_multiclass(np.repeat(bins, K, axis=1), [len(b) for b in borders],
                                np.tile(np.arange(K, dtype=np.int32), n), K, depth=4, iterations=4, learning_rate=0.2,
                                l2_leaf_reg=3.0 * K, bootstrap_type="No", random_seed=3, weights=q.reshape(-1))
    np.testing.assert_array_equal(got.split_feature, o.split_feature)
    np.testing.assert_array_equal(got.split_bin, o.split_bin)
    assert np.abs(got.leaf_values - o.leaf_values).max() <= 1e-9
    # the tail's bucket of one class is that class
    part = cb.top_logits(torch.from_numpy(z).cuda(), K - 1)
    same_trees(fit(X, borders, K, teacher=part), got)
    # temperature: probabilities of z / 2, leaves twice as large
    half = cb.TopLogits(top.index, top.value / 2.0)
    same_trees(fit(X, borders, K, teacher=cb.TopLogits(top.index, top.value), temperature=2.0),
               fit(X, borders, K, teacher=half), 2.0)
    # the loss of the staged approximants, as the device's own dim-major rows, against the definition
    rows = torch.from_numpy(np.ascontiguousarray(got.staged[-1].T)).cuda().t()
    check_distill(rows, cb.TopLogits(top.index, top.value), None, 1.0, "f64")
    labels = cb.sample_classes(rows, torch.rand((n,), device="cuda"), top_k=2)
    assert bool((cb.top_logits(rows, 2).index == labels[:, None]).any(dim=1).all())


def test_teacher_refusals():
    n, K = 50, 3
    X, borders, rs = columns(n, 3, 3)
    y = rs.randint(0, K, n)
    top = cb.TopLogits(y[:, None], np.zeros((n, 1)))
    with pytest.raises(ValueError):
        fit(X, borders, K, y=y, teacher=top)
    with pytest.raises(ValueError):
        fit(X, borders, K)
    with pytest.raises(RuntimeError, match="MultiClass"):
        fit(X, borders, K, teacher=top, loss="MultiClassOneVsAll")
    for bad in (cb.TopLogits(np.full((n, 1), K), np.zeros((n, 1))), cb.TopLogits(np.full((n, 1), -2), np.zeros((n, 1))),
                cb.TopLogits(y[:, None], np.full((n, 1), np.nan)), cb.TopLogits(y[:, None], np.full((n, 1), np.inf)),
                cb.TopLogits(y[:, None], np.zeros((n, 1)), np.full(n, np.nan)),
                cb.TopLogits(y[:, None], np.zeros((n, 2))), cb.TopLogits(y[:9, None], np.zeros((9, 1))),
                cb.TopLogits(y[:, None], np.zeros((n, 1)), np.zeros(n - 1)),
                cb.TopLogits(np.zeros((n, 257), dtype=np.int32), np.zeros((n, 257)))):
        with pytest.raises(cb.CbGpuError):
            fit(X, borders, K, teacher=bad)
    for t in (0.0, float("nan"), 1e4):
        with pytest.raises(cb.CbGpuError):
            fit(X, borders, K, teacher=top, temperature=t)
    # a session's turn of calls: no teacher after the first tree, no target with a teacher
    cfg = cb.DeviceTrainConfig()
    for first in ("teacher", "target"):
        rt = cb.B200MultiRuntime()
        assert rt.begin_device_training_raw("MultiClass", 2, True, 1, "Cosine", [X[:, f].copy() for f in range(3)],
                                            borders, None, n, 3, 33, 0.1, 3.0, cfg, approx_dim=K)
        grow = lambda t: rt.grow_tree_on_device(None, t, [], family=("MultiOutput", None, K),  # noqa: E731
                                                leaf_of_bytes=0, resident_approx=True)
        if first == "teacher":
            assert rt.set_teacher(top.index, top.value)
            with pytest.raises(cb.CbGpuError, match="no target"):
                grow(y)
            assert len(grow(None).splits) == 2
        else:
            with pytest.raises(cb.CbGpuError, match="first call needs the target"):
                grow(None)
            grow(y)
            with pytest.raises(cb.CbGpuError, match="target already"):
                rt.set_teacher(top.index, top.value)
        rt.end_device_training()
    with pytest.raises(cb.CbGpuError, match="no session"):
        cb.B200MultiRuntime().set_teacher(top.index, top.value)
