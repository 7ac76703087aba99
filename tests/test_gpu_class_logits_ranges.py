"""Class-logit operators at the ends of their ranges: finite masks, very small and very large
temperatures, parts of a row that weigh nothing, against the plain 64-bit forms.

Tolerances.  u is the unit roundoff (2^-24 for 16- and 32-bit logits, 2^-53 for f64).  An exponential's
argument is a difference that is rounded, times a scale that is rounded, rounded again: off by at most 3u times
its size r, which in a sum counts up to 40 (behind it the exponential is below u).  With 2 ulp of its own an
exponential is off by 3u r + 4u of itself, a sum by 124 u, a probability by u (3 r + 128), REL = 2 u 124 for those
that count beside 1; one far below is small, but as a share of itself off by its own r (up to 800, where it is 0 in
64 bits), and der1 of a class below shows it.  The 64-bit forms run on long doubles for f64 rows: their differences
of large logits keep the bits that the device's 64-bit differences keep.  A loss holds two logarithms of
sums (2 REL), the scaled differences that it adds up, whose rounding is 3u of their size each, and the q that
it weighs its terms with, each off by REL of itself: REL sum q |ln q / p|, of which the negative terms are
at most sum p (1 / e) in all, so it is at most REL (loss / T^2 + 2 / e) T^2.  Results that are below 2^-126 of
their unit are 0 in f32; numbers above the largest of a type are its infinity.
"""
from fractions import Fraction

import numpy as np
import pytest

import catboost_rs_b200 as cb
from tests import logits_reference as ref
from tests import test_gpu_class_logits as base

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DTYPES = base.DTYPES


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def teacher_of(index, value, tail, dtype):
    wide = torch.float64 if dtype == "f64" else torch.float32
    return cb.TopLogits(torch.tensor(np.asarray(index), dtype=torch.int32, device="cuda"),
                        torch.tensor(np.asarray(value, dtype=np.float64), dtype=DTYPES[dtype], device="cuda"),
                        None if tail is None else torch.tensor(np.asarray(tail, dtype=np.float64), dtype=wide, device="cuda"))


def check(x, teacher, T, dtype, out=None, lost=0.0):
    """Loss and derivatives against the definition, taken on rows from which their largest logit was
    subtracted first (so that the 64-bit form keeps its bits when the logits are large beside T)."""
    u, rel = base.unit(dtype), 2 * base.unit(dtype) * 124
    a, idx, val = base.host(x), teacher.index.cpu().numpy(), base.host(teacher.value)
    tail = np.full(len(a), -np.inf) if teacher.tail is None else base.host(teacher.tail)
    alone = base.host(cb.distill_loss(x, teacher, temperature=T))
    got = cb.distill_derivatives(x, teacher, temperature=T, out=out)
    loss, der1 = base.host(got.loss), base.host(got.der1)
    low = 0.0 if dtype == "f64" else 2.0 ** -126
    small = float(torch.finfo(x.dtype).smallest_normal) * float(torch.finfo(x.dtype).eps)
    wide = torch.finfo(torch.float64 if dtype == "f64" else torch.float32)
    real = np.longdouble if dtype == "f64" else np.float64
    for r in range(len(a)):
        row = a[r].astype(real) - max(a[r].max(), np.finfo(np.float64).min)
        z = val[r].astype(real)
        valid = (idx[r] >= 0) & (idx[r] < x.shape[1])
        top = z[valid].max() if valid.any() and z[valid].max() > -np.inf else 0.0
        # (tail T - z) / T exactly: the product has at most 106 bits
        beside_top = real(tail[r])
        if np.isfinite(tail[r]):
            exact = (Fraction(float(tail[r])) * Fraction(T) - Fraction(float(top))) / Fraction(T)
            most = Fraction(np.finfo(np.float64).max)
            beside_top = real(float(max(-most, min(most, exact))))
        wl, wd, p, q = ref.distill(row, idx[r], z - top, beside_top, 1.0, real(T))
        wl, wd = float(wl), wd.astype(np.float64)
        scaled = np.concatenate([[0.0], row[idx[r][valid]], (z - top)[valid]]) / T
        size = np.abs(scaled[np.isfinite(scaled)]).max()
        for g in (loss[r], alone[r]):
            if abs(wl) > float(wide.max):
                assert g == wl or np.isinf(g), (r, g, wl)
            elif np.isfinite(wl):
                assert abs(g - wl) <= T * T * (3 * rel + 6 * u * size) + (rel + 4 * u) * abs(wl) + float(wide.tiny), (r, g, wl)
            else:
                assert np.array_equal(g, wl, equal_nan=True), (r, g, wl)
        own = np.maximum(rel, u * (3 * np.minimum(-row / T, 800.0) + 128))
        bound = T * own * 2 * (p + q) + base.rounding(dtype) * np.abs(wd) + small + 2 * T * max(low, lost)
        beyond = np.abs(wd) + bound > float(torch.finfo(x.dtype).max)
        assert (np.isfinite(der1[r]) | beyond | np.isnan(wd)).all() and (der1[r] * np.sign(wd) >= 0)[beyond].all()
        off = np.where(beyond, 0.0, np.abs(der1[r] - wd) - bound)
        assert np.isnan(wd).any() or off.max() <= 0, (r, int(off.argmax()), der1[r][off.argmax()], wd[off.argmax()])
        assert np.isnan(der1[r]).all() or not np.isnan(wd).any()
    return got


# ---- finite masks ---------------------------------------------------------------------------------

MASKS = [("f64", -1e10), ("f64", -1e20), ("f64", -1e300), ("f32", -1e9), ("f32", -1e10), ("f32", -1e20), ("f32", -1e30),
         ("bf16", -1e10), ("bf16", -1e20), ("f16", -65504.0)]


@pytest.mark.parametrize("V", [14, 400, 513, 900, 6000, 40000, 131072])
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_distill_under_finite_masks(V, dtype, mask):
    rs = np.random.RandomState(V)
    a = rs.standard_normal((6, V)) * 2
    at = np.stack([rs.permutation(V // 2)[:5] + V // 2 for _ in a])  # the teacher's classes: in the second half
    a[0, :V // 2] = mask                                 # a part of the row, whole blocks of it
    keep = a[1, at[1]].copy()
    a[1] = mask                                          # all but the teacher's classes
    a[1, at[1]] = keep
    a[2] = mask                                          # all of them
    a[3, V // 2:] = mask                                 # the teacher's classes among them
    a[4, at[4]] += 30.0
    a[4, :V // 2] = mask
    z = rs.standard_normal((6, 5))
    for T in (1.0, 0.5, 2.0):
        for tail in (rs.uniform(-1, 2, 6), None):
            x, t = base.put(a, dtype), teacher_of(at, z, tail, dtype)
            got = check(x, t, T, dtype)
            assert not torch.isnan(got.loss).any() and not torch.isnan(got.der1).any()
            check(x, t, T, dtype, out=x)


@pytest.mark.parametrize("V", [14, 100, 400, 513, 900, 6000, 40000, 131072])
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_top_logits_under_finite_masks(V, dtype, mask):
    rs = np.random.RandomState(V)
    a = rs.standard_normal((5, V)) * 2
    for r, left in enumerate((3, 5, 7, 0)):  # unmasked classes
        masked = np.ones(V, dtype=bool)
        masked[rs.permutation(V)[:left]] = False
        a[r, masked] = mask
    a[4, :V // 2] = mask
    x = base.put(a, dtype)
    for T in (1.0, 0.5, 2.0):
        base.check_top(x, 5, T, dtype)


# ---- the ends of the temperature's range --------------------------------------------------------------

@pytest.mark.parametrize("V", [14, 100, 400, 513, 900, 6000, 40000])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,spread", [(1e-6, 1.0), (1e-6, 3000.0), (1e-6, 1e-6), (1e-3, 300.0), (1e6, 3.0), (1e6, 30000.0)])
def test_ends_of_the_temperature(V, dtype, T, spread):
    n = 3
    x = base.put(np.clip(np.random.RandomState(V).standard_normal((n, V)) * spread, -6e4, 6e4), dtype)
    base.check_top(x, 5, T, dtype)
    rs = np.random.RandomState(V + 1)  # a teacher whose logits are of the size of T
    at, z = np.stack([rs.permutation(V)[:5] for _ in range(n)]), rs.standard_normal((n, 5)) * min(T, 100.0)
    check(x, teacher_of(at, z, None, dtype), T, dtype)


# ---- teachers' logits that are large beside the temperature -----------------------------------------------

@pytest.mark.parametrize("V", [14, 100, 400, 513, 900, 6000, 40000])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,spread", [(1e-6, 1.0), (1e-6, 3000.0), (1e-3, 300.0), (0.3, 20000.0), (1.0, 60000.0), (1e6, 30000.0)])
def test_teachers_logits_large_beside_the_temperature(V, dtype, T, spread):
    x = base.put(np.random.RandomState(V).standard_normal((3, V)) * T, dtype)
    # (within the 16-bit type's range)
    y = base.put(np.clip(np.random.RandomState(V + 1).standard_normal((3, V)) * spread, -6e4, 6e4), dtype)
    y[:, V // 2] = y[:, 0] = y.max()  # several of much the same weight
    t = cb.top_logits(y, 5, temperature=T)
    check(x, t, T, dtype)
    check(x, cb.TopLogits(t.index, t.value), T, dtype)
    # the same by the logits of the teacher as they are: its entries lie where the tail puts them
    check(y, t, T, dtype)


@pytest.mark.parametrize("V", [14, 100, 400, 513, 900, 6000, 40000])
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_teachers_under_finite_masks(V, dtype, mask):
    # entries of a teacher's masked classes: a few, all of them beside a tail, all without one (they share it)
    rs = np.random.RandomState(V)
    x = base.put(rs.standard_normal((4, V)), dtype)
    at = np.stack([rs.permutation(V)[:5] for _ in range(4)])
    z = rs.standard_normal((4, 5))
    z[0, 3:], z[1] = mask, mask
    z[2] = float(torch.finfo(DTYPES[dtype]).min)
    for T in (1.0, 0.5, 2.0, 0.7):
        for tail in (None, np.array([0.3, 0.1, -0.5, 1.0]), np.array([0.3, mask / T, 0.3, 0.3])):
            t = teacher_of(at, z, tail, dtype)
            got = check(x, t, T, dtype)
            assert torch.isfinite(got.loss).all() and torch.isfinite(got.der1).all()
    # the teacher's top logits of rows that are masked but for some
    a = rs.standard_normal((4, V))
    for r, left in enumerate((3, 5, 0, V // 2)):
        masked = np.ones(V, dtype=bool)
        masked[rs.permutation(V)[:left]] = False
        a[r, masked] = mask
    t = cb.top_logits(base.put(a, dtype), 5)
    got = check(x, t, 1.0, dtype)
    assert torch.isfinite(got.loss).all() and torch.isfinite(got.der1).all()


# ---- parts of a row that weigh nothing ------------------------------------------------------------------

@pytest.mark.parametrize("V", [10, 14, 60, 400, 900, 6000, 40000, 131072])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T", [0.1, 1.0])
def test_distill_others_far_below_without_a_tail(V, dtype, T):
    # the others lie so far below the entries that their exponentials beside them are 0, and yet far above 0
    # (88.7 T is where a 32-bit exponential of the logit itself ends, 709 T a 64-bit one), in the whole row or
    # in one part of it while another part lies lower still
    rs = np.random.RandomState(V)
    a = rs.standard_normal((6, V)) * T
    at = np.stack([rs.permutation(V // 2)[:5] for _ in a])  # in the first half
    for r, (entries, others) in enumerate(((200, 100), (2000, 1000), (40000, 20000), (300, 0), (-100, -200), (120, 5))):
        a[r] += others * T
        a[r, at[r]] += (entries - others) * T
    a[3, :V // 2] += 150 * T     # the others of the entries' half of the row far above those of the other half
    a[5, V // 2:] += 90 * T      # and below them
    z = rs.standard_normal((6, 5)) * T
    for tail in (None, np.full(6, -np.inf), rs.uniform(-1, 2, 6)):
        x, t = base.put(a, dtype), teacher_of(at, z, tail, dtype)
        got = check(x, t, T, dtype)
        assert not torch.isnan(got.der1).any() and not torch.isnan(got.loss).any()
        check(x, t, T, dtype, out=x)


@pytest.mark.parametrize("V", [10, 14, 60, 400, 900, 6000, 40000, 131072])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T", [0.1, 1.0])
def test_distill_entries_of_no_weight_in_rows_far_below_0(V, dtype, T):
    # a part of the row whose entries the teacher rules out (-inf), or whose classes the student masks (-inf), has no
    # maximum of its own: beside maxima of -200 T (-1500 T in 64 bits) nothing may be taken relative to 0
    rs = np.random.RandomState(V)
    a = rs.standard_normal((5, V)) * T - 200 * T
    at = np.concatenate([np.stack([rs.permutation(V // 2)[:3] for _ in a]),
                         np.stack([rs.permutation(V // 2)[:2] + V // 2 for _ in a])], axis=1)
    z = rs.standard_normal((5, 5)) * T - 200 * T
    z[0, :3] = -np.inf                       # the entries of the first half
    a[1, :V // 2], z[1, :3] = -np.inf, -np.inf   # and the student masks that half
    a[2, :V // 2] = -np.inf                  # the student alone: loss +inf, der1 finite
    z[3, :4] = -np.inf
    a[4, V // 2:], z[4, 3:] = -np.inf, -np.inf
    lower = 1300 * T if dtype == "f64" else 0.0
    for tail in (None, rs.uniform(-1, 2, 5) - 200 - lower / T):
        x, t = base.put(a - lower, dtype), teacher_of(at, z - lower, tail, dtype)
        got = check(x, t, T, dtype)
        assert not torch.isnan(got.der1).any() and not torch.isnan(got.loss).any()
        assert torch.isinf(got.loss).tolist() == [False, False, True, False, False]
        check(x, t, T, dtype, out=x)


@pytest.mark.parametrize("V", [6, 60, 400, 900, 6000, 40000])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_teacher_without_an_entry_gives_0_whatever_the_row_holds(V, dtype):
    a = np.random.RandomState(V).standard_normal((6, V))
    a[0, V // 2], a[1, 0], a[2, V - 1], a[3, 1] = np.nan, np.inf, np.nan, -np.inf
    a[4] = np.nan
    index, value = np.full((6, 3), -1), np.zeros((6, 3))
    for tail in (None, np.full(6, -np.inf)):
        for i, z in ((index, value), (np.tile([0, 1, 2], (6, 1)), np.full((6, 3), -np.inf))):
            for layout in base.LAYOUTS:
                x, t = base.put(a, dtype, layout), teacher_of(i, z, tail, dtype)
                for out in (None, x):
                    got = cb.distill_derivatives(x, t, out=out)
                    assert (got.loss == 0).all() and (got.der1 == 0).all()


# ---- draws ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("V", [14, 30, 100, 400, 513, 1000, 5000])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T", [1e4, 1e6])
def test_cuts_of_masked_rows_at_large_temperatures(V, dtype, T):
    # many distinct logits of nearly the same weight, some classes masked: cuts in the middle of them, by count
    # and by mass, with classes by index in no order
    n = 40
    a = np.random.RandomState(V).standard_normal((n, V)) * 1000.0
    a[::2, ::3] = -np.inf
    a[1::4, 5] = float(torch.finfo(DTYPES[dtype]).min)
    x = base.put(a, dtype)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    for kw in (dict(top_k=max(2, V // 5)), dict(top_p=0.5), dict(top_k=20, top_p=0.5), dict(top_k=9), dict(top_p=0.05)):
        base.check_sample(x, u, temperature=T, **kw)


@pytest.mark.parametrize("V", [14, 100, 700, 1500, 5000, 140000])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16"])
def test_draws_at_temperatures_next_to_0(V, dtype):
    # row temperatures down to the smallest f32: what is below the largest logit weighs nothing, equal ones
    # share, and are cut by index
    T = [1e-3, 1e-20, 1e-36, 1e-37, 1e-38, 1.4e-45][::1 if V < 10000 else 2]
    rs = np.random.RandomState(V)
    a = np.floor(rs.uniform(0, 3, (2 * len(T), V)))  # a third of the classes each
    a[1::4] = 1.0
    x = base.put(a, dtype)
    t = torch.tensor(np.repeat(T, 2), dtype=torch.float32, device="cuda")
    for u0 in (0.1, 0.9)[:2 if V < 10000 else 1]:
        u = torch.full((len(a),), u0, device="cuda")
        for kw in (dict(), dict(top_k=3), dict(top_k=max(2, min(V // 4, 300))), dict(top_p=0.5), dict(top_k=min(V, 400), top_p=0.5),
                   dict(min_p=0.3)):
            base.check_sample(x, u, temperature=t, **kw)
    # logits that are such numbers themselves: a spread of 1e-38
    x = base.put(rs.uniform(-1e-38, 0, (3, V)), "f32" if dtype == "bf16" else dtype)
    u = torch.rand((3,), generator=torch.Generator("cuda").manual_seed(V), device="cuda")
    for kw in (dict(top_k=min(V, 300)), dict(top_p=0.5), dict(top_k=min(V, 400), top_p=0.5)):
        base.check_sample(x, u, **kw)


@pytest.mark.parametrize("V", [2, 3, 10, 16, 30, 100, 500])
@pytest.mark.parametrize("layout", ["rows", "dims"])
def test_numbers_next_to_a_border(V, layout):
    # a weight of V <= 512 classes is a multiple of 2^-52, off by half of it for its rounding; the exponential's
    # argument by 3 roundings (3 |x| e^x <= 1.2 of 2^-53) and its table and polynomial by 2 ulp at most (2 of
    # 2^-52): below 4 2^-52 in all, so a border moves by less than 8 V 2^-52 of the mass (border and mass).  What is
    # drawn beside it is what the definition draws.
    n = 64
    rs = np.random.RandomState(V)
    x = base.put(rs.standard_normal((n, V)) * 2, "f64", layout)
    a = base.host(x)
    share = np.exp((a - a.max(1, keepdims=True)).astype(np.longdouble))
    upto = np.cumsum(share, axis=1) / share.sum(1, keepdims=True)
    at = rs.randint(0, V - 1, n)
    for side in (-1, 1):
        u = (upto[np.arange(n), at] + side * (8 * V * 2.0 ** -52 + 2.0 ** -53)).astype(np.float64)
        got = cb.sample_classes(x, torch.from_numpy(u).cuda()).cpu().numpy()
        want = np.array([np.searchsorted(upto[r], u[r], side="right") for r in range(n)])
        assert (got == want).all(), (side, int((got != want).sum()))


@pytest.mark.parametrize("V", [6, 10, 16, 30, 100, 200, 400, 900, 6000, 40000])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("n", [4, 400])
def test_weights_below_32_bits_on_masked_classes(V, dtype, n):
    # a class that the student masks and the teacher does not gives +inf however little the teacher gives it (down
    # to e^-745, where it is 0 in 64 bits too), an entry as well as all others beside a tail
    rs = np.random.RandomState(V)
    below = [20.0, 80.0, 90.0, 150.0, 600.0, 900.0]
    a = rs.standard_normal((2 * len(below), V))
    index, value, tail = np.tile([0, 1, 2], (len(a), 1)), np.zeros((len(a), 3)), np.full(len(a), -np.inf)
    for r, d in enumerate(below):
        a[r, 1], value[r, 1] = -np.inf, -d
        a[len(below) + r, 3:], tail[len(below) + r] = -np.inf, -d
    want = np.array([d < 745 for d in below] * 2)
    at = np.arange(max(n, len(a))) % len(a)
    got = cb.distill_derivatives(base.put(a[at], dtype), teacher_of(index[at], value[at], tail[at], dtype))
    loss = base.host(got.loss)
    assert (loss[want[at]] == np.inf).all() and np.isfinite(loss[~want[at]]).all()
    assert torch.isfinite(got.der1).all()
    assert torch.equal(got.loss, cb.distill_loss(base.put(a[at], dtype), teacher_of(index[at], value[at], tail[at], dtype)))


@pytest.mark.parametrize("V", [10, 16, 30, 100, 200, 400, 900, 6000, 40000])
@pytest.mark.parametrize("dtype,far", [("f64", -1e10), ("f64", -1e200), ("f32", -300.0), ("f32", -1e10), ("f32", -1e38),
                                       ("bf16", -1e30), ("f16", -6e4)])
@pytest.mark.parametrize("n", [16, 400])
def test_weights_below_32_bits_on_classes_far_below(V, dtype, far, n):
    # as much below as the weight is small: their product is the loss, finite, of an entry and of all others
    rs = np.random.RandomState(V)
    below = [20.0, 80.0, 90.0, 150.0, 600.0, 700.0]
    a = rs.standard_normal((2 * len(below), V))
    index, value, tail = np.tile([0, 1, 2], (len(a), 1)), np.zeros((len(a), 3)), np.full(len(a), -np.inf)
    for r, d in enumerate(below):
        a[r, 1], value[r, 1] = far, -d
        a[len(below) + r, 3:], tail[len(below) + r] = far, -d
    at = np.arange(n) % len(a)
    x, t = base.put(a[at], dtype), teacher_of(index[at], value[at], tail[at], dtype)
    loss = cb.distill_loss(x, t)
    same = torch.from_numpy(at).cuda() if n > len(a) else None
    few = cb.TopLogits(*(v[:len(a)] for v in (t.index, t.value, t.tail)))
    lost = 0.0 if dtype == "f64" else 2.0 ** -126 * 1e20  # der1 beside a tail, as in test_distill_others_far_below
    got = check(x[:len(a)].contiguous(), few, 1.0, dtype, lost=lost)
    assert torch.isfinite(got.loss).all()
    if same is not None:  # both kernels are within the bound of check
        off = (loss.double() - got.loss.double()[same]).abs()
        u = base.unit(dtype)
        size = -far + 1000.0
        assert (off <= 2 * (3 * 248 * u + 252 * u * loss.double().abs() + 6 * u * size * (size < 1e6))).all()
