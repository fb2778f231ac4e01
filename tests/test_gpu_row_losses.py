"""The losses on rows of scores against their definitions in 64 bits and more (oracle/row_losses.py).

Tolerances.  A gradient entry is rounded to the scores' type once (half a step, eps / 2 relative, or half the smallest subnormal).
Before that it is computed in Float32 (Float64 for Float64 scores), u = 2^-24 (2^-53): an exponential exp2((x - m) c) is off by
(3 |x - m| c ln 2 + 3) u -- the difference, the constant, the product, the function --, the sum of a row by at most the same of its
largest terms and its tree of additions, and a listed entry subtracts a teacher's probability exp(l) that is off by (4 |l| + 8) u.
The oracle adds these up per entry (`size`: every term times 64 + 6 |x - m| c, or 64 + 4 |l|), the tests allow size * u.

The hardware's Float32 exponential gives 0 for results below 2^-126.  An entry is a coefficient times such an exponential, of a score
against one of the row's that is at most an exponent of 20 below the largest; where listed and other classes have references of
their own, the coefficient holds the exponential of their distance.  So at most exp(20) * 2^-126 < 2^-97 of the largest score's entry is
lost, whose `size` is 64 of it or more, hence max(size of the row) / 64 * 2^-97.  Where the coefficient is in the
exponent (the two-byte types) the loss is 2^-97 itself."""
import numpy as np
import pytest
import torch

from oracle import row_losses as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}


def pa():
    import proximalalgorithms.jl_amd as m

    return m


def flushed(size):
    return 2.0**-97 * np.maximum(1.0, size.max(axis=1, keepdims=True, initial=0.0) / 64)


def check(got, value, want, dtype):
    """gradient and value against the oracle's (f, grad, size, f_size)"""
    f, grad, size, f_size = want
    u = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    fin = torch.finfo(dtype)
    g = got.double().cpu().numpy()
    assert g.shape == grad.shape
    assert np.array_equal(np.isnan(g), np.isnan(grad))
    tol = np.abs(grad) * (fin.eps / 2) + size * u * 1.01 + fin.smallest_normal * fin.eps / 2
    if dtype != torch.float64:
        tol = tol + flushed(size)
    bad = np.abs(g - grad) > tol
    assert not bad.any(), (int(bad.sum()), g[bad][:5], grad[bad][:5], np.argwhere(bad)[:5])
    if np.isnan(f):
        assert np.isnan(value)
    elif np.isinf(f):
        assert value == f
    else:
        assert abs(value - f) <= f_size * u + abs(f) * (2.0**-24 if u > 1e-10 else u * 4) + 1e-300, (value, f, f_size)


def teacher(rng, n, v, k, absent=0.0, twice=False):
    idx = np.stack([rng.permutation(v)[:k] if k else np.zeros(0, int) for _ in range(n)]) if n else np.zeros((0, k), int)
    t = np.sort(rng.normal(size=(n, k)) * 2 + 6, axis=1)[:, ::-1].copy()
    if absent:
        idx[rng.random(idx.shape) < absent] = -1
    if twice and k > 2:
        idx[:, k // 2] = idx[:, 0]
        idx[:, -1] = idx[:, 0]
    return t, idx


def scores(rng, n, v, dtype, idx=None, t=None, gap=0, shift=0):
    """device scores (rows `gap` apart, first one `shift` elements into its buffer) and their exact values"""
    x = rng.normal(size=(n, v)) * 2
    if idx is not None and idx.size:
        for i in range(n):
            on = idx[i] >= 0
            x[i, idx[i][on]] = t[i][on] * 0.9 + rng.normal(size=on.sum())
    buf = torch.full((shift + n * (v + gap),), float("nan"), dtype=dtype, device="cuda")
    out = buf[shift:].view(n, v + gap)[:, :v]
    out.copy_(torch.from_numpy(x))
    return out, out.double().cpu().numpy()


def tdev(t, dtype):
    d = torch.from_numpy(t).to(dtype).cuda()
    return d, d.double().cpu().numpy()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 64, 1), (33, 100, 100), (7, 513, 20), (4, 1003, 5), (3, 4097, 64),
                                   (2, 20011, 300), (1, 50001, 20), (300, 31, 4)])
def test_distillation_sizes(dtype, n, v, k):
    rng = np.random.default_rng(n * 1000 + v)
    t, idx = teacher(rng, n, v, k)
    td, te = tdev(t, DT[dtype])
    x, xe = scores(rng, n, v, DT[dtype], idx, t)
    f = pa().DistillationLoss(td, torch.from_numpy(idx).int().cuda(), v, temperature=1.5, lam=2.25)
    val, g = f.value_and_gradient(x)
    check(g, val, ref.distillation(xe, te, idx, temperature=1.5, lam=2.25), DT[dtype])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("temperature", [1.0, 2.0, 0.25])
@pytest.mark.parametrize("rest,labelled", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("n,v,k,gap,shift", [(5, 300, 9, 0, 0), (4, 4101, 40, 3, 1), (9, 37, 37, 5, 3), (2, 70001, 130, 0, 5)])
def test_distillation_terms(dtype, temperature, rest, labelled, n, v, k, gap, shift):
    """the outside class, labels in and out of the list, absent and doubled entries, weights with zeros, strides, int64 and int32"""
    rng = np.random.default_rng(v + int(temperature * 8))
    t, idx = teacher(rng, n, v, k, absent=0.2 if k < v else 0.0, twice=k < v)
    td, te = tdev(t, DT[dtype])
    x, xe = scores(rng, n, v, DT[dtype], idx, t, gap, shift)
    lse = None
    if rest:
        with np.errstate(divide="ignore"):
            mass = np.where(idx >= 0, np.exp(te / temperature), 0).sum(1)
        lse = np.log(mass + 1e-30) + rng.random(n) * 0.5
        lse = torch.from_numpy(lse).to(torch.float64 if dtype == "f64" else torch.float32)
    w = rng.random(n).astype(np.float32)
    w[0] = 0.0
    x[0] = float("nan")  # a row of weight 0 is not looked at
    xe[0] = 0.0
    y = rng.integers(0, v, n)
    y[1] = -1
    y[2 % n] = max(idx[2 % n][0], 0)  # a label that is listed
    kw = dict(temperature=temperature, lam=0.7)
    dev = dict(kw, teacher_lse=None if lse is None else lse.cuda(), weights=torch.from_numpy(w).cuda())
    host = dict(kw, teacher_lse=None if lse is None else lse.double().numpy(), weights=w.astype(np.float64))
    if labelled:
        dev.update(labels=torch.from_numpy(y).cuda(), label_lam=0.3)
        host.update(labels=y, label_lam=0.3)
    f = pa().DistillationLoss(td, torch.from_numpy(idx).cuda(), v, **dev)
    val, g = f.value_and_gradient(x)
    want = ref.distillation(xe, te, idx, **host)
    check(g, val, want, DT[dtype])
    v2, g2 = f.value_and_gradient_async(x, out=x)  # in place
    assert g2 is x and torch.equal(g2, g)
    assert float(v2) == pytest.approx(val, rel=2.0**-23)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rest", [False, True])
def test_distillation_special_rows(dtype, rest):
    """masked classes (-inf, the type's lowest value), whole rows of them, NaN, infinities, lists without mass, indices out of range"""
    v, k = 261, 6
    dt = DT[dtype]
    rng = np.random.default_rng(5)
    n = 12
    t, idx = teacher(rng, n, v, k)
    x, xe = scores(rng, n, v, torch.float32, idx, t)
    xe = xe.copy()
    low = torch.finfo(dt).min
    xe[0] = -np.inf  # nothing left
    xe[1] = low  # everything at the lowest value: a uniform row
    xe[2, 10:] = -np.inf
    xe[2, :10] = np.arange(10)
    idx[2] = np.arange(k)
    xe[3, :] = low
    xe[3, 7] = 1.0
    idx[3] = 7 + np.arange(k) * 3
    t[3, 1:] = -np.inf  # the teacher is sure
    t[4] = -np.inf  # a list without mass
    idx[5] = -1  # no list
    xe[6, idx[6][2]] = -np.inf  # a listed class is masked: f = inf (checked alone below)
    xe[7, 3] = np.nan
    idx[8, 1] = v  # out of range
    xe[9] = 60000.0 if dtype == "f16" else 1e30  # large and equal
    xe[10] = np.where(np.arange(v) % 2, 3.0, low)
    xe[11, 5] = np.inf  # inf - inf
    lse = (np.log(np.where(np.isfinite(t), np.exp(t), 0).sum(1) + 1e-9) + 0.3).astype(np.float32)
    xd = torch.from_numpy(xe).to(dt).cuda()
    xe = xd.double().cpu().numpy()
    td, te = tdev(t, dt)
    for rows in ([0, 1, 2, 3, 4, 5, 9, 10], [6], [7], [8], [11], list(range(n))):
        sel = np.array(rows)
        f = pa().DistillationLoss(td[sel].contiguous(), torch.from_numpy(idx[sel]).cuda(), v, teacher_lse=torch.from_numpy(lse[sel]).cuda() if rest else None)
        val, g = f.value_and_gradient(xd[sel].contiguous())
        xr = np.where(np.isposinf(xe[sel]), np.nan, xe[sel])  # an infinite score is a NaN row by the formula
        check(g, val, ref.distillation(xr, te[sel], idx[sel], teacher_lse=lse[sel].astype(np.float64) if rest else None), dt)


def test_distillation_empty_and_vectors():
    m = pa()
    for n, v in ((0, 5), (0, 0), (4, 0)):
        f = m.DistillationLoss(np.zeros((n, 0), np.float32), np.zeros((n, 0), np.int64), v)
        val, g = f.value_and_gradient(torch.empty(n, v, device="cuda"))
        assert val == 0.0 and g.shape == (n, v)
    rng = np.random.default_rng(0)
    t, idx = teacher(rng, 6, 50, 4)
    for dt in (np.float32, np.float64):
        u = rng.normal(size=300).astype(dt)
        f = m.DistillationLoss(t, idx, 50)
        val, g = f.value_and_gradient(m.HIPVector.from_numpy(u))
        assert isinstance(val, dt) and isinstance(g, m.HIPVector)
        check(torch.from_numpy(g.numpy().reshape(6, 50)), val, ref.distillation(u.reshape(6, 50), t, idx), DT["f32" if dt == np.float32 else "f64"])
        assert f(m.HIPVector.from_numpy(u)) == val


# ---- balance ---------------------------------------------------------------------------------------------------------


def check_balance(loss, got, value, want, dtype):
    f, grad, counts, size, f_size = want
    assert np.array_equal(loss.counts.cpu().numpy(), counts)
    check(got, value, (f, grad, size, f_size), dtype)


def router(rng, n, e, dtype, gap=0, shift=0):
    buf = torch.full((shift + n * (e + gap),), float("nan"), dtype=dtype, device="cuda")
    out = buf[shift:].view(n, e + gap)[:, :e]
    out.copy_(torch.from_numpy(rng.normal(size=(n, e)) + rng.normal(size=e)))
    return out, out.double().cpu().numpy()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,e,k,gap,shift", [(1, 1, 1, 0, 0), (2, 4, 2, 0, 0), (7, 3, 3, 1, 1), (64, 64, 6, 0, 0), (300, 65, 8, 0, 3), (33, 127, 1, 5, 0),
                                             (700, 128, 8, 0, 0), (20, 200, 16, 0, 1), (1500, 256, 8, 0, 0), (9, 500, 40, 3, 0), (5, 1024, 1024, 0, 0)])
def test_balance_sizes(dtype, n, e, k, gap, shift):
    rng = np.random.default_rng(n + e)
    x, xe = router(rng, n, e, DT[dtype], gap, shift)
    loss = pa().BalanceLoss(n, e, k, lam=3.0)
    val, g = loss.value_and_gradient(x)
    want = ref.balance(xe, k, lam=3.0)
    check_balance(loss, g, val, want, DT[dtype])
    for _ in range(3):  # the counts start anew each time
        v2, g2 = loss.value_and_gradient_async(x)
        assert torch.equal(g2, g) and float(v2) == pytest.approx(val, rel=2.0**-23)
    assert np.array_equal(loss.counts.cpu().numpy(), want[2])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("e,k,offsets,n", [(16, 2, [0, 1, 1, 5, 40], 40), (60, 4, [0, 0, 0], 9), (64, 6, [0, 400, 401, 900], 1000), (130, 5, list(range(0, 301, 3)), 310),
                                           (8, 2, [0], 20)])
def test_balance_groups_and_masks(dtype, e, k, offsets, n):
    """ragged, empty and single-token groups, tokens behind the last one, masked tokens that hold NaN; chosen by the router itself"""
    rng = np.random.default_rng(len(offsets) + e)
    x, xe = router(rng, n, e, DT[dtype])
    mask = rng.random(n) < 0.7
    x[torch.from_numpy(~mask).cuda()] = float("nan")
    if offsets[-1] < n:
        x[offsets[-1]:] = float("inf")
    xe = x.double().cpu().numpy()
    loss = pa().BalanceLoss(n, e, k, offsets=offsets, mask=mask, lam=0.5)
    val, g = loss.value_and_gradient(x)
    check_balance(loss, g, val, ref.balance(xe, k, offsets=offsets, mask=mask, lam=0.5), DT[dtype])
    chosen = rng.integers(-1, e, (n, k))
    chosen[::3, -1] = chosen[::3, 0]  # named twice
    for idt in (np.int32, np.int64):
        loss = pa().BalanceLoss(n, e, k, offsets=offsets, mask=torch.from_numpy(mask).cuda(), chosen=torch.from_numpy(chosen.astype(idt)).cuda(), lam=0.5)
        val, g = loss.value_and_gradient(x)
        check_balance(loss, g, val, ref.balance(xe, k, offsets=offsets, mask=mask, chosen=chosen, lam=0.5), DT[dtype])
        v2, g2 = loss.value_and_gradient_async(x, out=x.clone())
        assert torch.equal(g2, g)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [9, 900])
def test_balance_special_rows(dtype, n):
    """equal scores, fewer live experts than k, the lowest value, NaN, infinities, a choice out of range"""
    e, k = 70, 5
    dt = DT[dtype]
    rng = np.random.default_rng(1)
    base = rng.normal(size=(n, e))
    base[0] = 0.0  # all equal: the first five
    base[1, 10:] = 1.0  # ties at the border
    base[2] = -np.inf
    base[3, 3:] = -np.inf  # three experts left
    base[4] = torch.finfo(dt).min
    base[5] = np.where(np.arange(e) % 3, -0.0, 0.0)  # equal in value, not in bits
    base[6] = np.repeat(rng.normal(size=e // 2), 2)
    base[7, :] = np.linspace(-60000, 60000, e)
    xd = torch.from_numpy(base).to(dt).cuda()
    loss = pa().BalanceLoss(n, e, k)
    val, g = loss.value_and_gradient(xd)
    check_balance(loss, g, val, ref.balance(xd.double().cpu().numpy(), k), dt)
    xd[8, 4] = float("nan")
    val, g = loss.value_and_gradient(xd)
    want = ref.balance(xd.double().cpu().numpy(), k)
    assert np.isnan(val)
    check_balance(loss, g, val, want, dt)
    xd[8, 4] = 0.0
    chosen = rng.integers(0, e, (n, k))
    chosen[n - 1, 0] = e
    loss = pa().BalanceLoss(n, e, k, offsets=[0, n // 2, n], chosen=torch.from_numpy(chosen).cuda())
    val, g = loss.value_and_gradient(xd)
    check_balance(loss, g, val, ref.balance(xd.double().cpu().numpy(), k, offsets=[0, n // 2, n], chosen=chosen), dt)
