"""The losses on rows of scores as they are used: every kernel form at full width, other layouts and types, streams, graphs, refusals,
and both together as terms of one objective under the package's iterations.  Oracle and tolerances: test_gpu_row_losses.py."""
import itertools

import numpy as np
import pytest
import torch

from oracle import proxgrad_oracle as o
from oracle import row_losses as ref
from .test_gpu_row_losses import DT, check, check_balance, flushed, pa, router, scores, tdev, teacher

pytestmark = pytest.mark.gpu
SIZE = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}


def repeated(n, base):
    """rows 0 .. n - 1 are the distinct rows 0 .. base - 1 over and over: many rows, few for the oracle"""
    return torch.arange(n, device="cuda") % base


def check_repeated(g, val, want, dtype, n):
    """each copy of a row against that row's gradient; the value is the rows' sum"""
    f, grad, size, f_size = want[0]
    base = grad.shape[0]
    u = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    fin = torch.finfo(dtype)
    for b in range(base):
        tol = torch.from_numpy(np.abs(grad[b]) * (fin.eps / 2) + size[b] * u * 1.01 + fin.smallest_normal * fin.eps / 2).cuda()
        if dtype != torch.float64:
            tol += flushed(size[b:b + 1]).item()
        off = (g[b::base].double() - torch.from_numpy(grad[b]).cuda()).abs_()
        assert bool((off <= tol).all()), b
    total = sum(w[0] * len(range(b, n, base)) for b, w in enumerate(want[1]))
    slack = sum(w[3] * len(range(b, n, base)) for b, w in enumerate(want[1]))
    assert abs(val - total) <= slack * u + abs(total) * (2.0**-24 if u > 1e-10 else 4 * u)


# bytes of a row that each form holds, one class short of full (an odd number: rows at every alignment); 300 rows for the smaller
# forms and 1100 for the larger, so that workgroups go on to further rows; the last one is longer than the registers
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rest,labelled", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("held,n", [(1024, 9000), (2048, 9000), (4096, 9000), (8192, 9000), (16384, 3000), (32768, 3000), (65536, 1100), (131072, 600),
                                    (262144, 300), (280000, 70)])
def test_every_form_at_full_width(dtype, rest, labelled, held, n):
    v = held // SIZE[dtype] - 1
    base, k, temperature = 3, 37, 2.0 if held % 3 else 1.25
    rng = np.random.default_rng(held + 2 * rest + labelled)
    t, idx = teacher(rng, base, v, k, twice=True)
    td, te = tdev(t, torch.float32 if dtype != "f64" else torch.float64)
    x, xe = scores(rng, base, v, DT[dtype], idx, t)
    y = rng.integers(0, v, base)
    y[1] = idx[1, 0]
    kw = dict(temperature=temperature, lam=1.25)
    lse = np.log(np.exp(te / temperature).sum(1) + 0.4) if rest else None
    lse = None if lse is None else torch.from_numpy(lse).to(td.dtype)
    each = repeated(n, base)
    dev = dict(kw, teacher_lse=None if lse is None else lse.cuda()[each])
    host = dict(kw, teacher_lse=None if lse is None else lse.double().numpy())
    if labelled:
        dev.update(labels=torch.from_numpy(y).cuda()[each], label_lam=0.5)
        host.update(labels=y, label_lam=0.5)
    f = pa().DistillationLoss(td[each], torch.from_numpy(idx).cuda()[each], v, **dev)
    u = x[each]
    val, g = f.value_and_gradient(u)
    one = lambda b: {q: (w[b:b + 1] if isinstance(w, np.ndarray) else w) for q, w in host.items()}  # noqa: E731
    alone = [ref.distillation(xe[b:b + 1], te[b:b + 1], idx[b:b + 1], **one(b)) for b in range(base)]
    want = (None, np.concatenate([w[1] for w in alone]), np.concatenate([w[2] for w in alone]), None)
    check_repeated(g, val, (want, alone), DT[dtype], n)
    v2, _ = f.value_and_gradient_async(u, out=u)
    assert torch.equal(u, g) and float(v2) == pytest.approx(val, rel=2.0**-23)  # in place, and the same again


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("temperature", [0.5, 1.0, 4.0])
@pytest.mark.parametrize("n,v", [(5, 700), (5, 9001), (70, 40001)])
def test_rising_scores(dtype, temperature, n, v):
    """every score above the ones before it, over a wide range: the sums' reference is raised again and again"""
    rng = np.random.default_rng(v)
    t, idx = teacher(rng, n, v, 6)
    xe = np.linspace(-300, 11, v) * np.linspace(0.1, 1, n)[:, None]
    xd = torch.from_numpy(xe).to(DT[dtype]).cuda()
    td, te = tdev(t, torch.float32)
    lse = torch.from_numpy(np.log(np.exp(te / temperature).sum(1) * 1.5)).float()
    y = rng.integers(0, v, n)
    kw = dict(temperature=temperature, label_lam=0.5)
    f = pa().DistillationLoss(td, torch.from_numpy(idx).cuda(), v, teacher_lse=lse.cuda(), labels=torch.from_numpy(y).cuda(), **kw)
    val, g = f.value_and_gradient(xd)
    rows = sorted({0, 1, n // 2, n - 1})
    want = ref.distillation(xd.double().cpu().numpy()[rows], te[rows], idx[rows], teacher_lse=lse.double().numpy()[rows], labels=y[rows], **kw)
    w = torch.zeros(n)
    w[rows] = 1.0
    f = pa().DistillationLoss(td, torch.from_numpy(idx).cuda(), v, teacher_lse=lse.cuda(), labels=torch.from_numpy(y).cuda(), weights=w.cuda(), **kw)
    val, g1 = f.value_and_gradient(xd)
    check(g1[rows], val, want, DT[dtype])
    assert torch.equal(g1[rows], g[rows]) and not g1[[i for i in range(n) if i not in rows]].any()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("n,v,k", [(3, 1100, 1024), (70, 1024, 1024), (66, 20000, 700), (2, 90001, 1024), (3, 50, 0)])
def test_long_and_empty_lists(dtype, rest, n, v, k):
    rng = np.random.default_rng(k + n)
    t, idx = teacher(rng, n, v, k, absent=0.1 if k < v else 0.0, twice=k < v)
    td, te = tdev(t, DT[dtype])
    x, xe = scores(rng, n, v, DT[dtype], idx, t)
    with np.errstate(divide="ignore"):
        lse = np.log(np.where(idx >= 0, np.exp(te), 0).sum(1) + 1e-3)
    lse = torch.from_numpy(lse).float() if rest else None
    w = np.zeros(n)
    rows = sorted({0, n // 3, n - 1})
    w[rows] = 1.5
    f = pa().DistillationLoss(td, torch.from_numpy(idx).cuda(), v, weights=torch.from_numpy(w).cuda(), teacher_lse=None if lse is None else lse.cuda())
    val, g = f.value_and_gradient(x)
    check(g, val, ref.distillation(xe, te, idx, weights=w, teacher_lse=None if lse is None else lse.double().numpy()), DT[dtype])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("logits", DT)
@pytest.mark.parametrize("n,v", [(9, 301), (2, 40000)])
def test_types_and_strides_of_the_teacher(dtype, logits, n, v):
    """logits of each type beside scores of each type; lists that are columns of a wider table; Float64 weights and lse; int32, int64"""
    rng = np.random.default_rng(7)
    k = 11
    t, idx = teacher(rng, n, v, k)
    wide = torch.full((n, k + 5), float("nan"), dtype=DT[logits], device="cuda")
    wide[:, 2:2 + k] = torch.from_numpy(t).to(DT[logits]).cuda()
    te = wide[:, 2:2 + k].double().cpu().numpy()
    wide_i = torch.full((n, k + 3), -7, dtype=torch.int32 if n > 2 else torch.int64, device="cuda")
    wide_i[:, 3:] = torch.from_numpy(idx).cuda()
    x, xe = scores(rng, n, v, DT[dtype], idx, t)
    w = rng.random(n)
    lse = np.log(np.exp(te).sum(1) * 1.25)
    y = torch.from_numpy(rng.integers(-1, v, n)).to(torch.int32)
    f = pa().DistillationLoss(wide[:, 2:2 + k], wide_i[:, 3:], v, teacher_lse=torch.from_numpy(lse).cuda(), weights=torch.from_numpy(w).cuda(),
                              labels=y.cuda(), label_lam=0.25)
    val, g = f.value_and_gradient(x)
    check(g, val, ref.distillation(xe, te, idx, teacher_lse=lse, weights=w, labels=y.numpy(), label_lam=0.25), DT[dtype])
    transposed = torch.from_numpy(np.ascontiguousarray(idx.T)).cuda().t()  # not dense along the list: copied
    f = pa().DistillationLoss(te.astype(np.float64), transposed, v, teacher_lse=lse, weights=w, labels=y.numpy(), label_lam=0.25)  # and from the host
    v2, g2 = f.value_and_gradient(x)
    check(g2, v2, ref.distillation(xe, te, idx, teacher_lse=lse, weights=w, labels=y.numpy(), label_lam=0.25), DT[dtype])


def both_losses(n=40, v=333, e=61, dt=torch.float32, ctx=None, seed=0):
    rng = np.random.default_rng(seed)
    t, idx = teacher(rng, n, v, 9)
    d = pa().DistillationLoss(t, idx, v, temperature=2.0, labels=rng.integers(0, v, n), label_lam=0.5, ctx=ctx)
    b = pa().BalanceLoss(n, e, 4, offsets=[0, n // 2, n - 1], ctx=ctx)
    gen = torch.Generator("cuda").manual_seed(seed)
    return (d, torch.randn(n, v, device="cuda", generator=gen).to(dt)), (b, torch.randn(n, e, device="cuda", generator=gen).to(dt))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("gap,shift", [(0, 1), (3, 0), (8, 5)])
def test_out_of_another_layout_and_what_lies_between_the_rows(dtype, which, gap, shift):
    loss, u = both_losses(dt=DT[dtype])[which]
    n, v = u.shape
    val, g = loss.value_and_gradient(u)
    buf = torch.full((shift + n * (v + gap) + 9,), 7.0, dtype=u.dtype, device="cuda")
    out = buf[shift:shift + n * (v + gap)].view(n, v + gap)[:, :v]
    v2, g2 = loss.value_and_gradient(u, out=out)
    assert g2 is out and torch.equal(out, g) and v2 == val
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[shift:shift + n * (v + gap)].view(n, v + gap)[:, :v] = False
    assert bool((buf[keep] == 7.0).all())
    # scores and gradient side by side in one buffer; in place in a padded one (its own alignment: sums in another order)
    pair = torch.full((n, 2 * v + gap), 7.0, dtype=u.dtype, device="cuda")
    pair[:, :v] = u
    loss.value_and_gradient(pair[:, :v], out=pair[:, v + gap:])
    assert torch.equal(pair[:, :v], u) and bool((pair[:, v:v + gap] == 7.0).all())
    out2 = pair[:, v + gap:].clone()
    loss.value_and_gradient(pair[:, :v], out=pair[:, :v])
    assert torch.equal(pair[:, :v], out2) and torch.equal(pair[:, v + gap:], out2)
    torch.testing.assert_close(out2, g, rtol=torch.finfo(u.dtype).eps, atol=2.0**-18)  # a rounding of each, and 64 * 2^-24 of terms up to 1 before


@pytest.mark.parametrize("which", [0, 1])
def test_rows_far_apart(which):
    """offsets that pass 32 bits, in elements and in bytes"""
    (d, ud), (b, ub) = both_losses(n=4, v=300, e=60, dt=torch.bfloat16)
    loss, u = ((d, ud), (b, ub))[which]
    n, v = u.shape
    ld = (1 << 30) + 24
    buf = torch.empty(3 * ld + v, dtype=u.dtype, device="cuda")
    far = buf.as_strided((n, v), (ld, 1))
    far.copy_(u)
    val, g = loss.value_and_gradient(u)
    v2, g2 = loss.value_and_gradient(far, out=torch.empty_like(u))
    torch.testing.assert_close(g2, g, rtol=2.0**-7, atol=1e-6)
    assert v2 == pytest.approx(val, rel=1e-6)
    loss.value_and_gradient(far, out=far)
    assert torch.equal(far, g2)


def test_another_current_stream():
    for loss, u in both_losses():
        val, g = loss.value_and_gradient(u)
        s = torch.cuda.Stream()
        for _ in range(4):
            out, value = torch.full_like(u, 9.0), torch.zeros((), device="cuda")
            late = torch.zeros_like(u)
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                big = torch.randn(2500, 2500, device="cuda")
                for _ in range(8):
                    big = big @ big * 1e-4
                late.copy_(u + 0 * big[0, 0].nan_to_num(0.0, 0.0, 0.0))  # u is ready late, on s
                value, out = loss.value_and_gradient_async(late, out=out, value=value)
                got = out.clone()  # on s, behind the loss
                v = value.clone()
            s.synchronize()
            assert torch.equal(got, g) and float(v) == pytest.approx(val, rel=2.0**-23)
    made = torch.cuda.Stream()  # a loss made under one stream, used under another
    with torch.cuda.stream(made):
        (d, ud), (b, ub) = both_losses(seed=3)
    torch.cuda.current_stream().wait_stream(made)
    for (loss, u), (same, _) in zip(((d, ud), (b, ub)), both_losses(seed=3)):
        assert torch.equal(loss.value_and_gradient(u)[1], same.value_and_gradient(u)[1])


def test_recorded_and_replayed():
    """each loss in two graphs, replayed in turn with eager calls of the same losses, and of others, between"""
    m = pa()
    ctx = m.Context.on_new_stream()
    losses = both_losses(ctx=ctx)
    big = both_losses(n=700, v=50, e=128, ctx=ctx, seed=1)  # the balance in tiles, with accumulators that take turns
    wide = both_losses(n=2, v=40000, e=8, ctx=ctx, seed=2)  # the distillation in parts
    torch.cuda.synchronize()
    with torch.cuda.stream(ctx._stream_owner):
        cases = []
        for loss, u in (*losses, *big, *wide):
            eager = loss.value_and_gradient(u)
            second = loss.value_and_gradient(u * 0.5)
            cases.append((loss, u.clone(), eager, second))
        torch.cuda.synchronize()
        graphs = []
        for turn in range(2):
            for loss, u, _, _ in cases:
                out, value = torch.zeros_like(u), torch.zeros((), device="cuda")
                torch.cuda.synchronize()
                ctx.capture_begin()
                loss.value_and_gradient_async(u, out=out, value=value)
                graphs.append((ctx.capture_end(), out, value))
        for k in range(4):
            order = range(len(graphs)) if k % 2 else reversed(range(len(graphs)))
            for i in order:
                loss, u, eager, second = cases[i % len(cases)]
                g, out, value = graphs[i]
                g.launch()
                torch.cuda.synchronize()
                assert torch.equal(out, eager[1]) and float(value) == pytest.approx(eager[0], rel=2.0**-23)
                out.fill_(3.0)
                value.fill_(3.0)
                if i % 3 == 0:
                    v2, g2 = loss.value_and_gradient(u * 0.5)
                    assert v2 == second[0] and torch.equal(g2, second[1])
                if i % 5 == 0:
                    float(u.sum())
    with pytest.raises(m.ProxGradError):
        ctx.capture_begin()
        try:
            losses[0][0].value_and_gradient_async(losses[0][1])  # needs an allocation
        finally:
            ctx.capture_end(abort=True)


def test_somebody_elses_capture_is_refused():
    m = pa()
    for loss, u in both_losses():
        want = loss.value_and_gradient(u)
        out, value = torch.empty_like(u), torch.zeros((), device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            w = u * 2
            with pytest.raises(m.ProxGradError):
                loss.value_and_gradient_async(u, out=out, value=value)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, u * 2)
        v2, g2 = loss.value_and_gradient(u)
        assert v2 == want[0] and torch.equal(g2, want[1])


def test_a_capture_of_the_contexts_own_stream_by_somebody_else_is_refused():
    m = pa()
    ctx = m.Context.on_new_stream()
    for loss, u in both_losses(ctx=ctx):
        out, value = torch.empty_like(u), torch.zeros((), device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=ctx._stream_owner):
            w = u * 3
            with pytest.raises(m.ProxGradError):
                loss.value_and_gradient_async(u, out=out, value=value)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, u * 3)
        torch.cuda.synchronize()
        with torch.cuda.stream(ctx._stream_owner):
            assert np.isfinite(loss.value_and_gradient(u)[0])
    ctx.capture_begin()
    try:
        with pytest.raises(m.ProxGradError):
            m.BalanceLoss(4, 4, 2, ctx=ctx)
        with pytest.raises(m.ProxGradError):
            m.DistillationLoss(np.zeros((2, 1)), np.zeros((2, 1), int), 4, ctx=ctx)
    finally:
        ctx.capture_end(abort=True)


def test_refusals_on_the_device():
    m = pa()
    (d, ud), (b, ub) = both_losses()
    for loss, u in ((d, ud), (b, ub)):
        n, v = u.shape
        buf = torch.zeros(4 * n * v, device="cuda")
        part = lambda at, ld=v: buf[at:].as_strided((n, v), (ld, 1), at)  # noqa: E731
        bad = [
            (ValueError, (u[:-1], None)), (ValueError, (u[:, :-1], None)), (ValueError, (u.cpu(), None)), (TypeError, (u.int(), None)), (TypeError, (None, None)),
            (TypeError, (u.cpu().numpy(), None)), (ValueError, (u, torch.empty(n + 1, v, device="cuda"))), (TypeError, (u, torch.empty_like(u, dtype=torch.float64))),
            (ValueError, (u, torch.empty_like(u, device="cpu"))), (ValueError, (u.t().contiguous().t(), None)), (ValueError, (u[:1].expand(n, v), None)),
            (ValueError, (part(0), part(4))), (ValueError, (part(4), part(0))), (ValueError, (part(0, v + 8), part(0))), (ValueError, (part(0), part(n * v - 1))),
            (ValueError, (m.HIPVector.zeros(n * v + 1, np.float32), None)),
            (TypeError, (u, m.HIPVector.zeros(n * v, np.float64))),
            (ValueError, (m.HIPVector.zeros(n * v, np.float32, m.Context.on_new_stream()), None)),
        ]
        for err, (x, out) in bad:
            with pytest.raises(err):
                loss.value_and_gradient(x, out=out)
        for value in (torch.zeros(2, device="cuda"), torch.zeros((), dtype=torch.float64, device="cuda"), torch.zeros(())):
            with pytest.raises(ValueError):
                loss.value_and_gradient_async(u, value=value)
        val, g = loss.value_and_gradient(part(0), out=part(n * v))  # next to each other is fine
        assert np.isfinite(val)
    with pytest.raises(ValueError):
        m.SlicedSeparableSum((d, b), ((0, ud.numel()), (0, ub.numel()))).value_and_gradient(m.HIPVector.zeros(ud.numel() + ub.numel(), np.float32))
    half = m.HIPVector.zeros(64, np.float32)
    with pytest.raises(ValueError):
        m.SlicedSeparableSum((m.SqrNormL2(),), ((0, 32),)).value_and_gradient(half, out=half)  # the rest of x would be lost


@pytest.mark.parametrize("n,e,k,groups", [(1, 1, 1, 1), (5000, 64, 6, 1), (3000, 256, 8, 1), (4000, 33, 2, 37), (2000, 1024, 16, 3)])
def test_balance_many_tiles(n, e, k, groups):
    """tiles in several accumulators, and the same bits each time"""
    rng = np.random.default_rng(e)
    x, xe = router(rng, n, e, torch.float32)
    cut = np.sort(rng.integers(0, n + 1, groups - 1))
    offsets = [0, *cut.tolist(), n]
    loss = pa().BalanceLoss(n, e, k, offsets=offsets if groups > 1 else None, lam=2.0)
    val, g = loss.value_and_gradient(x)
    check_balance(loss, g, val, ref.balance(xe, k, offsets=offsets, lam=2.0), torch.float32)
    for _ in range(5):
        v2, g2 = loss.value_and_gradient(x)
        assert v2 == val and torch.equal(g2, g)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,v", [(6, 300), (1, 70000)])
def test_masked_classes_and_terms_that_are_switched_off(dtype, n, v):
    """the list, the label or everything outside the list at -inf: an infinite value, unless that term's factor is zero; finite gradients"""
    rng = np.random.default_rng(3)
    t, idx = teacher(rng, n, v, 5)
    td, te = tdev(t, torch.float32)
    x, xe = scores(rng, n, v, DT[dtype], idx, t)
    y = idx[:, 1].copy()
    rows = np.arange(n)
    lse = np.log(np.exp(te).sum(1) + 3.0).astype(np.float32)
    for where in ("list", "outside"):
        xm = x.clone()
        if where == "list":
            xm[torch.from_numpy(rows).cuda(), torch.from_numpy(idx[:, 1]).cuda()] = float("-inf")  # a listed class, and the label
        else:
            keep = torch.zeros(n, v, dtype=torch.bool, device="cuda").scatter_(1, torch.from_numpy(idx).cuda(), True)
            xm[~keep] = float("-inf")
        xe = xm.double().cpu().numpy()
        for lam, label_lam, rest in itertools.product((0.0, 1.5), (0.0, 0.5), (False, True)):
            kw = dict(lam=lam, label_lam=label_lam)
            f = pa().DistillationLoss(td, torch.from_numpy(idx).cuda(), v, labels=torch.from_numpy(y).cuda(), teacher_lse=torch.from_numpy(lse).cuda() if rest else None, **kw)
            val, g = f.value_and_gradient(xm)
            want = ref.distillation(xe, te, idx, labels=y, teacher_lse=lse.astype(np.float64) if rest else None, **kw)
            assert np.isinf(want[0]) == bool((where == "list" and (lam or label_lam)) or (where == "outside" and rest and lam))
            check(g, val, want, DT[dtype])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,v", [(6, 300), (2, 70000), (300, 5000)])
@pytest.mark.parametrize("below", [60.0, 200.0, 5000.0])
def test_outside_class_far_below_the_listed_ones(dtype, n, v, below):
    """what the teacher leaves outside its list is divided by the softmax of the other classes, also where they have no share of the whole row's"""
    rng = np.random.default_rng(int(below))
    base = min(n, 4)
    t, idx = teacher(rng, base, v, 7)
    x, _ = scores(rng, base, v, DT[dtype])
    x.scatter_add_(1, torch.from_numpy(idx).cuda(), torch.full((base, 7), below, dtype=x.dtype, device="cuda"))
    xe = x.double().cpu().numpy()
    td, te = tdev(t, torch.float32)
    lse = np.log(np.exp(te / 2).sum(1) * 1.3).astype(np.float32)
    y = rng.integers(0, v, base)
    each = repeated(n, base)
    kw = dict(temperature=2.0, lam=1.5, label_lam=0.5)
    f = pa().DistillationLoss(td[each], torch.from_numpy(idx).cuda()[each], v, teacher_lse=torch.from_numpy(lse).cuda()[each], labels=torch.from_numpy(y).cuda()[each], **kw)
    val, g = f.value_and_gradient(x[each])
    alone = [ref.distillation(xe[b:b + 1], te[b:b + 1], idx[b:b + 1], teacher_lse=lse[b:b + 1].astype(np.float64), labels=y[b:b + 1], **kw) for b in range(base)]
    assert all(np.isfinite(w[0]) and (w[1] < 0).any() for w in alone)
    check_repeated(g, val, ((None, np.concatenate([w[1] for w in alone]), np.concatenate([w[2] for w in alone]), None), alone), DT[dtype], n)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,v,k", [(200, 900, 300), (70, 30000, 200), (2, 70000, 300)])
@pytest.mark.parametrize("rest", [False, True])
def test_classes_listed_many_times_give_the_same_bits_each_time(dtype, n, v, k, rest):
    rng = np.random.default_rng(k)
    t, idx = teacher(rng, n, v, k)
    idx[:, k // 3:] = idx[:, rng.integers(0, k // 3, k - k // 3)]  # three entries to a class on average
    td, te = tdev(t, torch.float32)
    x, xe = scores(rng, n, v, DT[dtype], idx, t)
    lse = np.log(np.exp(te).sum(1) * 1.2)
    f = pa().DistillationLoss(td, torch.from_numpy(idx).cuda(), v, teacher_lse=torch.from_numpy(lse).cuda() if rest else None)
    val, g = f.value_and_gradient(x)
    for _ in range(8):
        v2, g2 = f.value_and_gradient(x)
        assert v2 == val and torch.equal(g2, g)
    rows = [0, n - 1]
    want = ref.distillation(xe[rows], te[rows], idx[rows], teacher_lse=lse[rows] if rest else None)
    check(g[rows], want[0], want, DT[dtype])


@pytest.mark.parametrize("dtype,logits,n,v,k", [("f32", "f32", 150, 70000, 1024), ("bf16", "f64", 2000, 100, 50), ("f64", "f32", 1500, 40, 33), ("f16", "f16", 200, 140001, 700)])
@pytest.mark.parametrize("rest", [False, True])
def test_parts_of_more_rows_than_the_workspace_holds(dtype, logits, n, v, k, rest):
    rng = np.random.default_rng(n)
    base = 5
    t, idx = teacher(rng, base, v, k, absent=0.05)
    td, te = tdev(t, DT[logits])
    x, xe = scores(rng, base, v, DT[dtype], idx, t)
    lse = np.log(np.where(idx >= 0, np.exp(te), 0).sum(1) * 1.2)
    each = repeated(n, base)
    f = pa().DistillationLoss(td[each], torch.from_numpy(idx).cuda()[each], v, teacher_lse=torch.from_numpy(lse).cuda()[each] if rest else None)
    val, g = f.value_and_gradient(x[each])
    alone = [ref.distillation(xe[b:b + 1], te[b:b + 1], idx[b:b + 1], teacher_lse=lse[b:b + 1] if rest else None) for b in range(base)]
    check_repeated(g, val, ((None, np.concatenate([w[1] for w in alone]), np.concatenate([w[2] for w in alone]), None), alone), DT[dtype], n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 3])
def test_the_longest_row(dtype, shift):
    """2^24 classes, against the formula in Float64 on the device"""
    v = 1 << 24
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.empty(v + shift, device="cuda", dtype=DT[dtype])[shift:].view(1, v)
    x.copy_(torch.randn(1, v, device="cuda", generator=gen))
    idx = torch.tensor([[0, 1, v - 1, v // 2]], device="cuda")
    t = torch.tensor([[3.0, 2.0, 1.0, 0.0]], device="cuda")
    x[0, idx[0]] = 18.0
    f = pa().DistillationLoss(t, idx, v)
    val, g = f.value_and_gradient(x)
    p, lq = torch.softmax(t.double(), 1), torch.log_softmax(x.double(), 1)
    want = lq.exp()
    want[0, idx[0]] -= p[0]
    # a thread adds 128 vectors one after another: 128 roundings of the sum beside the 64 + 6 |x - m| log2(e), |x - m| < 25, of the others
    tol = want.abs() * torch.finfo(x.dtype).eps / 2 + lq.exp() * 2.0**-24 * (128 + 64 + 6 * 36) + 2.0**-97
    tol[0, idx[0]] += 2.0**-24 * 64  # the teacher's probabilities
    assert bool(((g.double() - want).abs() <= tol).all())
    kl = float((p * (p.log() - lq[0, idx[0]])).sum())
    assert abs(val - kl) <= 2.0**-24 * 64 * 40


def test_balance_of_very_many_groups():
    rng = np.random.default_rng(0)
    n, e, k = 20000, 8, 2
    x, xe = router(rng, n, e, torch.float32)
    for offsets in (list(range(n + 1)), sorted([0, n, *rng.integers(0, n, 3000).tolist()])):
        loss = pa().BalanceLoss(n, e, k, offsets=offsets)
        val, g = loss.value_and_gradient(x)
        check_balance(loss, g, val, ref.balance(xe, k, offsets=offsets), torch.float32)


def test_balance_of_nothing_and_positions_on_the_device():
    m = pa()
    for offsets in (None, [0], [0, 0, 0]):
        loss = m.BalanceLoss(0, 4, 2, offsets=offsets)
        val, g = loss.value_and_gradient(torch.empty(0, 4, device="cuda"))
        assert val == 0.0 and g.shape == (0, 4) and not loss.counts.any()
    rng = np.random.default_rng(0)
    x, xe = router(rng, 50, 12, torch.float32)
    offsets = torch.tensor([0, 7, 7, 50], device="cuda", dtype=torch.int32)
    mask = torch.from_numpy((rng.random(50) < 0.5).astype(np.uint8) * 255).cuda()
    loss = m.BalanceLoss(50, 12, 3, offsets=offsets, mask=mask)
    val, g = loss.value_and_gradient(x)
    check_balance(loss, g, val, ref.balance(xe, 3, offsets=[0, 7, 7, 50], mask=mask.cpu().numpy() > 0), torch.float32)
    mask.fill_(1)  # tensors on the device are used where they are
    val, g = loss.value_and_gradient(x)
    check_balance(loss, g, val, ref.balance(xe, 3, offsets=[0, 7, 7, 50]), torch.float32)
    empty = loss(x)
    assert empty == val
    mask.fill_(0)
    val, g = loss.value_and_gradient(x)
    assert val == 0.0 and not g.any() and not loss.counts.any()
    for dt in DT.values():  # one loss, scores of any type
        mask.fill_(1)
        xd = x.to(dt)
        val, g = loss.value_and_gradient(xd)
        check_balance(loss, g, val, ref.balance(xd.double().cpu().numpy(), 3, offsets=[0, 7, 7, 50]), dt)


class OracleLoss:
    is_generalized_quadratic = False

    def __init__(self, parts):
        self.parts = parts  # (lo, hi, rows -> (f, gradient))

    def value_and_gradient(self, u):
        f, g = 0.0, np.zeros_like(u)
        for lo, hi, rows, fn in self.parts:
            r = fn(u[lo:hi].reshape(rows, -1))
            f += r[0]
            g[lo:hi] = r[1].reshape(-1)
        return f, g

    def __call__(self, u):
        return self.value_and_gradient(u)[0]


def routed_student(rng, tokens=12, v=30, e=8, k=2, top=5, dim=25):
    """scores and router logits of one linear model: A x holds the distillation's rows, then a gap, then the router's"""
    t, idx = teacher(rng, tokens, v, top)
    y = rng.integers(0, v, tokens)
    lse = np.log(np.exp(t / 2).sum(1) + 0.5)
    a, b = tokens * v, tokens * v + 8
    kw = dict(temperature=2.0, lam=4.0, teacher_lse=lse, labels=y, label_lam=0.5)
    A = rng.normal(size=(b + tokens * e + 4, dim)) / np.sqrt(dim)
    dist = pa().DistillationLoss(t, idx, v, **{**kw, "teacher_lse": lse.astype(np.float64)})
    bal = pa().BalanceLoss(tokens, e, k, offsets=[0, 5, tokens], lam=0.1)
    f = pa().SlicedSeparableSum((dist, bal), ((0, a), (b, b + tokens * e)))
    fo = OracleLoss([(0, a, tokens, lambda r: ref.distillation(r, t, idx, **kw)[:2]),
                     (b, b + tokens * e, tokens, lambda r: ref.balance(r, k, offsets=[0, 5, tokens], lam=0.1)[:2])])
    return f, fo, A


def test_the_sum_of_both_on_one_vector():
    m = pa()
    f, fo, A = routed_student(np.random.default_rng(0))
    u = np.random.default_rng(1).normal(size=A.shape[0])
    want = fo.value_and_gradient(u)
    ud = m.HIPVector.from_numpy(u)
    val, g = f.value_and_gradient(ud)
    assert isinstance(val, np.float64) and val == pytest.approx(want[0], rel=1e-12) and f(ud) == val
    np.testing.assert_allclose(g.numpy(), want[1], rtol=1e-11, atol=1e-13)  # some hundred roundings of 2^-53 of terms up to 4
    assert not f.is_convex and not f.is_generalized_quadratic
    # against differences: second order in h, the third derivatives along d are below 30
    d = np.random.default_rng(2).normal(size=u.size)
    d /= np.linalg.norm(d)
    h = 1e-5
    diff = (f(m.HIPVector.from_numpy(u + h * d)) - f(m.HIPVector.from_numpy(u - h * d))) / (2 * h)
    assert abs(diff - float(want[1] @ d)) <= 30 * h * h / 6 + 2.0**-52 * 64 * abs(want[0]) / h


@pytest.mark.parametrize("name", ["ForwardBackwardIteration", "FastForwardBackwardIteration", "PANOCIteration"])
def test_iterations_on_both_together(name):
    """one objective of both losses behind a linear model, next to the same iteration in numpy on the oracle's losses"""
    m = pa()
    f, fo, A = routed_student(np.random.default_rng(4))
    x0 = np.zeros(A.shape[1])
    kw = dict(x0=x0, gamma=0.05)
    if name == "PANOCIteration":
        it = m.PANOCIteration(f=f, A=A, g=m.NormL1(0.01), adaptive=True, **kw)
        ora = o.PANOCIteration(f=fo, A=A, g=o.NormL1(0.01), adaptive=True, **kw)
    else:
        it = getattr(m, name)(f=m.Composed(f, A), g=m.NormL1(0.01), **kw)
        ora = getattr(o, name)(f=o.Composed(fo, A), g=o.NormL1(0.01), **kw)
    for a, b in itertools.islice(zip(it, ora), 12):
        assert float(a.gamma) == pytest.approx(float(b.gamma), rel=1e-12)
        np.testing.assert_allclose(a.z.numpy(), b.z, rtol=1e-8, atol=1e-9)
