"""The losses on rows of scores in numpy, straight from their definitions, in extended precision so that a Float64 kernel's error
is not compared with the same rounding here (test infrastructure only).

Each returns the value, the gradient and the sizes that rounding acts on, from which the tests derive their tolerances."""
import numpy as np

L = np.longdouble


def _log_softmax(z):
    with np.errstate(invalid="ignore", divide="ignore"):
        m = z.max()
        return z - m - np.log(np.exp(z - m).sum())


def distillation(x, t, idx, *, temperature=1.0, lam=1.0, teacher_lse=None, weights=None, labels=None, label_lam=0.0):
    """(f, gradient, size of the gradient's terms, size of the value's terms): rows of x one by one"""
    x = np.asarray(x, L)
    n, v = x.shape
    f, f_size = L(0), L(0)
    grad, size = np.zeros((n, v), L), np.zeros((n, v), L)
    log2e = L(1) / np.log(L(2))
    temperature, lam, label_lam = L(temperature), L(lam), L(label_lam)
    for i in range(n):
        w = L(1) if weights is None else L(weights[i])
        if w == 0:
            continue
        bad = np.isnan(x[i]).any() or (len(idx[i]) and (np.min(idx[i]) < -1 or np.max(idx[i]) >= v))
        y = -1 if labels is None else int(labels[i])
        if bad or y < -1 or y >= v:
            f = np.nan
            grad[i] = np.nan
            continue
        if np.all(x[i] == -np.inf):
            continue
        on = np.asarray(idx[i]) >= 0
        cls = np.asarray(idx[i])[on]
        tt = np.asarray(t[i], L)[on] / temperature
        lq = _log_softmax(x[i] / temperature)
        q = np.exp(lq)
        far = np.where(q > 0, (x[i][np.isfinite(x[i])].max() - x[i]) * log2e, 0.0)  # how far an entry's exponent is from the largest's
        if teacher_lse is not None:
            lp = tt - L(teacher_lse[i])
        else:
            lp = _log_softmax(tt) if len(tt) and tt.max() > -np.inf else np.full(len(tt), -np.inf)
        p = np.exp(lp)
        phat, ksize = np.zeros(v, L), np.zeros(v, L)
        np.add.at(phat, cls, p)
        with np.errstate(invalid="ignore"):
            np.add.at(ksize, cls, np.where(p > 0, p * (64 + 4 * np.abs(lp)), 0.0))
        pr, log_qr, left_size, share, near = L(0), L(0), L(0), np.zeros(v, L), np.zeros(v, L)
        outside = np.ones(v, bool)
        outside[cls] = False
        if teacher_lse is not None and len(tt) and outside.any():
            pr = max(L(0), L(1) - p.sum())
            top = lq[outside].max()
            log_qr = top + np.log(np.exp(lq[outside] - top).sum()) if top > -np.inf else -L(np.inf)
            if top > -np.inf:  # the outside class's mass is divided by the softmax of its own classes, however little q leaves them
                share[outside] = np.exp(lq[outside] - top) / np.exp(lq[outside] - top).sum()
                near[outside] = np.where(share[outside] > 0, (top - lq[outside]) * temperature * log2e, 0.0)
            # 1 - sum p is as far off as the sum is, (64 + 4 |log p|) roundings of each p, however little is left; an entry outside
            # the list gets q / Q of that, the value its slope log pr - log Q + 1 times that
            left_size = (p[p > 0] * (64 + 4 * np.abs(lp[p > 0]))).sum()
            ksize[outside] += left_size * share[outside]
        elif teacher_lse is not None and len(tt) == 0:
            pr, log_qr, share = L(1), L(0), q  # nothing listed: the outside class is everything on both sides
            near = far
        mass = p.sum() + pr
        with np.errstate(invalid="ignore", divide="ignore"):
            terms = np.where(p > 0, p * (lp - lq[cls]), 0.0)
            sizes = np.where(p > 0, p * (64 + 8 * (np.abs(lp) + np.abs(lq[cls]) + np.abs(x[i][cls]) / temperature)), 0.0)
            row = terms.sum() + (pr * (np.log(pr) - log_qr) if pr > 0 else 0.0)
            row_size = sizes[np.isfinite(sizes)].sum() + (64 * pr * (1 + abs(np.log(pr)) + abs(log_qr)) + 64 * (1 + abs(log_qr)) if pr > 0 and log_qr > -np.inf else 0.0)
            row_size += left_size * (1 + abs(np.log(pr)) + abs(log_qr)) if pr > 0 and log_qr > -np.inf else 0.0
        f += lam * w * row if lam else 0  # (a term that is switched off adds nothing, an infinite one neither)
        f_size += lam * w * row_size
        grad[i] = lam * w / temperature * (mass * q - phat - pr * share)
        size[i] = lam * w / temperature * (mass * q * (64 + 6 * far / temperature) + pr * share * (64 + 6 * near / temperature) + ksize)
        if y >= 0 and label_lam:
            ls = _log_softmax(x[i])
            one = np.zeros(v, L)
            one[y] = 1
            f -= label_lam * w * ls[y]
            if np.isfinite(ls[y]):
                f_size += label_lam * w * (64 + 8 * (abs(ls[y]) + 2 * abs(x[i][y])))
            grad[i] += label_lam * w * (np.exp(ls) - one)
            size[i] += label_lam * w * (np.exp(ls) * (64 + 6 * far) + one)
    return float(f), grad.astype(np.float64), size.astype(np.float64), float(f_size)


def balance(r, k, *, offsets=None, mask=None, chosen=None, lam=1.0):
    """(f, gradient, counts, size of the gradient's terms, size of the value's terms)"""
    r = np.asarray(r, L)
    n, e = r.shape
    offsets = [0, n] if offsets is None else offsets
    mask = np.ones(n, bool) if mask is None else np.asarray(mask, bool)
    counts = np.zeros((len(offsets) - 1, e), np.int64)
    f, f_size = L(0), L(0)
    grad, size = np.zeros((n, e), L), np.zeros((n, e), L)
    for g, (a, b) in enumerate(zip(offsets, offsets[1:])):
        tokens, bad = [t for t in range(a, b) if mask[t]], False
        for t in tokens:
            if chosen is not None:
                picks = [int(c) for c in chosen[t]]
                bad |= any(c < -1 or c >= e for c in picks)
                picks = [c for c in picks if 0 <= c < e]
            else:
                order = sorted((j for j in range(e) if r[t, j] > -np.inf), key=lambda j: (-r[t, j], j))  # NaN and -inf are never chosen
                picks = order[:k]
            for c in picks:
                counts[g, c] += 1
        if not tokens:
            continue
        ag = L(lam) * e / (L(k) * len(tokens) ** 2)
        c = counts[g].astype(L)
        for t in tokens:
            if bad or np.isnan(r[t]).any() or np.isposinf(r[t]).any():
                f = L(np.nan)
                grad[t] = np.nan
                continue
            if np.all(r[t] == -np.inf):
                continue
            p = np.exp(_log_softmax(r[t]))
            far = np.where(p > 0, (r[t].max() - r[t]) / np.log(L(2)), 0.0)
            d = (c * p).sum()
            f += ag * d
            spread = (c * p * (64 + 6 * far)).sum()
            f_size += ag * (spread + 64 * d)
            grad[t] = ag * p * (c - d)
            size[t] = ag * p * ((c + d) * (64 + 6 * far) + spread)
    return float(f), grad.astype(np.float64), counts, size.astype(np.float64), float(f_size)
