"""Measured cases of the losses on rows of scores: ``DistillationLoss`` and ``BalanceLoss``.

``own`` false: the operators in elementary torch operations, in 32 bits (totals over many rows in 64), rounded once at the end.
``own`` true: the calls a user's program makes.  Either way one pass is the value AND the gradient; a balance pass also returns
the counts per expert."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEVICE = "cuda"


def listed():
    """Sizes are generic: vocabularies around 32768 ... 131072, heads of a few hundred classes, 64 ... 256 experts."""
    return [
        # distillation ------------------------------------------------------------------------------------------------------
        # the answer tokens of one short prompt: a call is launch and latency
        distill("distill-answer", 8, 32768, 16, "f32"),
        # a line search on a few long rows: too few rows to fill the device one by one
        distill("distill-few-rows", 24, 131072, 64, "bf16", rest=True),
        # a classifier's head: many short rows of odd length, labels mixed in
        distill("distill-head", 65536, 1003, 5, "f32", labels=True),
        # odd vocabulary, rows at every alignment, padded rows, labels, temperature
        distill("distill-odd", 1021, 50001, 20, "f16", labels=True, temperature=2.0, padded=0.3),
        # one training step's tokens
        distill("distill-step", 4096, 32768, 64, "bf16"),
        # a solver's own precision, the teacher's mass outside its list as one class
        distill("distill-f32-rest", 2048, 65536, 50, "f32", rest=True, temperature=1.5),
        # the same with long lists, scores in a buffer wider than the vocabulary
        distill("distill-rest", 2048, 131000, 200, "bf16", rest=True, temperature=2.0, gap=72),
        # the largest: a full batch over a long vocabulary
        distill("distill-largest", 8192, 131072, 64, "bf16"),
        # balance -----------------------------------------------------------------------------------------------------------
        # the router of one small batch: latency
        balance("balance-small", 64, 64, 6, "f32"),
        # one training step's tokens, one group
        balance("balance-step", 16384, 128, 8, "bf16"),
        # the balance of each sequence by itself: ragged lengths, padded tokens
        balance("balance-sequences", 32771, 64, 6, "f32", groups=61, padded=0.2),
        # the largest: a full batch, many experts
        balance("balance-largest", 131072, 256, 8, "f32"),
    ]


def distill(name, rows, classes, top, dtype, rest=False, labels=False, temperature=1.0, padded=0.0, gap=0):
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "top": top, "dtype": dtype, "rest": rest,
            "labels": labels, "temperature": temperature, "padded": padded, "gap": gap}


def balance(name, tokens, experts, k, dtype, groups=1, padded=0.0):
    return {"name": name, "op": "balance", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "groups": groups,
            "padded": padded}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    dtype = rng.choice(["f32", "bf16", "f16"])
    if rng.random() < 0.6:
        classes = _spread(rng, 500, 131072)
        rows = _spread(rng, 1, max(1, min(65536, 8192 * 131072 * 2 // (classes * SIZE[dtype]))))
        c = distill("", rows, classes, min(classes, _spread(rng, 1, 256)), dtype, rest=rng.random() < 0.4, labels=rng.random() < 0.3,
                    temperature=rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]), padded=rng.choice([0.0, 0.0, 0.25]), gap=rng.choice([0, 0, 0, 8, 13]))
    else:
        experts = _spread(rng, 4, 512)
        tokens = _spread(rng, 16, max(16, min(131072, 131072 * 256 // experts)))
        c = balance("", tokens, experts, min(experts, _spread(rng, 1, 16)), dtype, groups=rng.choice([1, 1, _spread(rng, 1, 64)]),
                    padded=rng.choice([0.0, 0.0, 0.25]))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _per_row(case, n):
    """A mean over the rows; in half precision times a loss scale, without which most of a gradient's entries leave its range."""
    return 32.0 if case["dtype"] == "f16" else 1.0 / n


def prepare(case, seed):
    return (_prepare_distill if case["op"] == "distill" else _prepare_balance)(case, seed)


def _prepare_distill(case, seed):
    g = _generator(seed)
    n, v, k, dt = case["rows"], case["classes"], case["top"], TYPES[case["dtype"]]
    buffer = torch.empty(n, v + case["gap"], dtype=dt, device=DEVICE).normal_(0.0, 2.0, generator=g)
    scores = buffer[:, :v]
    # the listed classes: distinct, anywhere in the vocabulary; logits fall along the list as a sorted list's do
    first = torch.randint(0, v, (n, 1), device=DEVICE, generator=g)
    step = max(1, v // k)
    index = ((first + torch.arange(k, device=DEVICE) * step) % v).to(torch.int32)
    teacher = (torch.randn(n, k, device=DEVICE, generator=g) * 2.0 + 9.0).sort(dim=1, descending=True).values
    # the student has learnt something: its scores at the listed classes follow the teacher's, with noise
    seen = teacher * 0.9 + torch.randn(n, k, device=DEVICE, generator=g)
    scores.scatter_(1, index.long(), seen.to(dt))
    teacher = teacher.to(dt)
    state = {"case": case, "scores": scores, "teacher": teacher, "index": index, "lse": None, "weights": None, "labels": None,
             "temperature": case["temperature"], "lam": case["temperature"] ** 2 * _per_row(case, n), "label_lam": 0.0}
    if case["rest"]:  # the teacher's own normaliser: its list covers between 60 and 99 per cent of its mass
        covered = torch.rand(n, device=DEVICE, generator=g) * 0.39 + 0.6
        state["lse"] = torch.logsumexp(teacher.float() / case["temperature"], dim=1) - covered.log()
    if case["padded"]:
        state["weights"] = (torch.rand(n, device=DEVICE, generator=g) >= case["padded"]).float()
    if case["labels"]:
        labels = torch.randint(0, v, (n,), device=DEVICE, generator=g)
        state["labels"] = torch.where(torch.rand(n, device=DEVICE, generator=g) < 0.1, -1, labels).to(torch.int32)  # some unlabelled
        state["label_lam"] = 0.5 * _per_row(case, n)
    if own:
        import proximalalgorithms.jl_amd as pa

        state["loss"] = pa.DistillationLoss(teacher, index, v, temperature=state["temperature"], lam=state["lam"], teacher_lse=state["lse"],
                                            weights=state["weights"], labels=state["labels"], label_lam=state["label_lam"])
        state["grad"] = torch.empty_like(buffer)[:, :v]
    return state


def _prepare_balance(case, seed):
    g = _generator(seed)
    n, e, dt = case["tokens"], case["experts"], TYPES[case["dtype"]]
    lean = torch.randn(e, device=DEVICE, generator=g) * 0.7  # some experts are liked more than others
    scores = (torch.randn(n, e, device=DEVICE, generator=g) + lean).to(dt)
    offsets = None
    if case["groups"] > 1:
        cuts = torch.randint(0, n + 1, (case["groups"] - 1,), generator=torch.Generator().manual_seed(seed)).sort().values.tolist()
        offsets = [0] + cuts + [n]
    mask = (torch.rand(n, device=DEVICE, generator=g) >= case["padded"]) if case["padded"] else None
    state = {"case": case, "scores": scores, "offsets": offsets, "mask": mask, "lam": 0.01 * n * _per_row(case, n), "k": case["k"]}
    if own:
        import proximalalgorithms.jl_amd as pa

        state["loss"] = pa.BalanceLoss(n, e, case["k"], offsets=offsets, mask=mask, lam=state["lam"])
        state["grad"] = torch.empty_like(scores)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------------


def run(state):
    if own:
        value, grad = state["loss"].value_and_gradient_async(state["scores"], out=state["grad"])
        if state["case"]["op"] == "distill":
            return {"value": value, "grad": grad}
        return {"value": value, "grad": grad, "counts": state["loss"].counts}
    return (_plain_distill if state["case"]["op"] == "distill" else _plain_balance)(state)


def _plain_distill(s):
    x, index, inv_t = s["scores"].float(), s["index"].long(), 1.0 / s["temperature"]
    t = s["teacher"].float() * inv_t
    z = x * inv_t
    top = z.max(dim=1, keepdim=True).values
    q = torch.exp(z - top)
    total = q.sum(dim=1, keepdim=True)
    lse = top + torch.log(total)
    if s["lse"] is None:
        log_p = t - t.max(dim=1, keepdim=True).values
        log_p = log_p - torch.log(torch.exp(log_p).sum(dim=1, keepdim=True))
    else:
        log_p = t - s["lse"][:, None]
    p = torch.exp(log_p)
    loss = (p * (log_p - (z.gather(1, index) - lse))).sum(dim=1)
    if s["lse"] is None:
        grad = q / total
    else:
        # 64 bits: one minus a sum near one
        p_rest = (1.0 - torch.exp(t.double() - s["lse"].double()[:, None]).sum(dim=1)).clamp(min=0.0)
        others = q.scatter(1, index, 0.0).sum(dim=1, keepdim=True)
        q_rest = others / total
        inside = torch.where(p_rest > 0, p_rest * (torch.log(p_rest) - torch.log(q_rest[:, 0].double())), 0.0)
        loss = loss + inside.float()
        mass = p.sum(dim=1, keepdim=True) + p_rest[:, None].float()
        at = q.gather(1, index) / total * mass
        grad = (q / total) * (mass - p_rest[:, None].float() / q_rest)
        grad.scatter_(1, index, at)
    grad.scatter_add_(1, index, -p)
    w = torch.ones_like(loss) if s["weights"] is None else s["weights"]
    grad = grad * (w * (s["lam"] * inv_t))[:, None]
    value = s["lam"] * (w * loss).double().sum()
    if s["labels"] is not None:
        top = x.max(dim=1, keepdim=True).values
        q = torch.exp(x - top)
        total = q.sum(dim=1, keepdim=True)
        label = s["labels"].long()
        has = (label >= 0).float() * w
        at = label.clamp(min=0)[:, None]
        value = value + s["label_lam"] * (has * (top + torch.log(total) - x.gather(1, at))[:, 0]).double().sum()
        q = q / total
        q.scatter_add_(1, at, torch.full_like(total, -1.0))
        grad = grad + q * (s["label_lam"] * has)[:, None]
    return {"value": value.float(), "grad": grad.to(s["scores"].dtype)}


def _plain_balance(s):
    r, k, n = s["scores"].float(), s["k"], s["scores"].shape[0]
    e = r.shape[1]
    valid = torch.ones(n, dtype=torch.bool, device=r.device) if s["mask"] is None else s["mask"]
    alive = valid & (r > -math.inf).any(dim=1)
    # the k highest scores, the lowest index first among equals
    left, chosen, lanes = r.clone(), torch.zeros_like(r), torch.arange(e, device=r.device)
    for _ in range(k):
        best = left.max(dim=1, keepdim=True).values
        at = torch.where(left == best, lanes, e).min(dim=1, keepdim=True).values
        chosen.scatter_(1, at, (best > -math.inf).float())
        left.scatter_(1, at, -math.inf)
    chosen = chosen * valid[:, None]
    p = torch.exp(r - r.max(dim=1, keepdim=True).values)
    p = p / p.sum(dim=1, keepdim=True)
    p = torch.where(alive[:, None], p, 0.0)
    offsets = s["offsets"] or [0, n]
    lengths = torch.tensor([b - a for a, b in zip(offsets, offsets[1:])], device=r.device)
    group = torch.repeat_interleave(torch.arange(len(lengths), device=r.device), lengths)
    counts = torch.zeros(len(lengths), e, device=r.device).index_add_(0, group, chosen)
    tokens = torch.zeros(len(lengths), device=r.device).index_add_(0, group, valid.float())
    scale = torch.where(tokens > 0, s["lam"] * e / (k * tokens * tokens), 0.0)
    c = counts[group]
    d = (p * c).sum(dim=1, keepdim=True)
    value = (scale[group] * d[:, 0]).double().sum()
    grad = scale[group][:, None] * p * (c - d)
    return {"value": value.float(), "grad": grad.to(s["scores"].dtype), "counts": counts.to(torch.int32)}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "distill":
        n, v, k = case["rows"], case["classes"], case["top"]
        live = n * (1.0 - case["padded"])  # a padded row's scores are not needed, its gradient is zeros
        read = live * v * size + n * k * (size + 4) + (4 * n if case["rest"] else 0) + (4 * n if case["labels"] else 0) + (4 * n if case["padded"] else 0)
        # forward: subtract, exp, add; backward: subtract, exp, multiply; once more at temperature 1 for the labels
        return {"bytes": read + n * v * size + 4, "flops": live * v * (12 if case["labels"] and case["temperature"] != 1.0 else 6)}
    n, e, k = case["tokens"], case["experts"], case["k"]
    live = n * (1.0 - case["padded"])
    # softmax, the k largest, the product with the counts, the gradient
    return {"bytes": live * e * size + n * e * size + (n if case["padded"] else 0) + 4 * case["groups"] * e + 4, "flops": live * e * (8 + k)}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        return _exact_distill(s)
    return _exact_balance(s)


def _exact_distill(s):
    """Block by block of rows: KL(P || Q) with the classes outside the list as one more class where the normaliser is known."""
    n, v = s["scores"].shape
    big_t = float(s["temperature"])
    value, parts = 0.0, []
    block = max(1, (1 << 26) // v)
    for a in range(0, n, block):
        b = min(n, a + block)
        x = s["scores"][a:b].double()
        idx = s["index"][a:b].long()
        t = s["teacher"][a:b].double() / big_t
        norm = torch.logsumexp(t, 1) if s["lse"] is None else s["lse"][a:b].double()
        target = torch.zeros_like(x).scatter_add_(1, idx, torch.exp(t - norm[:, None]))
        log_q = torch.log_softmax(x / big_t, 1)
        q = log_q.exp()
        listed_p, listed_q = target.gather(1, idx), log_q.gather(1, idx)
        loss = (torch.special.xlogy(listed_p, listed_p) - listed_p * listed_q).sum(1)
        grad = q * target.sum(1, keepdim=True) - target
        if s["lse"] is not None:
            outside = torch.ones_like(x).scatter_(1, idx, 0.0)
            pr = torch.clamp(1.0 - target.sum(1), min=0.0)
            qr = (q * outside).sum(1)
            loss = loss + torch.special.xlogy(pr, pr) - torch.special.xlogy(pr, qr)
            grad = grad + pr[:, None] * (q - outside * q / qr[:, None])
        w = torch.ones_like(loss) if s["weights"] is None else s["weights"][a:b].double()
        grad = grad * (w * s["lam"] / big_t)[:, None]
        value += s["lam"] * float((w * loss).sum())
        if s["labels"] is not None:
            y = s["labels"][a:b].long()
            on = torch.where(y >= 0, w, 0.0) * s["label_lam"]
            logs = torch.log_softmax(x, 1)
            one = torch.zeros_like(x).scatter_(1, y.clamp(min=0)[:, None], 1.0)
            value -= float((on[:, None] * one * logs).sum())
            grad = grad + on[:, None] * (logs.exp() - one)
        parts.append(grad)
    return {"value": value, "grad": torch.cat(parts)}


def _exact_balance(s):
    r = s["scores"].double()
    n, e = r.shape
    k = s["k"]
    order = torch.sort(r, dim=1, descending=True, stable=True).indices[:, :k]
    valid = torch.ones(n, dtype=torch.bool, device=r.device) if s["mask"] is None else s["mask"]
    offsets = s["offsets"] or [0, n]
    probability = torch.softmax(r, 1)
    value, counts, grad = 0.0, [], torch.zeros_like(r)
    for a, b in zip(offsets, offsets[1:]):
        on = valid[a:b]
        m = int(on.sum())
        c = torch.bincount(order[a:b][on].reshape(-1), minlength=e)
        counts.append(c)
        if m == 0:
            continue
        scale = s["lam"] * e / (k * m * m)
        p = probability[a:b] * on[:, None]
        value += scale * float((p.sum(0) * c).sum())
        # d sum_e c_e p_e / d r_j = p_j c_j - p_j sum_e c_e p_e
        grad[a:b] = scale * (p * c - p * (p @ c.double())[:, None])
    return {"value": value, "grad": grad, "counts": torch.stack(counts)}
