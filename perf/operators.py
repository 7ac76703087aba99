"""Cases of the class-logit operators: top_logits, distill_loss, distill_derivatives and
sample_classes, with their plain forms.

Rows of class logits [n, classes] come from a booster (few classes, f64, stored
class by class) or from a neural teacher or student (up to a few hundred
thousand classes, 16 or 32 bits, stored row by row).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}

MAX_ELEMENTS = 4096 * 64000  # the largest listed case


def listed():
    return [
        # a step of training a student over a large class set on stored teacher logits
        dict(name="distill_train_bf16_64000", op="distill", n=4096, classes=64000, k=64, dtype="bf16",
             layout="rows", grad=True, tail=True, weight=True, masked=0.0, temperature=2.0),
        # its evaluation, 32-bit logits, a power of two of classes
        dict(name="distill_eval_f32_131072", op="distill", n=512, classes=131072, k=128, dtype="f32",
             layout="rows", grad=False, tail=True, weight=False, masked=0.0, temperature=1.0),
        # an odd class count (rows start at any alignment), masked classes, renormalised teacher
        dict(name="distill_train_f16_50021", op="distill", n=1021, classes=50021, k=20, dtype="f16",
             layout="rows", grad=True, tail=False, weight=False, masked=0.05, temperature=1.0),
        # a booster's approximants: 10 classes, class by class, 64 bits
        dict(name="distill_train_f64_10_dim_major", op="distill", n=1000003, classes=10, k=4, dtype="f64",
             layout="dims", grad=True, tail=True, weight=True, masked=0.0, temperature=1.0),
        # one small batch: latency
        dict(name="distill_train_f32_1000", op="distill", n=8, classes=1000, k=16, dtype="f32",
             layout="rows", grad=True, tail=True, weight=False, masked=0.0, temperature=1.0),
        # what a teacher run stores for each of its rows
        dict(name="top_logits_bf16_64000", op="top", n=2048, classes=64000, k=64, dtype="bf16", layout="rows",
             masked=0.0, temperature=2.0),
        # a few rows of many classes
        dict(name="top_logits_f32_131071", op="top", n=8, classes=131071, k=128, dtype="f32", layout="rows",
             masked=0.0, temperature=1.0),
        # many rows of few classes
        dict(name="top_logits_f32_100", op="top", n=200000, classes=100, k=8, dtype="f32", layout="rows",
             masked=0.1, temperature=1.0),
        # one answer: latency
        dict(name="sample_bf16_32000_single", op="sample", n=1, classes=32000, dtype="bf16", layout="rows",
             masked=0.0, temperature=0.8, top_k=0, top_p=0.95, min_p=0.0, per_row=False),
        # a batch of answers under every filter, each row with its own settings
        dict(name="sample_bf16_128000_filters", op="sample", n=256, classes=128000, dtype="bf16", layout="rows",
             masked=0.02, temperature=1.0, top_k=50, top_p=0.9, min_p=0.02, per_row=True),
        # the plain softmax draw over an odd class count
        dict(name="sample_f32_131071_plain", op="sample", n=64, classes=131071, dtype="f32", layout="rows",
             masked=0.0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=False),
        # labels drawn from a booster's predictions
        dict(name="sample_f64_10_dim_major", op="sample", n=100000, classes=10, dtype="f64", layout="dims",
             masked=0.0, temperature=1.0, top_k=5, top_p=0.95, min_p=0.0, per_row=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["distill", "distill", "top", "sample", "sample"])
    if rng.random() < 0.25:  # a booster's rows
        dtype, layout = "f64", rng.choice(["dims", "rows"])
        classes = _log_int(rng, 2, 64)
    else:
        dtype, layout = rng.choice(["bf16", "bf16", "f16", "f32"]), "rows"
        classes = _log_int(rng, 2, 200000)
    most = {"distill": MAX_ELEMENTS // 4, "top": MAX_ELEMENTS // 8, "sample": MAX_ELEMENTS // 8}[op]
    most = most * 2 // SIZES[dtype]
    n = _log_int(rng, 1, max(1, min(1000000, most // classes)))
    case = dict(op=op, n=n, classes=classes, dtype=dtype, layout=layout,
                masked=rng.choice([0.0, 0.0, 0.1]), temperature=rng.choice([0.5, 0.7, 1.0, 1.0, 1.5, 2.0]))
    if op == "sample":
        case.update(top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95]),
                    min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), per_row=rng.random() < 0.3)
    else:
        case["k"] = _log_int(rng, 1, min(128, classes))
    if op == "distill":
        case.update(grad=rng.random() < 0.7, tail=rng.random() < 0.5, weight=rng.random() < 0.5)
    return case


# ---- inputs ----------------------------------------------------------------

def _logits(case, gen, spread=2.0, shared=None):
    """f32 rows as a model gives them: classes of different popularity, rows around it, and a few
    classes of each row far above the rest."""
    n, V = case["n"], case["classes"]
    dev = gen.device
    x = torch.randn((n, V), generator=gen, device=dev)
    x.mul_(spread)
    if shared is not None:
        x.add_(shared, alpha=0.8)
        return x
    x.add_(torch.randn((V,), generator=gen, device=dev) * 1.5)
    if V >= 100:
        at = torch.randint(0, V, (n, 8), generator=gen, device=dev)
        x.scatter_add_(1, at, 4.0 + 8.0 * torch.rand((n, 8), generator=gen, device=dev))
    if case["masked"]:
        off = torch.rand((V,), generator=gen, device=dev) < case["masked"]
        off[0] = False
        x.masked_fill_(off, -math.inf)
    return x


def _stored(x, case):
    x = x.to(DTYPES[case["dtype"]])
    return x.t().contiguous().t() if case["layout"] == "dims" else x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * (seed + 1) + 17)
    n, V, T = case["n"], case["classes"], case["temperature"]
    state = dict(case=case)
    teacher = _logits(case, gen)
    if case["op"] == "distill":
        student = _stored(_logits(case, gen, 1.0, teacher), case)
        teacher = teacher.to(DTYPES[case["dtype"]])
        value, index = torch.topk(teacher, case["k"], dim=1)
        state.update(logits=student, top_index=index.to(torch.int32), top_value=value, tail=None, weight=None)
        if case["tail"]:
            rest = teacher.scatter(1, index, -math.inf)
            wide = torch.float64 if case["dtype"] == "f64" else torch.float32
            state["tail"] = torch.logsumexp(rest.to(wide) / T, dim=1)
        if case["weight"]:
            state["weight"] = 0.5 + torch.rand((n,), generator=gen, device="cuda", dtype=torch.float64).to(
                torch.float64 if case["dtype"] == "f64" else torch.float32)
        return state
    state["logits"] = _stored(teacher, case)
    if case["op"] == "sample":
        state["uniform"] = torch.rand((n,), generator=gen, device="cuda")
        for key in ("temperature", "top_k", "top_p", "min_p"):
            state[key] = case[key]
        if case["per_row"]:
            state["temperature"] = T * (0.75 + 0.5 * torch.rand((n,), generator=gen, device="cuda"))
            if case["top_p"] < 1.0:
                state["top_p"] = case["top_p"] * (0.9 + 0.1 * torch.rand((n,), generator=gen, device="cuda"))
            state["min_p"] = case["min_p"] * torch.rand((n,), generator=gen, device="cuda")
            if case["top_k"] > 0:
                state["top_k"] = torch.randint(1, case["top_k"] + 1, (n,), generator=gen, device="cuda",
                                               dtype=torch.int32)
    return state


# ---- one pass --------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "distill":
        return _plain_distill(case, state)
    if case["op"] == "top":
        return _plain_top(case, state)
    return _plain_sample(case, state)


def _run_own(case, s):
    import catboost_rs_b200 as cb
    if case["op"] == "top":
        top = cb.top_logits(s["logits"], case["k"], temperature=case["temperature"])
        return {"value": top.value, "index": top.index, "tail": top.tail}
    if case["op"] == "sample":
        return {"index": cb.sample_classes(s["logits"], s["uniform"], temperature=s["temperature"],
                                           top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])}
    teacher = cb.TopLogits(s["top_index"], s["top_value"], s["tail"])
    if case["grad"]:
        d = cb.distill_derivatives(s["logits"], teacher, weight=s["weight"], temperature=case["temperature"])
        return {"loss": d.loss, "der1": d.der1}
    return {"loss": cb.distill_loss(s["logits"], teacher, weight=s["weight"], temperature=case["temperature"])}


def _wide(case):
    return torch.float64 if case["dtype"] == "f64" else torch.float32


def _plain_distill(case, s):
    # the loss is a difference of logarithms that nearly agree once the student is close to the
    # teacher: its sums are taken in 64 bits; the derivative in 32
    wide, T = _wide(case), case["temperature"]
    index = s["top_index"].long()
    z = s["top_value"].double() / T
    n, k = index.shape
    if s["tail"] is not None:
        z = torch.cat([z, s["tail"].double()[:, None]], dim=1)
    z = z - z.max(dim=1, keepdim=True).values
    total = z.exp().sum(dim=1, keepdim=True)
    q = z.exp() / total
    log_q = z - total.log()
    a = s["logits"].double() / T
    a = a - a.max(dim=1, keepdim=True).values
    e = a.exp()
    tail_sum = e.scatter(1, index, 0.0).sum(dim=1, keepdim=True)
    norm = tail_sum + e.gather(1, index).sum(dim=1, keepdim=True)
    log_p = a.gather(1, index) - norm.log()
    if s["tail"] is not None:
        log_p = torch.cat([log_p, tail_sum.log() - norm.log()], dim=1)
    terms = torch.where(q > 0, q * (log_q - log_p), torch.zeros_like(q))
    w = torch.ones((n,), dtype=wide, device=a.device) if s["weight"] is None else s["weight"]
    loss = (w * (T * T) * terms.sum(dim=1)).to(wide)
    if not case["grad"]:
        return {"loss": loss}
    del a
    e = e.to(wide).div_(norm.to(wide))
    top_p = e.gather(1, index)
    if s["tail"] is not None:
        share = torch.where(q[:, k:] > 0, q[:, k:] * norm / tail_sum, torch.zeros_like(norm))
        e.mul_((1.0 - share).to(wide))
    e.neg_()
    e.scatter_(1, index, q[:, :k].to(wide) - top_p)
    e.mul_((w * T)[:, None])
    der1 = e.to(s["logits"].dtype)
    if case["layout"] == "dims":
        der1 = der1.t().contiguous().t()
    return {"loss": loss, "der1": der1}


def _plain_top(case, s):
    wide, k = _wide(case), case["k"]
    value, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    x = value.to(wide) / case["temperature"]
    peak = x[:, :1]
    tail = (x[:, k:] - peak).exp().sum(dim=1).log() + peak[:, 0]
    return {"value": value[:, :k].contiguous(), "index": order[:, :k].to(torch.int32), "tail": tail}


def _per_row(v, n, dev):
    if isinstance(v, torch.Tensor):
        return v.to(torch.float64)[:, None]
    return torch.full((n, 1), float(v), dtype=torch.float64, device=dev)


def _plain_sample(case, s):
    # which class is drawn turns on the order of sums next to the drawn number: 64 bits
    x = s["logits"].to(torch.float64)
    n, V = x.shape
    e = ((x - x.max(dim=1, keepdim=True).values) / _per_row(s["temperature"], n, x.device)).exp()
    u = s["uniform"].to(torch.float64)[:, None]
    if case["top_k"] > 0 or case["top_p"] < 1.0 or case["min_p"] > 0.0:
        order = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices
        ranked = e.gather(1, order)
        if case["top_k"] > 0:
            rank = torch.arange(V, device=x.device)[None, :]
            ranked = torch.where(rank < _per_row(s["top_k"], n, x.device), ranked, torch.zeros_like(ranked))
        if case["top_p"] < 1.0:
            upto = ranked.cumsum(dim=1)
            keep = upto - ranked < _per_row(s["top_p"], n, x.device) * upto[:, -1:]
            ranked = torch.where(keep, ranked, torch.zeros_like(ranked))
        if case["min_p"] > 0.0:
            ranked = torch.where(ranked >= _per_row(s["min_p"], n, x.device), ranked, torch.zeros_like(ranked))
        e = torch.zeros_like(e).scatter_(1, order, ranked)
    upto = e.cumsum(dim=1)
    drawn = (upto <= u * upto[:, -1:]).sum(dim=1)
    return {"index": drawn.to(torch.int32)}


# ---- the cost of a pass ----------------------------------------------------

def work(case):
    n, V, es = case["n"], case["classes"], SIZES[case["dtype"]]
    wide = 8 if case["dtype"] == "f64" else 4
    if case["op"] == "sample":
        return {"bytes": n * V * es + 8 * n + (16 * n if case["per_row"] else 0), "flops": 4 * n * V}
    k = case["k"]
    if case["op"] == "top":
        return {"bytes": n * V * es + n * k * (es + 4) + wide * n, "flops": 4 * n * V}
    small = n * k * (4 + es) + n * wide * (1 + int(case["tail"]) + int(case["weight"]))
    if case["grad"]:
        return {"bytes": 2 * n * V * es + small, "flops": 6 * n * V}
    return {"bytes": n * V * es + small, "flops": 4 * n * V}


# ---- from the definition, in 64 bits ---------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    step = max(1, (1 << 25) // case["classes"])
    pieces = []
    for r0 in range(0, case["n"], step):
        r = slice(r0, min(case["n"], r0 + step))
        part = {k: (v[r] if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
        pieces.append({"distill": _exact_distill, "top": _exact_top, "sample": _exact_sample}[case["op"]](case, part))
    return {k: torch.cat([p[k] for p in pieces]) for k in pieces[0]}


def _exact_distill(case, s):
    # KL divergence of the buckets (one for each top class, one for the others together); its
    # derivative from d log p_j / d a_i = ([i = j] - p_i) / T
    T = float(case["temperature"])
    x = s["logits"].double()
    log_p = torch.log_softmax(x / T, dim=1)
    index = s["top_index"].long()
    n, V = x.shape
    in_top = torch.zeros((n, V), dtype=torch.bool, device=x.device)
    in_top.scatter_(1, index, torch.ones_like(index, dtype=torch.bool))
    buckets = s["top_value"].double() / T
    if case["tail"]:
        buckets = torch.cat((buckets, s["tail"].double().view(n, 1)), 1)
    log_t = torch.log_softmax(buckets, dim=1)
    t = log_t.exp()
    k = index.size(1)
    w = s["weight"].double() if case["weight"] else torch.ones(n, dtype=torch.float64, device=x.device)
    part = torch.special.xlogy(t[:, :k], t[:, :k]) - torch.where(t[:, :k] > 0, t[:, :k] * log_p.gather(1, index), 0.0)
    kl = part.sum(1)
    rest = log_p.masked_fill(in_top, -math.inf)
    if case["tail"]:
        log_rest = torch.logsumexp(rest, dim=1)
        kl = kl + torch.where(t[:, k] > 0, t[:, k] * (log_t[:, k] - log_rest), 0.0)
    out = {"loss": w * T * T * kl}
    if case["grad"]:
        target = torch.zeros((n, V), dtype=torch.float64, device=x.device).scatter_add_(1, index, t[:, :k])
        if case["tail"]:  # the others' bucket pulls on each of them by its share of the bucket
            target = target + torch.where(t[:, k:] > 0, t[:, k:] * (rest - log_rest[:, None]).exp(), 0.0)
        out["der1"] = (target - log_p.exp()) * (w * T)[:, None]
    return out


def _exact_top(case, s):
    x = s["logits"].double()
    order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case["k"]]
    rest = x.scatter(1, order, -math.inf)
    return {"value": x.gather(1, order), "index": order.to(torch.int32),
            "tail": torch.logsumexp(rest / float(case["temperature"]), dim=1)}


def _exact_sample(case, s):
    # row by row on the host for a few rows, else the same steps on whole pieces
    x = s["logits"].double()
    n, V = x.shape

    def setting(key):
        v = s[key]
        return v.double() if isinstance(v, torch.Tensor) else torch.full((n,), float(v), dtype=torch.float64,
                                                                          device=x.device)

    p = torch.softmax(x / setting("temperature")[:, None], dim=1)
    top = p.max(dim=1).values
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    place = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=x.device).expand(n, V).contiguous())
    if case["top_k"] > 0:
        p = p * (place < setting("top_k")[:, None])
    if case["top_p"] < 1.0:
        in_order = p.gather(1, order)
        before = torch.cat((torch.zeros((n, 1), dtype=torch.float64, device=x.device),
                            in_order.cumsum(1)[:, :-1]), 1)
        p = p * (before < setting("top_p")[:, None] * p.sum(1, keepdim=True)).gather(1, place)
    if case["min_p"] > 0.0:
        p = p * (p >= setting("min_p")[:, None] * top[:, None])
    edges = np.cumsum(p.cpu().numpy(), axis=1)
    u = s["uniform"].double().cpu().numpy()
    drawn = [int(np.searchsorted(edges[i], u[i] * edges[i, -1], side="right")) for i in range(n)]
    return {"index": torch.tensor(drawn, dtype=torch.int32, device=x.device)}
