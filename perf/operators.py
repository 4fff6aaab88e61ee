"""Cases of the distillation operators: the teacher's best scores, the losses on a student's logits and on its last
linear layer, and their gradients.

A forest's scores over classes (or any teacher's logits) are cut down to the k best of each row, and a small network
is trained on those.  Four operators:

top          the k largest scores of each row in descending order (equal ones: lowest class first), their classes, and
             the row's log sum exp; scores may be probabilities, whose logarithms are then the values
distill      T^2 KL(teacher || student) over the teacher's top classes, from the student's logits
linear_ce    softmax cross entropy from a linear layer's input and weight, the logits not being kept
linear_top   `distill` from a linear layer's input and weight

With `own` false, `run` computes them in elementary torch operations in 32 bits; with `own` true it calls
`cuml_b200.distill`.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "fp64": torch.float64, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "fp64": 8, "bf16": 2, "fp16": 2}
_MOST = 8192 * 2048 * 131072  # rows x width x classes of the largest case on a linear layer


def _top(name, rows, classes, k, dtype, probabilities=False, temperature=1.0):
    return {"name": name, "op": "top", "rows": rows, "classes": classes, "k": k, "dtype": dtype,
            "probabilities": probabilities, "temperature": temperature}


def _distill(name, rows, classes, k, dtype, tail="renormalise", temperature=1.0, reduction="mean", train=True):
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "k": k, "dtype": dtype, "tail": tail,
            "temperature": temperature, "reduction": reduction, "train": train}


def _linear(name, op, rows, width, classes, k, dtype, temperature=1.0, reduction="mean", train=True):
    return {"name": name, "op": op, "rows": rows, "width": width, "classes": classes, "k": k, "dtype": dtype,
            "temperature": temperature, "reduction": reduction, "train": train}


def listed():
    return [
        # the answers of a ten-class forest to a large batch, most probable three classes of each row
        _top("top_forest_10", 1_000_003, 10, 3, "fp32", probabilities=True),
        # one row of a teacher with many classes, as a service asks for it: latency
        _top("top_one_row", 1, 50_001, 20, "fp32"),
        # a batch of teacher logits over many classes, cut down to what is stored for training
        _top("top_32k", 4096, 32_768, 64, "bf16", temperature=2.0),
        # a mini-batch of a ten-class student: latency of a training step's loss and gradient
        _distill("distill_batch_10", 64, 10, 3, "fp32", tail="bucket", temperature=2.0),
        # a student over a thousand classes, weights per row, odd sizes
        _distill("distill_1001", 8191, 1001, 16, "fp16", tail="bucket", reduction="none"),
        # the same loss without a gradient, as an evaluation takes it
        _distill("distill_eval_8k", 4096, 8192, 32, "fp32", train=False),
        # many classes: logits of 1 GB
        _distill("distill_128k", 4096, 131_072, 64, "bf16", temperature=2.0),
        # the last layer of a small student
        _linear("linear_ce_small", "linear_ce", 256, 128, 1000, 1, "bf16"),
        # odd sizes throughout
        _linear("linear_ce_odd", "linear_ce", 1999, 712, 10_007, 1, "fp16", reduction="sum"),
        # the largest: logits would take 2 GB in bf16 and 4 GB in fp32
        _linear("linear_ce_128k", "linear_ce", 8192, 2048, 131_072, 1, "bf16"),
        # distillation from a linear layer, ordinary and with many classes
        _linear("linear_top_1k", "linear_top", 2048, 512, 1000, 16, "bf16", temperature=2.0),
        _linear("linear_top_50k", "linear_top", 4096, 1024, 50_001, 32, "bf16", reduction="none"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["top", "distill", "linear_ce", "linear_top"])
    temperature = rng.choice([1.0, 1.0, 2.0, 4.0])
    reduction = rng.choice(["mean", "mean", "sum", "none"])
    train = rng.random() < 0.75
    if op in ("top", "distill"):
        classes = _spread(rng, 2, 131_072)
        rows = _spread(rng, 1, min(1_000_000, 2 ** 28 // classes))
        k = min(classes, _spread(rng, 1, 128))
        if op == "top":
            return _top(None, rows, classes, k, rng.choice(["fp32", "fp32", "bf16", "fp16", "fp64"]),
                        rng.random() < 0.3, temperature)
        return _distill(None, rows, classes, k, rng.choice(["fp32", "bf16", "fp16"]),
                        rng.choice(["renormalise", "bucket"]), temperature, reduction, train)
    width = _spread(rng, 32, 2048)
    if rng.random() < 0.8:
        width = (width + 7) // 8 * 8
    classes = _spread(rng, 2, 131_072)
    rows = min(_spread(rng, 1, 8192), max(1, _MOST // 8 // (width * classes)))
    k = 1 if op == "linear_ce" else min(classes, _spread(rng, 1, 64))
    return _linear(None, op, rows, width, classes, k, rng.choice(["bf16", "fp16"]),
                   1.0 if op == "linear_ce" else temperature, reduction, train)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _best(scores, k):
    """(values, classes) of the k largest of each row; here only to make inputs."""
    v, i = torch.topk(scores, k, dim=1)
    return v.float(), i.to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    n, c, k, op = case["rows"], case["classes"], case["k"], case["op"]
    dtype = _TYPES[case["dtype"]]
    state = {"case": case}
    if op == "top":
        if case["probabilities"]:
            # averaged votes of a forest: many classes have none
            x = torch.rand((n, c), generator=g, device=dev).mul_(30.0).sub_(10.0).clamp_(min=0).round_()
            x[:, 0].add_(1)
            state["scores"] = x.div_(x.sum(1, keepdim=True)).to(dtype)
        else:
            state["scores"] = torch.randn((n, c), generator=g, device=dev, dtype=torch.float32).mul_(3).to(dtype)
        return state
    if op == "distill":
        z = torch.randn((n, c), generator=g, device=dev, dtype=torch.float32).mul_(2)
        t = torch.randn((n, c), generator=g, device=dev, dtype=torch.float32).add_(z)
        state["values"], state["index"] = _best(t, k)
        state["logsumexp"] = torch.logsumexp(t.div_(case["temperature"]), 1)
        state["logits"] = z.to(dtype).requires_grad_(case["train"])
    else:
        d = case["width"]
        h = torch.randn((n, d), generator=g, device=dev)
        w = torch.randn((c, d), generator=g, device=dev).mul_(2 / math.sqrt(d))
        if op == "linear_ce":
            target = torch.randint(0, c, (n,), generator=g, device=dev)
            padded = torch.rand((n,), generator=g, device=dev) < 0.05
            padded[0] = False
            state["target"] = torch.where(padded, -100, target)
        else:
            i = torch.randint(0, c, (n, 1), generator=g, device=dev)
            step = torch.randint(0, c, (n, 1), generator=g, device=dev)
            # k different classes of each row, evenly spaced
            state["index"] = ((i + torch.arange(k, device=dev)) % c if c < 4 * k else
                              (i + torch.arange(k, device=dev) * (1 + step % (c // k - 1))) % c).to(torch.int32)
            state["values"] = torch.randn((n, k), generator=g, device=dev).mul_(3).sort(1, descending=True).values
        state["hidden"] = h.to(dtype).requires_grad_(case["train"])
        state["weight"] = w.to(dtype).requires_grad_(case["train"])
    if case["train"]:
        if case["reduction"] == "none":
            state["upstream"] = torch.rand((n,), generator=g, device=dev).add_(0.1)
        elif case["reduction"] == "mean" and case["dtype"] == "fp16":  # the loss scale of such a training
            state["upstream"] = torch.tensor(min(65536.0, 16.0 * n), device=dev)
    return state


# ---- the framework's operators -----------------------------------------------------------------------------------
def _own(state):
    from cuml_b200 import distill

    case = state["case"]
    op = case["op"]
    if op == "top":
        return tuple(distill.top_scores(state["scores"], case["k"], temperature=case["temperature"],
                                        probabilities=case["probabilities"]))
    if op == "distill":
        leaves = [state["logits"]]
        top = distill.TopScores(state["values"], state["index"], state["logsumexp"])
        loss = distill.distillation_loss(state["logits"], top, temperature=case["temperature"], tail=case["tail"],
                                         reduction=case["reduction"])
    else:
        leaves = [state["hidden"], state["weight"]]
        if op == "linear_ce":
            loss = distill.linear_cross_entropy(state["hidden"], state["weight"], state["target"],
                                                reduction=case["reduction"])
        else:
            top = distill.TopScores(state["values"], state["index"], None)
            loss = distill.linear_distillation_loss(state["hidden"], state["weight"], top,
                                                    temperature=case["temperature"], reduction=case["reduction"])
    if not case["train"]:
        return (loss,)
    grads = torch.autograd.grad(loss, leaves, state.get("upstream"))
    return (loss.detach(), *grads)


# ---- plain forms -------------------------------------------------------------------------------------------------
def _plain_top(state):
    case = state["case"]
    x = state["scores"]
    wide = x if x.dtype == torch.float64 else x.float()
    order = torch.sort(wide, dim=1, descending=True, stable=True)
    values, index = order.values[:, :case["k"]], order.indices[:, :case["k"]].to(torch.int32)
    if case["probabilities"]:
        # (the logarithm of a sum near 1 is a difference: in 64 bits)
        wide, values = wide.double().log(), values.log()
    y = wide / case["temperature"]
    m = y.max(1, keepdim=True).values
    lse = (y - m).exp().sum(1).log() + m[:, 0]
    return values.to(x.dtype), index, lse.to(order.values.dtype)


def _plain_rows(z, case, state):
    """Losses of the rows from 32-bit logits, and their gradients."""
    t = case["temperature"]
    if case["op"] == "linear_ce":
        target = state["target"]
        counted = target >= 0
        at = torch.where(counted, target, 0)[:, None]
        m = z.max(1, keepdim=True).values
        e = (z - m).exp()
        s = e.sum(1, keepdim=True)
        loss = (s.log() + m - z.gather(1, at))[:, 0]
        loss = torch.where(counted, loss, 0.0)
        if not case["train"]:
            return loss, None, counted
        d = e.div_(s)
        d.scatter_add_(1, at, torch.full_like(at, -1, dtype=d.dtype))
        return loss, d.mul_(counted[:, None]), counted
    at = state["index"].long()
    # (the two sides' logarithms nearly cancel: in 64 bits)
    v = state["values"].double() / t
    if case.get("tail") == "bucket":
        log_p = v - state["logsumexp"].double()[:, None]
    else:
        log_p = v - v.max(1, keepdim=True).values
        log_p = log_p - log_p.exp().sum(1, keepdim=True).log()
    p = log_p.exp().float()
    y = z / t
    m = y.max(1, keepdim=True).values
    e = (y - m).exp()
    s = e.sum(1, keepdim=True)
    log_q = (z.gather(1, at).double() - z.max(1, keepdim=True).values) / t - s.double().log()
    loss = (p * (log_p - log_q)).sum(1).float()
    q = e.div_(s)
    if case.get("tail") == "bucket":
        # (what is left of the teacher is a difference from 1: in 64 bits)
        p_rest = (1 - log_p.exp().sum(1)).clamp(min=0).float()
        if case["k"] == case["classes"]:
            p_rest = torch.zeros_like(p_rest)  # no class is left
        q_top = q.gather(1, at)
        q_rest = q.scatter(1, at, 0.0).sum(1)
        loss = loss + torch.where(p_rest > 0, p_rest * (p_rest.log() - q_rest.log()), 0.0)
        if case["train"]:
            q.mul_((1 - torch.where(p_rest > 0, p_rest / q_rest, 0.0))[:, None])
            q.scatter_(1, at, q_top)
    counted = torch.ones_like(loss, dtype=torch.bool)
    if not case["train"]:
        return loss * t * t, None, counted
    q.scatter_add_(1, at, -p)
    return loss * t * t, q.mul_(t), counted


def _plain(state):
    case = state["case"]
    if case["op"] == "top":
        return _plain_top(state)
    with torch.no_grad():
        linear = case["op"] != "distill"
        if linear:
            h, w = state["hidden"].float(), state["weight"].float()
            z = h @ w.t()
        else:
            z = state["logits"].float()
        loss, d, counted = _plain_rows(z, case, state)
        count = counted.sum()
        scale = 1.0
        if case["reduction"] == "mean":
            scale = 1.0 / count
        if case["reduction"] != "none":
            loss = loss.sum() * scale
        if not case["train"]:
            return (loss,)
        d = d * (state["upstream"][:, None] if case["reduction"] == "none" else scale * state.get("upstream", 1.0))
        if not linear:
            return loss, d.to(state["logits"].dtype)
        return loss, (d @ w).to(state["hidden"].dtype), (d.t() @ h).to(state["weight"].dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def _exact_gradient(z, case, state, a, b):
    """Losses of rows a to b and their gradients by the logits, from logits in 64 bits."""
    t = case["temperature"]
    y = (z / t).detach()
    log_q = torch.log_softmax(y, 1)
    q = log_q.exp()
    if case["op"] == "linear_ce":
        target = state["target"][a:b]
        keep = target.ge(0)
        p = torch.zeros_like(q)
        p[torch.arange(b - a, device=q.device), target.clamp(min=0)] = 1.0
        loss = -(p * log_q).sum(1)
        return loss * keep, (q - p) * keep[:, None]
    at = state["index"][a:b].long()
    v = state["values"][a:b].double() / t
    if case.get("tail") != "bucket":
        log_p = torch.log_softmax(v, 1)
        p = torch.zeros_like(q).scatter_(1, at, log_p.exp())
        loss = (log_p.exp() * (log_p - log_q.gather(1, at))).sum(1)
        return loss * t * t, (q - p) * t
    log_p = v - state["logsumexp"][a:b].double()[:, None]
    p_top = log_p.exp()
    p_rest = (1.0 - p_top.sum(1)).clamp(min=0) * float(case["k"] < case["classes"])
    best = torch.zeros_like(q, dtype=torch.bool).scatter_(1, at, True)
    q_rest = q.masked_fill(best, 0.0).sum(1)
    loss = (p_top * (log_p - log_q.gather(1, at))).sum(1) + torch.special.xlogy(p_rest, p_rest) \
        - torch.special.xlogy(p_rest, q_rest)
    d = torch.where(best, q, q - q * (torch.where(p_rest > 0, p_rest / q_rest, 0.0))[:, None])
    d.scatter_add_(1, at, -p_top)
    return loss * t * t, d * t


def exact(case, seed):
    state = prepare(case, seed)
    n, c, t = case["rows"], case["classes"], case["temperature"]
    step = max(1, min(n, 2 ** 27 // c))
    if case["op"] == "top":
        x = state["scores"]
        value, index, lse = [], [], []
        for a in range(0, n, step):
            y = x[a:a + step].double()
            # by class first, then (stably) by score: equal scores stay in the order of their classes
            order = torch.argsort(-y, dim=1, stable=True)[:, :case["k"]]
            y = y.log() if case["probabilities"] else y
            value.append(y.gather(1, order))
            index.append(order.to(torch.int32))
            lse.append(torch.logsumexp(y / t, 1))
        return torch.cat(value), torch.cat(index), torch.cat(lse)
    weight = torch.ones(n, dtype=torch.float64, device="cuda")
    if case["op"] == "linear_ce":
        weight = (state["target"] >= 0).double()
    if case["reduction"] == "mean":
        weight = weight / weight.sum()
    upstream = weight * state["upstream"].double() if "upstream" in state else weight
    linear = case["op"] != "distill"
    if linear:
        h, w = state["hidden"].detach().double(), state["weight"].detach().double()
        dw = torch.zeros_like(w)
    losses, grads = [], []
    for a in range(0, n, step):
        b = min(n, a + step)
        z = h[a:b] @ w.t() if linear else state["logits"][a:b].detach().double()
        loss, d = _exact_gradient(z, case, state, a, b)
        losses.append(loss)
        if case["train"]:
            d = d * upstream[a:b, None]
            grads.append(d @ w if linear else d if n * c <= 2 ** 28 else d.float())
            if linear:
                dw += d.t() @ h[a:b]
    loss = torch.cat(losses)
    if case["reduction"] != "none":
        loss = (loss * weight).sum()
    if not case["train"]:
        return (loss,)
    return (loss, torch.cat(grads), dw) if linear else (loss, torch.cat(grads))


def work(case):
    n, c, k, e = case["rows"], case["classes"], case["k"], _BYTES[case["dtype"]]
    if case["op"] == "top":
        return {"bytes": n * c * e + n * k * (e + 4) + n * max(4, e // 8 * 8), "flops": 3 * n * c}
    if case["op"] == "distill":
        both = 2 if case["train"] else 1
        return {"bytes": both * n * c * e + n * (8 * k + 8), "flops": 4 * both * n * c}
    d = case["width"]
    both = 2 if case["train"] else 1
    return {"bytes": both * (n + c) * d * e + n * (8 * k + 4), "flops": (6 if case["train"] else 2) * n * c * d}
