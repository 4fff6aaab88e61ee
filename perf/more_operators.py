"""Cases of scoring a classifier's answers and of clipping gradients.

A student (or any classifier) that answers over classes is scored, trained on the scores and its gradients are
clipped before the optimizer takes them.  Three operators:

log_probs   log probability of each row's given class, the row's entropy and its best alternatives, from logits;
            rows whose class is ignored, or whose classes are all masked, give 0 (alternatives: 0 and class -1)
linear      the same without alternatives from a linear layer's input and weight, the logits not being kept
clip        the norm of all gradients of a model together, and the gradients scaled down to a largest norm, in place
            or to tensors of their own

With `own` false, `run` computes them in elementary torch operations in 32 bits; with `own` true it calls
`cuml_b200.distill`.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_MOST = 8192 * 2048 * 131072  # rows x width x classes of the largest case on a linear layer


def _logits(name, rows, classes, dtype, top=0, masked=False, temperature=1.0, train=True):
    return {"name": name, "op": "log_probs", "rows": rows, "classes": classes, "dtype": dtype, "top": top,
            "masked": masked, "temperature": temperature, "train": train}


def _linear(name, rows, width, classes, dtype, temperature=1.0, train=True):
    return {"name": name, "op": "linear", "rows": rows, "width": width, "classes": classes, "dtype": dtype,
            "temperature": temperature, "train": train}


def _clip(name, features, width, layers, classes, dtype, out, clipped, flat=False, largest=False):
    return {"name": name, "op": "clip", "features": features, "width": width, "layers": layers, "classes": classes,
            "dtype": dtype, "out": out, "clipped": clipped, "flat": flat, "largest": largest}


def listed():
    return [
        # one answer over many classes with its alternatives, as a service gives it: latency
        _logits("score_one_row", 1, 50_001, "fp32", top=20, train=False),
        # a mini-batch of a policy over ten actions, some of them masked: latency of a step's scores and gradient
        _logits("score_policy_10", 64, 10, "fp32", masked=True),
        # a ten-class forest's or student's answers to a large batch, with the best three classes
        _logits("score_eval_10", 1_000_003, 10, "fp32", top=3, train=False),
        # a batch over many classes, evaluated with alternatives
        _logits("score_eval_32k", 4096, 32_768, "bf16", top=8, train=False),
        # a training step over a thousand classes, odd sizes
        _logits("score_train_1001", 8191, 1001, "fp16", temperature=2.0),
        # the largest: logits of 1 GB
        _logits("score_train_128k", 4096, 131_072, "bf16"),
        # the last layer of a small student, trained on its own scores
        _linear("linear_small", 256, 128, 1000, "bf16"),
        # evaluation of a layer with many classes, odd sizes throughout
        _linear("linear_eval_50k", 1999, 712, 50_001, "fp16", temperature=2.0, train=False),
        # the largest layer: logits would take 2 GB in bf16 and 4 GB in fp32
        _linear("linear_train_128k", 8192, 2048, 131_072, "bf16"),
        # gradients of a small student in place, not above the largest norm: latency of an ordinary step
        _clip("clip_small", 64, 128, 2, 10, "fp32", "", False),
        # some hundred tensors of odd sizes that lie one after the other in a buffer, as they are exchanged; clipped
        # copies in 32 bits for an optimizer of 32-bit weights
        _clip("clip_deep", 333, 1001, 96, 1003, "fp16", "fp32", True, flat=True),
        # the largest: a billion gradients
        _clip("clip_billion", 1024, 8192, 16, 1000, "bf16", "bf16", True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["log_probs", "log_probs", "linear", "clip"])
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    train = rng.random() < 0.7
    if op == "log_probs":
        classes = _spread(rng, 2, 131_072)
        rows = _spread(rng, 1, min(1_000_000, 2 ** 28 // classes))
        masked = rng.random() < 0.3
        top = 0 if rng.random() < 0.5 else min(classes, _spread(rng, 1, 128))
        return _logits(None, rows, classes, rng.choice(["fp32", "bf16", "fp16"]), top, masked, temperature, train)
    if op == "linear":
        width = _spread(rng, 32, 2048)
        if rng.random() < 0.8:
            width = (width + 7) // 8 * 8
        classes = _spread(rng, 2, 131_072)
        rows = min(_spread(rng, 1, 8192), max(1, _MOST // 8 // (width * classes)))
        return _linear(None, rows, width, classes, rng.choice(["bf16", "fp16"]), temperature, train)
    width = _spread(rng, 8, 4096)
    flat = rng.random() < 0.5
    layers = min(_spread(rng, 1, 128 if flat else 30), max(1, 2 ** 28 // width ** 2))
    dtype, clipped = rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5
    # (in place only what is not clipped: a pass then leaves the same work for the next)
    out = rng.choice([dtype, "fp32"]) if clipped or rng.random() < 0.5 else ""
    return _clip(None, _spread(rng, 2, 1000), width, layers, _spread(rng, 2, 10_000), dtype, out, clipped,
                 flat, rng.random() < 0.2)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _shapes(case):
    """Weights and biases of a network of `layers` hidden layers."""
    sizes = [case["features"]] + [case["width"]] * case["layers"] + [case["classes"]]
    return [s for a, b in zip(sizes, sizes[1:]) for s in ((b, a), (b,))]


def _tensors(state, flat, shapes, dtype, dev):
    """Tensors of their own, or one after the other in the buffer state[flat]."""
    if not state["case"]["flat"]:
        return [torch.zeros(s, dtype=dtype, device=dev) for s in shapes]
    state[flat] = torch.zeros(sum(math.prod(s) for s in shapes), dtype=dtype, device=dev)
    return [x.view(s) for x, s in zip(state[flat].split([math.prod(s) for s in shapes]), shapes)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "clip":
        shapes = _shapes(case)
        unit = 1024.0 if case["dtype"] == "fp16" else 1.0  # the loss scale of such a training
        each = (2.5 if case["clipped"] else 0.4) * unit / math.sqrt(sum(math.prod(s) for s in shapes))
        state["gradients"] = _tensors(state, "flat", shapes, dtype, dev)
        for x in state["gradients"]:
            size = each * (0.5 + torch.rand((), generator=g, device=dev))
            x.copy_(torch.randn(x.shape, generator=g, device=dev).mul_(size))
        if case["out"]:
            state["out"] = _tensors(state, "flat_out", shapes, _TYPES[case["out"]], dev)
        state["most"] = unit if not case["largest"] else each * (1.5 if case["clipped"] else 10.0)
        return state
    n, c = case["rows"], case["classes"]
    target = torch.randint(0, c, (n,), generator=g, device=dev)
    if case["op"] == "log_probs":
        z = torch.randn((n, c), generator=g, device=dev, dtype=torch.float32).mul_(2.5).to(dtype)
        if case["masked"]:
            mask = torch.rand((n, c), generator=g, device=dev) < 0.4
            mask[:, :max(1, case["top"])] = False
            mask.scatter_(1, target[:, None], False)
            if n > 2:
                mask[n // 2] = True  # a row that is masked altogether
            z.masked_fill_(mask, float("-inf"))
        state["logits"] = z.requires_grad_(case["train"])
    else:
        d = case["width"]
        h = torch.randn((n, d), generator=g, device=dev)
        w = torch.randn((c, d), generator=g, device=dev).mul_(2 / math.sqrt(d))
        state["hidden"] = h.to(dtype).requires_grad_(case["train"])
        state["weight"] = w.to(dtype).requires_grad_(case["train"])
    padded = torch.rand((n,), generator=g, device=dev) < 0.05
    padded[0] = False
    state["target"] = torch.where(padded, -100, target)
    if case["train"]:
        # a policy's loss: advantages per row, and one weight for all entropies (fp16: times the loss scale)
        scale = 16.0 if case["dtype"] == "fp16" else 1.0 / n
        state["of_log_prob"] = torch.randn((n,), generator=g, device=dev).mul_(-scale)
        state["of_entropy"] = torch.full((), -0.1 * scale, device=dev).expand(n)
    return state


# ---- the framework's operators -----------------------------------------------------------------------------------
def _own(state):
    from cuml_b200 import distill

    case = state["case"]
    if case["op"] == "clip":
        norm = distill.clip_gradients(state["gradients"], state["most"], out=state.get("out"),
                                      norm_type=math.inf if case["largest"] else 2.0)
        if case["flat"]:
            return norm, state["flat_out" if case["out"] else "flat"]
        return (norm, *state.get("out", state["gradients"]))
    if case["op"] == "log_probs":
        leaves = [state["logits"]]
        scored = distill.log_probs(state["logits"], state["target"], temperature=case["temperature"], top=case["top"])
    else:
        leaves = [state["hidden"], state["weight"]]
        scored = distill.linear_log_probs(state["hidden"], state["weight"], state["target"],
                                          temperature=case["temperature"])
    best = () if scored.top is None else (scored.top.values, scored.top.index)
    if not case["train"]:
        return (scored.log_prob, scored.entropy, *best)
    grads = torch.autograd.grad((scored.log_prob, scored.entropy), leaves, (state["of_log_prob"], state["of_entropy"]))
    return (scored.log_prob.detach(), scored.entropy.detach(), *best, *grads)


# ---- plain forms -------------------------------------------------------------------------------------------------
def _plain_clip(state):
    case = state["case"]
    # (long sums: in 64 bits)
    if case["largest"]:
        norm = torch.stack([x.float().abs().max() for x in state["gradients"]]).max()
    else:
        norm = torch.stack([x.double().square().sum() for x in state["gradients"]]).sum().sqrt().float()
    factor = torch.where(norm > state["most"], state["most"] / norm, torch.ones_like(norm))
    to = _TYPES[case["out"] or case["dtype"]]
    clipped = ((x.float() * factor).to(to) for x in state["gradients"])
    return (norm, torch.cat([x.view(-1) for x in clipped])) if case["flat"] else (norm, *clipped)


def _plain(state):
    case = state["case"]
    with torch.no_grad():
        if case["op"] == "clip":
            return _plain_clip(state)
        linear, target, c, k = case["op"] == "linear", state["target"], case["classes"], case.get("top", 0)
        if linear:
            h, w = state["hidden"].float(), state["weight"].float()
            z = h @ w.t()
        else:
            z = state["logits"].float()
        m = z.max(1, keepdim=True).values
        counted = (target >= 0) & (target < c) & (m[:, 0] > -math.inf)
        y = (z - torch.where(m > -math.inf, m, 0.0)) / case["temperature"]
        e = y.exp()
        s = e.sum(1, keepdim=True)
        e.div_(s)
        log_s = s.log()
        e_y = torch.where(e > 0, e * y, 0.0).sum(1)
        entropy = torch.where(counted, log_s[:, 0] - e_y, 0.0)
        at = torch.where(counted, target, 0)[:, None]
        log_prob = torch.where(counted, (y.gather(1, at) - log_s)[:, 0], 0.0)
        best = ()
        if k:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
            value = y.gather(1, order) - log_s
            best = (torch.where(counted[:, None], value, 0.0),
                    torch.where(counted[:, None], order, -1).to(torch.int32))
        if not case["train"]:
            return (log_prob, entropy, *best)
        g, b = state["of_log_prob"][:, None], state["of_entropy"][:, None]
        log_q = torch.where(e > 0, y.sub_(log_s), 0.0)
        d = e.neg_().mul_(log_q.add_(entropy[:, None]).mul_(b).add_(g))
        d.scatter_add_(1, at, g)
        d = torch.where(counted[:, None], d.div_(case["temperature"]), 0.0)
        if not linear:
            return (log_prob, entropy, *best, d.to(state["logits"].dtype))
        return (log_prob, entropy, (d @ w).to(state["hidden"].dtype), (d.t() @ h).to(state["weight"].dtype))


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        if case["largest"]:
            norm = max(x.double().abs().max() for x in state["gradients"])
        else:
            norm = sum((x.double().pow(2).sum() for x in state["gradients"]), torch.zeros((), dtype=torch.float64,
                                                                                          device="cuda")).sqrt()
        down = min(1.0, state["most"] / float(norm))
        if case["flat"]:
            return norm, state["flat"].double() * down
        return (norm, *(x.double() * down for x in state["gradients"]))
    n, c, t, k = case["rows"], case["classes"], case["temperature"], case.get("top", 0)
    linear, step = case["op"] == "linear", max(1, min(n, 2 ** 26 // c))
    if linear:
        h, w = state["hidden"].detach().double(), state["weight"].detach().double()
        dw = torch.zeros_like(w)
    scores, entropies, values, index, grads = [], [], [], [], []
    for a in range(0, n, step):
        b = min(n, a + step)
        z = h[a:b] @ w.t() if linear else state["logits"][a:b].detach().double()
        target = state["target"][a:b]
        counts = target.ge(0) & ~torch.isneginf(z).all(1)
        log_q = torch.log_softmax(torch.where(counts[:, None], z, 0.0) / t, 1)
        q = log_q.exp()
        log_q = log_q.masked_fill(torch.isneginf(log_q), 0.0)
        named = torch.zeros_like(q).scatter_(1, target.clamp(min=0)[:, None], 1.0)
        entropy = -(q * log_q).sum(1)
        scores.append((named * log_q).sum(1) * counts)
        entropies.append(entropy * counts)
        if k:
            # stably by score: equal scores stay in the order of their classes
            order = torch.argsort(-z, dim=1, stable=True)[:, :k]
            values.append(log_q.gather(1, order) * counts[:, None])
            index.append(torch.where(counts[:, None], order, -1).to(torch.int32))
        if case["train"]:
            g = state["of_log_prob"][a:b, None].double()
            down = state["of_entropy"][a:b, None].double()
            d = (g * (named - q) - down * q * (log_q + entropy[:, None])) * counts[:, None] / t
            grads.append(d @ w if linear else d if n * c <= 2 ** 28 else d.float())
            if linear:
                dw += d.t() @ h[a:b]
    out = (torch.cat(scores), torch.cat(entropies))
    if k:
        out += (torch.cat(values), torch.cat(index))
    if case["train"]:
        out += (torch.cat(grads), dw) if linear else (torch.cat(grads),)
    return out


def work(case):
    if case["op"] == "clip":
        count = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": count * (_BYTES[case["dtype"]] + (_BYTES[case["out"]] if case["out"] else 0)) + 4,
                "flops": (3 if case["clipped"] else 2) * count}
    n, c, e = case["rows"], case["classes"], _BYTES[case["dtype"]]
    both = 2 if case["train"] else 1
    few = n * 16 + (n * 8 if case["train"] else 0)  # targets, scores, gradients by them
    if case["op"] == "log_probs":
        return {"bytes": both * n * c * e + few + n * case["top"] * 8, "flops": 6 * both * n * c}
    d = case["width"]
    return {"bytes": both * (n + c) * d * e + few, "flops": (6 if case["train"] else 2) * n * c * d}
