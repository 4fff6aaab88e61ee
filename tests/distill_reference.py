"""The distillation operators from their definitions, in 64 bits on the CPU (test oracle)."""
import torch

NEG = float("-inf")


def top(scores, k, temperature=1.0, probabilities=False):
    x = scores.detach().cpu().double()
    # NaN first, then descending, equal ones (and the two zeros) by class
    key = torch.where(x.isnan(), torch.full_like(x, float("inf")), x + 0.0)
    first = torch.argsort(torch.stack([~x.isnan()]).float()[0], dim=1, stable=True)
    order = first.gather(1, torch.argsort(-key.gather(1, first), dim=1, stable=True))
    nan_first = order.gather(1, torch.argsort((~x.isnan()).gather(1, order).to(torch.int8), dim=1, stable=True))
    index = nan_first[:, :k]
    y = x.log() if probabilities else x
    return y.gather(1, index), index.to(torch.int32), torch.logsumexp(y / temperature, 1)


def teacher(values, index, lse, n_cols, temperature, ignore=None):
    """(target probabilities (n, n_cols), which classes are named, rest (n,), rows that count)."""
    n, k = index.shape
    p = torch.zeros((n, n_cols), dtype=torch.float64)
    named = torch.zeros((n, n_cols), dtype=torch.bool)
    rest = torch.zeros(n, dtype=torch.float64)
    counts = torch.zeros(n, dtype=torch.bool)
    for i in range(n):
        entries = [(int(c), 0.0 if values is None else float(values[i, j]) / temperature) for j, c in enumerate(index[i])
                   if 0 <= int(c) < n_cols and int(c) != ignore]
        v = torch.tensor([e[1] for e in entries], dtype=torch.float64)
        norm = float(lse[i]) if lse is not None else float(torch.logsumexp(v, 0)) if len(entries) else NEG
        counts[i] = norm != NEG
        if not counts[i]:
            continue
        for (c, _), q in zip(entries, (v - norm).exp().tolist()):
            p[i, c] += q
            named[i, c] = True
        if lse is not None and not named[i].all():
            left = 1.0 - float(p[i].sum())
            rest[i] = left if not left < 2.0 ** -20 else 0.0
    return p, named, rest, counts


def loss(z, values, index, lse=None, temperature=1.0, ignore=None):
    """(loss per row, gradient by the logits, rows that count) of rows of logits."""
    z = z.detach().cpu().double()
    cpu = lambda t: None if t is None else t.detach().cpu().double() if t.is_floating_point() else t.cpu()  # noqa: E731
    p, named, rest, counts = teacher(cpu(values), cpu(index), cpu(lse), z.shape[1], temperature, ignore)
    counts = counts & ~(z == NEG).all(1)
    log_q = torch.log_softmax(z / temperature, 1)
    q = log_q.exp()
    each = torch.where(p > 0, torch.special.xlogy(p, p) - p * log_q, torch.zeros_like(p))
    each = torch.where(p.isnan(), p, each)
    out = each.sum(1)
    q_rest = q.masked_fill(named, 0.0).sum(1)
    has = rest != 0
    out = torch.where(has, out + rest * (rest.log() - q_rest.log()), out)
    factor = torch.where(has, 1 - rest / q_rest, torch.ones_like(rest))
    grad = torch.where(named, q, q * factor[:, None]) - p
    zero = torch.zeros((), dtype=torch.float64)
    return (torch.where(counts, out * temperature ** 2, zero), torch.where(counts[:, None], grad * temperature, zero),
            counts)


def reduced(rows, counts, reduction):
    """(loss, factor of the rows' gradients)."""
    if reduction == "none":
        return rows, 1.0
    factor = 1.0 if reduction == "sum" else 1.0 / max(1, int(counts.sum()))
    return rows.sum() * factor, factor
