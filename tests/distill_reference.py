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
    index = index.long()
    valid = (index >= 0) & (index < n_cols)
    if ignore is not None:
        valid &= index != ignore
    v = torch.zeros((n, k), dtype=torch.float64) if values is None else values / temperature
    v = v.masked_fill(~valid, NEG)
    norm = torch.logsumexp(v, 1) if lse is None else lse.reshape(-1)
    counts = norm != NEG
    at = torch.where(valid, index, 0)
    each = torch.where(valid & counts[:, None], (v - norm[:, None]).exp(), torch.zeros_like(v))
    p = torch.zeros((n, n_cols), dtype=torch.float64).scatter_add_(1, at, each)
    named = torch.zeros((n, n_cols), dtype=torch.float64).scatter_add_(1, at, valid.double()) > 0
    rest = torch.zeros(n, dtype=torch.float64)
    if lse is not None:
        left = 1.0 - p.sum(1)
        rest = torch.where(counts & ~named.all(1) & ~(left < 2.0 ** -20), left, rest)
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
