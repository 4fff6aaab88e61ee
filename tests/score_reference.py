"""Scores of given classes from their definitions, in 64 bits on the CPU (test oracle)."""
import torch

NEG = float("-inf")


def scores(z, target, temperature=1.0, ignore=-100):
    """(log probability of the target, entropy, log q, q, rows that count) of rows of logits."""
    z = z.detach().cpu().double()
    n, c = z.shape
    target = torch.zeros(n, dtype=torch.int64) if target is None else target.detach().cpu().long()
    counts = (target >= 0) & (target < c) & (target != ignore) & ~(z == NEG).all(1)
    log_q = torch.log_softmax(torch.where(counts[:, None], z, torch.zeros_like(z)) / temperature, 1)
    q = log_q.exp()
    each = torch.where(q > 0, q * log_q, torch.zeros_like(q))
    each = torch.where(q.isnan(), q, each)
    at = torch.where(counts, target, 0)
    zero = torch.zeros((), dtype=torch.float64)
    return (torch.where(counts, log_q.gather(1, at[:, None])[:, 0], zero), torch.where(counts, -each.sum(1), zero), log_q, q,
            counts)


def gradient(z, target, g, h, temperature=1.0, ignore=-100):
    """Gradient by the logits of sum(g log_prob + h entropy); g, h: (n,) in 64 bits or None."""
    _, entropy, log_q, q, counts = scores(z, target, temperature, ignore)
    n, c = q.shape
    g = torch.zeros(n, dtype=torch.float64) if g is None else g
    h = torch.zeros(n, dtype=torch.float64) if h is None else h
    one = torch.zeros_like(q)
    if target is not None:
        one[torch.arange(n), torch.where(counts, target.detach().cpu().long(), 0)] = 1.0
    else:
        g = torch.zeros_like(g)
    d = g[:, None] * (one - q)
    d = d - torch.where(q > 0, q * (log_q + entropy[:, None]), torch.zeros_like(q)) * h[:, None]
    return torch.where(counts[:, None], d / temperature, torch.zeros((), dtype=torch.float64))


def top(z, k, counts, log_q):
    """(log q, classes) of the k largest logits of each row, equal ones by class; 0 and -1 where a row does not count."""
    z = z.detach().cpu().double()
    order = torch.argsort(-(z + 0.0), dim=1, stable=True)[:, :k]
    zero = torch.zeros((), dtype=torch.float64)
    return (torch.where(counts[:, None], log_q.gather(1, order), zero),
            torch.where(counts[:, None], order, torch.full((), -1)).to(torch.int32))
