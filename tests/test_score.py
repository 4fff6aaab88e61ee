"""Log probabilities, entropies and alternatives of rows of logits: refusals (CPU), and the kernels against 64 bits (GPU).

Tolerances count roundings; u = 2^-24 and S, what a row's sum of powers is off by relative to itself, are as in
test_distill.py.  log q is off by S (the difference of logits is taken in 64 bits) and half a step of fp32.  The mean exponent is
a sum of the same powers times their exponents, of which each is off by S times its size: at most the entropy's largest
value, log n_classes, plus the 6 log 2 by which the sum's reference may differ from the maximum (at most 5): E = S (7 + log n).  A
gradient's q is off by 2 S relative, log q + H by E plus 4 u of its size.  A power of two below 2^-126 is 0, of a sum that is 2^-6 at
least, as the reference may be 2^6 above 1: q below 2^-120 may be 0, and q (log q + H) with it, of which the second factor there is
below 120 log 2 + log n < 128 (and the product falls with q)."""
import ctypes as C
import math

import pytest
import torch

from tests import score_reference as ref
from tests.conftest import has_gpu
from tests.test_distill import HALF_STEP, S, TINY, TYPES, U, check_values, gen

gpu = pytest.mark.gpu
TRAINED = ["fp32", "bf16", "fp16"]


def entropy_error(c):
    return S * (7 + math.log(c))


def wide(x):
    return None if x is None else x.detach().cpu().double()


def check(z, target, temperature=1.0, k=0, g=None, h=None, ignore=-100):
    """Scores and, with g or h, gradients of `log_probs` against 64 bits."""
    from cuml_b200 import distill

    n, c = z.shape
    z = z.detach().requires_grad_(g is not None or h is not None)
    got = distill.log_probs(z, target, temperature=temperature, top=k, ignore_index=ignore)
    log_prob, entropy, log_q, q, counts = ref.scores(z, target, temperature, ignore)
    e = entropy_error(c)
    assert got.entropy.dtype == torch.float32 and got.entropy.shape == (n,)
    if target is None:
        assert got.log_prob is None
    else:
        check_values(got.log_prob, log_prob, 4 * U, S, U)
        assert not (got.log_prob > 0).any()
    check_values(got.entropy, entropy, 4 * U, e, U)
    assert not (got.entropy < 0).any()
    if k:
        values, index = ref.top(z, k, counts, log_q)
        assert torch.equal(got.top.index.cpu(), index) and got.top.logsumexp is None
        check_values(got.top.values, values, 4 * U, S, U)
        assert not got.top.values.requires_grad
    else:
        assert got.top is None
    if not z.requires_grad:
        return got, None
    pairs = [(s, u) for s, u in ((got.log_prob, g), (got.entropy, h)) if u is not None]
    (grad,) = torch.autograd.grad([s for s, _ in pairs], z, [u for _, u in pairs])
    want = ref.gradient(z, target, wide(g), wide(h), temperature, ignore)
    one = torch.zeros_like(q)
    if target is not None:
        one[torch.arange(n), torch.where(counts, target.cpu().long(), 0)] = 1.0
    size = lambda x: torch.zeros(n, 1, dtype=torch.float64) if x is None else wide(x).abs()[:, None]  # noqa: E731
    centred = torch.where(q > 0, (log_q + entropy[:, None]).abs(), torch.zeros_like(q))
    allowed = (size(g) * 2 * S * (q + one) + size(h) * q * (centred * (2 * S + 4 * U) + e)) / temperature + 4 * U * want.abs()
    allowed = allowed + 2.0 ** -120 * (size(g) + 128 * size(h)) / temperature
    allowed = torch.where(counts[:, None], allowed, torch.zeros_like(allowed)) + TINY[z.dtype]
    assert grad.dtype == z.dtype
    check_values(grad, want, 0.0, allowed, HALF_STEP[z.dtype])
    return got, grad


def logits(n, c, dtype, seed=0, scale=2.5):
    return (torch.randn((n, c), generator=gen(seed + n + c), device="cuda") * scale).to(TYPES[dtype])


def targets(n, c, seed=0):
    return torch.randint(0, c, (n,), generator=gen(seed + c), device="cuda")


def upstreams(n, seed=5, scale=1.0):
    g = gen(seed)
    return torch.randn((n,), generator=g, device="cuda") * scale, torch.randn((n,), generator=g, device="cuda") * scale


# ---- refusals ------------------------------------------------------------------------------------------------
def test_python_refusals_without_a_gpu():
    from cuml_b200 import distill

    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        distill.log_probs(x, t)
    with pytest.raises(TypeError):
        distill.log_probs([[1.0]], t)
    with pytest.raises(ValueError, match="CUDA"):
        distill.linear_log_probs(x.bfloat16(), x.bfloat16(), t)
    with pytest.raises(ValueError, match="temperature"):
        distill.log_probs(x, t, temperature=0.0)


def test_c_refusals_without_a_gpu(lib):
    from cuml_b200.distill import CTarget

    def score(dtype=2, logits=64, n=4, c=8, stride=8, index=64, log_prob=64, t=1.0, k=2, entropy=64, kept=64, top=64,
              top_index=64, target=True, index64=1):
        given = CTarget(index, 1, -100, index64)
        return lib.b2fil_log_probs(dtype, logits, n, c, stride, C.byref(given) if target else None, t, k, log_prob, entropy,
                                   kept, top, top_index, None, 0, 0, None)

    for bad in (dict(dtype=1), dict(dtype=7), dict(logits=None), dict(logits=65), dict(n=-1), dict(c=0), dict(c=1 << 31),
                dict(stride=7), dict(index=68), dict(index=66, index64=0), dict(log_prob=None), dict(log_prob=66),
                dict(t=0.0), dict(t=float("nan")), dict(k=-1), dict(k=9), dict(k=257, c=300, stride=300), dict(entropy=None),
                dict(kept=None), dict(kept=72), dict(top=None), dict(top_index=None), dict(top_index=66), dict(target=False)):
        assert score(**bad) == -1, bad
        assert lib.b2fil_last_error()
    assert score(n=0) == 0
    assert lib.b2fil_log_probs_workspace(2, 4, 8, 9, 0) == -1
    assert lib.b2fil_log_probs_workspace(1, 4, 8, 0, 0) == -1

    def grad(logits=64, kept=64, g=64, h=64, out=64, stride=8, t=1.0, n=4):
        return lib.b2fil_log_probs_grad(2, logits, n, 8, 8, t, kept, g, 1, h, 1, out, stride, 0, None)

    for bad in (dict(logits=None), dict(kept=None), dict(kept=72), dict(g=66), dict(h=66), dict(out=None), dict(out=65),
                dict(stride=7), dict(t=-1.0), dict(n=-1)):
        assert grad(**bad) == -1, bad
    assert grad(n=0) == 0

    def linear(dtype=2, hidden=64, weight=64, hs=16, ws=16, n=4, c=10, width=16, log_prob=64, entropy=64, kept=64, t=1.0):
        return lib.b2fil_linear_log_probs(dtype, hidden, hs, weight, ws, n, c, width, C.byref(CTarget(64, 1, -100, 1)), t,
                                          log_prob, entropy, kept, None, 0, 0, None)

    for bad in (dict(dtype=0), dict(hidden=None), dict(weight=65), dict(hs=8), dict(n=(1 << 31) - 1), dict(c=0), dict(width=0),
                dict(log_prob=None), dict(entropy=None), dict(kept=68), dict(t=0.0)):
        assert linear(**bad) == -1, bad
    assert linear(n=0) == 0

    def linear_grad(kept=64, g=64, dh=64, dw=64, t=1.0, width=16):
        return lib.b2fil_linear_log_probs_grad(2, 64, 16, 64, 16, 4, 10, width, t, kept, g, 1, None, 0, dh, dw, None, 0, 0, None)

    for bad in (dict(kept=None), dict(kept=72), dict(g=66), dict(dh=72), dict(dw=8), dict(t=0.0), dict(width=17)):
        assert linear_grad(**bad) == -1, bad
    assert linear_grad(dh=None, dw=None) == 0


@pytest.mark.skipif(has_gpu(), reason="checks the behaviour on a box without a GPU")
def test_workspace_needs_a_device(lib):
    assert lib.b2fil_log_probs_workspace(0, 4, 8, 2, 0) == -4
    assert lib.b2fil_linear_log_probs_workspace(2, 64, 16, 64, 16, 4, 10, 16, 99) == -1


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_python_refusals(monkeypatch, compiled):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z, t = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for k in (-1, 9):
        with pytest.raises(ValueError, match="top must be"):
            distill.log_probs(z, t, top=k)
    with pytest.raises(ValueError, match="top must be"):
        distill.log_probs(torch.zeros(1, 500, device="cuda"), top=257)
    for bad, text in ((t[:3], "target must have shape"), (t[:, None], "target must have shape"),
                      (t.float(), "target must be one of"), (t.cpu(), "CUDA")):
        with pytest.raises(ValueError, match=text):
            distill.log_probs(z, bad)
        with pytest.raises(ValueError, match=text):
            distill.linear_log_probs(z.bfloat16(), z.bfloat16(), bad)
    with pytest.raises(ValueError, match="logits must be one of"):
        distill.log_probs(z.double(), t)
    with pytest.raises(ValueError, match="logits"):
        distill.log_probs(z[:, :0], t)
    with pytest.raises(TypeError):
        distill.log_probs(z, [0, 0, 0, 0])
    h = z.bfloat16()
    for args, text in (((z, z, t), "hidden must be one of"), ((h, h.half(), t), "differ in type"), ((h, h[:, :4], t), "width"),
                       ((h.cpu(), h, t), "CUDA")):
        with pytest.raises(ValueError, match=text):
            distill.linear_log_probs(*args)
    with pytest.raises((RuntimeError, NotImplementedError)):  # forward-mode derivatives
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z))
            distill.log_probs(dual, t)


# ---- scores and gradients --------------------------------------------------------------------------------------
SHAPES = [(1, 1, 0), (1, 2, 2), (3, 7, 1), (64, 10, 3), (1003, 10, 0), (37, 33, 5), (130, 1001, 16), (9, 2048, 256),
          (9, 2049, 40), (5, 6000, 0), (500, 3000, 8), (1, 50_001, 20), (2, 131_072, 64), (301, 9001, 2), (1, 300_000, 33),
          (9001, 2, 2), (5003, 13, 3), (6000, 64, 16), (5000, 65, 0), (1300, 4097, 1), (1200, 2500, 30)]


@gpu
@pytest.mark.parametrize("n,c,k", SHAPES)
@pytest.mark.parametrize("dtype", TRAINED)
def test_log_probs(n, c, k, dtype):
    z, t = logits(n, c, dtype), targets(n, c)
    if n > 4:
        t[1], t[3], t[4] = -100, c, -1
    g, h = upstreams(n, scale=16.0 if dtype == "fp16" else 1.0)
    check(z, t, 2.0 if n % 2 else 1.0, k, g, h)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("n,c", [(33, 10), (6, 5000)])
def test_one_of_the_two_scores_and_no_target(monkeypatch, compiled, n, c):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z, t = logits(n, c, "fp32"), targets(n, c).int()
    g, h = upstreams(n)
    check(z, t, 0.7, 0, g, None)
    check(z, t, 0.7, 3, None, h)
    check(z, None, 0.7, 3, None, h)
    check(z, t, 1.0, 0, g, h, ignore=3)
    assert not distill.log_probs(z, t).entropy.requires_grad
    with torch.no_grad():
        assert not distill.log_probs(z.requires_grad_(), t).log_prob.requires_grad


@gpu
@pytest.mark.parametrize("c", [40, 700, 5000, 40_000])
@pytest.mark.parametrize("dtype", TRAINED)
def test_masks(c, dtype):
    """Masked classes, rows that are masked altogether, all equal ones, ties; one class that has all."""
    n, k = 8, 20
    z, t = logits(n, c, dtype), targets(n, c)
    lowest = torch.finfo(z.dtype).min
    z[0, 5::2] = float("-inf")
    z[1] = float("-inf")
    z[2] = lowest
    z[3] = lowest
    z[3, 1::2] = float("-inf")
    z[4, 3:] = lowest
    z[5] = torch.where(torch.arange(c, device="cuda") == 7, 200.0, -200.0).to(z.dtype)
    z[6] = 0.25
    z[7, ::3] = float("-inf")
    z[7, 1::3] = lowest
    t[0], t[3], t[4], t[5], t[7] = 2, 4, 1, 7, 2
    g, h = upstreams(n)
    for m, rows in ((1, slice(None)), (1, slice(3, 4)), (700, slice(None))):
        if m > 1 and c > 5000:
            continue
        many = lambda x: x[rows].repeat(m, *[1] * (x.ndim - 1))  # noqa: E731
        check(many(z), many(t), 1.0, k, many(g), many(h))
    # a given class that is masked: log q is -inf, its gradient that of the formula
    t[0] = 5
    check(z, t, 1.0, 0, g, h)


@gpu
@pytest.mark.parametrize("dtype", TRAINED)
@pytest.mark.parametrize("c", [2049, 4001, 20_000])
@pytest.mark.parametrize("k", [1, 7, 24, 25])
def test_best_of_many_rows_of_thousands_of_classes(c, k, dtype):
    """As many rows as belong to a warp each: ordinary ones, ties, both zeros, infinities, NaN, fewer classes than k above a mask, rows in
    order, and the best all in one lane's pieces; rows off the 16-byte boundaries."""
    t = TYPES[dtype]
    x = torch.randn((1200, c + 5), generator=gen(c + k), device="cuda").to(t)[:, 1:c + 1]
    place, per = torch.arange(c, device="cuda"), 16 // t.itemsize
    x[10] = 0.0
    x[10, 1::2] = -0.0
    x[20] = float("-inf")
    x[30, ::3] = torch.finfo(t).min
    x[40] = place / c
    x[50] = torch.finfo(t).min
    x[50, c // 2] = 3.0
    x[60, 3:] = float("-inf")
    x[70, 3:] = torch.finfo(t).min
    x[80] = torch.where(place // per % 32 < 3, 1.0, -1.0)
    x[90] = torch.where(place // per % 256 == 5, (place % 401) / 401.0, -1.0)
    x[100] = torch.where(place // per % 256 < 20, 2.0 + (place % 97) / 97.0, -1.0)
    x[110] = torch.where(place % 2 == 0, 1.5, 1.25)
    x[120] = -place / c
    x[130, :c - 2] = float("-inf")
    target = targets(1200, c)
    target[5] = -100
    target[[50, 60, 130]] = torch.tensor([c // 2, 1, c - 1], device="cuda")
    check(x, target, 1.0, k)
    from cuml_b200 import distill

    x[30, 5] = x[30, c - 1] = float("nan")
    x[50, 7] = float("inf")
    x[90] = float("nan")
    got = distill.log_probs(x, target, top=k)
    want = distill_top(x, k)
    counts = ref.scores(x, target)[-1]
    assert torch.equal(got.top.index.cpu(), torch.where(counts[:, None], want, torch.full_like(want, -1)))
    assert got.top.values[[30, 50, 90]].isnan().all() and got.entropy[[30, 50, 90]].isnan().all()


def distill_top(x, k):
    from tests import distill_reference

    return distill_reference.top(x, k)[1]


@gpu
def test_rows_that_do_not_count_are_not_read():
    from cuml_b200 import distill

    for c in (10, 50, 3000, 20_000):
        for n in (4, 6000 if c < 100 else 400):
            z, t = logits(n, c, "bf16"), targets(n, c)
            z[1] = float("nan")
            t[1] = -100
            z = z.requires_grad_()
            got = distill.log_probs(z, t, top=4)
            assert got.log_prob[1] == 0 and got.entropy[1] == 0 and (got.top.index[1] == -1).all() and (got.top.values[1] == 0).all()
            assert got.entropy.isfinite().all() and got.log_prob.isfinite().all()
            (d,) = torch.autograd.grad(got.log_prob.sum() + got.entropy.sum(), z)
            assert (d[1] == 0).all() and d.isfinite().all()
    empty = distill.log_probs(z[:0], t[:0], top=3)
    assert empty.log_prob.shape == (0,) and empty.top.index.shape == (0, 3)
    (d,) = torch.autograd.grad(empty.entropy.sum(), z)
    assert d.abs().sum() == 0


@gpu
@pytest.mark.parametrize("c", [12, 300, 3000, 50_000])
def test_infinite_and_nan_logits_as_in_a_softmax(c):
    from cuml_b200 import distill

    for n in (4, 400):
        z, t = logits(n, c, "fp32"), targets(n, c)
        z[0, 7] = float("nan")
        z[1, 8] = float("inf")
        z[2] = float("inf")
        z.requires_grad_()
        for k in (0, 3):
            got = distill.log_probs(z, t, top=k)
            (d,) = torch.autograd.grad(got.log_prob.sum() + got.entropy.sum(), z)
            for r in (0, 1, 2):
                assert got.log_prob[r].isnan() and got.entropy[r].isnan() and d[r].isnan().all()
            assert got.log_prob[3:].isfinite().all() and got.entropy[3:].isfinite().all() and d[3:].isfinite().all()
            if k:
                assert got.top.values[:3].isnan().all() and got.top.index[0, 0] == 7 and got.top.index[1, 0] == 8


@gpu
@pytest.mark.parametrize("dtype", TRAINED)
def test_logits_far_apart_and_far_from_zero(dtype):
    """log q is a difference of logits: where these are far from zero, what counts is how far they are apart."""
    for n in (5, 5000):
        for c in (8, 20, 3000):
            if n * c > 200_000:
                continue
            z, t = logits(n, c, dtype, scale=1.0), targets(n, c)
            far = 1e4 if dtype == "fp16" else 1e6
            g, h = upstreams(n)
            check(z + far, t, 1.0, 3, g, h)
            check(z - far, t, 100.0, 3, g, h)
            check((z.float() * 1e4).to(z.dtype), t, 1.0, 3, g, h)


@gpu
@pytest.mark.parametrize("dtype", TRAINED)
@pytest.mark.parametrize("k", [0, 3])
def test_logits_that_the_paired_sums_do_not_take(dtype, k):
    """Rows below and around the border of what counts as ordinary, masked parts of a row beside ordinary ones, and very high and low
    temperatures, by which a mask of the type's lowest value may count."""
    border = 30_000.0 if dtype == "fp16" else 1e29
    for n, c in ((6, 3000), (6, 20_000), (1200, 2500)):
        z, t = logits(n, c, dtype, scale=1.0), targets(n, c)
        lowest = torch.finfo(z.dtype).min
        low = z.float()
        low[0] = -border + low[0] * border / 1000
        low[1, : c // 2] = -border * 0.999
        low[1, c // 2:] = -border * 1.001
        low[2, : c - 50] = lowest
        low[3] = lowest if dtype == "fp16" else -2 * border
        low[4, : c // 2] = float("-inf")
        low[4, c // 2:] = -border * 1.5
        t[:5] = c - 1
        z = low.to(z.dtype)
        g, h = upstreams(n)
        for temperature in (1.0, 50.0, 1e4, 1e6, 1e-3):
            if temperature == 1e-3 and dtype == "fp16":
                continue  # (gradients beyond 65504)
            check(z, t, temperature, k, g, h)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_strides_and_shapes(monkeypatch, compiled):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z = logits(60, 1000, "bf16")
    for view in (z[:, 1:900], z[::2], z.t().contiguous().t(), z[:1].expand(60, 1000), z[:, ::3], z[:, 3:12]):
        n, c = view.shape
        g, h = upstreams(n)
        check(view, targets(n, c), 1.0, 7, g, h)
    t = targets(60, 1000)
    both = torch.stack([t, t + 1], 1)[:, 0]
    assert both.stride(0) == 2
    got, grad = check(z, both, 1.0, 4, torch.ones(1, device="cuda").expand(60), torch.randn(120, device="cuda")[::2])
    cube = z.view(3, 20, 1000).requires_grad_()
    shaped = distill.log_probs(cube, t.view(3, 20), top=4)
    assert shaped.log_prob.shape == (3, 20) and shaped.top.index.shape == (3, 20, 4)
    assert torch.equal(shaped.log_prob.view(60), got.log_prob) and torch.equal(shaped.top.values.view(60, 4), got.top.values)
    (d,) = torch.autograd.grad(shaped.log_prob.sum(), cube)
    assert d.shape == cube.shape
    one = distill.log_probs(z[0], t[0])
    assert one.log_prob.shape == () and torch.equal(one.log_prob, got.log_prob[0])
    half = torch.randn((40, 131), generator=gen(3), device="cuda").half()[:, 1:]  # 2-byte alignment
    g, h = upstreams(40)
    check(half, targets(40, 130), 1.0, 9, g, h)


@gpu
def test_gradient_against_differences():
    """Central differences of the scores themselves, h = 2^-5: their own error is h^2 / 6 of the third derivatives (of log q
    below 1, of the entropy below 2 + log 12), and of the scores' roundings, over 2 h."""
    from cuml_b200 import distill

    z, t = logits(3, 12, "fp32", 4, 1.0), targets(3, 12)
    g, w = upstreams(3)
    f = lambda x: (distill.log_probs(x, t, temperature=1.3)[0].double() * g.double()).sum() + (  # noqa: E731
        distill.log_probs(x, t, temperature=1.3)[1].double() * w.double()).sum()
    z.requires_grad_()
    (d,) = torch.autograd.grad(f(z), z)
    h = 2.0 ** -5
    size = float(g.abs().sum() + w.abs().sum())
    for r in range(3):
        for c in range(12):
            step = torch.zeros_like(z)
            step[r, c] = h
            slope = (f(z.detach() + step) - f(z.detach() - step)) / (2 * h)
            assert abs(slope.item() - d[r, c].item()) < size * (h * h / 6 * 5 + (S + entropy_error(12)) / h)


@gpu
def test_the_same_as_the_losses():
    """log_prob is minus the cross entropy, alternatives are a teacher's, an entropy bonus is a KL to the uniform distribution
    less log n."""
    from cuml_b200 import distill

    z, t = logits(200, 1000, "fp32"), targets(200, 1000)
    got = distill.log_probs(z, t, top=6)
    check_values(got.log_prob, -wide(distill.cross_entropy(z, t, reduction="none")), 4 * U, 2 * S, U)
    few = distill.log_probs(z[:, :200], None, top=200)
    uniform = distill.distillation_loss(torch.zeros_like(z[:, :200]), few.top, reduction="none")
    check_values(few.entropy, math.log(200) - wide(uniform), 4 * U, entropy_error(200) + 4 * S, U)
    student = torch.zeros_like(z).requires_grad_()
    t[3] = -100
    taught = distill.distillation_loss(student, distill.log_probs(z, t, top=6).top, reduction="none")
    assert taught[3] == 0 and (taught[:3] > 0).all()


# ---- a linear layer ----------------------------------------------------------------------------------------------
def adds(n):
    return (n / 8 + 16) * 2 * U


def check_linear(h, w, target, temperature=1.0, g=None, b=None, wants=(True, True)):
    """As in test_distill_linear.py: a logit's sum is off by e_z, log q by 2 e_z / T more than above, an entropy by that
    times E|log q + H| <= 2 H, log q + H by both."""
    from cuml_b200 import distill

    n, c = h.shape[0], w.shape[0]
    half = HALF_STEP[h.dtype]
    h, w = h.detach().requires_grad_(wants[0]), w.detach().requires_grad_(wants[1])
    got = distill.linear_log_probs(h, w, target, temperature=temperature)
    hd, wd = wide(h), wide(w)
    z = hd @ wd.t()
    e_z = 2 * adds(h.shape[1]) * (hd.abs() @ wd.abs().t()).amax(1) / temperature  # per row
    log_prob, entropy, log_q, q, counts = ref.scores(z, target, temperature)
    check_values(got.log_prob, log_prob, 4 * U, S + e_z, U)
    e = entropy_error(c) + e_z * (1 + 2 * entropy)
    check_values(got.entropy, entropy, 4 * U, e, U)
    assert not (got.log_prob > 0).any() and not (got.entropy < 0).any()
    leaves = [x for x, is_wanted in zip((h, w), wants) if is_wanted]
    pairs = [(s, u) for s, u in ((got.log_prob, g), (got.entropy, b)) if u is not None]
    grads = list(torch.autograd.grad([s for s, _ in pairs], leaves, [u for _, u in pairs]))
    d = ref.gradient(z, target, wide(g), wide(b), temperature)
    one = torch.zeros_like(q)
    one[torch.arange(n), torch.where(counts, target.cpu().long(), 0)] = 1.0
    size = lambda x: torch.zeros(n, 1, dtype=torch.float64) if x is None else wide(x).abs()[:, None]  # noqa: E731
    centred = (log_q + entropy[:, None]).abs()
    e_d = (size(g) * (q + one) * (2 * S + e_z[:, None]) +
           size(b) * q * (centred * (2 * S + 4 * U + e_z[:, None]) + e[:, None] + e_z[:, None])) / temperature
    e_d = torch.where(counts[:, None], e_d, torch.zeros_like(e_d)) + d.abs() * (half + 4 * U)
    if h.dtype == torch.float16:  # below 2^-14 of the scaled differences, steps are 2^-24; the scale is up to twice what it need be
        e_d = e_d + 2.0 ** -25 / 2.0 ** 14 * 2 * float((size(g) + 8 * size(b)).max()) / temperature
    tiny = 2.0 ** -25 if h.dtype == torch.float16 else 0.0
    for is_hidden, is_wanted in zip((True, False), wants):
        if not is_wanted:
            continue
        x = grads.pop(0)
        other, dd, ee = (wd, d, e_d) if is_hidden else (hd, d.t(), e_d.t())
        allowed = ee @ other.abs() + adds(dd.shape[1]) * (dd.abs() @ other.abs())
        assert x.dtype == h.dtype and x.is_contiguous()
        check_values(x, dd @ other, 2 * U, allowed + tiny, half)


SIZES = [(1, 8, 1), (1, 64, 2), (3, 16, 7), (128, 64, 256), (129, 72, 257), (256, 256, 256), (257, 264, 300),
         (64, 128, 1000), (200, 520, 1003), (513, 200, 2050), (40, 96, 20_011), (300, 33, 130), (70, 1001, 515),
         (5000, 64, 40), (9000, 264, 513), (3, 1, 5), (1, 512, 30_000)]


def layer(n, width, c, dtype, seed=0):
    g = gen(seed + n + width + c)
    h = torch.randn((n, width), generator=g, device="cuda")
    w = torch.randn((c, width), generator=g, device="cuda") * (2 / width ** 0.5)
    return h.to(TYPES[dtype]), w.to(TYPES[dtype])


@gpu
@pytest.mark.parametrize("n,width,c", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_log_probs(n, width, c, dtype):
    from cuml_b200 import distill

    h, w = layer(n, width, c, dtype)
    t = targets(n, c, 1)
    if n > 2:
        t[::5] = -100
        t[1] = c
    g, b = upstreams(n, scale=3.0)
    check_linear(h, w, t, 1.0, g, b)
    check_linear(h, w, t.int(), 2.0, g, None, wants=(True, False))
    check_linear(h, w, t, 0.5, None, b, wants=(False, True))
    distill.check_status()


@gpu
def test_several_pieces_of_the_classes():
    """(20,000 x 7,000 differences are more than one piece holds.)"""
    h, w = layer(20_000, 16, 7000, "bf16")
    g, b = upstreams(20_000)
    check_linear(h, w, targets(20_000, 7000), 1.0, g, b)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_linear_shapes_strides_and_autocast(monkeypatch, compiled):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    h, w = layer(60, 64, 200, "bf16")
    t = targets(60, 200)
    want = distill.linear_log_probs(h, w, t)
    padded = torch.zeros((60, 80), dtype=torch.bfloat16, device="cuda")
    for at in (8, 3):
        padded[:, at:at + 64] = h
        for a, b in zip(distill.linear_log_probs(padded[:, at:at + 64], w, t)[:2], want[:2]):
            assert torch.equal(a, b)
    assert torch.equal(distill.linear_log_probs(h.t().contiguous().t(), w.t().contiguous().t(), t)[1], want[1])
    none = distill.linear_log_probs(h, w)
    counted = t >= 0
    assert none.log_prob is None and torch.equal(none.entropy[counted], want.entropy[counted])
    cube = h.view(3, 20, 64).detach().requires_grad_()
    got = distill.linear_log_probs(cube, w, t.view(3, 20))
    assert got.log_prob.shape == (3, 20) and torch.autograd.grad(got.entropy.sum(), cube)[0].shape == cube.shape
    h32, w32 = h.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = distill.linear_log_probs(h32, w32, t)
    assert torch.equal(got.log_prob, want.log_prob)
    a, b = torch.autograd.grad(got.log_prob.sum() + got.entropy.sum(), (h32, w32))
    assert a.dtype == b.dtype == torch.float32
    empty = distill.linear_log_probs(h[:0], w.requires_grad_(), t[:0])
    (d,) = torch.autograd.grad(empty.entropy.sum(), w)
    assert empty.log_prob.shape == (0,) and d.shape == w.shape and (d == 0).all()


# ---- call paths ----------------------------------------------------------------------------------------------------
@gpu
def test_without_the_compiled_call_path(monkeypatch):
    """The same numbers and gradients through ctypes."""
    from cuml_b200 import distill

    z, t = logits(50, 300, "bf16"), targets(50, 300)
    h, w = layer(50, 64, 300, "bf16")

    def everything():
        out = []
        for target in (t, None):
            x = z.detach().requires_grad_()
            got = distill.log_probs(x, target, top=5, temperature=1.5)
            a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
            of_layer = distill.linear_log_probs(a, b, target, temperature=2.0)
            total = got.entropy.sum() + (0 if target is None else (2 * got.log_prob).sum())
            of_both = of_layer.entropy.sum() + (0 if target is None else (2 * of_layer.log_prob).sum())
            out += [got.log_prob, got.entropy, *got.top[:2], *torch.autograd.grad(total, x), *of_layer[:2],
                    *torch.autograd.grad(of_both, (a, b))]
        return out

    assert distill._native()
    compiled = everything()
    monkeypatch.setattr(distill, "_call", False)
    for x, y in zip(compiled, everything()):
        assert (x is None) == (y is None)
        assert x is None or (x.dtype == y.dtype and torch.equal(x, y))


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_autograd_rules(monkeypatch, compiled):
    """A graph is used once unless it is retained, inputs are not changed in between, there is no second derivative; the targets may
    change."""
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z, t = logits(5, 30, "fp32"), targets(5, 30)
    h, w = layer(5, 16, 30, "bf16")
    for leaves, f in (([z], lambda a: distill.log_probs(a, t)), ([h, w], lambda a, b: distill.linear_log_probs(a, b, t))):
        leaves = [x.detach().requires_grad_() for x in leaves]
        got = f(*leaves)
        loss = got.log_prob.sum() + got.entropy.sum()
        first = torch.autograd.grad(loss, leaves, retain_graph=True)
        kept = t.clone()
        t.zero_()
        again = torch.autograd.grad(loss, leaves)
        t.copy_(kept)
        assert all(torch.equal(x, y) for x, y in zip(first, again))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(loss, leaves)
        got = f(*leaves)
        with torch.no_grad():
            leaves[0].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(got.entropy.sum(), leaves)
        grads = torch.autograd.grad(f(*leaves).entropy.sum(), leaves, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grads[0].sum(), leaves)
        got = f(*leaves)
        (got.log_prob.double().mean() + got.entropy.half().sum()).backward()  # (upstreams of other types)
        assert all(x.grad is not None and x.grad.shape == x.shape and x.grad.isfinite().all() for x in leaves)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_saved_tensors_under_hooks_and_checkpoints(monkeypatch, compiled):
    from torch.utils.checkpoint import checkpoint

    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z, t = logits(20, 300, "fp32").requires_grad_(), targets(20, 300)
    h, w = (x.requires_grad_() for x in layer(20, 64, 300, "bf16"))

    def step(z, h, w):
        a, b = distill.log_probs(z, t, top=2), distill.linear_log_probs(h, w, t)
        return a.log_prob.sum() + 2 * a.entropy.sum() + 3 * b.log_prob.sum() + 4 * b.entropy.sum()

    want = torch.autograd.grad(step(z, h, w), (z, h, w))
    pack, unpack = (lambda x: x.t().contiguous().cpu()), (lambda x: x.cuda().t())  # (given back in another order of rows)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        loss = step(z, h, w)
    for a, b in zip(torch.autograd.grad(loss, (z, h, w)), want):
        assert torch.equal(a, b)
    loss = checkpoint(step, z, h, w, use_reentrant=False)
    for a, b in zip(torch.autograd.grad(loss, (z, h, w)), want):
        assert torch.equal(a, b)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[:1] if x.dim() == 2 else x):
        loss = step(z, h, w)
    with pytest.raises(RuntimeError, match="hook gave back another tensor"):
        torch.autograd.grad(loss, (z, h, w))


@gpu
def test_captured_and_replayed():
    """A captured step runs again on other values of its inputs."""
    from cuml_b200 import distill

    z, t = logits(300, 5000, "bf16"), targets(300, 5000)
    h, w = layer(300, 64, 5000, "fp16")
    g, b = upstreams(300)
    held = [z.clone(), h.clone(), w.clone(), t.clone()]

    def step(z, h, w, t):
        leaves = [x.detach().requires_grad_() for x in (z, h, w)]
        a, c = distill.log_probs(leaves[0], t, top=3), distill.linear_log_probs(*leaves[1:], t)
        grads = torch.autograd.grad([a.log_prob, a.entropy, c.log_prob, c.entropy], leaves, [g, b, g, b])
        return [a.log_prob.detach(), a.entropy.detach(), *a.top[:2], c.log_prob.detach(), c.entropy.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for shift in (0, 1):
        fresh = [z.roll(shift, 0), h.roll(shift, 0), w.roll(shift, 0), t.roll(shift, 0)]
        for x, y in zip(held, fresh):
            x.copy_(y)
        graph.replay()
        for x, y in zip(out, step(*fresh)):
            assert torch.equal(x, y)
    del graph


@gpu
def test_more_than_two_to_the_31_elements():
    """The last rows of large logits against the same rows alone, which may be summed in another order: each is off by what the
    head of this file says, the gradient by q (4 S + 2 E) <= 4 S + 2 E (and 2 S for the given class) and two roundings."""
    from cuml_b200 import distill

    n, c = 66_000, 32_800
    x = torch.randn((n, c), generator=gen(1), device="cuda", dtype=torch.bfloat16).requires_grad_()
    t = targets(n, c)
    got = distill.log_probs(x, t, top=7)
    (d,) = torch.autograd.grad((got.log_prob, got.entropy), x, (torch.ones_like(got.entropy), torch.ones_like(got.entropy)))
    few = x.detach()[-900:].clone().requires_grad_()
    want = distill.log_probs(few, t[-900:].clone(), top=7)
    (e,) = torch.autograd.grad((want.log_prob, want.entropy), few, (torch.ones_like(want.entropy), torch.ones_like(want.entropy)))
    check_values(got.log_prob[-900:], wide(want.log_prob), 8 * U, 2 * S, 2 * U)
    check_values(got.entropy[-900:], wide(want.entropy), 8 * U, 2 * entropy_error(c), 2 * U)
    assert torch.equal(got.top.index[-900:], want.top.index)
    check_values(got.top.values[-900:], wide(want.top.values), 8 * U, 2 * S, 2 * U)
    check_values(d[-900:], wide(e), 8 * U, 6 * S + 2 * entropy_error(c), 2 * HALF_STEP[torch.bfloat16])
    assert (d[0] != 0).any()
