"""The distillation operators at the ends of their ranges, against 64 bits: low temperatures, logits far apart, teachers
whose log-sum-exp is large, the largest scores; and what autograd offers beside a plain backward pass.

u, S and the counting of roundings are those of test_distill.py."""
import pytest
import torch

from tests.test_distill import HALF_STEP, S, TINY, TYPES, U, check_top, check_values, gen, gpu

NEG = float("-inf")
# rows, classes, entries: a thread per row, a warp per short row, parts of a row, a block per row, a warp per long row
KERNELS = [(5000, 12, 4), (6000, 64, 16), (7, 12, 4), (300, 130, 20), (9, 3000, 8), (400, 3000, 8), (1300, 2500, 5),
           (3, 50_001, 20)]


def bucket(z, values, index, lse, temperature, least=0.0):
    """(losses, gradients, allowed errors of both without the gradients' own rounding) with the rest as one more class, of
    rows that all count and whose entries name no class twice; a rest below `least` is none.

    With s the softmax over the classes that are not named, p_r what is left of 1 and P the sum of all of p,
    d loss / d z_c = T (P q_c - p_c) for named classes and T (P q_c - p_r s_c) for the others.  Each logarithm is off
    by S; q, p_r s and p by 2 S relative (of s and q: an exponent of up to 127, rounded twice, beside S)."""
    z, v, lse = z.detach().cpu().double(), values.cpu().double() / temperature, lse.cpu().double()
    index, (n, c) = index.cpu().long(), z.shape
    inside = (index >= 0) & (index < c)
    at = torch.where(inside, index, 0)
    each = torch.where(inside, (v - lse[:, None]).exp(), torch.zeros_like(v))
    p = torch.zeros((n, c), dtype=torch.float64).scatter_add_(1, at, each)
    named = torch.zeros((n, c)).scatter_add_(1, at, inside.float()) > 0
    rest = 1 - each.sum(1)
    rest = torch.where((rest < least) | named.all(1), torch.zeros_like(rest), rest)
    y = z / temperature
    all_of, others = torch.logsumexp(y, 1), y.masked_fill(named, NEG)
    left = torch.logsumexp(others, 1)
    log_q = y - all_of[:, None]
    loss = torch.where(p > 0, p * (p.log() - log_q), torch.zeros_like(p)).sum(1)
    loss = loss + torch.where(rest > 0, rest * (rest.log() - (left - all_of)), torch.zeros_like(rest))
    s = torch.where(rest[:, None] > 0, (others - left[:, None]).exp(), torch.zeros_like(p)).nan_to_num()
    mass = (each.sum(1) + rest)[:, None]
    grad = mass * log_q.exp() - p - rest[:, None] * s
    size = mass * log_q.exp() + p + rest[:, None] * s
    t2 = temperature ** 2
    return loss * t2, grad * temperature, 3 * S * t2 + (loss * t2).abs() * 4 * U, 2 * S * size * temperature


def check_bucket(z, values, index, lse, temperature, upstream=None, least=0.0, reduction="none"):
    from cuml_b200 import distill

    z = z.detach().requires_grad_()
    loss = distill.distillation_loss(z, (values, index, lse), temperature=temperature, tail="bucket", reduction=reduction)
    rows, grad, off, grad_off = bucket(z, values, index, lse, temperature, least)
    factor = 1.0
    if reduction == "mean":
        factor = 1 / len(rows)
        check_values(loss, rows.mean(), 4 * U, off.mean(), U)
    else:
        check_values(loss, rows, 0.0, off, U)
    upstream = torch.ones_like(loss) if upstream is None else upstream
    (got,) = torch.autograd.grad(loss, z, upstream)
    up = upstream.detach().cpu().double().reshape(-1, 1) * factor
    assert torch.isfinite(got.float()).all()
    # (a power of less than 2^-126 is 0: q, s and p are each off by up to that, times what multiplies them, at most 1)
    none = 3 * 2.0 ** -126 * temperature * up
    check_values(got, grad * up, 0.0, grad_off * up + none + TINY[z.dtype], HALF_STEP[z.dtype])
    return loss


@pytest.mark.parametrize("temperature", [1.0, 0.1])
@pytest.mark.parametrize("c,k,more", [(9, 3, 0.4), (9, 3, 0.0), (6, 6, 0.0), (6, 8, 0.7)])
def test_the_oracles_gradient_is_that_of_its_loss(c, k, more, temperature):
    """Central differences of the 64-bit loss, h = 2^-10 T: off by h^2 / 6 of the third derivative, below 4 / T,
    and by 2^-52 of losses below 100 over h (3e-10)."""
    g = gen(c, "cpu")
    z = torch.randn((4, c), generator=g, dtype=torch.float64) * temperature
    z[1, :k // 2] += 30 * temperature
    v = torch.randn((4, k), generator=g, dtype=torch.float64) * temperature
    i = torch.stack([torch.randperm(max(c, k), generator=g)[:k] for _ in range(4)])
    lse = torch.logsumexp(v / temperature, 1) + more
    loss = lambda x: bucket(x, v, i, lse, temperature, least=1e-9)[0]  # noqa: E731
    grad, h = bucket(z, v, i, lse, temperature, least=1e-9)[1], 2.0 ** -10 * temperature
    for j in range(c):
        d = torch.zeros_like(z)
        d[:, j] = h
        slope = (loss(z + d) - loss(z - d)) / (2 * h)
        assert ((slope - grad[:, j]).abs() <= 2.0 ** -20 / 6 * temperature * 4 + 1e-9).all()


def apart(n, c, k, dtype, temperature, gap, seed=0):
    """Logits whose named classes lie `gap` temperatures above the others (below them in every third row); a teacher that
    leaves about a tenth."""
    g = gen(seed + c)
    order = torch.rand((n, c), generator=g, device="cuda").argsort(1)[:, :k]
    z = torch.randn((n, c), generator=g, device="cuda")
    sign = torch.where(torch.arange(n, device="cuda") % 3 == 1, -gap, gap)[:, None]
    z = z.scatter_add_(1, order, sign.expand(n, k).to(z.dtype)) * temperature
    v = torch.randn((n, k), generator=g, device="cuda") * temperature
    return z.to(TYPES[dtype]), v, order.int(), torch.logsumexp(v.double() / temperature, 1).float() + 0.1


# ---- the rest as one more class --------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n,c,k", KERNELS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("gap", [60.0, 90.0, 1e4])
def test_losses_of_named_classes_far_from_the_others(n, c, k, dtype, gap):
    """The loss is finite and the same whichever kernel takes the row."""
    from cuml_b200 import distill

    for temperature in (1.0, 0.1, 0.01):
        z, v, i, lse = apart(n, c, k, dtype, temperature, gap)
        loss = distill.distillation_loss(z, (v, i, lse), temperature=temperature, tail="bucket", reduction="none")
        rows, _, off, _ = bucket(z, v, i, lse, temperature)
        check_values(loss, rows, 0.0, off, U)
        few = distill.distillation_loss(z[:3], (v[:3], i[:3], lse[:3]), temperature=temperature, tail="bucket",
                                        reduction="none")
        check_values(loss[:3], few.cpu().double(), 0.0, 2 * off[:3], 2 * U)


@gpu
@pytest.mark.parametrize("n,c,k", KERNELS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("gap", [9.0, 60.0, 90.0, 1e4])
def test_gradients_of_named_classes_far_from_the_others(n, c, k, dtype, gap):
    for temperature in (1.0, 0.1, 0.01):
        z, v, i, lse = apart(n, c, k, dtype, temperature, gap)
        check_bucket(z, v, i, lse, temperature)
        check_bucket(z, v, i, lse, temperature, torch.tensor(65536.0 if dtype != "fp16" else 8.0 * n, device="cuda"),
                     reduction="mean")


@gpu
@pytest.mark.parametrize("n,c,k", [(5000, 12, 4), (6000, 64, 16), (7, 12, 4), (300, 130, 20), (133, 3000, 8), (400, 3000, 8),
                                   (1300, 2500, 5), (133, 60_000, 10)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("less", [3.0, 7.0])
def test_rests_of_nearly_one(n, c, k, dtype, less):
    """Few classes named of many, as at high temperatures: the loss is a difference of numbers near 1.  With M the named classes'
    probabilities of both sides together, what the sums are off by (64 additions of a thread, 20 of threads, 16 u of a term) weighs with M,
    and each p, and each logarithm of 1 - M, is off by 2 u of itself."""
    from cuml_b200 import distill

    for temperature in (1.0, 4.0):
        z, v, i, _ = apart(n, c, k, dtype, temperature, 0.0)
        z = z.float().scatter_add_(1, i.long(), torch.full_like(v, -less * temperature)).to(z.dtype)
        lse = torch.logsumexp(v.double() / temperature, 1).float() + less
        loss = distill.distillation_loss(z, (v, i, lse), temperature=temperature, tail="bucket", reduction="none")
        rows = bucket(z, v, i, lse, temperature)[0]
        p = (v.double() / temperature - lse.double()[:, None]).exp()
        log_q = torch.log_softmax(z.double() / temperature, 1).gather(1, i.long())
        m = p.sum(1) + log_q.exp().sum(1)
        off = 100 * U * m + 2 * U * (p * (p.log() - log_q).abs()).sum(1) + 4 * U * m
        check_values(loss, rows, 0.0, (off * temperature ** 2).cpu(), U)


@gpu
@pytest.mark.parametrize("n,c,k", [(5, 6, 6), (5000, 6, 8), (5000, 1, 3), (40, 200, 203), (3, 250, 256)])
def test_a_teacher_of_more_classes_than_the_student(n, c, k):
    """All of the student's classes are named, and a part of the teacher's mass is on none of them."""
    from cuml_b200 import distill

    g = gen(c)
    z = torch.randn((n, c), generator=g, device="cuda") * 2
    v = torch.randn((n, k), generator=g, device="cuda")
    i = torch.rand((n, max(c, k)), generator=g, device="cuda").argsort(1)[:, :k].int()  # (k above c: some are outside)
    for more in (0.0, 0.7):
        lse = torch.logsumexp(v.double(), 1).float() + more
        check_bucket(z, v, i, lse, 1.0, least=2.0 ** -20)
    # the gradient is that of the loss that is returned: differences, off by 3 S / h and h^2 / 6 of the third derivative
    h, x = 0.25, z[:1].detach().requires_grad_()
    f = lambda x: distill.distillation_loss(x, (v[:1], i[:1], lse[:1]), tail="bucket", reduction="sum")  # noqa: E731
    d = torch.zeros_like(x)
    d[0, 0] = h
    slope = (f(x.detach() + d) - f(x.detach() - d)) / (2 * h)
    assert abs(slope.item() - torch.autograd.grad(f(x), x)[0][0, 0].item()) < h * h / 6 * 0.2 + 3 * S / h


@gpu
@pytest.mark.parametrize("n,c,k", [(7, 40, 16), (5000, 40, 16), (300, 700, 100), (9, 3000, 40), (400, 3000, 40), (1300, 2500, 24)])
@pytest.mark.parametrize("shift", [50.0, -100.0, 700.0])
@pytest.mark.parametrize("dtype", ["fp32", "fp64"])
def test_teachers_whose_logits_are_far_from_zero(n, c, k, shift, dtype):
    """A 32-bit log-sum-exp of that size says 1 to some 2^-19 only; where the teacher names all that it has, and the student
    masks the same classes, nothing is left, and the masked classes have no gradient."""
    from cuml_b200 import distill

    t = torch.randn((n, c), generator=gen(c), device="cuda").add_(shift).to(TYPES[dtype])
    t[:, k:] = NEG
    z = torch.randn((n, c), generator=gen(c + 1), device="cuda")
    z[:, k:] = NEG
    z = z.requires_grad_()
    top = distill.top_scores(t, k)
    loss = distill.distillation_loss(z, top, tail="bucket", reduction="none")
    rows = distill.distillation_loss(z, top, reduction="none")
    assert torch.isfinite(loss).all()
    # p is off by the log-sum-exp's half step, 2^-24 of its size, and so is a loss whose logarithms are below 16
    off = 6 * S + 16 * (abs(shift) + 16) * U
    check_values(loss, rows.detach().cpu().double(), 4 * U, off, U)
    (g,) = torch.autograd.grad(loss, z, torch.ones_like(loss))
    (want,) = torch.autograd.grad(rows, z, torch.ones_like(rows))
    assert (g[:, k:] == 0).all()
    check_values(g, want.cpu().double(), 4 * S, 4 * S + 2 * (abs(shift) + 16) * U, U)


def test_scalars_off_their_elements_are_refused(lib):
    """(On the CPU: a kernel would write to an address that is none of a 32-bit number's.)"""
    import ctypes as C

    from cuml_b200.distill import CTeacher

    teacher = CTeacher(64, 64, None, 2, 2, -100, 2, 0)
    for loss, factor in ((66, 64), (64, 65), (None, 64), (64, None)):
        for reduction in (1, 2):
            assert lib.b2fil_distill_loss(2, 64, 4, 8, 8, C.byref(teacher), 1.0, reduction, 64, 64, 64, 64, loss, factor, None,
                                          0, 0, None) == -1, (loss, factor)
            assert lib.b2fil_linear_loss(2, 64, 16, 64, 16, 4, 10, 16, C.byref(teacher), 1.0, reduction, 64, 64, 64, 64, 64,
                                         loss, factor, None, 0, 0, None) == -1, (loss, factor)
        assert b"loss and factor" in lib.b2fil_last_error()


@gpu
@pytest.mark.parametrize("precision", ["single", "double"])
@pytest.mark.parametrize("n", [60, 6000])
def test_a_student_of_a_forest_at_a_low_temperature(precision, n):
    """A forest's probabilities, whose powers leave the range of 32 bits, with the rest as one more class; what counts as
    one is 2^-20, or 2^-22 of the log-sum-exp's size."""
    from tests.helpers import random_rows
    from tests.test_distill_forest import N_CLASSES, forest

    fi = forest(precision)
    X = torch.as_tensor(random_rows(4, n, 6), device="cuda")
    z = torch.randn((n, N_CLASSES), generator=gen(1), device="cuda")
    for temperature in (0.02, 0.1):
        top = fi.teach(X, 4, temperature=temperature)
        assert torch.isfinite(top.logsumexp).all()
        least = (top.logsumexp.cpu().double().abs() * 2.0 ** -22).clamp(min=2.0 ** -20)
        check_bucket(z, top.values.float(), top.index, top.logsumexp.float(), temperature, least=least)
        loss = fi.distillation_loss(X, z, k=4, temperature=temperature, tail="bucket", reduction="none")
        rows = bucket(z, top.values.float(), top.index, top.logsumexp.float(), temperature, least)[0]
        check_values(loss, rows, 4 * U, 3 * S * temperature ** 2, U)


@gpu
@pytest.mark.parametrize("n,c", [(6, 12), (5000, 12), (6, 5000)])
def test_rows_without_an_entry(n, c):
    """They do not count where the named classes are scaled to 1.  With the rest as one more class all of a teacher's mass
    may be there: such a row counts, with a loss of 0, unless its log-sum-exp is -inf."""
    from cuml_b200 import distill

    z = torch.randn((n, c), generator=gen(1), device="cuda")
    v = torch.randn((n, 3), generator=gen(2), device="cuda")
    i = torch.arange(3, device="cuda", dtype=torch.int32).repeat(n, 1)
    lse = torch.logsumexp(v, 1) + 0.5
    i[1::2] = -1
    full = distill.distillation_loss(z, (v, i, lse), tail="bucket", reduction="none")
    assert (full[1::2] == 0).all()
    total = full.double().sum().item()
    mean = distill.distillation_loss(z, (v, i, lse), tail="bucket")
    assert abs(mean.item() - total / n) <= 4 * U * total
    lse[1::2] = NEG
    mean = distill.distillation_loss(z, (v, i, lse), tail="bucket")
    assert abs(mean.item() - total / (n - n // 2)) <= 4 * U * total
    rows = distill.distillation_loss(z, (v, i), reduction="none").double()
    mean = distill.distillation_loss(z, (v, i))
    assert (rows[1::2] == 0).all() and abs(mean.item() - rows.sum().item() / (n - n // 2)) <= 4 * U * rows.sum().item()


# ---- best scores -----------------------------------------------------------------------------------------------
TOPS = [(1000, 10, 3), (5000, 60, 20), (9, 200, 40), (64, 1000, 9), (33, 2000, 30), (1300, 3000, 10), (2, 40_000, 100),
        (1, 140_000, 20), (700, 5000, 30)]


@gpu
@pytest.mark.parametrize("n,c,k", TOPS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.05, 0.2, 0.5, 1000.0])
def test_probabilities_at_other_temperatures(n, c, k, dtype, temperature):
    """x^(1/T) leaves the range of 32 bits, its logarithm does not.  (log x is off by 2 u of its size and the factor 1 / T by
    u; flat rows, nearly flat ones, rows with zeros and with one sure class.)"""
    x = torch.ones((n, c), device="cuda")
    x[n // 3:] += torch.rand((n - n // 3, c), generator=gen(c), device="cuda")
    x[n // 2:, ::3] = 0.0
    x[-1, 1:] = 0.0
    check_top((x / x.sum(1, keepdim=True)).to(TYPES[dtype]), k, temperature, probabilities=True)


@gpu
@pytest.mark.parametrize("n,c,k", TOPS)
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_a_types_largest_value(n, c, k, dtype):
    """The largest value times log2(e) is no number of the type."""
    t = TYPES[dtype]
    x = torch.randn((n, c), generator=gen(c), device="cuda").to(t)
    x[0, c // 2] = torch.finfo(t).max
    x[-1, ::2] = torch.finfo(t).max
    x[n // 2] = torch.finfo(t).max * 0.75
    check_top(x, k)
    check_top(x, k, 4.0)


@gpu
@pytest.mark.parametrize("n,c,k", TOPS)
@pytest.mark.parametrize("dtype", ["fp32", "fp64", "bf16"])
@pytest.mark.parametrize("size", [1e7, 1e9, 3e10, 1e20, 1e36])
def test_scores_far_from_zero(n, c, k, dtype, size):
    """Scores of which one step is more than all exponents; masks of that size on whole rows, and on the first, the last and most
    of the classes of rows."""
    x = torch.randn((n, c), generator=gen(c), device="cuda")
    x[n // 2] *= size
    x[n - 1] = -size
    x[0, :c // 2] = -size
    if n > 2:
        x[1, c // 2:] = -size
        x[n - 2, torch.arange(c, device="cuda") % 256 > 3] = -size
    check_top(x.to(TYPES[dtype]), k)
    check_top(x.to(TYPES[dtype]), k, 2.0)


@gpu
@pytest.mark.parametrize("c", [2, 10, 300, 2000, 40_000])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_the_sum_of_probabilities_keeps_what_additions_drop(c, dtype):
    """At T = 1 log sum p is off by a few u whatever the number of classes: the sum's own rounding to 64 bits, the
    logarithm's, 1 u each, and 2 u where the sum is nearly 1."""
    from cuml_b200 import distill

    x = torch.rand((600, c), generator=gen(c), device="cuda")
    x = (x / x.sum(1, keepdim=True)).to(TYPES[dtype])
    want = x.double().sum(1).log()
    got = distill.top_scores(x, 2, probabilities=True).logsumexp.double()
    assert ((got - want).abs() <= 4 * U * (want.abs() + 2.0 ** -6)).all()


# ---- autograd --------------------------------------------------------------------------------------------------
def students(dtype=torch.float32):
    """(leaves, loss of them) of each operator."""
    from cuml_b200 import distill

    n, c, width = 24, 40, 32
    z = torch.randn((n, c), generator=gen(1), device="cuda")
    h = torch.randn((n, width), generator=gen(2), device="cuda").bfloat16()
    w = torch.randn((c, width), generator=gen(3), device="cuda").bfloat16()
    top = distill.top_scores(torch.randn((n, c), generator=gen(4), device="cuda"), 5)
    target = torch.randint(0, c, (n,), generator=gen(5), device="cuda")
    return [([z], lambda a: distill.distillation_loss(a * 2, top, tail="bucket")),
            ([z], lambda a: distill.cross_entropy(a * 2, target)),
            ([h, w], lambda a, b: distill.linear_distillation_loss(a * 2, b * 2, top)),
            ([h, w], lambda a, b: distill.linear_cross_entropy(a * 2, b * 2, target, reduction="sum"))]


@pytest.fixture(params=["compiled", "ctypes"])
def path(request, monkeypatch):
    from cuml_b200 import distill

    if request.param == "ctypes":
        monkeypatch.setattr(distill, "_call", False)
    return request.param


def fresh(leaves):
    return [x.detach().clone().requires_grad_() for x in leaves]


@gpu
def test_under_an_activation_checkpoint(path):
    """What is saved is computed again in the backward pass."""
    from torch.utils.checkpoint import checkpoint

    for leaves, f in students():
        a = fresh(leaves)
        want = torch.autograd.grad(f(*a), a)
        for reentrant in (False, True):
            b = fresh(leaves)
            checkpoint(f, *b, use_reentrant=reentrant).backward()
            assert all(torch.equal(x, y.grad) for x, y in zip(want, b))


@gpu
def test_under_hooks_that_move_what_is_saved(path):
    """Saved on the host; and given back with its columns first."""
    for leaves, f in students():
        a = fresh(leaves)
        want = torch.autograd.grad(f(*a), a)
        columns = torch.autograd.graph.saved_tensors_hooks(
            lambda x: x, lambda x: x.t().contiguous().t() if x.ndim == 2 else x)
        for hooks in (torch.autograd.graph.save_on_cpu(), columns):
            b = fresh(leaves)
            with hooks:
                loss = f(*b)
            got = torch.autograd.grad(loss, b)
            assert all(torch.equal(x, y) for x, y in zip(want, got))
        for other in (lambda x: x[:5], lambda x: x.double(), lambda x: x.cpu()):
            with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: other(x) if x.ndim == 2 else x):
                loss = f(*fresh(leaves))
            with pytest.raises(RuntimeError, match="hook"):
                loss.backward()


@gpu
def test_forward_mode_is_refused(path):
    """There is no forward-mode derivative: an error, not a tangent that is left out."""
    import torch.autograd.forward_ad as fw

    for leaves, f in students():
        for which in range(len(leaves)):
            with fw.dual_level():
                duals = [fw.make_dual(x, torch.ones_like(x)) if j == which else x for j, x in enumerate(leaves)]
                with pytest.raises(NotImplementedError):
                    f(*duals)


@gpu
def test_the_compiled_path_takes_every_shape_and_autocast():
    """(batch, position, class) logits with their targets, and layers that are cast: no slower than flat ones."""
    from cuml_b200 import distill

    assert distill._native()
    z = torch.randn((4, 6, 50), generator=gen(1), device="cuda").requires_grad_()
    target = torch.randint(0, 50, (4, 6), generator=gen(2), device="cuda")
    for t in (target, target.int(), target.t().contiguous().t()):
        loss = distill.cross_entropy(z, t)
        assert loss.grad_fn.name() == "DistillLossBackward"
        assert torch.equal(loss, distill.cross_entropy(z.detach().view(24, 50), target.reshape(24)))
    h = torch.randn((4, 6, 32), generator=gen(3), device="cuda").requires_grad_()
    w = torch.randn((50, 32), generator=gen(4), device="cuda").requires_grad_()
    top = distill.top_scores(z.detach(), 5)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        losses = [distill.linear_cross_entropy(h, w, target), distill.linear_distillation_loss(h, w, top),
                  distill.linear_cross_entropy(h[0], w, target[0])]
    for loss in losses:
        assert loss.grad_fn.name() == "LinearDistillLossBackward"
        assert all(g.dtype == torch.float32 for g in torch.autograd.grad(loss, (h, w)))
    assert torch.equal(losses[0], distill.linear_cross_entropy(h.bfloat16(), w.bfloat16(), target))


@gpu
def test_a_wait_that_ran_out_is_seen_in_what_is_returned():
    """Until `check_status` has reported it, the losses and gradients of a linear layer are NaN."""
    from cuml_b200 import distill
    from cuml_b200.fil import _lib

    distill.check_status()
    sizes = [(24, 40, 32), (300, 600, 64), (300, 20, 33)]
    layers = [(torch.randn((n, w), generator=gen(1), device="cuda").bfloat16().requires_grad_(),
               torch.randn((c, w), generator=gen(2), device="cuda").bfloat16().requires_grad_(),
               torch.randint(0, c, (n,), generator=gen(3), device="cuda")) for n, c, w in sizes]

    def everything():
        out = []
        for h, w, target in layers:
            loss = distill.linear_cross_entropy(h, w, target)
            out.append((loss, *torch.autograd.grad(loss, (h, w))))
        return out

    want = everything()
    assert _lib.load().b2fil_distill_selftest_timeout(0, torch.cuda.current_stream().cuda_stream) == 0
    for (_, c, _), (loss, *grads) in zip(sizes, everything()):
        assert loss.isnan() or c <= 128  # (logits of few classes are dot products, which wait for nothing)
        assert all(g.isnan().all() for g in grads)
    with pytest.raises(_lib.B2FilError):
        distill.check_status()
    for a, b in zip(want, everything()):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,width,c", [(64, 256, 1000), (64, 256, 100), (600, 1024, 2000)])
def test_a_linear_layer_at_the_lowest_temperatures(n, width, c, dtype):
    """Logits are off by some 1e-6 of their size, which at such temperatures decides between classes: the gradients are
    those of one of the choices, never infinite."""
    from cuml_b200 import distill

    h = torch.randn((n, width), generator=gen(1), device="cuda").to(TYPES[dtype]).requires_grad_()
    w = torch.randn((c, width), generator=gen(2), device="cuda").to(TYPES[dtype]).requires_grad_()
    top = distill.top_scores(h.detach().float() @ w.detach().float().t(), 6)
    for temperature in (1e-6, 1e-5, 1e-4):
        loss = distill.linear_distillation_loss(h, w, top, temperature=temperature)
        up = torch.tensor(1 / temperature, device="cuda")
        grads = torch.autograd.grad(loss, (h, w), up)
        assert torch.isfinite(loss) and all(torch.isfinite(g).all() for g in grads)
