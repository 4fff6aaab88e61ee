"""Best scores and the losses on logits: refusals (CPU), and the kernels against 64 bits (GPU).

Tolerances count roundings.  u = 2^-24 is half a step of fp32.  A term of a softmax is off by 4 u (power of
two), plus u of its exponent's size, which weighs at most 1/e; adding the terms of a thread one after the
other and then those of threads costs at most one u per addition: 64 pieces of 8 in a segment of 16,384
elements, or 4 x 131,072 / (256 x 8) where a block takes a row.  S = 600 u covers every case below; a stored
value is off by half a step of its type."""
import ctypes as C
import math

import pytest
import torch

from tests import distill_reference as ref
from tests.conftest import has_gpu

gpu = pytest.mark.gpu
U = 2.0 ** -24
S = 600 * U
TYPES = {"fp32": torch.float32, "fp64": torch.float64, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}
TINY = {torch.float32: 0.0, torch.float64: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # below normal fp16


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def check_values(got, want, rel, absolute, half):
    got, want = got.detach().cpu().double(), torch.as_tensor(want, dtype=torch.float64)
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    same = got == want
    off = (got - want).abs()
    allowed = torch.as_tensor(rel) * want.abs() + torch.as_tensor(absolute) + half * want.abs()
    bad = ~(same | want.isnan() | (off <= allowed))
    assert not bad.any(), (int(bad.sum()), float((off / allowed)[bad].max()), got[bad][:4], want[bad][:4])


# ---- refusals ------------------------------------------------------------------------------------------------
def test_python_refusals_without_a_gpu():
    from cuml_b200 import distill

    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        distill.top_scores(x, 2)
    with pytest.raises(TypeError):
        distill.top_scores([[1.0]], 1)
    with pytest.raises(ValueError, match="CUDA"):
        distill.distillation_loss(x, (x[:, :2], torch.zeros(4, 2, dtype=torch.int32)))


def test_c_refusals_without_a_gpu(lib):
    from cuml_b200.distill import CTeacher

    def top(dtype=0, n=4, c=8, stride=8, k=2, t=1.0, values=64, ws=None):
        return lib.b2fil_top_scores(dtype, 64, n, c, stride, k, 0, t, values, 64, 64, ws, 0, 0, None)

    for bad in (dict(dtype=9), dict(n=-1), dict(c=0), dict(k=0), dict(k=9), dict(k=257, c=300), dict(t=0.0),
                dict(t=float("nan")), dict(values=None), dict(values=65), dict(stride=7), dict(c=1 << 31)):
        assert top(**bad) == -1, bad
        assert lib.b2fil_last_error()
    assert top(n=0) == 0
    assert lib.b2fil_top_scores_workspace(0, 4, 8, 9, 0) == -1

    def loss(dtype=2, n=4, c=8, stride=8, k=2, index=64, t=1.0, reduction=2, stats=64, out=64, lse=None):
        teacher = CTeacher(64, index, lse, k, k, -100, k, 0)
        return lib.b2fil_distill_loss(dtype, 64, n, c, stride, C.byref(teacher), t, reduction, 64, stats, 64, 64, out, 64,
                                      None, 0, 0, None)

    for bad in (dict(dtype=1), dict(n=-1), dict(c=0), dict(stride=3), dict(k=0), dict(k=257), dict(index=None),
                dict(index=66), dict(t=0.0), dict(t=1e9), dict(reduction=3), dict(stats=72), dict(out=None),
                dict(c=(1 << 20) + 1, stride=1 << 21, lse=64)):
        assert loss(**bad) == -1, bad
    assert lib.b2fil_distill_loss(2, 64, 4, 8, 8, None, 1.0, 0, 64, 64, 64, 64, None, None, None, 0, 0, None) == -1

    def grad(g=64, stride=8, k=2, at=64):
        return lib.b2fil_distill_loss_grad(2, 64, 4, 8, 8, k, 1.0, 64, 64, at, 64, 0, None, g, stride, 0, None)

    for bad in (dict(g=None), dict(g=65), dict(stride=7), dict(k=0), dict(at=None), dict(at=66)):
        assert grad(**bad) == -1, bad


@pytest.mark.skipif(has_gpu(), reason="checks the behaviour on a box without a GPU")
def test_workspace_needs_a_device(lib):
    assert lib.b2fil_top_scores_workspace(0, 4, 8, 2, 0) == -4
    assert lib.b2fil_distill_loss_workspace(0, 4, 8, 2, 99) == -1


@gpu
def test_python_refusals():
    from cuml_b200 import distill

    z = torch.zeros(4, 8, device="cuda")
    v, i = torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, device="cuda", dtype=torch.int32)
    for k in (0, 9):
        with pytest.raises(ValueError, match="k must be"):
            distill.top_scores(z, k)
    with pytest.raises(ValueError, match="k must be"):
        distill.top_scores(torch.zeros(1, 500, device="cuda"), 257)
    with pytest.raises(ValueError, match="must be one of"):
        distill.top_scores(z.int(), 2)
    with pytest.raises(ValueError, match="temperature"):
        distill.top_scores(z, 2, temperature=0)
    for bad, text in (((v, i[:, :1]), "differ in shape"), ((v[:3], i[:3]), "rows"), ((v, i.float()), "index"),
                      ((v.cpu(), i), "CUDA"), ((v[:, :0], i[:, :0]), "k must be")):
        with pytest.raises(ValueError, match=text):
            distill.distillation_loss(z, bad)
    with pytest.raises(ValueError, match="logsumexp"):
        distill.distillation_loss(z, (v, i), tail="bucket")
    with pytest.raises(ValueError, match="tail"):
        distill.distillation_loss(z, (v, i), tail="none")
    with pytest.raises(ValueError, match="reduction"):
        distill.distillation_loss(z, (v, i), reduction="max")
    with pytest.raises(ValueError, match="logits"):
        distill.distillation_loss(z.double(), (v, i))
    with pytest.raises(TypeError):
        distill.distillation_loss(z, v)
    with pytest.raises(ValueError, match="2\\^20"):
        distill.distillation_loss(torch.zeros(1, (1 << 20) + 1, device="cuda"), (v[:1], i[:1], v[:1, 0]), tail="bucket")


@gpu
@pytest.mark.parametrize("columns", [1, 2])
def test_a_target_with_columns_is_refused(columns):
    """One class per row is a target's whole shape, also where the columns could be read as a teacher's entries."""
    from cuml_b200 import distill

    z = torch.zeros(4, 8, device="cuda")
    target = torch.zeros(4, columns, device="cuda", dtype=torch.int64)
    with pytest.raises(ValueError, match="target must have shape"):
        distill.cross_entropy(z, target)
    with pytest.raises(ValueError, match="target must have shape"):
        distill.linear_cross_entropy(z.bfloat16(), torch.zeros(5, 8, device="cuda", dtype=torch.bfloat16), target)
    for index in (target, target[:, 0]):
        with pytest.raises(TypeError, match="values"):
            distill.distillation_loss(z, distill.TopScores(None, index, None))
        with pytest.raises(TypeError, match="values"):
            distill.linear_distillation_loss(z.bfloat16(), z.bfloat16(), distill.TopScores(None, index, None))


# ---- best scores ---------------------------------------------------------------------------------------------
def check_top(x, k, temperature=1.0, probabilities=False):
    from cuml_b200 import distill

    got = distill.top_scores(x, k, temperature=temperature, probabilities=probabilities)
    values, index, lse = ref.top(x, k, temperature, probabilities)
    assert got.index.dtype == torch.int32 and got.values.dtype == x.dtype
    assert torch.equal(got.index.cpu(), index)
    wide = x.dtype == torch.float64
    half = HALF_STEP[x.dtype]
    if not probabilities:
        check_values(got.values, values, 0.0, 0.0, 0.0)
    else:
        check_values(got.values, values, 1e-15 if wide else 2 * U, TINY[x.dtype], half)
    scale = 2.0 ** -53 / U if wide else 1.0
    check_values(got.logsumexp, lse, 4 * U * scale, S * scale, 0.0)


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 7, 7), (1000, 10, 3), (257, 33, 5), (5, 255, 64), (4, 1000, 256), (300, 1001, 17),
          (2, 2049, 100), (3, 16_385, 256), (700, 5000, 8), (1, 50_001, 20), (2, 131_072, 128), (650, 20_000, 33),
          (40, 513, 3), (40, 1024, 24), (40, 1025, 7), (40, 2048, 30), (9, 2047, 256)]


@gpu
@pytest.mark.parametrize("n,c,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_top_scores(n, c, k, dtype):
    x = torch.randn((n, c), generator=gen(n + c + k), device="cuda").mul_(3).to(TYPES[dtype])
    check_top(x, k, temperature=2.0 if k % 2 else 1.0)


@gpu
@pytest.mark.parametrize("n,c,k", [(1000, 10, 3), (64, 300, 40), (2, 40_000, 256), (33, 2000, 9)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 3.0])
def test_top_of_probabilities(n, c, k, dtype, temperature):
    x = torch.rand((n, c), generator=gen(c), device="cuda").mul_(30).sub_(20).clamp_(min=0).round_()
    x[:, 0] += 1
    check_top((x / x.sum(1, keepdim=True)).to(TYPES[dtype]), k, temperature, probabilities=True)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c,k", [(6, 12, 12), (6, 700, 100), (6, 5000, 256), (6, 40_000, 200)])
def test_top_of_hard_rows(n, c, k, dtype):
    """Ties, both zeros, infinities, NaN, masked rows, rows in order, and the best all in one thread's group."""
    t = TYPES[dtype]
    x = torch.randn((n, c), generator=gen(c), device="cuda").to(t)
    x[0] = 0.0
    x[0, 1::2] = -0.0
    x[1] = float("-inf")
    x[2, ::3] = torch.finfo(t).min
    x[2, 5] = float("nan")
    x[2, 9] = float("nan")
    x[3] = torch.arange(c, device="cuda") / c  # ascending, many equal in 16 bits
    x[4] = torch.finfo(t).min
    x[4, 7] = float("inf")
    per = 16 // t.itemsize
    x[5] = -1.0
    for step in range(c // (256 * per)):  # one thread's pieces
        x[5, step * 256 * per:step * 256 * per + per] = 1.0
    check_top(x, k)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [1025, 2049, 4001, 8192])
@pytest.mark.parametrize("k", [1, 7, 24, 25])
def test_top_of_many_rows_of_thousands_of_classes(c, k, dtype):
    """As many rows as belong to a warp each, whose lanes' best give the bound: ordinary ones, ties, both zeros,
    infinities, NaN, fewer scores than k above a mask, rows in order, and the best all in one lane's pieces."""
    t = TYPES[dtype]
    x = torch.randn((1200, c + 5), generator=gen(c + k), device="cuda").to(t)[:, 1:c + 1]  # (rows off the 16-byte boundaries)
    x[10] = 0.0
    x[10, 1::2] = -0.0
    x[20] = float("-inf")
    x[30, ::3] = torch.finfo(t).min
    x[30, 5] = x[30, c - 1] = float("nan")
    x[40] = torch.arange(c, device="cuda") / c
    x[50] = torch.finfo(t).min
    x[50, 7] = float("inf")
    x[60, 3:] = float("-inf")
    x[70, 3:] = torch.finfo(t).min
    x[80] = -1.0
    x[80, torch.arange(c, device="cuda") // (16 // t.itemsize) % 32 < 3] = 1.0
    x[90] = float("nan")
    x[100] = torch.where(torch.arange(c, device="cuda") % 32 < 16, (torch.arange(c, device="cuda") % 401) / 401.0, -1.0).to(t)
    check_top(x, k)
    x[20] = x[10]
    check_top(torch.softmax(x.float().nan_to_num(0.0, 5.0, -5.0), 1).to(t), k, 2.0, probabilities=True)


@gpu
def test_top_where_the_candidates_overflow_their_list():
    """A row whose best 8 x 200 + 2000 scores lie in the groups of few threads: the k-th key is found by bits."""
    for dtype, per in ((torch.float32, 4), (torch.float64, 2), (torch.bfloat16, 8)):
        x = torch.zeros((700, 16_384), device="cuda", dtype=dtype)  # (as many rows as give one block per row)
        place = torch.arange(16_384, device="cuda") // per % 256
        x[:, place < 200] = 1.0
        x[3] = torch.where(place < 200, (torch.arange(16_384, device="cuda") % 97) / 97.0, -1.0).to(dtype)
        check_top(x, 256)


@gpu
def test_top_of_views_and_other_shapes():
    from cuml_b200 import distill

    base = torch.randn((40, 131), generator=gen(5), device="cuda")
    for x in (base[:, 3:110], base.t(), base[::3], base[5:6].expand(7, 131), base[:, ::2]):
        check_top(x, 9)
    cube = base[:, :130].reshape(4, 10, 130)
    got = distill.top_scores(cube, 4)
    assert got.values.shape == (4, 10, 4) and got.logsumexp.shape == (4, 10)
    assert torch.equal(got.index.reshape(40, 4).cpu(), ref.top(base[:, :130], 4)[1])
    one = distill.top_scores(base[0], 4)
    assert one.index.shape == (4,) and one.logsumexp.shape == ()
    none = distill.top_scores(base[:0], 4)
    assert none.values.shape == (0, 4) and none.logsumexp.shape == (0,)
    half = base.half()[:, 1:]  # 2-byte alignment
    check_top(half, 30)


# ---- loss on logits ------------------------------------------------------------------------------------------
def make(n, c, k, dtype, seed, temperature=1.0, index64=False):
    z = torch.randn((n, c), generator=gen(seed), device="cuda").mul_(2)
    t = torch.randn((n, c), generator=gen(seed + 1), device="cuda").add_(z)
    v, i = torch.topk(t, min(k, c), dim=1)
    return z.to(TYPES[dtype]), v, i if index64 else i.int(), torch.logsumexp(t / temperature, 1)


def check_loss(z, values, index, lse, temperature, reduction, upstream=None):
    """`lse` given: with the rest as one more class."""
    from cuml_b200 import distill

    z = z.detach().requires_grad_()
    tail = "renormalise" if lse is None else "bucket"
    loss = distill.distillation_loss(z, (values, index, lse), temperature=temperature, tail=tail, reduction=reduction)
    rows, grad, counts = ref.loss(z, values, index, lse, temperature)
    want, factor = ref.reduced(rows, counts, reduction)
    k = index.shape[1]
    # each logarithm is off by S; the probabilities add to 1; the rest is off by the additions of k entries
    t2 = temperature ** 2
    per_row = t2 * (3 * S) + rows.abs() * 4 * U
    allowed = per_row if reduction == "none" else (per_row * counts).sum() * factor + 4 * U * torch.as_tensor(want).abs()
    check_values(loss, want, 0.0, allowed, U)
    if upstream is None:
        upstream = torch.ones_like(loss)
    (got,) = torch.autograd.grad(loss, z, upstream)
    up = upstream.detach().cpu().double().reshape(-1, 1) * factor
    scale = (up.abs() * temperature).expand(z.shape[0], 1)
    p, _, rest, _ = ref.teacher(values.cpu().double(), index.cpu(), None if lse is None else lse.cpu().double(), z.shape[1],
                                temperature)
    q = (torch.softmax(z.detach().cpu().double() / temperature, 1)).nan_to_num()
    # q and p are off by S relative; the factor of the rest by S of both its sides
    allowed = scale * (2 * S * (q + p)) + 4 * S * (grad * up).abs() + TINY[z.dtype]
    if lse is not None:
        others = (q * (p == 0)).sum(1, keepdim=True)
        allowed = allowed + scale * q * (rest[:, None] * 4 * S + k * 4 * U) / others.clamp(min=1e-30)
    check_values(got, grad * up, 0.0, allowed, HALF_STEP[z.dtype])
    return loss, got


LOSSES = [(1, 1, 1), (1, 2, 1), (64, 10, 3), (1003, 10, 10), (37, 33, 5), (130, 1001, 16), (9, 2048, 256), (9, 2049, 40),
          (500, 3000, 8), (3, 50_001, 20), (2, 131_072, 64), (301, 9001, 2),
          (9001, 2, 2), (5003, 13, 3), (6000, 64, 16), (5000, 64, 17), (5000, 65, 4)]


@gpu
@pytest.mark.parametrize("n,c,k", LOSSES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tail", ["renormalise", "bucket"])
def test_distillation_loss(n, c, k, dtype, tail):
    temperature = 2.0 if n % 2 else 1.0
    z, v, i, lse = make(n, c, k, dtype, n + c, temperature, index64=bool(c % 2))
    for reduction in ("mean", "sum", "none"):
        up = torch.rand((n,), generator=gen(3), device="cuda") if reduction == "none" else None
        if reduction == "mean" and dtype == "fp16":
            up = torch.tensor(8.0 * n, device="cuda")
        check_loss(z, v, i, lse if tail == "bucket" else None, temperature, reduction, up)


@gpu
@pytest.mark.parametrize("c", [40, 700, 5000, 40_000])
@pytest.mark.parametrize("tail", ["renormalise", "bucket"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_masks_of_teacher_and_student(c, tail, dtype):
    n, k = 8, 20
    z, v, i, lse = make(n, c, k, dtype, c)
    i[0, 3] = i[0, 1]          # named twice
    i[0, 7] = i[0, 1]
    i[1, 5:] = -1              # fewer than k
    i[2] = -1                  # none named
    v[3] = float("-inf")       # a teacher without a class
    lse[3] = float("-inf")
    i[4, 0] = c                # outside
    z[5] = float("-inf")       # a student without a class
    lowest = torch.finfo(z.dtype).min
    z[6] = lowest              # all equal
    z[6, 1::2] = float("-inf")
    i[6, :] = torch.arange(0, 2 * k, 2, device="cuda", dtype=torch.int32)
    z[7] = torch.where(torch.arange(c, device="cuda") % 3 == 0, z[7], lowest)
    i[7, :] = torch.arange(0, k, device="cuda", dtype=torch.int32)[torch.randperm(k)].int() % c
    v[7] = torch.where(i[7] % 3 == 0, v[7], float("-inf"))
    if tail == "bucket":
        lse[7] = torch.logsumexp(v[7], 0) + 0.3
    for reduction in ("mean", "none"):
        check_loss(z, v, i, lse if tail == "bucket" else None, 1.0, reduction)
    if c == 40:  # as many rows as belong to a thread each, with sixteen entries
        many = lambda x: x.repeat(700, *[1] * (x.ndim - 1))  # noqa: E731
        check_loss(many(z), many(v[:, :16]), many(i[:, :16]), many(lse) if tail == "bucket" else None, 1.0, "mean")


@gpu
@pytest.mark.parametrize("n,c,k,dtype", [(1300, 2049, 40, "bf16"), (1300, 4096, 3, "fp32"), (1211, 4097, 9, "fp32"),
                                         (1200, 8191, 16, "fp16"), (1200, 8193, 2, "bf16"), (1183, 6000, 5, "bf16")])
@pytest.mark.parametrize("tail", ["renormalise", "bucket"])
def test_many_rows_of_thousands_of_classes(n, c, k, dtype, tail):
    """On both sides of where such rows belong to a warp each (at most 256 terms per lane); rows 3 elements apart."""
    z, v, i, lse = make(n, c + 3, k, dtype, c, 2.0)
    z, i = z[:, :c], i % c  # (some classes may be named twice)
    lse = torch.logsumexp(v.double() / 2.0, 1).float() + 0.25
    check_loss(z, v, i, lse if tail == "bucket" else None, 2.0, "mean")
    up = torch.rand((n,), generator=gen(4), device="cuda")
    check_loss(z, v, i, lse if tail == "bucket" else None, 2.0, "none", up)


@gpu
def test_rows_that_do_not_count_have_no_gradient_whatever_is_in_them():
    from cuml_b200 import distill

    for c in (50, 3000):
        z, v, i, _ = make(4, c, 4, "bf16", 1)
        z[1] = float("nan")
        i[1] = -1
        z = z.requires_grad_()
        loss = distill.distillation_loss(z, (v, i))
        (g,) = torch.autograd.grad(loss, z)
        assert torch.isfinite(loss) and (g[1] == 0).all() and torch.isfinite(g).all()
        none = distill.distillation_loss(z, (v, torch.full_like(i, -1)))
        assert none.item() == 0.0 and (torch.autograd.grad(none, z)[0] == 0).all()
        empty = distill.distillation_loss(z[:0], (v[:0], i[:0]))
        assert empty.item() == 0.0 and torch.autograd.grad(empty, z)[0].abs().sum() == 0


@gpu
def test_infinite_and_nan_logits_as_in_a_softmax():
    from cuml_b200 import distill

    z, v, i, _ = make(4, 300, 4, "fp32", 1)
    z[0, i[0, 0].item()] = float("-inf")  # the teacher gives it mass
    z[1, 17] = float("nan")
    z[2, 18] = float("inf")
    rows = distill.distillation_loss(z, (v, i), reduction="none")
    assert rows[0] == float("inf") and rows[1].isnan() and rows[2].isnan() and rows[3].isfinite()


@gpu
def test_logits_of_other_strides_and_shapes():
    from cuml_b200 import distill

    z, v, i, lse = make(60, 1000, 7, "bf16", 9)
    for view in (z[:, 1:900], z[::2], z.t().contiguous().t(), z[:1].expand(60, 1000)):
        n, c = view.shape
        ii = i[:n] % c
        check_loss(view, v[:n], ii, None, 1.0, "mean")
    wide = torch.randn((60, 50), generator=gen(2), device="cuda")
    check_loss(z, wide[:, 3:43:4][:, :7], torch.cat([i, i], 1)[:, 7:], lse, 1.0, "sum")
    cube = z.view(3, 20, 1000).requires_grad_()
    rows = distill.distillation_loss(cube, (v.view(3, 20, 7), i.view(3, 20, 7), lse.view(3, 20)), tail="bucket",
                                     reduction="none")
    assert rows.shape == (3, 20)
    flat, grad, _ = ref.loss(z, v, i, lse, 1.0)
    check_values(rows.reshape(-1), flat, 0.0, 3 * S, 4 * U)
    (g,) = torch.autograd.grad(rows, cube, torch.ones(1, device="cuda").expand(3, 20))
    check_values(g.reshape(60, 1000), grad, 4 * S, 1e-5, HALF_STEP[torch.bfloat16])


@gpu
def test_gradient_against_differences():
    """Central differences of the loss itself, h = 2^-5: their own error is h^2/6 of the third derivative (below
    1), and 3 S / h of the loss's roundings."""
    from cuml_b200 import distill

    z, v, i, lse = make(3, 12, 4, "fp32", 4, 2.0)
    z = z.requires_grad_()
    h = 2.0 ** -5
    for tail in ("renormalise", "bucket"):
        f = lambda x: distill.distillation_loss(x, (v, i, lse), temperature=2.0, tail=tail, reduction="sum")  # noqa: E731
        (g,) = torch.autograd.grad(f(z), z)
        for r in range(3):
            for c in range(12):
                d = torch.zeros_like(z)
                d[r, c] = h
                slope = (f(z.detach() + d) - f(z.detach() - d)) / (2 * h)
                assert abs(slope.item() - g[r, c].item()) < h * h / 6 + 3 * 4 * 3 * S / h


@gpu
def test_without_the_compiled_call_path(monkeypatch):
    """The same numbers, gradients and errors through ctypes."""
    from cuml_b200 import distill

    z, v, i, lse = make(50, 300, 7, "bf16", 9)
    h = torch.randn((50, 64), generator=gen(1), device="cuda").bfloat16()
    w = torch.randn((300, 64), generator=gen(2), device="cuda").bfloat16()

    def everything():
        out = list(distill.top_scores(z, 5))
        for reduction in ("mean", "none"):
            x = z.detach().requires_grad_()
            loss = distill.distillation_loss(x, distill.TopScores(v, i, lse), tail="bucket", reduction=reduction)
            a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
            of_layer = distill.linear_distillation_loss(a, b, (v, i), reduction=reduction, temperature=2.0)
            out += [loss, *torch.autograd.grad(loss.sum(), x), of_layer, *torch.autograd.grad(of_layer.sum(), (a, b))]
        return out

    assert distill._native()
    compiled = everything()
    monkeypatch.setattr(distill, "_call", False)
    for x, y in zip(compiled, everything()):
        assert x.dtype == y.dtype and torch.equal(x, y)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_autograd_rules(monkeypatch, compiled):
    """A graph is used once unless it is retained, inputs are not changed in between, there is no second derivative."""
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z, v, i, lse = make(5, 30, 4, "fp32", 9)
    h = torch.randn((5, 16), generator=gen(1), device="cuda").bfloat16()
    w = torch.randn((30, 16), generator=gen(2), device="cuda").bfloat16()
    top = distill.TopScores(v, i, lse)
    for leaves, f in (([z], lambda a: distill.distillation_loss(a, top)),
                      ([h, w], lambda a, b: distill.linear_distillation_loss(a, b, top))):
        leaves = [x.detach().requires_grad_() for x in leaves]
        loss = f(*leaves)
        first = torch.autograd.grad(loss, leaves, retain_graph=True)
        again = torch.autograd.grad(loss, leaves)
        assert all(torch.equal(x, y) for x, y in zip(first, again))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(loss, leaves)
        loss = f(*leaves)
        with torch.no_grad():
            leaves[0].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, leaves)
        grads = torch.autograd.grad(f(*leaves), leaves, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grads[0].sum(), leaves)
        with torch.no_grad():
            assert not f(*leaves).requires_grad
        assert not f(*[x.detach() for x in leaves]).requires_grad
        (2 * f(*leaves)).backward()
        assert all(x.grad is not None and x.grad.shape == x.shape for x in leaves)
        # an upstream gradient of another type and stride
        rows = distill.distillation_loss(leaves[0], top, reduction="none") if len(leaves) == 1 else \
            distill.linear_distillation_loss(*leaves, top, reduction="none")
        up = torch.arange(10, device="cuda", dtype=torch.float32)[::2]
        a = torch.autograd.grad(rows, leaves, up, retain_graph=True)
        b = torch.autograd.grad(rows, leaves, up.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("n,c", [(1, 2), (64, 10), (33, 1001), (5, 5000)])
def test_cross_entropy(monkeypatch, compiled, n, c):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    z = (torch.randn((n, c), generator=gen(c), device="cuda") * 2).requires_grad_()
    target = torch.randint(0, c, (n,), generator=gen(n), device="cuda")
    if n > 4:
        target[1], target[2], target[3] = -100, c, -1
    rows, grad, counts = ref.loss(z, None, target[:, None])
    for reduction in ("mean", "sum", "none"):
        want, factor = ref.reduced(rows, counts, reduction)
        loss = distill.cross_entropy(z, target, reduction=reduction)
        check_values(loss, want, 4 * U, 3 * S * (n if reduction == "sum" else 1), U)
        (g,) = torch.autograd.grad(loss, z, torch.ones_like(loss))
        check_values(g, grad * factor, 4 * S, 4 * S * factor, U)
    assert torch.equal(distill.cross_entropy(z, target.int(), ignore_index=0, reduction="none"),
                       distill.cross_entropy(z, torch.where(target == 0, -5, target), reduction="none"))
    cube = z.detach().reshape(n, 1, c)
    assert torch.equal(distill.cross_entropy(cube, target[:, None], reduction="none")[:, 0],
                       distill.cross_entropy(z, target, reduction="none"))
    for bad, text in ((target[:0], "target must have shape"), (target.float(), "target must be one of"), (target.cpu(), "CUDA")):
        with pytest.raises(ValueError, match=text):
            distill.cross_entropy(z, bad)
    with pytest.raises(ValueError, match="reduction"):
        distill.cross_entropy(z, target, reduction="max")


@gpu
@pytest.mark.parametrize("dtype", ["fp64", "bf16", "fp16"])
@pytest.mark.parametrize("compiled", [True, False])
def test_teachers_of_other_types(monkeypatch, dtype, compiled):
    """The scores that `top_scores` returns go into a loss as they are."""
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    t = torch.randn((40, 300), generator=gen(1), device="cuda").to(TYPES[dtype])
    z = torch.randn((40, 300), generator=gen(2), device="cuda")
    top = distill.top_scores(t, 9)
    check_loss(z, top.values.float(), top.index, top.logsumexp.float(), 1.0, "mean")
    for tail in ("renormalise", "bucket"):
        given = distill.distillation_loss(z, top, tail=tail, reduction="none")
        in_floats = distill.TopScores(top.values.float(), top.index, top.logsumexp.float())
        assert torch.equal(given, distill.distillation_loss(z, in_floats, tail=tail, reduction="none"))


@gpu
def test_more_than_two_to_the_31_elements():
    """The last rows of large arrays, and the last classes of a large layer, against the same rows alone."""
    from cuml_b200 import distill

    n, c = 66_000, 32_800
    x = torch.randn((n, c), generator=gen(1), device="cuda", dtype=torch.bfloat16)
    top = distill.top_scores(x, 7)
    few = distill.top_scores(x[-900:].clone(), 7)
    for a, b in zip(top, few):
        assert torch.equal(a[-900:], b)
    z = x.requires_grad_()
    loss = distill.distillation_loss(z, top, reduction="none")
    (g,) = torch.autograd.grad(loss, z, torch.ones_like(loss))
    tail = x.detach()[-900:].clone().requires_grad_()
    rows = distill.distillation_loss(tail, few, reduction="none")
    assert torch.equal(loss[-900:], rows)
    assert torch.equal(g[-900:], torch.autograd.grad(rows, tail, torch.ones_like(rows))[0])
    assert (g[0] != 0).any()
