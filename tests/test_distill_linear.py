"""Losses on a linear layer's output: refusals (CPU), and the kernels against 64 bits (GPU).

Tolerances count roundings; u = 2^-24, S as in test_distill.py.  A product's sum of width terms is off by at most
2 u for each of width / 8 + 16 additions, of the sum of the terms' sizes: e_z.  So are both sums of the
gradients, over classes and over rows.  A difference softmax - teacher is off by 2 e_z / T + 2 S relative in each of its
parts, and half a step of the layer's type; each enters the sums with the size of what it is multiplied by."""
import ctypes as C

import pytest
import torch

from tests import distill_reference as ref
from tests.test_distill import HALF_STEP, S, TYPES, U, check_values, gen, gpu


def layer(n, width, c, dtype, seed=0):
    g = gen(seed + n + width + c)
    h = torch.randn((n, width), generator=g, device="cuda")
    w = torch.randn((c, width), generator=g, device="cuda") * (2 / width ** 0.5)
    return h.to(TYPES[dtype]), w.to(TYPES[dtype])


def adds(n):
    return (n / 8 + 16) * 2 * U


def check(h, w, values, index, temperature, reduction, upstream=None, wants=(True, True), call=None):
    from cuml_b200 import distill

    n, c, k = h.shape[0], w.shape[0], index.shape[1]
    half = HALF_STEP[h.dtype]
    h, w = h.detach().requires_grad_(wants[0]), w.detach().requires_grad_(wants[1])
    if call is None:
        call = lambda: distill.linear_distillation_loss(h, w, (values, index), temperature=temperature,  # noqa: E731
                                                        reduction=reduction)
        loss = call()
    else:
        loss = call(h, w)
    hd, wd = h.detach().cpu().double(), w.detach().cpu().double()
    z = hd @ wd.t()
    e_z = adds(h.shape[1]) * (hd.abs() @ wd.abs().t()).amax(1)  # per row
    rows, grad, counts = ref.loss(z, values, index, None, temperature)
    want, factor = ref.reduced(rows, counts, reduction)
    per_row = temperature ** 2 * (3 * S + 2 * e_z / temperature) + rows.abs() * 4 * U
    allowed = per_row if reduction == "none" else (per_row * counts).sum() * factor + 4 * U * torch.as_tensor(want).abs()
    check_values(loss, want, 0.0, allowed, U)
    leaves = [x for x, is_wanted in zip((h, w), wants) if is_wanted]
    if not leaves:
        return
    if upstream is None:
        upstream = torch.ones_like(loss)
    got = list(torch.autograd.grad(loss, leaves, upstream))
    up = upstream.detach().cpu().double().reshape(-1, 1) * factor
    d = grad * up
    p = ref.teacher(None if values is None else values.cpu().double(), index.cpu(), None, c, temperature)[0]
    q = torch.softmax(z / temperature, 1)
    scale = (up.abs() * temperature).expand(n, 1) * counts[:, None]
    e_d = scale * (q + p) * (2 * S + (2 * e_z / temperature)[:, None]) + d.abs() * half
    if h.dtype == torch.float16:  # below 2^-14 of the scaled differences, steps are 2^-24
        e_d = e_d + up.abs().max() * temperature * 2.0 ** -25 / 2.0 ** 14 * 2
    tiny = 2.0 ** -25 if h.dtype == torch.float16 else 0.0
    for x, is_hidden in zip(("h", "w"), (True, False)):
        if not wants[0 if is_hidden else 1]:
            continue
        g = got.pop(0)
        other, dd, ee = (wd, d, e_d) if is_hidden else (hd, d.t(), e_d.t())
        exact = dd @ other
        allowed = ee @ other.abs() + adds(dd.shape[1]) * (dd.abs() @ other.abs())
        assert g.dtype == h.dtype and g.is_contiguous()
        check_values(g, exact, 2 * U, allowed + tiny, half)


def entries(n, c, k, seed=0, index64=False):
    g = gen(seed + c)
    i = torch.stack([torch.randperm(c, generator=g, device="cuda")[:k] for _ in range(n)])
    v = torch.randn((n, k), generator=g, device="cuda").mul_(2).sort(1, descending=True).values
    return v, i if index64 else i.int()


# rows, width, classes: one tile and less, its borders, several tiles, sums over classes and over rows in several
# parts, odd widths
SIZES = [(1, 8, 1), (1, 64, 2), (3, 16, 7), (128, 64, 256), (129, 72, 257), (256, 256, 256), (257, 264, 300),
         (64, 128, 1000), (200, 520, 1003), (513, 200, 2050), (40, 96, 20_011), (300, 33, 130), (70, 1001, 515),
         (5000, 64, 40), (9000, 264, 513), (3, 1, 5), (500, 1003, 2100)]


@gpu
@pytest.mark.parametrize("n,width,c", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_distillation(n, width, c, dtype):
    from cuml_b200 import distill

    h, w = layer(n, width, c, dtype)
    k = min(c, 9)
    v, i = entries(n, c, k, index64=bool(n % 2))
    for reduction, t in (("mean", 1.0), ("sum", 2.0), ("none", 4.0)):
        up = torch.rand((n,), generator=gen(3), device="cuda") * 3 if reduction == "none" else None
        if reduction == "mean" and dtype == "fp16":
            up = torch.tensor(8.0 * n, device="cuda")
        check(h, w, v, i, t, reduction, up)
    distill.check_status()


@gpu
@pytest.mark.parametrize("n,width,c", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_cross_entropy(n, width, c, dtype):
    from cuml_b200 import distill

    h, w = layer(n, width, c, dtype, seed=7)
    target = torch.randint(0, c, (n,), generator=gen(1), device="cuda")
    if n > 2:
        target[::5] = -100
        target[1] = c
    for reduction in ("mean", "sum", "none"):
        up = torch.tensor(8.0 * n, device="cuda") if reduction == "mean" and dtype == "fp16" else None
        check(h, w, None, target[:, None], 1.0, reduction, up,
              call=lambda a, b: distill.linear_cross_entropy(a, b, target, reduction=reduction))
    check(h, w, None, target[:, None].int(), 1.0, "sum", wants=(True, False),
          call=lambda a, b: distill.linear_cross_entropy(a, b, target.int(), reduction="sum"))
    check(h, w, None, target[:, None], 1.0, "sum", wants=(False, True),
          call=lambda a, b: distill.linear_cross_entropy(a, b, target, reduction="sum"))
    distill.check_status()


@gpu
@pytest.mark.parametrize("k", [2, 5])
def test_several_pieces_of_the_classes(k):
    """(20,000 x 7,000 differences are more than one piece holds; few enough for the CPU to check.)"""
    h, w = layer(20_000, 16, 7000, "bf16")
    v, i = entries(20_000, 7000, k)
    check(h, w, v, i, 1.0, "mean")


@gpu
def test_no_row_counts_and_no_rows():
    from cuml_b200 import distill

    h, w = layer(5, 32, 40, "bf16")
    h, w = h.requires_grad_(), w.requires_grad_()
    target = torch.full((5,), -100, device="cuda")
    loss = distill.linear_cross_entropy(h, w, target)
    a, b = torch.autograd.grad(loss, (h, w))
    assert loss.item() == 0.0 and (a == 0).all() and (b == 0).all()
    loss = distill.linear_cross_entropy(h[:0], w, target[:0])
    a, b = torch.autograd.grad(loss, (h, w))
    assert loss.item() == 0.0 and (a == 0).all() and (b == 0).all()
    rows = distill.linear_cross_entropy(h, w, target.clone().fill_(3), ignore_index=3, reduction="none")
    assert rows.shape == (5,) and (rows == 0).all()


@gpu
def test_shapes_strides_and_autocast():
    from cuml_b200 import distill

    h, w = layer(60, 64, 200, "bf16")
    wide = torch.zeros((60, 80), dtype=torch.bfloat16, device="cuda")
    wide[:, 8:72] = h
    target = torch.randint(0, 200, (60,), generator=gen(1), device="cuda")
    want = distill.linear_cross_entropy(h, w, target)
    assert torch.equal(distill.linear_cross_entropy(wide[:, 8:72], w, target), want)
    assert torch.equal(distill.linear_cross_entropy(h.t().contiguous().t(), w.t().contiguous().t(), target), want)
    wide[:, 3:67] = h
    assert torch.equal(distill.linear_cross_entropy(wide[:, 3:67], w, target), want)  # rows not on 16 bytes
    cube = h.view(3, 20, 64).detach().requires_grad_()
    rows = distill.linear_cross_entropy(cube, w, target.view(3, 20), reduction="none")
    assert rows.shape == (3, 20) and torch.autograd.grad(rows.sum(), cube)[0].shape == cube.shape
    h32, w32 = h.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = distill.linear_cross_entropy(h32, w32, target)
    assert torch.equal(loss, want)
    a, b = torch.autograd.grad(loss, (h32, w32))
    assert a.dtype == b.dtype == torch.float32


@gpu
def test_python_refusals():
    from cuml_b200 import distill

    h, w = layer(4, 16, 10, "bf16")
    target = torch.zeros(4, dtype=torch.int64, device="cuda")
    for args, text in (((h.float(), w.float(), target), "hidden must be one of"), ((h, w.half(), target), "differ in type"),
                       ((h, w[:, :8], target), "width"), ((h, w, target[:3]), "target must have shape"),
                       ((h, w, target.float()), "target must be one of"), ((h.cpu(), w, target), "CUDA"),
                       ((h, w[:0], target), "n_classes")):
        with pytest.raises(ValueError, match=text):
            distill.linear_cross_entropy(*args)
    with pytest.raises(ValueError, match="reduction"):
        distill.linear_cross_entropy(h, w, target, reduction="all")
    with pytest.raises(ValueError, match="rows"):
        distill.linear_distillation_loss(h, w, (torch.zeros(3, 2, device="cuda"), torch.zeros(3, 2, device="cuda").int()))


def test_c_refusals_without_a_gpu(lib):
    from cuml_b200.distill import CTeacher

    def call(dtype=2, hidden=64, weight=64, hs=16, ws=16, n=4, c=10, width=16, k=2, lse=None, reduction=2, stats=64, at=64,
             t=1.0):
        teacher = CTeacher(64, 64, lse, k, k, -100, k, 0)
        return lib.b2fil_linear_loss(dtype, hidden, hs, weight, ws, n, c, width, C.byref(teacher), t, reduction, 64, stats,
                                     64, 64, at, 64, 64, None, 0, 0, None)

    for bad in (dict(dtype=0), dict(hidden=None), dict(weight=65), dict(hs=8), dict(ws=15), dict(n=-1), dict(n=(1 << 31) - 1),
                dict(c=0), dict(width=0), dict(width=(1 << 20) + 1), dict(k=0), dict(k=257), dict(lse=64), dict(reduction=5),
                dict(stats=68), dict(at=None), dict(t=0.0)):
        assert call(**bad) == -1, bad
        assert lib.b2fil_last_error()

    def grad(n=4, width=16, k=2, up=64, dh=64, dw=64, t=1.0):
        return lib.b2fil_linear_loss_grad(2, 64, 16, 64, 16, n, 10, width, k, t, 64, 64, 64, 64, up, 0, None, dh, dw, None,
                                          0, 0, None)

    for bad in (dict(n=-1), dict(width=17), dict(k=0), dict(up=None), dict(dh=72), dict(dw=8), dict(t=-1.0)):
        assert grad(**bad) == -1, bad
    assert grad(dh=None, dw=None) == 0
    assert lib.b2fil_distill_status(0, None) == -1


@gpu
def test_a_wait_that_runs_out_is_reported_once():
    from cuml_b200 import distill
    from cuml_b200.fil import _lib

    distill.check_status()
    lib = _lib.load()
    assert lib.b2fil_distill_selftest_timeout(0, torch.cuda.current_stream().cuda_stream) == 0
    with pytest.raises(_lib.B2FilError) as e:
        distill.check_status()
    assert e.value.code == -7
    distill.check_status()


_FIRST_BACKWARD = """
import torch
from cuml_b200 import distill
h = torch.ones(256, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
w = torch.ones(1000, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
loss = distill.linear_cross_entropy(h, w, torch.zeros(256, dtype=torch.int64, device="cuda"))
torch.autograd.grad(loss, (h, w))
distill.check_status()
print("first", loss.item())
"""


@gpu
def test_the_first_thing_that_autograds_thread_does():
    """The thread of a process's first backward pass has no CUDA context yet."""
    import subprocess
    import sys

    from tests.conftest import ROOT

    r = subprocess.run([sys.executable, "-c", _FIRST_BACKWARD], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("first 6.9"), r.stderr[-800:]


@gpu
def test_a_layer_of_more_than_two_to_the_31_weights():
    """(4 x 1040 x 2,100,000.)  The logits' sums of 1040 terms are off by e_z = 2 u (1040 / 8 + 16) of the sum of their
    terms' sizes, here below 60; the gradients as above."""
    from cuml_b200 import distill

    n, width, c = 4, 1040, 2_100_000
    h = torch.randn((n, width), generator=gen(1), device="cuda").bfloat16().requires_grad_()
    w = torch.randn((c, width), generator=gen(2), device="cuda", dtype=torch.bfloat16).mul_(2 / width ** 0.5).requires_grad_()
    target = torch.tensor([c - 1, 5, c - 300, c // 2], device="cuda")
    loss = distill.linear_cross_entropy(h, w, target, reduction="none")
    dh, dw = torch.autograd.grad(loss, (h, w), torch.ones_like(loss))
    distill.check_status()
    with torch.no_grad():
        z = torch.cat([h.double() @ part.double().t() for part in w.split(300_000)], 1)
        rows, grad, _ = ref.loss(z, None, target[:, None])
        e_z = adds(width) * 60
        check_values(loss, rows, 4 * U, 3 * S + 2 * e_z, U)
        half = HALF_STEP[torch.bfloat16]
        e_d = grad.abs() * (half + 2 * S + 2 * e_z) + 1e-12
        for at in (slice(0, 10), slice(c - 310, c)):
            exact = grad[:, at].t() @ h.cpu().double()
            check_values(dw[at], exact, 2 * U, (e_d[:, at].t() + adds(n) * grad[:, at].t().abs()) @ h.cpu().double().abs(), half)
        exact = sum(grad[:, a:a + 300_000] @ w[a:a + 300_000].cpu().double() for a in range(0, c, 300_000))
        allowed = sum((e_d[:, a:a + 300_000] + adds(c) * grad[:, a:a + 300_000].abs()) @ w[a:a + 300_000].cpu().double().abs()
                      for a in range(0, c, 300_000))
        check_values(dh, exact, 2 * U, allowed, half)
