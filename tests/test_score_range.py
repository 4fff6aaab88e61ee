"""Scores and clipping at the ends of their ranges: low temperatures, many sums per tile, shared memory of tensors."""
import math

import pytest
import torch

from tests import score_reference as ref
from tests.test_distill import HALF_STEP, S, TYPES, U, check_values, gen
from tests.test_score import adds, check, entropy_error, layer, logits, targets, upstreams, wide

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,width,c", [(64, 2048, 300), (64, 2048, 200), (64, 2048, 2000), (500, 1024, 1000), (3, 520, 20)])
@pytest.mark.parametrize("sign", [-1, 1])
def test_entropy_of_a_layer_at_the_lowest_temperature(n, width, c, dtype, sign):
    """The logits' roundings over T are exponents of tens there, so a class of many that are equal may seem to have all of the row in the
    backward pass.  Whatever q <= 1 is taken for it, its difference is h q (log q + H) / T with q |log q| <= 1 / e and H <= log n_classes:
    at most |h| log n_classes / T, which bounds both gradients (and rounding takes at most half a step more, of the differences
    and of the sums)."""
    from cuml_b200 import distill

    t, temperature, up = TYPES[dtype], 1e-6, 1e-8
    h = (torch.rand((n, width), generator=gen(1), device="cuda") + 0.5).to(t).requires_grad_()
    w = ((torch.rand((1, width), generator=gen(2), device="cuda") + 0.5) * (sign / 8)).to(t).repeat(c, 1).requires_grad_()
    got = distill.linear_log_probs(h, w, temperature=temperature)
    dh, dw = torch.autograd.grad(got.entropy, (h, w), torch.full((n,), up, device="cuda"))
    each = up / temperature * math.log(c) * (1 + 4 * HALF_STEP[t])
    assert (wide(dh).abs() <= each * wide(w).abs().sum(0)).all()
    assert (wide(dw).abs() <= each * wide(h).abs().sum(0)).all()
    distill.check_status()


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_tensors_that_share_memory_until_one_is_written(monkeypatch, compiled):
    """A clone that is made when it is written (copy on write) is made before it is clipped, or taken as `out`: what it was made from stays.
    Measuring a norm makes none."""
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    for n in (1000, 300_000):
        source = torch.full((n,), 2.0, device="cuda")
        x, y = torch._lazy_clone(source), torch._lazy_clone(source)
        norm = distill.clip_gradients([x], 1.0)
        assert (source == 2).all() and (y == 2).all() and torch.allclose(x, source / norm)
        kept = torch.full((n,), 5.0, device="cuda")
        out = torch._lazy_clone(kept)
        distill.clip_gradients([source], 1.0, out=[out])
        assert (kept == 5).all() and (source == 2).all() and torch.equal(out, x)
        z = torch._lazy_clone(source)
        assert torch.equal(distill.gradient_norm([z, y]), distill.gradient_norm([source, source]))
        if compiled:
            assert torch._C._is_cow_tensor(z)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
def test_few_gradients_clipped_by_one_launch_after_the_other(dtype, kind):
    """A launch reads what the launch before has written, and what it writes itself only after all of it has been read.  Halved each time, so
    that nothing is rounded: powers of two that fp16 holds, 50,000 of them and few, on and off the 16-byte boundaries."""
    from cuml_b200 import distill

    for n in (7, 3001, 50_000):
        flat = torch.zeros(n + 11, dtype=TYPES[dtype], device="cuda")
        parts = list(flat[3:3 + n].split((n + 2) // 3))
        start = [2.0 ** torch.randint(0, 6, x.shape, generator=gen(n), device="cuda") for x in parts]

        def clip():
            for x, y in zip(parts, start):
                x.copy_(y)
            return [distill.clip_gradients(parts, m, norm_type=kind) for m in limits]

        size = torch.cat(start).double()
        norm = float(size.max() if kind == math.inf else size.sum() if kind == 1.0 else size.square().sum().sqrt())
        limits = [norm / 2 ** i for i in range(1, 6)]
        clip()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms = clip()
        for _ in range(3):
            graph.replay()
            for i, got in enumerate(norms):
                assert abs(got.item() - norm / 2 ** i) <= 12 * (i + 1) * 2.0 ** -24 * norm / 2 ** i
            for x, y in zip(parts, start):
                # (a factor is off by 12 steps of fp32 at most, an element by half a step of its type for each of the five)
                assert ((wide(x) * 32 - wide(y)).abs() <= wide(y) * 5 * (12 * 2.0 ** -24 + HALF_STEP[x.dtype])).all()
            assert not flat[:3].any() and not flat[3 + n:].any()
        del graph


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_norm_of_mostly_zero_gradients(dtype):
    """Zeros of both signs are left out at once; what is so small that its square is zero in 32 bits is not.  (9 u of the norm, as in
    test_gradients.py, and for norms below 2^-126, which are multiples of 2^-149 in fp32, half of that: 2^-150.)"""
    from cuml_b200 import distill

    for size in (1.0, 1e-30, 2.0 ** -133):
        for n in (5, 4099, 100_003):
            x = torch.zeros(n, dtype=TYPES[dtype], device="cuda")
            x[1::3] = -0.0
            assert distill.gradient_norm([x]) == 0
            x[:: 997] = size
            x[n - 1] = -3 * size
            want = float(wide(x).square().sum().sqrt())
            assert abs(distill.gradient_norm([x]).item() - want) <= 9 * 2.0 ** -24 * want + 2.0 ** -150
            assert distill.gradient_norm([x], norm_type=math.inf) == wide(x).abs().max()
            x[n // 2] = float("nan")
            assert distill.gradient_norm([x]).isnan()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,width,c", [(7000, 3, 40), (7000, 12, 300), (3000, 17, 5000), (6000, 20, 300), (300, 20, 9000), (2000, 29, 300),
                                       (257, 33, 300), (5000, 50, 515), (300, 100, 9001), (300, 1001, 20_011), (1500, 250, 700)])
def test_gradients_of_odd_widths_are_those_of_wider_rows_of_zeros(n, width, c, dtype):
    """Rows that are no whole pieces of 16 bytes are copied with zeros behind them.  Those zeros given by the caller take part in the same
    products and sums, so what comes out for the other columns is the same, bit for bit."""
    from cuml_b200 import distill

    t, line = TYPES[dtype], 16
    h, w = (torch.randn(s, generator=gen(width + s[0]), device="cuda").to(t) for s in ((n, width), (c, width)))
    pad = (width + line - 1) // line * line - width
    target = torch.randint(0, c, (n,), generator=gen(c), device="cuda")
    up = torch.randn(n, generator=gen(9), device="cuda")

    def grads(h, w):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(distill.linear_cross_entropy(h, w, target, reduction="none"), (h, w), up)

    odd = grads(h, w)
    wide_rows = grads(*(torch.nn.functional.pad(x, (0, pad)) for x in (h, w)))
    for a, b in zip(odd, wide_rows):
        assert torch.equal(a, b[:, :width])
        assert not b[:, width:].any()


@gpu
@pytest.mark.parametrize("n,c", [(4, 10), (6000, 10), (6000, 50), (200_000, 40), (400, 600), (1300, 4000), (400, 20_000), (20, 50_000),
                                 (400, 3000)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rows_that_do_not_count_may_hold_anything(n, c, dtype):
    """Scores alone, with and without gradients: NaN and infinities of such rows reach no other row's, and nothing kept of the memory."""
    from cuml_b200 import distill

    z, t = torch.randn((n, c), generator=gen(c), device="cuda").to(TYPES[dtype]), torch.randint(0, c, (n,), generator=gen(n), device="cuda")
    t[1::3] = -100
    counts = t >= 0
    plain, odd = z.clone(), z.clone()
    plain[~counts] = 0.5
    odd[1::3, ::2] = float("nan")
    odd[1::3, 1::2] = float("inf")
    odd[4::6] = float("-inf")
    up = torch.randn((2, n), generator=gen(3), device="cuda")
    out = []
    for x in (plain, odd):
        torch.empty((1 << 26,), device="cuda").fill_(float("nan"))  # (what a workspace is made from)
        x.requires_grad_()
        got = distill.log_probs(x, t)
        out.append((got.log_prob, got.entropy, *torch.autograd.grad((got.log_prob, got.entropy), x, (up[0], up[1]))))
    for a, b in zip(*out):
        assert torch.equal(a, b) and (b[~counts] == 0).all()


@gpu
@pytest.mark.parametrize("n,c", [(9000, 13), (9000, 16), (7200, 3), (24_000, 40), (24_000, 14), (90_000, 47), (90_000, 49), (90_000, 60),
                                 (60_000, 33)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_rows_of_few_classes_by_threads_in_one_pass_and_by_lanes_in_the_other(n, c, dtype):
    z, t = logits(n, c, dtype), targets(n, c)
    t[::11] = -100
    z[5] = float("-inf")
    g, h = upstreams(n)
    check(z, t, 1.5, 0, g, h)
    check(torch.nn.functional.pad(z, (1, 2))[:, 1:c + 1], t, 1.5, 0, g, h)


def scores_of_layer(h, w, target, temperature=1.0):
    """In 64 bits on the GPU: log q of the targets, entropies, and per row the sum of |h| |w| of its largest class."""
    z = h.double() @ w.double().t() / temperature
    log_q = torch.log_softmax(z, 1)
    size = (h.double().abs() @ w.double().abs().t()).amax(1) / temperature
    return log_q.gather(1, target[:, None])[:, 0].cpu(), -(log_q.exp() * log_q).sum(1).cpu(), size.cpu()


@gpu
@pytest.mark.parametrize("width", [704, 768, 776, 1024, 1536, 1544, 2048, 2312, 3200])
@pytest.mark.parametrize("n,c", [(1300, 5000), (5000, 1300), (130, 60_000)])
def test_layers_whose_tiles_are_several_sums(width, n, c):
    """A tile's sum of 768 terms is handed on while its next begins, and a pair of blocks takes several tiles: one sum, two, three and more per
    tile, with depths at and behind the ends of the sums, where tiles are more than the pairs of blocks.  Logits are off as in
    test_score.py."""
    from cuml_b200 import distill

    for dtype in ("bf16", "fp16"):
        h, w = layer(n, width, c, dtype, 1)
        t = targets(n, c)
        got = distill.linear_log_probs(h, w, t)
        log_prob, entropy, size = scores_of_layer(h, w, t)
        e_z = 2 * adds(width) * size
        check_values(got.log_prob, log_prob, 4 * U, S + e_z, U)
        check_values(got.entropy, entropy, 4 * U, entropy_error(c) + e_z * (1 + 2 * entropy), U)
        again = distill.linear_log_probs(h, w, t)
        assert torch.equal(got.log_prob, again.log_prob) and torch.equal(got.entropy, again.entropy)
    distill.check_status()


@gpu
@pytest.mark.parametrize("dtype,border", [("bf16", 1.7e-6), ("fp16", 8.5e-6)])
def test_sums_of_a_layer_are_not_cut_short_over_their_whole_length(dtype, border):
    """Of products that are all positive, the tensor cores' sum is cut short with each addition of 16 of them, on average by 0.36 2^-23 (half a
    step; a step is 0.72 2^-23 of a number on average).  In parts of 48 additions that makes (24.5 x 48 + 24.5 x 48 + 16.5 x 32) / 128 = 22.5
    of these, 1.0e-6 of a sum of 2048 terms; in one sum it would be 64.5, 2.8e-6.  The border is between the two.  Products of fp16 have 22
    bits, and what of these lies below the sum's last place is cut, too: with two places more that are kept on the way, sixteen times a
    quarter of a step for each addition, so five times as much with the sum's own (4.8e-6 and 1.4e-5; those of bf16 have 16 bits, which lie above
    that).  One class has the sum z and the others 0, so log q of one of these is -z less next to nothing."""
    from cuml_b200 import distill

    n, width, c = 4096, 2048, 300
    h = (torch.rand((n, width), generator=gen(1), device="cuda") + 0.5).to(TYPES[dtype])
    w = torch.zeros((c, width), dtype=TYPES[dtype], device="cuda")
    w[7] = ((torch.rand(width, generator=gen(2), device="cuda") + 0.5) / 64).to(TYPES[dtype])
    t = torch.full((n,), 250, device="cuda")
    got = distill.linear_log_probs(h, w, t).log_prob
    want = scores_of_layer(h, w, t)[0]
    off = wide(got) - want
    assert float(off.norm() / want.norm()) < border


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_views_of_the_negatives_of_what_lies_in_memory(monkeypatch, compiled):
    """Gradients that come from a part of a conjugate, and inputs that are such views, have the other sign than their memory."""
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    n, c = 40, 300
    z, t = logits(n, c, "fp32"), targets(n, c)
    h, w = layer(n, 64, c, "bf16")
    a, b = upstreams(n)
    teacher = distill.log_probs(logits(n, c, "fp32", 3), top=5).top
    both = [(distill.log_probs, (z,), (t,)), (distill.linear_log_probs, (h, w), (t,))]
    one = [(distill.cross_entropy, (z,), (t,)), (distill.distillation_loss, (z,), (teacher,)), (distill.linear_cross_entropy, (h, w), (t,)),
           (distill.linear_distillation_loss, (h, w), (teacher,))]
    for f, leaves, rest in both + one:
        leaves = [x.detach().requires_grad_() for x in leaves]

        def run(*args):
            out = f(*args) if f in (distill.log_probs, distill.linear_log_probs) else (f(*args, reduction="none"),)
            return out[0], out[1] if len(out) > 1 else out[0] * 0

        x, y = run(*leaves, *rest)
        want = torch.autograd.grad((x, y), leaves, (a, b))
        x, y = run(*leaves, *rest)
        seen = []
        x.register_hook(lambda g: seen.append(g.is_neg()))
        y.register_hook(lambda g: seen.append(g.is_neg()))
        got = torch.autograd.grad(torch.complex(x, y).conj().mul(torch.complex(a, b)).real.sum(), leaves)
        assert any(seen) and all(torch.equal(p, q) for p, q in zip(want, got))
        negative = [torch._neg_view(-p.detach()).requires_grad_() for p in leaves]
        flipped = [torch._neg_view(-p) if isinstance(p, torch.Tensor) else
                   type(p)(*(q if q is None else torch._neg_view(-q) for q in p)) for p in rest]
        x2, y2 = run(*negative, *flipped)
        assert torch.equal(x, x2) and torch.equal(y, y2)
        for p, q in zip(want, torch.autograd.grad((x2, y2), negative, (torch._neg_view(-a), torch._neg_view(-b)))):
            assert torch.equal(p, q)
    assert torch.equal(distill.top_scores(z, 3).values, distill.top_scores(torch._neg_view(-z), 3).values)
    tail = distill.top_scores(z, 3)
    odd = distill.TopScores(tail.values, tail.index, torch._neg_view(-tail.logsumexp))
    other = logits(n, c, "fp32", 4)
    assert torch.equal(*(distill.distillation_loss(other, x, tail="bucket") for x in (tail, odd)))
    # gradients
    x = torch._neg_view(-z)
    norm = distill.gradient_norm([z])
    assert torch.equal(distill.gradient_norm([x]), norm)
    plain, out = z.clone(), torch.empty_like(z)
    distill.clip_gradients([plain], 1.0)
    distill.clip_gradients([x], 1.0, out=[out])
    assert torch.equal(out, plain)
    distill.clip_gradients([x], 1.0)
    assert x.is_neg() and torch.equal(x, plain)
    with pytest.raises(ValueError, match="negative view"):
        distill.clip_gradients([z], 1.0, out=[torch._neg_view(torch.empty_like(z))])


@gpu
@pytest.mark.parametrize("n,c,dtype", [(2500, 16_500, "bf16"), (3000, 20_001, "bf16"), (2500, 8200, "fp32"), (5000, 16_500, "fp32"),
                                       (10_000, 33_001, "fp16")])
@pytest.mark.parametrize("k", [1, 8, 24])
def test_best_of_many_long_rows(n, c, dtype, k):
    """As many rows as let a warp take long ones: the same rows few at a time, which are shared by blocks, and some against 64 bits.  The
    largest logit is many times there, at the row's ends among them."""
    from cuml_b200 import distill

    z, t = logits(n, c, dtype), targets(n, c)
    z[::7, ::97] = 11.0
    z[3::7, -2:] = z[3::7, :1] = 12.5
    z[5::50, 40:] = float("-inf")
    t[::9] = -100
    got = distill.log_probs(z, t, top=k)
    for first in (0, n // 3, n - 250):
        rows = slice(first, first + 250)
        few = distill.log_probs(z[rows].clone(), t[rows].clone(), top=k)
        assert torch.equal(got.top.index[rows], few.top.index)
        check_values(got.log_prob[rows], wide(few.log_prob), 8 * U, 2 * S, 2 * U)
        check_values(got.entropy[rows], wide(few.entropy), 8 * U, 2 * entropy_error(c), 2 * U)
        check_values(got.top.values[rows], wide(few.top.values), 8 * U, 2 * S, 2 * U)
    some = torch.arange(0, n, n // 30, device="cuda")
    log_prob, entropy, log_q, _, counts = ref.scores(z[some], t[some])
    values, index = ref.top(z[some], k, counts, log_q)
    assert torch.equal(got.top.index[some].cpu(), index)
    check_values(got.top.values[some], values, 4 * U, S, U)
    check_values(got.log_prob[some], log_prob, 4 * U, S, U)
    check_values(got.entropy[some], entropy, 4 * U, entropy_error(c), U)
