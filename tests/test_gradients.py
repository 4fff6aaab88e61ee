"""The norm of many gradients and clipping: refusals (CPU), and the kernels against 64 bits (GPU).

Tolerances count roundings, u = 2^-24.  Sums of up to eight numbers are taken in fp32 (8 u, of a square one u more each), the rest in
64 bits; a root halves that, and the result is rounded: 9 u of the norm at most.  A factor is off by that and its own rounding,
a scaled gradient by 12 u and half a step of its type."""
import ctypes as C
import math

import pytest
import torch

from tests.test_distill import HALF_STEP, TYPES, U, check_values, gen

gpu = pytest.mark.gpu
MADE = ["fp32", "bf16", "fp16"]
KINDS = [2.0, 1.0, math.inf]


def norm_of(tensors, kind):
    parts = [x.detach().cpu().double().abs().reshape(-1) for x in tensors]
    flat = torch.cat(parts) if parts else torch.zeros(0, dtype=torch.float64)
    if kind == math.inf:
        return flat.max() if flat.numel() else torch.zeros((), dtype=torch.float64)
    return flat.sum() if kind == 1.0 else flat.square().sum().sqrt()


def made(shapes, dtypes, seed=0, scale=0.01):
    g = gen(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(TYPES[dtypes[i % len(dtypes)]])
            for i, s in enumerate(shapes)]


def check_clip(tensors, most, kind, out=None, given=None):
    """In place, or to `out`; `given`: what is passed in the tensors' place."""
    from cuml_b200 import distill

    before = [x.detach().cpu().double() for x in tensors]
    norm = norm_of(tensors, kind)
    alone = distill.gradient_norm(given if given is not None else tensors, norm_type=kind)
    assert all(torch.equal(x.detach().cpu().double(), y) for x, y in zip(tensors, before))
    got = distill.clip_gradients(given if given is not None else tensors, most, norm_type=kind, out=out)
    assert got.shape == () and got.dtype == torch.float32 and torch.equal(got, alone)
    check_values(got, norm, 9 * U, 0.0, U)
    factor = float(most / norm) if norm > most else 1.0
    for x, y in zip(before, tensors if out is None else [o for o in out if o is not None]):
        exact = factor == 1.0 and (out is None or y.dtype == torch.float32)
        tiny = 2.0 ** -25 if y.dtype == torch.float16 else 2.0 ** -134 if y.dtype == torch.bfloat16 else 2.0 ** -150
        tiny = torch.tensor(tiny, dtype=torch.float64)  # (as a 32-bit number it would be 0)
        check_values(y, x * factor, 0.0 if exact else 12 * U, 0.0 if exact else tiny, 0.0 if exact else HALF_STEP[y.dtype])


# ---- refusals ------------------------------------------------------------------------------------------------
def test_python_refusals_without_a_gpu():
    from cuml_b200 import distill

    x = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        distill.gradient_norm([x])
    with pytest.raises(TypeError, match="list"):
        distill.clip_gradients(x, 1.0)
    with pytest.raises(TypeError, match="list"):
        distill.clip_gradients([x], 1.0, out=x)
    with pytest.raises(TypeError, match="torch tensor"):
        distill.clip_gradients([1.0], 1.0)
    for most in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            distill.clip_gradients([x], most)
    for kind in (3.0, 0.0, "two", None):
        with pytest.raises(ValueError, match="norm_type"):
            distill.gradient_norm([x], norm_type=kind)
    with pytest.raises(ValueError, match="out has 2"):
        distill.clip_gradients([x], 1.0, out=[x, x])


def test_c_refusals_without_a_gpu(lib):
    from cuml_b200.distill import CGradient

    def entry(at=4096, to=None, rows=1, cols=8, from_row=8, from_col=1, to_row=8, to_col=1, kind=0, to_kind=0, tensor=0):
        return CGradient(at, at if to is None else to, rows, cols, from_row, from_col, to_row, to_col, kind, to_kind, tensor)

    def clip(*entries, n=None, kind=2, scales=1, most=1.0, norm=64):
        array = (CGradient * max(1, len(entries)))(*entries)
        return lib.b2fil_clip_gradients(array, len(entries) if n is None else n, kind, scales, most, norm, None, 0, 0, None)

    def text():
        return lib.b2fil_last_error().decode()

    for bad in (entry(at=0), entry(at=4098), entry(kind=1), entry(kind=9), entry(to_kind=1), entry(to=8192 + 2),
                entry(rows=-1), entry(cols=1 << 41), entry(rows=1 << 30, cols=1 << 30), entry(from_col=-1), entry(to_col=2),
                entry(to_kind=2)):
        assert clip(bad) == -1 and text()
    for bad in (dict(n=-1), dict(kind=3), dict(kind=-1), dict(most=-1.0), dict(most=float("nan")), dict(norm=None), dict(norm=66)):
        assert clip(entry(), **bad) == -1, bad
    # what overlaps
    strided = dict(rows=4, cols=4, from_row=8, to_row=8)
    for bad in ([entry(), entry(tensor=1)], [entry(), entry(at=4096 + 28, tensor=1)],
                [entry(to=8192), entry(at=8192 + 16, to=16384, tensor=1)],  # writes what another reads
                [entry(to=4096 + 16)], [entry(rows=4, cols=4, from_row=2, to_row=2)], [entry(cols=4, from_col=0, to_col=0)],
                [entry(**strided), entry(at=4096 + 12, tensor=1, **strided)],
                [entry(**strided), entry(at=4096 + 32 * 2 + 20, tensor=1, **strided)]):
        assert clip(*bad) == -1 and "overlap" in text(), bad
    # what does not (a device is asked for next)
    for good in ([entry(), entry(at=4096 + 32, tensor=1)], [entry(**strided), entry(at=4096 + 16, tensor=1, **strided)],
                 [entry(to=8192), entry(to=16384, tensor=1)], [entry(rows=0, at=0)], [entry(), entry()],
                 [entry(rows=4, cols=4, from_row=1, from_col=4, to_row=1, to_col=4)],
                 [entry(cols=4, from_col=2, to_col=2), entry(at=4100, cols=4, from_col=2, to_col=2, tensor=1)]):
        assert clip(*good) != 0 and "overlap" not in text(), good
    assert lib.b2fil_clip_gradients_workspace(None, 3, 0) == -1
    assert lib.b2fil_clip_gradients_workspace(None, -1, 0) == -1


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_python_refusals(monkeypatch, compiled):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    x = torch.ones(4, 8, device="cuda")
    for bad, text in (([x.double()], "must be one of"), ([x.int()], "must be one of"), ([x, x.cpu()], "CUDA"),
                      ([x.to_sparse()], "strided"), ([x, x], "overlap"), ([x, x[1:3]], "overlap"), ([x[:1].expand(4, 8)], "overlap"),
                      ([x.view(-1).as_strided((4, 4), (2, 1))], "overlap"), ([x.view(-1)[:20], x.view(-1)[19:]], "overlap")):
        with pytest.raises((ValueError, RuntimeError), match=text):
            distill.clip_gradients(bad, 1.0)
        assert (x == 1).all()
    for out, text in (([torch.zeros(8, 4, device="cuda")], "shape"), ([None], "torch tensor"), ([x.view(-1)[:1].expand(4, 8)], "overlap"),
                      ([torch.zeros(4, 8, device="cuda", requires_grad=True)], "requires grad"), ([x.double()], "must be one of")):
        with pytest.raises((ValueError, TypeError, RuntimeError), match=text):
            distill.clip_gradients([x], 1.0, out=out)
    y = torch.ones(64, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        distill.clip_gradients([y[:32]], 1.0, out=[y[16:48]])
    assert (y == 1).all()
    # a norm only reads: the same tensor twice counts twice, expanded ones count as they are seen
    assert abs(distill.gradient_norm([x, x]).item() - 8.0) < 1e-5
    assert abs(distill.gradient_norm([x[:1].expand(400, 8)], norm_type=1).item() - 3200.0) < 1e-2


# ---- norms and clipping ------------------------------------------------------------------------------------------
SHAPES = {
    "one": [(1,)],
    "scalar": [()],
    "few": [(7,), (128, 64), (128,), (10, 128), (10,)],
    "odd": [(333, 101), (101,), (1, 1), (3, 5, 7), (0,), (50_001,), (17, 0, 4)],
    "many": [(i % 37 + 1, i % 11 + 1) for i in range(1300)],
    "long": [(3_000_001,), (4097,)],
}


@gpu
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtypes", [["fp32"], ["bf16"], ["fp16"], MADE])
def test_clip(shapes, kind, dtypes):
    tensors = made(SHAPES[shapes], dtypes)
    norm = float(norm_of(tensors, kind))
    check_clip(tensors, norm * 2, kind)
    check_clip([x.clone() for x in tensors], norm / 3, kind)
    for to in MADE:
        check_clip(tensors, norm / 3, kind, out=[torch.full_like(x, 7.0, dtype=TYPES[to]) for x in tensors])
        check_clip(tensors, norm * 3, kind, out=[torch.full_like(x, 7.0, dtype=TYPES[to]) for x in tensors])


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_strides_and_places(monkeypatch, compiled):
    """Transposed, sliced, interleaved and misaligned tensors; what lies between them stays as it is."""
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    for dtype in MADE:
        def views():
            base = made([(64, 96), (24, 10, 14), (5001,)], [dtype], 3)
            a, b, c = base
            parts = [a[:, :31], a[:, 31:50], a[:32, 60:].t(), a[32:, 61::3], b[::2, 1:8, ::2], b[1::2, :, 3].t(), c[1:1001], c[1001:1012],
                     c[1013:5000:2]]
            return base, parts

        base, parts = views()
        kept = [x.clone() for x in base]
        touched = [torch.zeros_like(x) for x in base]
        for x, y in zip(base, touched):
            for p in parts:
                if p.untyped_storage().data_ptr() == x.untyped_storage().data_ptr():
                    y.as_strided(p.shape, p.stride(), p.storage_offset()).fill_(1)
        check_clip(parts, float(norm_of(parts, 2.0)) / 2, 2.0)
        for x, y, z in zip(base, kept, touched):
            assert torch.equal(x[z == 0], y[z == 0]) and not torch.equal(x[z == 1], y[z == 1])
        # to tensors of other layouts, and from and to different places within 16 bytes
        base, parts = views()
        out = [torch.empty(p.numel() + 1, device="cuda")[1:].view(p.shape) if p.ndim < 2 else
               torch.empty(p.shape[::-1], device="cuda").permute(*reversed(range(p.ndim))) for p in parts]
        check_clip(parts, float(norm_of(parts, 2.0)) / 2, 2.0, out=out)
        flat = torch.empty(sum(p.numel() for p in parts) + 3, dtype=torch.bfloat16, device="cuda")[3:]
        out = [f.view(p.shape) for f, p in zip(flat.split([p.numel() for p in parts]), parts)]
        check_clip(parts, float(norm_of(parts, 1.0)) / 2, 1.0, out=out)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_parameters_none_and_nothing(monkeypatch, compiled):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    net = torch.nn.Sequential(torch.nn.Linear(13, 31), torch.nn.ReLU(), torch.nn.Linear(31, 7)).cuda()
    net(torch.randn(50, 13, device="cuda")).square().mean().backward()
    net[0].bias.grad = None
    weights = [p.detach().clone() for p in net.parameters()]
    grads = [p.grad for p in net.parameters() if p.grad is not None]
    check_clip(grads, float(norm_of(grads, 2.0)) / 2, 2.0, given=list(net.parameters()))
    assert all(torch.equal(a, b) for a, b in zip(weights, net.parameters()))
    assert distill.clip_gradients(net.parameters(), 1e-9).item() > 0  # (a generator)
    out = [None if p.grad is None else torch.empty_like(p.grad) for p in net.parameters()]
    check_clip(grads, 1e-12, 2.0, given=list(net.parameters()), out=out)
    for nothing in ([], [None], (), [net[0].bias], [torch.zeros(0, device="cuda")]):
        assert distill.clip_gradients(nothing, 1.0).item() == 0.0
        assert distill.gradient_norm(nothing, norm_type=math.inf).item() == 0.0
    zeros = [torch.zeros(100, device="cuda")]
    check_clip(zeros, 0.0, 2.0)
    ones = [torch.ones(100, device="cuda")]
    check_clip(ones, 0.0, 2.0)
    assert (ones[0] == 0).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_not_finite_and_out_of_the_usual_range(kind):
    from cuml_b200 import distill

    for odd in (float("nan"), float("inf"), float("-inf")):
        for dtype in MADE:
            for n in (100, 100_000):
                x, y = made([(n,), (33,)], [dtype])
                x[n // 2] = odd
                kept = x.clone()
                norm = distill.clip_gradients([x, y], 1e-3, norm_type=kind)
                assert norm.isnan() if odd != odd else norm == float("inf")
                assert torch.equal(x.isnan(), kept.isnan()) and torch.equal(x.nan_to_num(1.0), kept.nan_to_num(1.0))
                out = [torch.zeros_like(x), torch.zeros_like(y)]
                distill.clip_gradients([x, y], 1e-3, norm_type=kind, out=out)
                assert torch.equal(out[0].nan_to_num(1.0), kept.nan_to_num(1.0)) and torch.equal(out[1], y)
    # squares that 32 bits do not hold
    for scale in (1e-38, 1e-30, 1e-22, 1e18, 1e30, 1e36):
        for dtype in ("fp32", "bf16"):
            tensors = made([(300, 7), (5,), (20_001,)], [dtype], 1, scale)
            tensors[0][100:200] = 0
            norm = float(norm_of(tensors, kind))
            if norm < 3e38:
                check_clip(tensors, norm / 2, kind)
    # a norm that 32 bits do not hold is infinite to its caller, and changes nothing
    large = [torch.full((1000,), 3e38, device="cuda") for _ in range(2)]
    norm = distill.clip_gradients(large, 1.0, norm_type=kind)
    if kind != math.inf:
        assert norm == float("inf") and all((x == 3e38).all() for x in large)
    mixed = made([(5000,), (5000,)], ["fp32"], 2, 1.0)
    mixed[0].mul_(1e-25)
    mixed[1][::2] = 1e20
    check_clip(mixed, 1.0, kind)


@gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_autograd_sees_what_is_written(monkeypatch, compiled):
    from cuml_b200 import distill

    if not compiled:
        monkeypatch.setattr(distill, "_call", False)
    x = torch.ones(5, device="cuda")
    y = torch.ones(5, device="cuda", requires_grad=True)
    product = (x * y).sum()
    distill.gradient_norm([x])
    product.backward(retain_graph=True)
    distill.clip_gradients([x], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    product = (x * y).sum()
    distill.clip_gradients([y.grad], 1.0, out=[x])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():
        z = torch.ones(4, device="cuda")
        assert distill.clip_gradients([z], 1.0).item() == 2.0 and torch.equal(z, torch.full_like(z, 0.5))


@gpu
def test_the_same_every_time_and_on_other_streams():
    from cuml_b200 import distill

    tensors = made([(1001, 333), (7,), (77_777,)] * 9, MADE, 1)
    most = float(norm_of(tensors, 2.0)) / 2
    norm, results = None, None
    side = torch.cuda.Stream()
    for i in range(6):
        own = [x.clone() for x in tensors]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got = distill.clip_gradients(own, most)
        torch.cuda.current_stream().wait_stream(side)
        if norm is None:
            norm, results = got, own
        assert torch.equal(got, norm) and all(torch.equal(a, b) for a, b in zip(own, results))
    torch.cuda.synchronize()


@gpu
def test_captured_and_replayed():
    """Captured calls keep addresses, not numbers: replayed on other gradients they clip those."""
    from cuml_b200 import distill

    for shapes in (SHAPES["few"], SHAPES["many"], [(700, 1000)] * 3):
        held = made(shapes, ["fp32", "bf16"], 1)
        fresh = [made(shapes, ["fp32", "bf16"], s) for s in (2, 3)]
        distill.clip_gradients([x.clone() for x in held], 0.001)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = distill.clip_gradients(held, 0.001)
        for values in fresh:
            for x, y in zip(held, values):
                x.copy_(y)
            graph.replay()
            want = distill.clip_gradients(values, 0.001)
            assert torch.equal(norm, want) and all(torch.equal(x, y) for x, y in zip(held, values))
        del graph


@gpu
def test_more_strided_tensors_than_a_launch_takes():
    """600 columns of a matrix, between flat tensors, and a view of five dimensions none of which are neighbours."""
    base = made([(700, 601), (40_000,), (6, 5, 8, 9, 4)], MADE, 8)
    odd = base[2][::2, ::3, 1::3, 2::4, :3]
    parts = [base[0][:, i] for i in range(600)] + [base[1], odd]
    kept = base[0][:, 600].clone()
    check_clip(parts, float(norm_of(parts, 2.0)) / 2, 2.0)
    assert torch.equal(base[0][:, 600], kept)


@gpu
def test_without_the_compiled_call_path(monkeypatch):
    """The same numbers through ctypes."""
    from cuml_b200 import distill

    def everything():
        out = []
        for name, shapes in SHAPES.items():
            for kind in KINDS:
                x = made(shapes, MADE)
                to = [torch.zeros_like(t, dtype=torch.bfloat16) for t in x]
                out += [distill.gradient_norm(x, norm_type=kind), distill.clip_gradients(x, 0.01, norm_type=kind, out=to), *to]
                out += [distill.clip_gradients(x, 0.01, norm_type=kind), *x]
        return out

    assert distill._native()
    compiled = everything()
    monkeypatch.setattr(distill, "_call", False)
    for x, y in zip(compiled, everything()):
        assert x.dtype == y.dtype and torch.equal(x, y)


@gpu
def test_more_than_two_to_the_31_elements():
    from cuml_b200 import distill

    n = (1 << 31) + 12_345
    x = torch.full((n,), 2.0 ** -10, dtype=torch.bfloat16, device="cuda")
    x[-1] = 3.0
    norm = distill.clip_gradients([x], 1.0)
    want = math.sqrt((n - 1) * 2.0 ** -20 + 9)
    check_values(norm, want, 9 * U, 0.0, U)
    half = HALF_STEP[torch.bfloat16]
    check_values(x[-1], 3.0 / want, 12 * U, 0.0, half)
    check_values(x[:5], torch.full((5,), 2.0 ** -10 / want), 12 * U, 0.0, half)
    check_values(x[-6:-1], torch.full((5,), 2.0 ** -10 / want), 12 * U, 0.0, half)
    assert (x[:-1] == x[0]).all()


# ---- together ------------------------------------------------------------------------------------------------------
class _Policy(torch.nn.Module):
    def __init__(self, classes):
        super().__init__()
        self.body = torch.nn.Linear(32, 64)
        self.head = torch.nn.Parameter(torch.randn(classes, 64) * 0.1)

    def forward(self, x):
        return torch.relu(self.body(x))


@gpu
@pytest.mark.parametrize("from_layer", [True, False])
def test_a_step_of_a_policy(from_layer):
    """Scores, their gradients and clipping one after the other, against the same step in 64 bits from elementary operations on the
    rounded weights.  The gradients' tolerance: the layer's products and differences are rounded to bf16 three times (2^-8 each), of
    sums of 500 rows: 2^-6 of the gradients' norm."""
    from cuml_b200 import distill

    torch.manual_seed(3)
    classes, n = 300, 500
    net = _Policy(classes).cuda()
    x = torch.randn((n, 32), generator=gen(1), device="cuda")
    actions, advantage = targets(n, classes), torch.randn((n,), generator=gen(2), device="cuda")
    actions[::7] = -100
    hidden = net(x).bfloat16()
    if from_layer:
        scored = distill.linear_log_probs(hidden, net.head.bfloat16(), actions)
    else:
        scored = distill.log_probs(hidden @ net.head.bfloat16().t(), actions)
    loss = -(advantage * scored.log_prob).mean() - 0.05 * scored.entropy.mean()
    loss.backward()
    wide = [p.detach().double().requires_grad_() for p in net.parameters()]
    order = dict(zip((name for name, _ in net.named_parameters()), wide))
    h = torch.relu(x.double() @ order["body.weight"].t() + order["body.bias"])
    log_q = torch.log_softmax(h @ order["head"].t(), 1)
    counts = actions >= 0
    named = log_q.gather(1, actions.clamp(min=0)[:, None])[:, 0] * counts
    entropy = -(log_q.exp() * log_q).sum(1) * counts
    (-(advantage * named).mean() - 0.05 * entropy.mean()).backward()
    total = norm_of([p.grad for p in wide], 2.0)
    norm = distill.clip_gradients(net.parameters(), float(total) / 4)
    off = math.sqrt(sum(float((a.grad.double() * 4 - b.grad).square().sum()) for a, b in zip(net.parameters(), wide)))
    assert abs(norm.item() - float(total)) < 2.0 ** -6 * float(total)
    assert off < 2 * 2.0 ** -6 * float(total)
    distill.check_status()


def targets(n, c):
    return torch.randint(0, c, (n,), generator=gen(c), device="cuda")
