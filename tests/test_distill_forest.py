"""Forests as teachers: their best classes, and the losses of a student on them; the operators together, captured into
graphs, on other streams."""
import numpy as np
import pytest
import torch

from tests import distill_reference as ref
from tests.helpers import random_forest_desc, random_rows
from tests.test_distill import HALF_STEP, S, U, check_values, gen, gpu
from tests.test_distill_linear import check as check_layer

N_CLASSES = 11


def forest(precision="single", n_outputs=N_CLASSES, **kw):
    from cuml_b200.fil import ForestInference

    desc = random_forest_desc(3, n_trees=4 * n_outputs, n_features=6, max_depth=5, n_outputs=n_outputs, postproc="softmax")
    return ForestInference.load_from_treelite_model(desc, precision=precision, is_classifier=True, **kw)


@gpu
@pytest.mark.parametrize("precision", ["single", "double"])
@pytest.mark.parametrize("n,k", [(1, 1), (257, 3), (1000, N_CLASSES)])
def test_predict_top(precision, n, k):
    fi = forest(precision)
    X = random_rows(1, n, 6, np.float32 if precision == "single" else np.float64)
    proba = fi.predict_proba(X)
    values, index, _ = ref.top(torch.as_tensor(proba), k)
    got = fi.predict_top(X, k)
    assert all(isinstance(g, np.ndarray) for g in got) and got[0].dtype == proba.dtype and got[1].dtype == np.int32
    assert np.array_equal(got[1], index.numpy()) and np.array_equal(got[0], values.numpy().astype(proba.dtype))
    for x in (torch.as_tensor(X), torch.as_tensor(X, device="cuda")):
        v, i = fi.predict_top(x, k)
        assert v.device == x.device and i.device == x.device
        assert torch.equal(i.cpu(), index) and np.array_equal(v.cpu().numpy(), got[0])
    fi.output_type = "numpy"
    assert isinstance(fi.predict_top(torch.as_tensor(X, device="cuda"), k)[0], np.ndarray)


@gpu
def test_predict_top_of_a_binary_forest_and_labels():
    from sklearn.datasets import make_classification
    from sklearn.ensemble import RandomForestClassifier as SkForest

    from cuml_b200.ensemble import RandomForestClassifier
    from cuml_b200.fil import ForestInference

    desc = random_forest_desc(5, n_trees=9, postproc="sigmoid")
    fi = ForestInference.load_from_treelite_model(desc, is_classifier=True)
    X = random_rows(2, 50, 6)
    v, i = fi.predict_top(X, 2)
    proba = fi.predict_proba(X)
    assert np.array_equal(v, -np.sort(-proba, axis=1)) and np.array_equal(i[:, 0], proba.argmax(1))

    x, y = make_classification(400, 8, n_informative=6, n_classes=4, random_state=0)
    model = SkForest(20, max_depth=5, random_state=0).fit(x, np.array(["a", "b", "c", "d"])[y])
    ours = RandomForestClassifier.from_sklearn(model)
    v, labels = ours.predict_top(x.astype(np.float32), 2)
    assert labels.shape == (400, 2) and np.array_equal(labels[:, 0], ours.predict(x.astype(np.float32)))
    assert (v[:, 0] >= v[:, 1]).all()


@gpu
def test_refusals():
    from cuml_b200.fil import ForestInference

    fi = forest()
    X = torch.as_tensor(random_rows(1, 5, 6), device="cuda")
    z = torch.zeros(5, N_CLASSES, device="cuda")
    h, w = torch.zeros(5, 16, device="cuda").bfloat16(), torch.zeros(N_CLASSES, 16, device="cuda").bfloat16()
    for k in (0, N_CLASSES + 1):
        with pytest.raises(ValueError, match="k must be"):
            fi.predict_top(X, k)
    with pytest.raises(ValueError, match="shape"):
        fi.predict_top(X[:, :5], 2)
    for kw in (dict(), dict(logits=z, hidden=h, weight=w), dict(hidden=h), dict(weight=w)):
        with pytest.raises(ValueError, match="hidden and weight"):
            fi.distillation_loss(X, **kw)
    with pytest.raises(ValueError, match="bucket"):
        fi.distillation_loss(X, hidden=h, weight=w, tail="bucket")
    with pytest.raises(ValueError, match="classes"):
        fi.distillation_loss(X, z[:, 1:])
    with pytest.raises(ValueError, match="rows"):
        fi.distillation_loss(X, z[1:])
    regressor = ForestInference.load_from_treelite_model(random_forest_desc(0), is_classifier=False)
    with pytest.raises(RuntimeError, match="classifiers"):
        regressor.predict_top(X, 1)
    with pytest.raises(RuntimeError, match="classifiers"):
        regressor.teach(X, 1)


def dense_teacher(fi, X, k, temperature):
    """(values, index, logsumexp) of the forest's log-probabilities in 64 bits."""
    return ref.top(fi.predict_proba(X), k, temperature, probabilities=True)


@gpu
@pytest.mark.parametrize("precision", ["single", "double"])
def test_loss_of_a_student_of_a_forest(precision):
    """Teacher and student together: loss and gradients against 64 bits.  The forest's probabilities are common to
    both sides; their logarithms in fp32 are off by 2 U of their size, which is below 32."""
    fi = forest(precision)
    n, k, t = 300, 4, 2.0
    X = torch.as_tensor(random_rows(4, n, 6), device="cuda")
    v, i, lse = dense_teacher(fi, X, k, t)
    z = torch.randn((n, N_CLASSES), generator=gen(1), device="cuda").requires_grad_()
    extra = 64 * U * t * t
    for tail in ("renormalise", "bucket"):
        loss = fi.distillation_loss(X, z, k=k, temperature=t, tail=tail, reduction="none")
        rows, grad, _ = ref.loss(z, v, i, lse if tail == "bucket" else None, t)
        check_values(loss, rows, 4 * U, 3 * S * t * t + extra, U)
        (g,) = torch.autograd.grad(loss, z, torch.ones_like(loss))
        check_values(g, grad, 4 * S, 4 * S * t + extra, U)
    # as many entries as there are classes at most, labels beside the forest, and the linear layer
    labels = torch.randint(0, N_CLASSES, (n,), generator=gen(2), device="cuda")
    loss = fi.distillation_loss(X, z, k=100, temperature=t, labels=labels, label_weight=0.25)
    v, i, _ = dense_teacher(fi, X, N_CLASSES, t)
    soft, hard = ref.loss(z, v, i, None, t)[0], ref.loss(z, None, labels[:, None])[0]
    check_values(loss, 0.75 * soft.mean() + 0.25 * hard.mean(), 4 * U, 3 * S * t * t + extra, U)
    h = torch.randn((n, 32), generator=gen(3), device="cuda").bfloat16()
    w = torch.randn((N_CLASSES, 32), generator=gen(4), device="cuda").bfloat16()
    top = fi.teach(X, k, temperature=t)
    check_layer(h, w, top.values.float(), top.index, t, "mean",
                call=lambda a, b: fi.distillation_loss(X, hidden=a, weight=b, k=k, temperature=t))
    a, b = h.requires_grad_(), w.requires_grad_()
    both = fi.distillation_loss(X, hidden=a, weight=b, k=k, temperature=t, labels=labels, label_weight=0.5)
    assert all(torch.isfinite(x.float()).all() for x in torch.autograd.grad(both, (a, b)))


@gpu
@pytest.mark.parametrize("linear", [False, True])
def test_a_student_learns_a_forest(linear):
    """A training loop as a user writes it runs, and every parameter gets a gradient."""
    torch.manual_seed(0)
    fi = forest()
    X = torch.as_tensor(random_rows(7, 512, 6, nan_frac=0.0), device="cuda")
    body = torch.nn.Sequential(torch.nn.Linear(6, 64), torch.nn.GELU()).cuda()
    head = torch.nn.Linear(64, N_CLASSES, bias=False).cuda()
    parameters = [*body.parameters(), *head.parameters()]
    optimiser = torch.optim.AdamW(parameters, lr=1e-2)
    for _ in range(4):
        for part in X.split(200):
            optimiser.zero_grad()
            if linear:
                with torch.autocast("cuda", dtype=torch.bfloat16):
                    loss = fi.distillation_loss(part, hidden=body(part), weight=head.weight, k=4, temperature=2.0)
            else:
                loss = fi.distillation_loss(part, head(body(part)), k=4, temperature=2.0, tail="bucket")
            loss.backward()
            assert all(p.grad is not None and torch.isfinite(p.grad).all() and (p.grad != 0).any() for p in parameters)
            optimiser.step()


def step(kind, state):
    from cuml_b200 import distill

    if kind == "top":
        return tuple(distill.top_scores(state["z"], 20))
    top = distill.TopScores(state["v"], state["i"], state["lse"])
    if kind == "loss":
        loss = distill.distillation_loss(state["z"], top, tail="bucket", reduction="mean")
        return loss, *torch.autograd.grad(loss, state["z"])
    loss = distill.linear_distillation_loss(state["h"], state["w"], top, reduction=kind)
    up = None if kind == "mean" else state["up"]
    return loss, *torch.autograd.grad(loss, (state["h"], state["w"]), up)


def inputs(seed, n=300, c=1500, width=64):
    g = gen(seed)
    t = torch.randn((n, c), generator=g, device="cuda") * 2
    v, i = torch.topk(t, 6, dim=1)
    return {"z": torch.randn((n, c), generator=g, device="cuda").requires_grad_(), "v": v, "i": i.int(),
            "lse": torch.logsumexp(t, 1), "up": torch.rand((n,), generator=g, device="cuda"),
            "h": torch.randn((n, width), generator=g, device="cuda").bfloat16().requires_grad_(),
            "w": torch.randn((c, width), generator=g, device="cuda").bfloat16().requires_grad_()}


KINDS = ["top", "loss", "mean", "none"]


def plain(out):
    return [x.detach().clone() for x in out]


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_two_captured_graphs(kind):
    """Forward and backward captured twice and replayed in turns with new inputs give what eager calls give.  (No
    autograd graph of the same leaves that was made outside is alive: torch refuses to capture then, whatever
    the operator.)"""
    first, second = inputs(1), inputs(2)
    want = [plain(step(kind, inputs(seed))) for seed in (1, 2, 3, 4)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in (first, second):
            step(kind, s)
    torch.cuda.current_stream().wait_stream(side)
    for s in (first, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(kind, s)
        graphs.append(graph)
        outs.append(out)
    for round_of in ((0, 1), (2, 3)):
        for s, seed in zip((first, second), round_of):
            with torch.no_grad():
                for name, x in inputs(seed + 1).items():
                    s[name].copy_(x)
        graphs[0].replay()
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for out, which in zip(outs, round_of):
            assert all(torch.equal(x, y) for x, y in zip(plain(out), want[which])), (kind, which)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_at_once(kind):
    states = [inputs(seed) for seed in (1, 2)]
    want = [plain(step(kind, s)) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    outs = [[], []]
    for _ in range(10):
        for j, (stream, s) in enumerate(zip(streams, states)):
            with torch.cuda.stream(stream):
                outs[j].append(step(kind, s))
    torch.cuda.synchronize()
    for j in (0, 1):
        for out in outs[j]:
            assert all(torch.equal(x, y) for x, y in zip(plain(out), want[j]))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_threads_at_once(kind):
    import threading

    states = [inputs(seed) for seed in (1, 2, 3)]
    want = [plain(step(kind, s)) for s in states]
    got, errors = [None] * 3, []

    def work(j):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[j] = plain(step(kind, states[j]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(j,)) for j in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_the_same_call_twice_gives_the_same_bits(kind):
    a, b = plain(step(kind, inputs(5))), plain(step(kind, inputs(5)))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_rows_behind_the_last_are_left_alone():
    """Outputs that a C caller gives are written in their n rows only."""
    import ctypes as C

    from cuml_b200 import distill
    from cuml_b200.fil import _lib

    lib = _lib.load()
    s = inputs(1)
    n, c, k = 37, 1500, 6
    stream = torch.cuda.current_stream().cuda_stream
    values = torch.full((64, 20), 7.0, device="cuda")
    index = torch.full((64, 20), 7, device="cuda", dtype=torch.int32)
    lse = torch.full((64,), 7.0, device="cuda")
    ws = torch.empty(max(1, lib.b2fil_top_scores_workspace(0, n, c, 20, 0)), dtype=torch.uint8, device="cuda")
    z = s["z"].detach()
    assert lib.b2fil_top_scores(0, z.data_ptr(), n, c, c, 20, 0, 1.0, values.data_ptr(), index.data_ptr(), lse.data_ptr(),
                                ws.data_ptr(), ws.numel(), 0, stream) == 0
    assert (values[n:] == 7).all() and (index[n:] == 7).all() and (lse[n:] == 7).all() and (lse[:n] != 7).all()
    teacher = distill.CTeacher(s["v"].data_ptr(), s["i"].data_ptr(), None, k, k, -1, k, 0)
    rows = torch.full((64,), 7.0, device="cuda")
    stats, p = torch.full((64, 4), 7.0, device="cuda"), torch.full((64, k), 7.0, device="cuda")
    logit, at = p.clone(), torch.full((64, k), 7, device="cuda", dtype=torch.int32)
    h, w = s["h"].detach(), s["w"].detach()
    layer = (h.data_ptr(), 64, w.data_ptr(), 64, n, c, 64)
    ws = torch.empty(lib.b2fil_linear_loss_workspace(2, *layer, k, 0), dtype=torch.uint8, device="cuda")
    assert lib.b2fil_linear_loss(2, h.data_ptr(), 64, w.data_ptr(), 64, n, c, 64, C.byref(teacher), 1.0, 0, rows.data_ptr(),
                                 stats.data_ptr(), logit.data_ptr(), p.data_ptr(), at.data_ptr(), None, None,
                                 ws.data_ptr(), ws.numel(), 0, stream) == 0
    up = torch.ones(n, device="cuda")
    dh = torch.full((64, 64), 7.0, device="cuda").bfloat16()
    dw = torch.full((c + 27, 64), 7.0, device="cuda").bfloat16()
    ws = torch.empty(lib.b2fil_linear_loss_grad_workspace(2, *layer, k, 1, 1, 0), dtype=torch.uint8, device="cuda")
    assert lib.b2fil_linear_loss_grad(2, h.data_ptr(), 64, w.data_ptr(), 64, n, c, 64, k, 1.0, stats.data_ptr(),
                                      logit.data_ptr(), p.data_ptr(), at.data_ptr(), up.data_ptr(), 1, None,
                                      dh.data_ptr(), dw.data_ptr(), ws.data_ptr(), ws.numel(), 0, stream) == 0
    for x in (rows, stats, p, at, logit):
        assert (x[n:] == 7).all()
    assert (dh[n:] == 7).all() and (dw[c:] == 7).all() and (dh[:n] != 7).all()
    grad = torch.full((64, c + 100), 7.0, device="cuda")
    rows2, ws = rows.clone(), torch.empty(lib.b2fil_distill_loss_workspace(0, n, c, k, 0), dtype=torch.uint8, device="cuda")
    assert lib.b2fil_distill_loss(0, z.data_ptr(), n, c, c, C.byref(teacher), 1.0, 0, rows2.data_ptr(), stats.data_ptr(),
                                  p.data_ptr(), at.data_ptr(), None, None, ws.data_ptr(), ws.numel(), 0, stream) == 0
    assert lib.b2fil_distill_loss_grad(0, z.data_ptr(), n, c, c, k, 1.0, stats.data_ptr(), p.data_ptr(), at.data_ptr(),
                                       up.data_ptr(), 1, None, grad.data_ptr(), c + 100, 0, stream) == 0
    assert (grad[n:] == 7).all() and (grad[:, c:] == 7).all() and (rows2[n:] == 7).all() and (stats[n:] == 7).all()
    assert lib.b2fil_distill_loss(0, z.data_ptr(), n, c, c, C.byref(teacher), 1.0, 0, rows2.data_ptr(), stats.data_ptr(),
                                  p.data_ptr(), at.data_ptr(), None, None, ws.data_ptr(), ws.numel() - 1, 0, stream) == -1


def test_half_steps():
    """The tolerances' half steps are those of the types."""
    assert HALF_STEP[torch.bfloat16] == 2.0 ** -8 and HALF_STEP[torch.float16] == 2.0 ** -11
