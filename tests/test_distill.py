"""Distillation from a teacher's lists: engine.distill / distill_loss against the definition in float64.

Tolerances.  A logit is a sum of f products of fp32 values carried to at least 22 bits: with S = max sum |x y| / T it is
off by at most dz = (8 sqrt(f) 2^-24 + 2 * 2^-22) S, eight standard deviations of f roundings of half a step and both
operands' truncation.  A probability is then off by a factor 1 + 2 dz + 8 * 2^-24 (the logit's and the log-sum's error,
exponential and division), and a sum of m (or n) such terms by 8 sqrt(m) 2^-24 of the sum of their magnitudes on top.
The weights of the sums are held as two fp16 numbers: the smallest step of fp16 is 2^-24, so each is off by 2^-25 at
most where it is too small for its 22 bits.  With the largest weight grad_b T scaled to at least 2^14 that is 2^-39 of it
per row of dY; with a row's largest probability scaled to at least 2^7 it is 2^-32 of that probability per item of dX."""

import math

import numpy as np
import pytest
import torch

from movie_recommender_system_amd import _lib
from movie_recommender_system_amd import engine as E

LOW = torch.finfo(torch.float32).min
HALF = 2.0 ** -24


def statement(X, Y, ids, scores, T, tlse=None, grad=None):
    """(loss, dX, dY, gradient of the logits at weight one, rows that have entries) by the definition, float64 on the
    CPU, row by row."""
    X, Y = X.double().cpu(), Y.double().cpu()
    ids, scores = ids.cpu(), scores.double().cpu()
    n, m = X.shape[0], Y.shape[0]
    logq = torch.log_softmax(X @ Y.T / T, dim=1)
    G = torch.zeros(n, m, dtype=torch.float64)
    loss = torch.zeros(n, dtype=torch.float64)
    has = torch.zeros(n, dtype=torch.bool)
    for b in range(n):
        use = [(int(i), float(s)) for i, s in zip(ids[b], scores[b]) if 0 <= i < m and s > LOW]
        if not use:
            continue
        has[b] = True
        t = torch.tensor([s for _, s in use], dtype=torch.float64) / T
        lse = torch.logsumexp(t, 0) if tlse is None else tlse[b].double().cpu()
        p = torch.zeros(m, dtype=torch.float64)
        for (i, _), v in zip(use, torch.exp(t - lse)):
            p[i] += v
        items = sorted({i for i, _ in use})
        on = torch.zeros(m, dtype=torch.bool)
        on[items] = True
        q = logq[b].exp()
        pos = on & (p > 0)
        kl = (p[pos] * (p[pos].log() - logq[b][pos])).sum()
        a = 1.0
        if tlse is not None:
            pr = max(0.0, 1.0 - float(p.sum()))
            qr = max(2.0 ** -24, float(q[~on].sum()))
            if pr > 0:
                kl += pr * math.log(pr / qr)
                a = 1.0 - pr / qr
        loss[b] = T * T * kl
        G[b] = T * torch.where(on, q - p, a * q)
    W = G if grad is None else G * grad.double().cpu()[:, None]
    return loss, W @ Y, W.T @ X, G, has


def tolerances(X, Y, T, G, has, tlse, loss, grad):
    X, Y = X.double().cpu(), Y.double().cpu()
    n, f = X.shape
    m = Y.shape[0]
    S = float((X.abs() @ Y.abs().T).max()) / T if n and m else 0.0
    dz = (8 * math.sqrt(f) * HALF + 2 * 2.0 ** -22) * S
    q = torch.softmax(X @ Y.T / T, dim=1)
    # What carries an error is the student's probability and the teacher's, not their difference: an item with q = p has
    # gradient zero and still the error of q (with one item both are 1, and the device's q is off by dz).
    mag = (G.abs() + 2 * T * q * has[:, None]) * (1.0 if grad is None else grad.double().cpu().abs()[:, None])
    rel = 2 * dz + 16 * HALF
    if tlse is not None:
        rel = rel * 4 + 1e-6   # p_r / q_r: both are differences from one
    w = torch.ones(n, dtype=torch.float64) if grad is None else grad.double().cpu().abs()
    tx = (rel + 8 * math.sqrt(m) * HALF) * (mag @ Y.abs())
    tx = tx + m * 2.0 ** -32 * (T * w * has * q.amax(1))[:, None] * Y.abs().amax()
    ty = (rel + 8 * math.sqrt(n) * HALF) * (mag.T @ X.abs()) + n * 2.0 ** -39 * T * w.max() * X.abs().amax()
    tl = T * T * (2 * dz + 64 * HALF) * (1 + loss.abs() / (T * T)) * (4 if tlse is not None else 1) + 4 * HALF * loss.abs()
    return tl, tx, ty


def compare(X, Y, ids, scores, T, tlse, grad, got):
    loss, dX, dY, G, has = statement(X, Y, ids, scores, T, tlse, grad)
    for name, a, b, t in zip(("loss", "dX", "dY"), got, (loss, dX, dY), tolerances(X, Y, T, G, has, tlse, loss, grad)):
        off = (a.double().cpu() - b).abs()
        assert torch.all(off <= t), f"{name}: {float((off / t).max())} times the tolerance"


def problem(seed, n, m, f, k, dev="cpu", spread=2.0, ragged=False, T=1.0, tail=False):
    g = torch.Generator().manual_seed(seed)
    a = math.sqrt(spread / math.sqrt(f))
    X = torch.randn(n, f, generator=g) * a
    Y = torch.randn(m, f, generator=g) * a
    t = (X + 0.5 * a * torch.randn(n, f, generator=g)) @ Y.T
    scores, ids = torch.topk(t, min(k, m), dim=1)
    tlse = torch.logsumexp(t / T, dim=1) if tail else None
    if k > m:
        ids = torch.cat([ids, torch.full((n, k - m), -1)], 1)
        scores = torch.cat([scores, torch.full((n, k - m), LOW)], 1)
    if ragged:
        length = torch.randint(0, k + 1, (n, 1), generator=g)
        length[::5] = 0
        ids = torch.where(torch.arange(k) < length, ids, -1)
        scores = torch.where(ids < 0, LOW, scores)
    grad = 0.5 + torch.rand(n, generator=g)
    to = lambda v: None if v is None else v.contiguous().to(dev)
    return to(X), to(Y), to(ids.to(torch.int32)), to(scores), to(tlse), to(grad)


# ------------------------------------------------------------------------------------------------ refusals (no GPU)

def c_call(entry, X=256, n=4, Y=256, m=8, f=32, ids=256, scores=256, k=3, T=1.0, loss=256, grad=256, ws=256, ws_bytes=1 << 40):
    """The C entries with made-up device addresses: every call here is refused before anything is launched."""
    lib = _lib.require()
    if entry == "loss":
        rc = lib.mirec_distill_loss(X, n, Y, m, f, ids, scores, k, T, None, 1, loss, ws, ws_bytes, None)
    else:
        rc = lib.mirec_distill_grad(X, n, Y, m, f, k, T, grad, None, None, ws, ws_bytes, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("entry", ["loss", "grad"])
@pytest.mark.parametrize("change,code,text", [
    ({"n": -1}, -1, "negative"), ({"m": -1}, -1, "negative"), ({"f": 16}, -4, "width"), ({"f": 100}, -4, "width"),
    ({"f": 224}, -4, "width"), ({"k": 0}, -1, "entry"), ({"k": 257}, -4, "256"), ({"T": 0.0}, -1, "temperature"),
    ({"T": -1.0}, -1, "temperature"), ({"T": float("nan")}, -1, "temperature"), ({"T": float("inf")}, -1, "temperature"),
    ({"m": 0}, -1, "empty"), ({"X": None}, -1, "null"), ({"Y": None}, -1, "null"), ({"X": 260}, -1, "aligned"),
    ({"Y": 264}, -1, "aligned"), ({"ws": None}, -2, "workspace"), ({"ws": 320}, -2, "workspace"), ({"ws_bytes": 100}, -2, "workspace"),
    ({"n": (1 << 26) + 1}, -4, "2^26"), ({"m": (1 << 26) + 1}, -4, "2^26"),
])
def test_the_c_entries_refuse(entry, change, code, text):
    rc, msg = c_call(entry, **change)
    assert rc == code and text in msg, (rc, msg)


@pytest.mark.parametrize("entry,change", [("loss", {"ids": None}), ("loss", {"scores": None}), ("loss", {"loss": None}),
                                          ("grad", {"grad": None})])
def test_the_c_entries_refuse_null(entry, change):
    rc, msg = c_call(entry, **change)
    assert rc == -1 and "null" in msg


def test_nothing_to_do_is_no_error():
    assert c_call("loss", n=0)[0] == 0 and c_call("grad", n=0)[0] == 0


def test_the_wrapper_refuses_host_tensors():
    X, Y, ids, scores, _, _ = problem(1, 4, 10, 32, 3)
    with pytest.raises(_lib.MirecError):
        E.distill(X, Y, ids, scores)


def test_the_statement_against_differences():
    """The oracle's gradients are those of its loss (float64, central differences along random directions)."""
    for tail in (False, True):
        X, Y, ids, scores, tlse, grad = problem(3, 5, 40, 32, 6, ragged=not tail, T=1.5, tail=tail)
        loss, dX, dY, _, _ = statement(X, Y, ids, scores, 1.5, tlse, grad)
        g = torch.Generator().manual_seed(9)
        DX, DY = torch.randn(X.shape, generator=g).double(), torch.randn(Y.shape, generator=g).double()
        h = 1e-5
        f = lambda s: float((grad.double() * statement(X.double() + s * DX, Y.double() + s * DY, ids, scores, 1.5, tlse)[0]).sum())
        want = float((dX * DX).sum() + (dY * DY).sum())
        assert abs((f(h) - f(-h)) / (2 * h) - want) <= 1e-6 * (1 + abs(want))


# ------------------------------------------------------------------------------------------------------- on the GPU

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda", 0)


@gpu
@pytest.mark.parametrize("f", [32, 64, 96, 128, 160, 192])
@pytest.mark.parametrize("n,m,k", [(1, 1, 1), (1, 33, 5), (31, 32, 20), (33, 500, 100), (65, 1000, 20), (130, 129, 256), (257, 2111, 64)])
def test_sizes_and_widths(dev, n, m, f, k):
    X, Y, ids, scores, _, grad = problem(n + m + f, n, m, f, k, dev)
    got = E.distill(X, Y, ids, scores, grad=grad)
    compare(X, Y, ids, scores, 1.0, None, grad, got)


@gpu
@pytest.mark.parametrize("T", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_temperature_tail_and_ragged_lists(dev, T, tail, ragged):
    X, Y, ids, scores, tlse, grad = problem(17, 90, 700, 64, 40, dev, ragged=ragged, T=T, tail=tail)
    got = E.distill(X, Y, ids, scores, temperature=T, teacher_lse=tlse, grad=grad)
    compare(X, Y, ids, scores, T, tlse, grad, got)
    if ragged:
        assert torch.all(got[0][::5] == 0) and torch.all(got[1][::5] == 0)
    # without weights of the rows
    got = E.distill(X, Y, ids, scores, temperature=T, teacher_lse=tlse)
    compare(X, Y, ids, scores, T, tlse, None, got)


@gpu
@pytest.mark.parametrize("n,m", [(1, 5000), (2, 20000), (600, 40), (1500, 7), (3, 1)])
def test_few_rows_and_few_items(dev, n, m):
    X, Y, ids, scores, _, grad = problem(n * m, n, m, 96, 10, dev)
    got = E.distill(X, Y, ids, scores, grad=grad)
    compare(X, Y, ids, scores, 1.0, None, grad, got)


@gpu
def test_entries_that_are_no_items_are_left_out(dev):
    X, Y, ids, scores, _, _ = problem(5, 8, 50, 32, 6, dev)
    ids[0, 0] = 50                         # one behind the last
    ids[1, 1] = (1 << 31) - 1
    ids[2, :] = -1
    ids[3, 2] = -(1 << 31)
    scores[4, 3] = float("nan")
    scores[5, 0] = -math.inf
    scores[6, :] = LOW
    got = E.distill(X, Y, ids, scores)
    compare(X, Y, ids, scores, 1.0, None, None, got)
    assert got[0][2] == 0 and got[0][6] == 0 and torch.all(got[1][[2, 6]] == 0)


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_the_same_item_twice_adds_up(dev, tail):
    X, Y, ids, scores, tlse, grad = problem(6, 12, 300, 64, 20, dev, tail=tail)
    if tail:
        tlse = tlse + 1.0    # the doubled entries must not hold more than all the mass
    ids[:, 7] = ids[:, 3]
    ids[0, :] = 17
    ids[1, 10:] = ids[1, 0]
    got = E.distill(X, Y, ids, scores, teacher_lse=tlse, grad=grad)
    compare(X, Y, ids, scores, 1.0, tlse, grad, got)


@gpu
@pytest.mark.parametrize("k", [1, 64, 65, 192, 256])
@pytest.mark.parametrize("n", [40, 2100])
@pytest.mark.parametrize("twice", [False, True])
def test_lists_of_every_length(dev, k, n, twice):
    """The list kernel of few and of many rows; in every third row some items are listed again."""
    X, Y, ids, scores, _, grad = problem(71, n, 300, 32, k, dev, ragged=True)
    if twice:
        ids[::3, k // 2:] = torch.where(ids[::3, k // 2:] >= 0, ids[::3, :k - k // 2], -1)
    compare(X, Y, ids, scores, 1.0, None, grad, E.distill(X, Y, ids, scores, grad=grad))


@gpu
def test_a_list_of_the_whole_catalogue(dev):
    """With every item listed the class of the others is empty on both sides."""
    X, Y, ids, scores, tlse, grad = problem(8, 20, 100, 32, 100, dev)
    got = E.distill(X, Y, ids, scores, grad=grad)
    compare(X, Y, ids, scores, 1.0, None, grad, got)


@gpu
@pytest.mark.parametrize("spread", [0.01, 8.0, 60.0])
def test_flat_and_peaked_rows(dev, spread):
    X, Y, ids, scores, _, grad = problem(11, 64, 900, 64, 16, dev, spread=spread)
    got = E.distill(X, Y, ids, scores, grad=grad)
    compare(X, Y, ids, scores, 1.0, None, grad, got)


@gpu
def test_rows_and_items_of_very_different_size(dev):
    """Factor rows whose entries span twelve decades, zero rows among them."""
    X, Y, ids, scores, _, grad = problem(12, 70, 800, 64, 16, dev, spread=1.0)
    g = torch.Generator().manual_seed(2)
    X *= (10.0 ** (-6 * torch.rand(70, 1, generator=g))).to(dev)
    Y *= (10.0 ** (-6 * torch.rand(800, 1, generator=g))).to(dev)
    X[3] = 0
    Y[5] = 0
    Y[9] *= 0
    got = E.distill(X, Y, ids, scores, grad=grad)
    compare(X, Y, ids, scores, 1.0, None, grad, got)


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("m", [900, 928, 5])
@pytest.mark.parametrize("scale", [1e-15, 1e-20, 1e-25])
def test_factors_whose_products_vanish(dev, scale, m, tail):
    """Logits of 1e-30 and less, and of zero in fp32: a uniform softmax, and gradients of the factors' size."""
    X, Y, ids, scores, _, grad = problem(18, 70, m, 64, 16, dev)
    X, Y = X * scale, Y * scale
    tlse = torch.logsumexp(scores, 1) + 0.5 if tail else None
    got = E.distill(X, Y, ids, scores, teacher_lse=tlse, grad=grad)
    compare(X, Y, ids, scores, 1.0, tlse, grad, got)


@gpu
def test_weights_of_very_different_size(dev):
    X, Y, ids, scores, _, grad = problem(13, 100, 600, 32, 12, dev)
    grad = grad * torch.logspace(-12, 0, 100, device=dev)
    grad[7] = 0
    grad[8] = -1.0
    got = E.distill(X, Y, ids, scores, grad=grad)
    loss, dX, dY, _, _ = statement(X, Y, ids, scores, 1.0, None, grad)
    # dX row by row, whatever its weight; dY where the largest weights decide it
    rel = (got[1].double().cpu() - dX).norm(dim=1) / dX.norm(dim=1).clamp(min=1e-300)
    rel[7] = 0
    assert float(rel.max()) < 1e-5 and torch.all(got[1][7] == 0)
    assert float((got[2].double().cpu() - dY).norm() / dY.norm()) < 1e-5


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_gradients_against_differences(dev, tail):
    """Along the gradient's own direction: d = <g, D> h is large against the loss's rounding."""
    T = 1.5
    X, Y, ids, scores, tlse, grad = problem(14, 40, 300, 64, 20, dev, T=T, tail=tail)
    loss, dX, dY = E.distill(X, Y, ids, scores, temperature=T, teacher_lse=tlse, grad=grad)
    norm = float(torch.sqrt(dX.double().square().sum() + dY.double().square().sum()))
    h = 1e-2
    f = lambda s: float((grad.double() * E.distill(X + s * dX / norm, Y + s * dY / norm, ids, scores, temperature=T,
                                                   teacher_lse=tlse)[0].double()).sum())
    # second order is h^2 / 6 of the third derivative (the loss has scale T^2 n); rounding 40 rows x 1e-6 / h
    assert abs((f(h) - f(-h)) / (2 * h) - norm) <= 5e-3 * norm + 40 * 1e-6 / h


@gpu
def test_autograd(dev):
    X, Y, ids, scores, _, grad = problem(15, 50, 400, 32, 10, dev)
    want = E.distill(X, Y, ids, scores, temperature=2.0, grad=grad)
    X, Y = X.requires_grad_(), Y.requires_grad_()
    loss = E.distill_loss(X, Y, ids, scores, temperature=2.0)
    assert torch.equal(loss.detach(), want[0])
    (loss * grad).sum().backward()
    assert torch.equal(X.grad, want[1]) and torch.equal(Y.grad, want[2])
    # a broadcast incoming gradient, one side only, and no gradient at all
    (dy,) = torch.autograd.grad(E.distill_loss(X.detach(), Y, ids, scores).sum(), Y)
    ones = E.distill(X.detach(), Y.detach(), ids, scores)
    assert torch.equal(dy, ones[2])
    (dx,) = torch.autograd.grad(E.distill_loss(X, Y.detach(), ids, scores).sum(), X)
    assert torch.equal(dx, ones[1])
    with torch.no_grad():
        assert torch.equal(E.distill_loss(X, Y, ids, scores), ones[0])
    # factors changed between the passes are noticed
    loss = E.distill_loss(X, Y, ids, scores)
    with torch.no_grad():
        Y.mul_(2.0)
    with pytest.raises(RuntimeError):
        loss.sum().backward()


@gpu
def test_empty_steps_and_refusals(dev):
    X, Y, ids, scores, _, grad = problem(16, 6, 50, 32, 5, dev)
    loss, dX, dY = E.distill(X[:0], Y, ids[:0], scores[:0])
    assert loss.numel() == 0 and dX.shape == (0, 32) and torch.all(dY == 0) and dY.shape == Y.shape
    for bad in ((X.double(), Y, ids, scores), (X, Y[:, :16], ids, scores), (X, Y, ids.long(), scores), (X, Y, ids[:3], scores),
                (X, Y, ids, scores[:, :3]), (X[::2], Y, ids[:3], scores[:3]), (X, Y.cpu(), ids, scores), (X[0], Y, ids, scores)):
        with pytest.raises(ValueError):
            E.distill(*bad)
    with pytest.raises(ValueError):
        E.distill(X, Y, ids, scores, grad=grad[:3])
    with pytest.raises(ValueError):
        E.distill(X, Y, ids, scores, ws=torch.zeros(1, dtype=torch.uint8, device=dev).expand(1 << 20))
    with pytest.raises(ValueError):
        E.distill(X, Y, ids, scores, teacher_lse=grad.double())
    with pytest.raises(_lib.MirecError):
        E.distill(X, Y, ids, scores, temperature=0.0)
    with pytest.raises(_lib.MirecError):
        E.distill(torch.zeros(2, 48, device=dev), torch.zeros(5, 48, device=dev), ids[:2], scores[:2])


@gpu
def test_streams_and_a_workspace_reused(dev):
    """Steps on streams of their own at once, a workspace used again for smaller steps: the same bits."""
    a = problem(21, 150, 900, 64, 30, dev)
    b = problem(22, 40, 333, 64, 7, dev)
    step = lambda p, ws=None: E.distill(*p[:4], temperature=1.3, grad=p[5], ws=ws)
    want = [step(a), step(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    outs = []
    for st, p in zip(streams, (a, b)):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([step(p) for _ in range(3)])
    torch.cuda.synchronize()
    for w, os in zip(want, outs):
        for o in os:
            assert all(torch.equal(x, y) for x, y in zip(o, w))
    lib = _lib.require()
    ws = torch.full((int(lib.mirec_distill_workspace_bytes(150, 900, 64, 30)),), 255, dtype=torch.uint8, device=dev)
    for p, w in ((a, want[0]), (b, want[1]), (a, want[0])):
        assert all(torch.equal(x, y) for x, y in zip(step(p, ws), w))


@gpu
def test_captured_steps_replay(dev):
    """Two captured steps over the same input buffers, replayed between eager ones."""
    n, m, f, k = 200, 1500, 64, 20
    static = [v.clone() if v is not None else None for v in problem(31, n, m, f, k, dev, T=2.0, tail=True)]
    step = lambda p: E.distill(p[0], p[1], p[2], p[3], temperature=2.0, teacher_lse=p[4], grad=p[5])
    step(static)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(static))
        graphs.append(gr)
    for rep in range(3):
        p = problem(100 + rep, n, m, f, k, dev, T=2.0, tail=True)
        for s, v in zip(static, p):
            s.copy_(v)
        want = step(p)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(x, y) for x, y in zip(o, want))


@gpu
def test_captured_steps_share_a_workspace(dev):
    """Two captured steps of different sizes in one workspace, replayed in turn with an eager step between them."""
    big, small = problem(41, 300, 1100, 64, 30, dev), problem(42, 70, 260, 64, 9, dev)
    ws = torch.empty(int(_lib.require().mirec_distill_workspace_bytes(300, 1100, 64, 30)), dtype=torch.uint8, device=dev)
    step = lambda p: E.distill(*p[:4], temperature=0.7, grad=p[5], ws=ws)
    want = [[v.clone() for v in step(p)] for p in (big, small)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for p in (big, small):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(p))
            with pytest.raises(_lib.MirecError):   # autograd inside a capture is refused
                E.distill_loss(p[0].detach().requires_grad_(), p[1], p[2], p[3])
        graphs.append(gr)
    for _ in range(3):
        for gr, o, w, p in zip(graphs, outs, want, (big, small)):
            for v in o:
                v.fill_(float("nan"))
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(o, w))
            assert all(torch.equal(x, y) for x, y in zip(step(p), w))


@gpu
def test_gradients_without_a_loss_that_prepared_them(dev):
    """A workspace of arbitrary bytes, or one left by a loss without gradients: wrong numbers, but in their places."""
    X, Y, ids, scores, _, grad = problem(43, 90, 700, 96, 12, dev)
    ws = torch.randint(0, 256, (int(_lib.require().mirec_distill_workspace_bytes(90, 700, 96, 12)),), dtype=torch.uint8, device=dev)
    guard = torch.full((700 + 90 + 2, 96), 7.0, device=dev)
    dX, dY = guard[1:91], guard[91:791]
    lib = _lib.require()
    grad_call = lambda: lib.mirec_distill_grad(X.data_ptr(), 90, Y.data_ptr(), 700, 96, 12, 1.0, grad.data_ptr(), dX.data_ptr(),
                                               dY.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert grad_call() == 0
    E._distill_loss(X, Y, ids, scores, 1.0, None, False, ws)
    assert grad_call() == 0
    torch.cuda.synchronize()
    assert torch.all(guard[0] == 7.0) and torch.all(guard[791] == 7.0)
    loss, _ = E._distill_loss(X, Y, ids, scores, 1.0, None, True, ws)
    assert grad_call() == 0
    compare(X, Y, ids, scores, 1.0, None, grad, (loss, dX, dY))


@gpu
def test_rows_beyond_32_bit_offsets(dev):
    """17 million rows of 128 columns: element offsets pass 2^31.  Weights are zero but for rows at both ends and around
    the offset 2^31, so that the gradient of the items is those rows' alone."""
    n, m, f, k = 17_000_000, 40, 128, 3
    at = torch.cat([torch.arange(0, 5), torch.arange(2 ** 24 - 3, 2 ** 24 + 3), torch.arange(n - 5, n)])
    g = torch.Generator(device=dev).manual_seed(51)
    X = torch.empty(n, f, device=dev).normal_(0.0, 0.4, generator=g)
    Y = torch.empty(m, f, device=dev).normal_(0.0, 0.4, generator=g)
    ids = torch.randint(0, m, (n, k), generator=g, device=dev, dtype=torch.int32)
    scores = torch.empty(n, k, device=dev).normal_(0.0, 1.0, generator=g)
    grad = torch.zeros(n, device=dev)
    grad[at.to(dev)] = 1.0
    loss, dX, dY = E.distill(X, Y, ids, scores, grad=grad)
    sub = at.to(dev)
    want = statement(X[sub], Y, ids[sub], scores[sub], 1.0)
    tol = tolerances(X[sub], Y, 1.0, want[3], want[4], None, want[0], None)
    for a, b, t in zip((loss[sub], dX[sub], dY), want, tol):
        assert torch.all((a.double().cpu() - b).abs() <= t)
    assert int((dX.abs().amax(1) > 0).sum()) == len(at)


@gpu
def test_items_beyond_32_bit_offsets(dev):
    """17 million items of 128 columns, all zero but for 48 at both ends and around the offset 2^31: the softmax over all
    of them is that of the 48 and 17 million - 48 logits of zero.  The sum of a range's equal terms is a chain of at most
    ytiles / 64 + 16 additions in fp32, each off by half a step of the sum: what a probability is off by on top."""
    n, m, f, k = 8, 17_000_000, 128, 12
    at = torch.cat([torch.arange(0, 16), torch.arange(2 ** 24 - 8, 2 ** 24 + 8), torch.arange(m - 16, m)])
    g = torch.Generator().manual_seed(52)
    X, some = torch.randn(n, f, generator=g) * 0.8, torch.randn(48, f, generator=g) * 0.8
    pick = torch.stack([torch.randperm(48, generator=g)[:k] for _ in range(n)])
    scores = torch.randn(n, k, generator=g)
    Y = torch.zeros(m, f, device=dev)
    Y[at.to(dev)] = some.to(dev)
    loss, dX, dY = E.distill(X.to(dev), Y, at[pick].to(torch.int32).to(dev), scores.to(dev))
    x, y = X.double(), some.double()
    z = x @ y.T
    lse = torch.logaddexp(torch.logsumexp(z, 1), torch.full((n,), math.log(m - 48), dtype=torch.float64))
    logp = torch.log_softmax(scores.double(), 1)
    q = (z - lse[:, None]).exp()
    p = torch.zeros(n, 48, dtype=torch.float64).scatter_(1, pick, logp.exp())
    chain = ((m + 31) // 32 / 64 + 16) * 16 * HALF
    dz = (8 * math.sqrt(f) * HALF + 2 * 2.0 ** -22) * float((x.abs() @ y.abs().T).max())
    rel = chain + 2 * dz + 16 * HALF
    want = (logp.exp() * (logp - (z - lse[:, None]).gather(1, pick))).sum(1)
    assert torch.all((loss.double().cpu() - want).abs() <= rel + 64 * HALF * (1 + want.abs()))
    mag = (q - p).abs() + 2 * q
    small = 2.0 ** -32 * float(q.amax().clamp(min=1.0 / m)) * 48 * float(y.abs().amax())
    assert torch.all((dX.double().cpu() - (q - p) @ y).abs() <= (rel + 64 * HALF) * (mag @ y.abs()) + small)
    tiny = n * 2.0 ** -39 * float(x.abs().amax())
    assert torch.all((dY[at.to(dev)].double().cpu() - (q - p).T @ x).abs() <= (rel + 16 * HALF) * (mag.T @ x.abs()) + tiny)
    zero = torch.tensor([16, 2 ** 23, 2 ** 24 - 9, 2 ** 24 + 8, m - 17])
    qz = (-lse).exp()[:, None]
    assert torch.all((dY[zero.to(dev)].double().cpu() - (qz * x).sum(0)).abs() <= (rel + 16 * HALF) * (qz * x.abs()).sum(0) + tiny)


def compare_with_rest(X, Y, ids, scores, T, tlse, grad, got):
    """``compare`` for rows whose students leave little outside their lists.  A probability q (on the list or off it), and
    with it the share q_r, is off by a factor 1 + rel: twice dz, the exponential and division, and 8 sqrt(m) 2^-24 for the
    sums.  The teacher's p is fp32: its logarithm lp is rounded once (half a step, 2^-24 |lp|) and the exponential is within
    4 of those steps; p_r = 1 - sum p carries the sum of these, dp.  Off the list the weight of an item is q - p_r q / q_r:
    both terms' rel, and dp q / q_r.  The two fp16 numbers that hold a weight are off by 2^-32 of the row's largest
    (dX, off the list), by 2^-39 of the largest T grad (dY)."""
    loss, dX, dY, G, has = statement(X, Y, ids, scores, T, tlse, grad)
    X, Y, ids, scores, grad = X.double().cpu(), Y.double().cpu(), ids.cpu(), scores.double().cpu(), grad.double().cpu()
    n, f = X.shape
    m = Y.shape[0]
    logq = torch.log_softmax(X @ Y.T / T, 1)
    p = torch.zeros(n, m, dtype=torch.float64)
    on = torch.zeros(n, m, dtype=torch.bool)
    for b in range(n):
        for i, v in zip(ids[b].tolist(), scores[b].tolist()):
            if 0 <= i < m and v > LOW:
                p[b, i] += math.exp(v / T - float(tlse[b]))
                on[b, i] = True
    lp = torch.where(on, p.clamp(min=1e-300).log(), 0.0)
    pr = (1.0 - p.sum(1)).clamp(min=0.0)
    qr = torch.where(on, 0.0, logq.exp()).sum(1).clamp(min=2.0 ** -24)
    dz = (8 * math.sqrt(f) * HALF + 2 * 2.0 ** -22) * float((X.abs() @ Y.abs().T).max()) / T
    rel = 2 * dz + 16 * HALF + 8 * math.sqrt(m) * HALF
    ep = p * (lp.abs() + 4) * HALF
    dp = ep.sum(1)
    q = logq.exp()
    share = q / qr[:, None]
    off = T * torch.where(on, rel * q + ep, rel * (q + pr[:, None] * share) + dp[:, None] * share) * has[:, None]
    weigh = T * torch.where(on, 0.0, q + pr[:, None] * share).amax(1) * has
    w = grad.abs()
    tx = w[:, None] * (off @ Y.abs() + (8 * math.sqrt(m) + 16) * HALF * (G.abs() @ Y.abs()) + m * 2.0 ** -32 * weigh[:, None] * Y.abs().amax())
    ty = (off * w[:, None]).T @ X.abs() + (8 * math.sqrt(n) + 16) * HALF * ((G.abs() * w[:, None]).T @ X.abs())
    ty = ty + n * 2.0 ** -39 * T * w.max() * X.abs().amax()
    part = torch.where(on, p * rel + ep * (lp - logq).abs(), 0.0).sum(1)
    rest = torch.where(pr > 0, pr * rel + dp * (1 + (pr.clamp(min=1e-300) / qr).log().abs()), 0.0)
    tl = T * T * (part + rest + 4 * HALF) + 4 * HALF * loss.abs()
    for name, a, b, t in zip(("loss", "dX", "dY"), got, (loss, dX, dY), (tl, tx, ty)):
        assert torch.all(torch.isfinite(a)), f"{name} is not finite"
        over = (a.double().cpu() - b).abs() / t.clamp(min=1e-300)
        assert torch.all(over <= 1), f"{name}: {float(over.max())} times the tolerance"


def certain_student(seed, n, m, f, T, top, rest, noise, k=5):
    """Logits (over T) of `top` for item 7, which is on every list, and about `rest` of the probability for all others
    together, spread with a standard deviation of `noise`; half of the teacher's mass is off its list."""
    g = torch.Generator().manual_seed(seed)
    s = math.sqrt(noise * T / math.sqrt(f - 2))
    X, Y = torch.randn(n, f, generator=g) * s, torch.randn(m, f, generator=g) * s
    gap = math.log(m / rest) + noise * noise / 2
    X[:, 0], Y[:, 0] = math.sqrt(T * gap), 0.0
    Y[7, 0] = math.sqrt(T * gap)
    common = T * (top - gap)
    X[:, 1], Y[:, 1] = math.sqrt(abs(common)), math.copysign(math.sqrt(abs(common)), common)
    ids = torch.stack([torch.cat([torch.tensor([7]), 8 + torch.randperm(m - 8, generator=g)[:k - 1]]) for _ in range(n)])
    ids[::3, 1] = -1
    scores = torch.randn(n, k, generator=g) * T
    tlse = torch.logsumexp(torch.where(ids < 0, -math.inf, scores) / T, 1) + math.log(2.0)
    return X, Y, ids.to(torch.int32), scores, tlse, 0.5 + torch.rand(n, generator=g)


@gpu
@pytest.mark.parametrize("f,T,noise", [(64, 1.0, 1.0), (64, 0.05, 3.0), (32, 1.0, 3.0), (160, 2.0, 1.0)])
@pytest.mark.parametrize("rest", [1e-9, 1e-7, 1e-6, 1e-5, 1e-4, 1e-2])
@pytest.mark.parametrize("top", [20.0, 48.0, 100.0])
def test_a_student_certain_of_its_list(dev, top, rest, f, T, noise):
    """What the student gives all items off the list is small beside what it gives the list, and its own sum."""
    X, Y, ids, scores, tlse, grad = (v.to(dev) for v in certain_student(81, 70, 900, f, T, top, rest, noise))
    got = E.distill(X, Y, ids, scores, temperature=T, teacher_lse=tlse, grad=grad)
    compare_with_rest(X, Y, ids, scores, T, tlse, grad, got)
    with torch.no_grad():
        assert torch.equal(E.distill_loss(X, Y, ids, scores, T, tlse), got[0])


@gpu
@pytest.mark.parametrize("spread", [6.0, 8.0, 12.0])
@pytest.mark.parametrize("n,m,f,k", [(1500, 900, 64, 50), (80, 5000, 128, 100), (40, 300, 96, 256)])
def test_a_sharp_student_and_a_flat_teacher(dev, n, m, f, k, spread):
    """Lists of the student's own best items, a teacher that hardly tells them apart and keeps up to a third or almost all of
    its mass elsewhere; few and many rows, lists of every item of a tile."""
    X, Y, _, _, _, grad = problem(82, n, m, f, 1, spread=spread)
    g = torch.Generator().manual_seed(83)
    ids = torch.topk(X @ Y.T, k, dim=1).indices
    ids[1] = torch.arange(32, 32 + k)           # whole tiles of items
    ids[2] = torch.arange(k).flip(0)
    ids[3, k // 2:] = ids[3, :k - k // 2]       # items listed twice
    ids[4] = -1
    scores = torch.randn(n, k, generator=g)
    tlse = torch.logsumexp(scores, 1) + 0.02 + 3 * torch.rand(n, generator=g)
    X, Y, ids, scores, tlse, grad = (v.to(dev) for v in (X, Y, ids.to(torch.int32), scores, tlse, grad))
    got = E.distill(X, Y, ids, scores, teacher_lse=tlse, grad=grad)
    compare_with_rest(X, Y, ids, scores, 1.0, tlse, grad, got)


@gpu
@pytest.mark.parametrize("m", [1, 32, 100, 256])
def test_nothing_off_the_list(dev, m):
    """Every item listed and mass of the teacher elsewhere: the student's share is taken to be 2^-24."""
    X, Y, ids, scores, tlse, grad = problem(84, 40, m, 64, m, dev, tail=True)
    tlse = tlse + 0.5
    got = E.distill(X, Y, ids, scores, teacher_lse=tlse, grad=grad)
    compare_with_rest(X, Y, ids, scores, 1.0, tlse, grad, got)


@gpu
@pytest.mark.parametrize("liked", [False, True])
def test_a_model_learns_from_a_models_lists(dev, liked):
    """AlternatingLeastSquares.distill: the loss is the statement's, and the first step of Adam moves every factor by the
    rate against its gradient's sign (where that is certain)."""
    from scipy import sparse as sp
    from movie_recommender_system_amd.als import AlternatingLeastSquares
    users, items, rate = 120, 500, 0.02
    g = np.random.default_rng(61)
    teacher = AlternatingLeastSquares(factors=48)
    teacher.user_factors, teacher.item_factors = (g.normal(0, 0.5, (c, 48)).astype(np.float32) for c in (users, items))
    rows = sp.random(users, items, 0.05, format="csr", dtype=np.float32, random_state=3) if liked else None
    student = AlternatingLeastSquares(factors=20, random_state=5)
    assert student.distill(teacher, rows, epochs=0) == []
    x0, y0 = student.user_factors.copy(), student.item_factors.copy()
    assert x0.shape == (users, 20) and y0.shape == (items, 20)
    (loss,) = student.distill(teacher, rows, N=30, temperature=0.5, epochs=1, batch=1000, learning_rate=rate)
    ids, scores = teacher.recommend_all(rows, N=30, filter_already_liked_items=liked)
    ids, scores = torch.from_numpy(ids), torch.from_numpy(scores)
    X, Y = torch.from_numpy(x0), torch.from_numpy(y0)
    want = statement(X, Y, ids, scores, 0.5)
    tl, tx, ty = tolerances(X, Y, 0.5, want[3], want[4], None, want[0], None)
    assert abs(loss - float(want[0].mean())) <= float(tl.mean())
    for before, after, grad, tol in ((x0, student.user_factors, want[1], tx), (y0, student.item_factors, want[2], ty)):
        moved = torch.from_numpy(after - before).double()
        sure = grad.abs() > tol + 1e-6    # 1e-8 in Adam's denominator is then 1e-2 of the step at most
        assert bool(sure.any()) and torch.all(moved.abs() <= rate * (1 + 1e-4) + 1e-6)
        assert torch.all((moved + rate * grad.sign())[sure].abs() <= rate * 1.1e-2 + 1e-6)
    # batches and more epochs run; the students' own lists and draws
    losses = student.distill(teacher, rows, N=30, epochs=2, batch=50)
    assert len(losses) == 2 and all(math.isfinite(v) for v in losses)
    got, lp = student.sample(np.arange(5), rows[:5] if liked else None, N=3, filter_already_liked_items=liked, random_state=1)
    assert got.shape == (5, 3) and np.all(got >= 0) and np.all(lp <= 0)
    for bad in (dict(N=0), dict(batch=0), dict(learning_rate=0.0), dict(epochs=-1)):
        with pytest.raises(ValueError):
            student.distill(teacher, rows, **bad)
    with pytest.raises(ValueError):
        student.distill(AlternatingLeastSquares(factors=8))
    other = AlternatingLeastSquares(factors=8)
    other.user_factors, other.item_factors = np.zeros((3, 8), np.float32), np.zeros((4, 8), np.float32)
    with pytest.raises(ValueError):
        student.distill(other)


@gpu
def test_a_refused_distillation_leaves_the_model_as_it_was(dev):
    from scipy import sparse as sp
    from movie_recommender_system_amd.als import AlternatingLeastSquares
    g = np.random.default_rng(62)
    teacher = AlternatingLeastSquares(factors=16)
    teacher.user_factors, teacher.item_factors = (g.normal(0, 0.5, (c, 16)).astype(np.float32) for c in (30, 400))
    bad = [dict(N=300), dict(temperature=0.0), dict(temperature=float("nan")), dict(N=0), dict(learning_rate=-1.0),
           dict(user_items=sp.csr_matrix((30, 399), dtype=np.float32))]
    new = AlternatingLeastSquares(factors=8, random_state=3)
    old = AlternatingLeastSquares(factors=8, random_state=3)
    x, y = (g.normal(0, 0.5, (c, 8)).astype(np.float32) for c in (30, 400))
    old.user_factors, old.item_factors = x, y
    half = AlternatingLeastSquares(factors=8, random_state=3)
    half.item_factors = np.zeros((7, 8), np.float32)     # not the teacher's items
    for kw in bad:
        for model in (new, old, half):
            with pytest.raises((ValueError, _lib.MirecError)):
                model.distill(teacher, **kw)
        assert new.user_factors is None and new.item_factors is None
        assert old.user_factors is x and old.item_factors is y and half.user_factors is None
    with pytest.raises(ValueError):
        half.distill(teacher)
    with pytest.raises(ValueError):                      # still a model that was never fitted
        new.sample(0, None, filter_already_liked_items=False)
    with pytest.raises(_lib.MirecError):                 # wider than the kernels
        wide = AlternatingLeastSquares(factors=200)
        wide.distill(teacher)
    assert wide.user_factors is None and wide.item_factors is None


@gpu
def test_the_list_of_the_best_items_to_draws(dev):
    """The operators together, as they are used: a teacher's top-K lists, a student's step, its own lists, draws."""
    g = torch.Generator().manual_seed(3)
    XT, YT = (torch.randn(300, 64, generator=g) * 0.4).to(dev), (torch.randn(2000, 64, generator=g) * 0.4).to(dev)
    ids, scores = E.topk(XT, YT, 50)
    X, Y = XT[:, :32].contiguous(), YT[:, :32].contiguous()
    loss, dX, dY = E.distill(X, Y, ids, scores, temperature=1.0)
    compare(X, Y, ids, scores, 1.0, None, None, (loss, dX, dY))
    sid, ssc = E.topk(X, Y, 20)
    u = torch.rand(300, 4, generator=g).to(dev)
    got, lp = E.sample_scores(ssc, u, ids=sid, temperature=0.5, top_p=0.9, replacement=False)
    for r in range(300):
        mine = [i for i in got[r].tolist() if i >= 0]
        assert mine and set(mine) <= set(sid[r].tolist()) and len(set(mine)) == len(mine)
