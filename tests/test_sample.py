"""Drawing items from scores: engine.sample_scores / mirec_sample against a float64 statement of its definition.

A draw is checked by the interval of (0, 1) that belongs to the item: the device's running sum may sit off the float64 one
by the weights' own error.  A weight is 2^f by a polynomial within 1.6e-14 of it, its exponent a product of float64 numbers
below 2^7 (2^-46 ln 2 of it at most) in float64 arithmetic (a dozen roundings, each 2^-53), rounded to S = min(51, 62 -
ceil(log2 m)) fraction bits; with the largest weight 1 the borders of the normalised running sum are off by at most 2 (3e-13
+ m 2^-(S+1)).  The logarithm of the probability carries the same and one rounding to fp32 (half a step: 2^-24 of it)."""

import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

from movie_recommender_system_amd import _lib
from movie_recommender_system_amd import engine as E

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def border_error(m):
    bits = min(51, 62 - max(0, math.ceil(math.log2(max(m, 1)))))
    return 2 * (3e-13 + m * 2.0 ** -(bits + 1))


def keep_row(s, ok, T, top_k, top_p, min_p):
    """Weights (float64, zero where not kept) of one row by the definition."""
    m = len(s)
    w = np.zeros(m)
    if not ok.any():
        return w
    if not T >= 1e-37:
        top_k, T = 1, 1.0
    best = s[ok].max()
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(s == best, 0.0, (s - best) / T)
    w[ok] = np.exp(d[ok])
    order = np.array(sorted(np.flatnonzero(ok), key=lambda i: (-s[i], i)))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = w[order]
        before = np.concatenate([[0.0], np.cumsum(mass)[:-1]])
        inside = before < top_p * mass.sum()
        inside[0] = True
        order = order[inside]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    out = np.zeros(m)
    out[order] = w[order]
    return out


def check(scores, uniforms, got_ids, got_lp, ids=None, liked=None, T=1.0, top_k=0, top_p=1.0, min_p=0.0, replacement=True):
    """Every draw of every row against the definition; `liked`: list of index arrays."""
    low = float(torch.finfo(scores.dtype).min)
    s = scores.detach().double().cpu().numpy()
    u = uniforms.double().cpu().numpy()
    got_ids, got_lp = got_ids.cpu().numpy(), got_lp.cpu().numpy()
    n, m = s.shape
    tol = border_error(m)
    par = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else v
    for r in range(n):
        with np.errstate(invalid="ignore"):
            ok = s[r] > low
        if ids is not None:
            lid = ids[r].cpu().numpy()
            ok &= lid >= 0
        if liked is not None:
            ok[liked[r]] = False
        w = keep_row(s[r], ok, par(T, r), int(par(top_k, r)), par(top_p, r), par(min_p, r))
        for j in range(u.shape[1]):
            total = w.sum()
            where = f"row {r} draw {j}"
            if total <= 0:
                assert got_ids[r, j] == -1 and got_lp[r, j] == -np.inf, where
                continue
            i = got_ids[r, j]
            if ids is not None:
                i = np.flatnonzero(lid == i)
                assert i.size == 1, where
                i = i[0]
            assert 0 <= i < m and w[i] > 0, f"{where}: item {i} is not kept"
            hi = w[:i + 1].sum() / total
            lo = hi - w[i] / total
            assert lo - tol <= u[r, j] < hi + tol, f"{where}: item {i} holds [{lo}, {hi}), drawn with {u[r, j]}"
            lp = math.log(w[i] / total)
            assert abs(got_lp[r, j] - lp) <= 2.0 ** -24 * abs(lp) + 2 * tol / 1.0 + 1e-12, f"{where}: {got_lp[r, j]} {lp}"
            if not replacement:
                w[i] = 0.0


# ------------------------------------------------------------------------------------------------ refusals (no GPU)

def call(scores=16, dtype=0, n=2, m=4, stride=4, ids=None, ids_stride=0, indptr=None, indices=None, uniforms=16, draws=1,
         T=1.0, k=0, p=1.0, q=0.0, out_ids=16, out_lp=16):
    """mirec_sample with made-up device addresses: every call here is refused before anything is launched."""
    lib = _lib.require()
    rc = lib.mirec_sample(scores, dtype, n, m, stride, ids, ids_stride, indptr, indices, uniforms, draws, 1, T, None, k,
                          None, p, None, q, None, out_ids, out_lp, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("change,code,text", [
    ({"n": -1}, -1, "negative"), ({"m": -1}, -1, "negative"), ({"draws": -1}, -1, "negative"),
    ({"dtype": 3}, -1, "type"), ({"draws": 1025}, -4, "1024"), ({"m": (1 << 30) + 1}, -4, "2^30"),
    ({"T": -0.5}, -1, "temperature"), ({"T": float("nan")}, -1, "temperature"), ({"T": float("inf")}, -1, "temperature"),
    ({"p": -0.1}, -1, "top_p"), ({"p": 1.1}, -1, "top_p"), ({"p": float("nan")}, -1, "top_p"),
    ({"q": -0.1}, -1, "min_p"), ({"q": 1.1}, -1, "min_p"), ({"k": -1}, -1, "top_k"),
    ({"scores": None}, -1, "null"), ({"uniforms": None}, -1, "null"), ({"out_ids": None}, -1, "null"),
    ({"out_lp": None}, -1, "null"), ({"stride": -4}, -1, "stride"), ({"scores": 18}, -1, "aligned"),
    ({"ids": 16, "indptr": 16}, -1, "ids"), ({"indptr": 16, "m": 524289}, -4, "524288"),
])
def test_the_c_entry_refuses(change, code, text):
    rc, msg = call(**change)
    assert rc == code and text in msg, (rc, msg)


def test_nothing_to_do_is_no_error():
    assert call(n=0)[0] == 0 and call(draws=0)[0] == 0


def test_the_wrapper_refuses_on_the_host():
    s = torch.zeros(2, 4)
    with pytest.raises(_lib.MirecError):
        E.sample_scores(s, torch.zeros(2, 1))
    with pytest.raises(ValueError):
        E.sample_scores(s.double(), torch.zeros(2, 1))
    with pytest.raises(ValueError):
        E.sample_scores(s[0], torch.zeros(2, 1))


def waits_missing(source):
    """Instructions written out in a HIP source that read vcc as a carry, or a register by a data-parallel move, less than
    two wait states behind the vector instruction that wrote it.  The macros' steps follow each other, so every step is
    read twice in a row."""
    bad = []
    for block in re.findall(r"#define SM_\w+_STEP(?:.*\\\n)*.*", source):
        step = [i.strip() for text in re.findall(r'"((?:[^"\\]|\\.)*)"', block) for i in text.split("\\n")]
        step = [i for i in step if re.match(r"[sv]_", i)]
        written = {}     # register -> wait states since
        for ins in step * 2:
            nop = re.match(r"s_nop (\d+)", ins)
            if nop:
                written = {r: w + int(nop.group(1)) + 1 for r, w in written.items()}
                continue
            name, ops = ins.split(None, 1)
            ops = re.findall(r"%\d|\bvcc\b", ops)
            outs = 2 if "_co_" in name else 1
            bad += [ins for r in ops[outs:] if written.get(r, 9) < 2]
            written = {r: w + 1 for r, w in written.items()}
            written.update({r: 0 for r in ops[:outs]})
    return bad


def test_cross_lane_steps_keep_their_wait_states():
    text = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "sample_kernel.h")).read()
    assert len(re.findall(r"#define SM_\w+_STEP", text)) == 2
    assert waits_missing(text) == []
    # what the check is for: a carry read directly behind its write, a move directly behind a write
    assert waits_missing('#define SM_A_STEP(M) "s_nop 0\\n" "v_add_co_u32_dpp %0, vcc, %0, %0 " M "\\n" "v_addc_co_u32_dpp %1, vcc, %1, %1, vcc " M "\\n"')
    assert waits_missing('#define SM_B_STEP(M) "s_nop 0\\nv_max_f32_dpp %0, %0, %0 " M "\\n"')


# ------------------------------------------------------------------------------------------------------- on the GPU

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda", 0)


def make(seed, n, m, dtype, draws, dev, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    s = (torch.randn(n, m, generator=g) * spread).to(TORCH[dtype])
    u = torch.rand(n, draws, generator=g)
    return s.to(dev), u.to(dev)


def filter_rows(seed, n, m, share, dev):
    rng = np.random.default_rng(seed)
    rows = [np.sort(rng.choice(m, int(rng.integers(0, int(share * m) + 1)), replace=False)) for _ in range(n)]
    indptr = np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int64)
    flat = np.concatenate(rows + [np.zeros(0, np.int64)]).astype(np.int32)
    flat = np.concatenate([flat, np.zeros(1, np.int32)])[:max(1, flat.size)]
    csr = E.DeviceCSR(torch.from_numpy(indptr).to(dev), torch.from_numpy(flat).to(dev),
                      torch.ones(flat.size, device=dev), (n, m))
    return rows, csr


CUTS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_p=0.6), dict(min_p=0.1), dict(top_k=40, top_p=0.8, min_p=0.02),
        dict(T=0.3, top_p=0.95), dict(T=0.0), dict(T=5.0, top_k=1 << 30, top_p=0.999), dict(top_p=0.0), dict(min_p=1.0)]


@gpu
@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,m", [(3, 1), (4, 2), (5, 63), (4, 64), (6, 65), (3, 255), (3, 257), (5, 1000), (2, 4099)])
def test_draws_follow_the_definition(dev, n, m, dtype, cut):
    s, u = make(n * 7919 + m, n, m, dtype, 5, dev)
    kw = {{"T": "temperature"}.get(k, k): v for k, v in cut.items()}
    ids, lp = E.sample_scores(s, u, **kw)
    check(s, u, ids, lp, **cut)


@gpu
@pytest.mark.parametrize("n,m,dtype", [(2, 27000, "f32"), (1, 32768, "f32"), (1, 33001, "f32"), (2, 65537, "bf16"), (1, 200000, "bf16"),
                                       (1, 300001, "f32"), (1, 131072, "f16")])
@pytest.mark.parametrize("cut", [dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_p=0.5, min_p=0.01), dict(top_k=5000)])
def test_long_rows(dev, n, m, dtype, cut):
    s, u = make(m, n, m, dtype, 16, dev, spread=1.3)
    ids, lp = E.sample_scores(s, u, **cut)
    check(s, u, ids, lp, **cut)


@gpu
@pytest.mark.parametrize("cut", [dict(), dict(top_k=10), dict(top_p=0.7), dict(top_k=33, top_p=0.9, min_p=0.05)])
@pytest.mark.parametrize("levels", [1, 2, 5])
@pytest.mark.parametrize("m", [64, 777, 5000])
def test_ties_rank_by_index(dev, m, levels, cut):
    """Scores of few distinct values: every cut falls inside a group of equal scores."""
    g = torch.Generator().manual_seed(m + levels)
    s = torch.randint(0, levels, (4, m), generator=g).float().to(dev)
    u = torch.rand(4, 9, generator=g).to(dev)
    ids, lp = E.sample_scores(s, u, **cut)
    check(s, u, ids, lp, **cut)


@gpu
@pytest.mark.parametrize("cut", [dict(top_k=1), dict(top_k=129), dict(top_k=300), dict(top_k=700), dict(top_k=5000), dict(top_p=0.37),
                                 dict(top_k=6000, top_p=0.37), dict(top_p=0.37, min_p=0.9999999), dict(top_k=200, top_p=0.9)])
@pytest.mark.parametrize("n,m", [(2, 7000), (3, 20011)])
@pytest.mark.parametrize("spread", [3e-7, 1e-4])
def test_cuts_among_nearly_equal_scores(dev, n, m, spread, cut):
    """All scores in one bin of the first histogram (1/32 octave): cuts by the finer ones, ties by index."""
    s, u = make(m + n, n, m, "f32", 4, dev, spread)
    s = s + 1.0
    ids, lp = E.sample_scores(s, u, **cut)
    check(s, u, ids, lp, **cut)


@gpu
@pytest.mark.parametrize("cut", [dict(), dict(top_k=20), dict(top_k=1000, top_p=0.8), dict(top_p=0.7), dict(min_p=0.3)])
@pytest.mark.parametrize("n,m,dtype", [(1, 300_007, "f32"), (2, 1_000_003, "f16")])
def test_rows_of_more_than_1024_chunks(dev, n, m, dtype, cut):
    s, u = make(m, n, m, dtype, 3, dev)
    ids, lp = E.sample_scores(s, u, replacement=False, **cut)
    check(s, u, ids, lp, replacement=False, **cut)


@gpu
def test_a_model_draws_from_its_lists(dev):
    """AlternatingLeastSquares.sample: every draw by the definition on the model's own list, repeatable, refusals."""
    from scipy import sparse as sp
    from movie_recommender_system_amd.als import AlternatingLeastSquares
    g = np.random.default_rng(8)
    model = AlternatingLeastSquares(factors=24)
    with pytest.raises(ValueError):
        model.sample(0, None)
    model.user_factors, model.item_factors = (g.normal(0, 0.6, (c, 24)).astype(np.float32) for c in (60, 800))
    liked = sp.random(60, 800, 0.1, format="csr", dtype=np.float32, random_state=4)
    users = np.array([3, 59, 3, 0])
    kw = dict(N=6, pool=50, temperature=0.4, top_p=0.95, min_p=0.01)
    ids, lp = model.sample(users, liked[users], random_state=11, **kw)
    again = model.sample(users, liked[users], random_state=np.random.RandomState(11), **kw)
    assert np.array_equal(ids, again[0]) and np.array_equal(lp, again[1]) and ids.dtype == np.int32 and lp.dtype == np.float32
    best, scores = model.recommend(users, liked[users], N=50)
    u = np.random.RandomState(11).randint(0, 1 << 24, size=(4, 6)).astype(np.float32) * np.float32(2.0 ** -24)
    check(torch.from_numpy(scores), torch.from_numpy(u), torch.from_numpy(ids), torch.from_numpy(lp), ids=torch.from_numpy(best),
          T=0.4, top_p=0.95, min_p=0.01, replacement=False)
    # one user; the attached matrix; temperature zero; a pool that the filter empties
    model.attach_user_items(liked)
    one, p1 = model.sample(3, N=6, pool=50, temperature=0.0, random_state=1)
    assert one.shape == (6,) and one[0] == best[0, 0] and np.all(one[1:] == -1) and np.all(np.isneginf(p1[1:]))
    with pytest.raises(_lib.MirecError):     # longer than the lists of the top-K kernels
        model.sample([5], N=4, pool=10 ** 6, filter_already_liked_items=False, random_state=2)
    wide, _ = model.sample([5], N=4, pool=224, filter_already_liked_items=False, random_state=2)
    assert wide.shape == (1, 4) and np.all(wide >= 0)
    everything = sp.csr_matrix(np.ones((1, 800), np.float32))
    none, p0 = model.sample([5], everything, N=2, random_state=2)
    assert np.all(none == -1) and np.all(np.isneginf(p0))
    with pytest.raises(IndexError):
        model.sample(60)
    for bad in (dict(N=0), dict(pool=0)):
        with pytest.raises(ValueError):
            model.sample(1, **bad)
    with pytest.raises(ValueError):
        model.sample([1, 2], liked[:1])
    with pytest.raises(_lib.MirecError):
        model.sample(1, temperature=-1.0)


@gpu
def test_borders_belong_to_the_next_item(dev):
    """Equal weights over a power of two of items: the borders are multiples of 1/m, and a number on a border takes the
    item that begins there."""
    m = 4096
    s = torch.full((1, m), 0.25, device=dev)
    u = (torch.arange(0, m, 5, device=dev, dtype=torch.float32) / m)[None]
    ids, lp = E.sample_scores(s, u[:, :800].contiguous())
    assert torch.equal(ids[0].long(), torch.arange(0, m, 5, device=dev)[:800])
    assert torch.all(lp == -math.log(m))
    # half of them by top_p: the mass before item m/2 is not below one half
    ids, lp = E.sample_scores(s, torch.tensor([[0.0, 0.999]], device=dev), top_p=0.5)
    assert ids[0, 0] == 0 and ids[0, 1] == int(0.999 * m / 2) and torch.all(lp == -math.log(m / 2))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_excluded_scores(dev, dtype):
    t = TORCH[dtype]
    low = torch.finfo(t).min
    nan, inf = float("nan"), float("inf")
    s = torch.tensor([[nan, 1.0, -inf, low, 2.0, nan, 0.5, low],
                      [nan, nan, -inf, low, low, -inf, nan, nan],
                      [low, low, low, low, low, low, low, 3.0],
                      [inf, 1.0, inf, 0.0, inf, -inf, nan, low],
                      [-0.0, 0.0, -0.0, 0.0, low, low, low, low]], dtype=t, device=dev)
    u = torch.rand(5, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    for cut in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=3, top_p=0.99), dict(temperature=0.0)):
        ids, lp = E.sample_scores(s, u, **cut)
        if "temperature" in cut:
            cut = dict(T=0.0)
        check(s, u, ids, lp, **cut)
        assert torch.all(ids[1] == -1) and torch.all(ids[2] == 7) and torch.all(lp[2] == 0)
        assert set(ids[3].tolist()) <= {0, 2, 4}


@gpu
@pytest.mark.parametrize("m", [50, 1000, 9001])
@pytest.mark.parametrize("cut", [dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.8)])
def test_filtered_items_are_never_drawn(dev, m, cut):
    n = 6
    s, u = make(m, n, m, "f32", 8, dev)
    for share in (0.0, 0.1, 0.9, 1.0):
        rows, csr = filter_rows(m + int(10 * share), n, m, share, dev)
        ids, lp = E.sample_scores(s, u, mask=csr, **cut)
        check(s, u, ids, lp, liked=rows, **cut)
    # a filter that holds everything, in no order and with entries named twice
    flat = np.concatenate([np.random.default_rng(0).permutation(m), np.arange(m)]).astype(np.int32)
    csr = E.DeviceCSR(torch.arange(n + 1, device=dev) * (2 * m), torch.from_numpy(np.tile(flat, n)).to(dev),
                      torch.ones(2 * m * n, device=dev), (n, m))
    ids, lp = E.sample_scores(s, u, mask=csr, **cut)
    assert torch.all(ids == -1) and torch.all(lp == -math.inf)


@gpu
@pytest.mark.parametrize("k", [1, 20, 64, 100, 224])
@pytest.mark.parametrize("replacement", [True, False])
def test_ranked_lists(dev, k, replacement):
    """Lists as topk returns them, with empty slots at the tail and whole rows empty."""
    g = torch.Generator().manual_seed(k)
    n = 70
    s = torch.sort(torch.randn(n, k, generator=g), dim=1, descending=True).values
    ids = torch.stack([torch.randperm(5000, generator=g)[:k] for _ in range(n)]).to(torch.int32)
    length = torch.randint(0, k + 1, (n, 1), generator=g)
    empty = torch.arange(k)[None] >= length
    ids[empty & (torch.rand(n, k, generator=g) < 0.5)] = -1
    s[empty] = torch.finfo(torch.float32).min
    u = torch.rand(n, 7, generator=g)
    s, ids, u = s.to(dev), ids.to(dev), u.to(dev)
    for cut in (dict(), dict(top_k=5), dict(top_p=0.7, min_p=0.1)):
        got, lp = E.sample_scores(s, u, ids=ids, replacement=replacement, **cut)
        check(s, u, got, lp, ids=ids, replacement=replacement, **cut)


@gpu
@pytest.mark.parametrize("k", [300, 1000, 9000])
@pytest.mark.parametrize("replacement", [True, False])
def test_long_and_unordered_lists(dev, k, replacement):
    """Lists longer than the short rows' kernels take, in any order, with empty slots in between."""
    g = torch.Generator().manual_seed(k)
    s = torch.randn(6, k, generator=g)
    ids = torch.stack([torch.randperm(20000, generator=g)[:k] for _ in range(6)]).to(torch.int32)
    ids[torch.rand(6, k, generator=g) < 0.3] = -1
    ids[5] = -1
    u = torch.rand(6, 5, generator=g)
    s, ids, u = s.to(dev), ids.to(dev), u.to(dev)
    for cut in (dict(), dict(top_k=5), dict(top_p=0.7, min_p=0.001), dict(top_k=200)):
        got, lp = E.sample_scores(s, u, ids=ids, replacement=replacement, **cut)
        check(s, u, got, lp, ids=ids, replacement=replacement, **cut)


@gpu
@pytest.mark.parametrize("m", [1, 32, 33, 64, 65, 100, 128, 129, 256])
@pytest.mark.parametrize("lists", [False, True])
def test_rows_that_share_a_wavefront(dev, m, lists):
    """Many short rows: each draws what it draws alone, whatever shares its wavefront (parameters and filters per row, rows
    that are in order beside rows that are not)."""
    n = 29993
    g = torch.Generator().manual_seed(m)
    s = torch.randn(n, m, generator=g)
    s = torch.where(torch.rand(n, 1, generator=g) < 0.6, torch.sort(s, dim=1, descending=True).values, s).to(dev)
    u = torch.rand(n, 3, generator=g).to(dev)
    T = (0.2 + torch.rand(n, generator=g)).to(dev)
    k = torch.randint(0, 80, (n,), generator=g, dtype=torch.int32).to(dev)
    p = (torch.rand(n, generator=g) * 1.3).to(dev)
    rows, csr = filter_rows(m, n, m, 0.3, dev)
    ids = (torch.randint(0, 1 << 20, (n, m), generator=g, dtype=torch.int32) * 1024 + torch.arange(m, dtype=torch.int32)).to(dev)
    ids[::7, ::3] = -1
    for replacement in (True, False):
        kw = dict(temperature=T, top_k=k, top_p=p, replacement=replacement)
        got, lp = E.sample_scores(s, u, **kw, **(dict(ids=ids) if lists else dict(mask=csr)))
        for r in (0, 1, 2, 3, 777, 14976, 14977, n - 2, n - 1):
            one = slice(r, r + 1)
            extra = dict(ids=ids[one]) if lists else dict(mask=E.DeviceCSR(csr.indptr[r:r + 2], csr.indices, csr.data, (1, m)))
            alone = E.sample_scores(s[one], u[one], temperature=T[one], top_k=k[one], top_p=p[one], replacement=replacement, **extra)
            assert torch.equal(got[one], alone[0]) and torch.equal(lp[one], alone[1]), r
        pick = torch.arange(0, n, 997)
        at = pick.to(dev)
        pc = p[at].cpu().clamp(max=1.0)
        check(s[at], u[at], got[at], lp[at], ids=ids[at] if lists else None, liked=None if lists else [rows[r] for r in pick.tolist()],
              T=T[at].cpu(), top_k=k[at].cpu(), top_p=pc, replacement=replacement)


@gpu
@pytest.mark.parametrize("m", [5, 300, 3001, 30000])
def test_without_replacement_no_item_twice(dev, m):
    n, draws = 5, 12
    s, u = make(m, n, m, "f32", draws, dev)
    for cut in (dict(), dict(top_k=8), dict(top_p=0.5), dict(min_p=0.2)):
        ids, lp = E.sample_scores(s, u, replacement=False, **cut)
        check(s, u, ids, lp, replacement=False, **cut)
        for r in ids.tolist():
            r = [i for i in r if i >= 0]
            assert len(set(r)) == len(r)
    # as many draws as items, and more: every item once, then nothing
    if m <= 300:
        s, u = make(m + 1, 3, m, "f32", m + 3, dev, spread=0.5)
        ids, lp = E.sample_scores(s, u, replacement=False)
        check(s, u, ids, lp, replacement=False)
        assert torch.equal(torch.sort(ids[:, :m], dim=1).values, torch.arange(m, dtype=torch.int32, device=dev).expand(3, m))
        assert torch.all(ids[:, m:] == -1)


def check_leaving(scores, uniforms, got_ids, got_lp, ids=None, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draws without replacement against the definition in logarithms, so that an item counts however unlikely it was beside
    those that have left.  The device forms its weights anew once their sum is below 2^(ceil(log2 m) + 23) units (m up to
    2^19): m roundings of half a unit are 2^-24 of it at most, the border error on top."""
    low = float(torch.finfo(scores.dtype).min)
    s, u = scores.double().cpu().numpy(), uniforms.double().cpu().numpy()
    got_ids, got_lp = got_ids.cpu().numpy(), got_lp.cpu().numpy()
    n, m = s.shape
    tol = 2.0 ** -24 + border_error(m)
    for r in range(n):
        ok = s[r] > low
        if ids is not None:
            lid = ids[r].cpu().numpy()
            ok &= lid >= 0
        t = float(T[r]) if isinstance(T, torch.Tensor) else T
        best = s[r][ok].max() if ok.any() else 0.0
        d = (s[r] - best) / t
        left = [i for i in sorted(np.flatnonzero(ok), key=lambda i: (-s[r][i], i))]
        if top_k > 0:
            left = left[:top_k]
        if top_p < 1:
            mass = np.exp(d[left])
            before = np.concatenate([[0.0], np.cumsum(mass)[:-1]])
            left = [i for j, i in enumerate(left) if j == 0 or before[j] < top_p * mass.sum()]
        if min_p > 0:
            left = [i for i in left if d[i] >= math.log(min_p)]
        left = np.array(sorted(left), dtype=np.int64)
        for j in range(u.shape[1]):
            where = f"row {r} draw {j}"
            if left.size == 0:
                assert got_ids[r, j] == -1 and got_lp[r, j] == -np.inf, where
                continue
            i = got_ids[r, j]
            if ids is not None:
                i = np.flatnonzero(lid == i)[0]
            at = np.flatnonzero(left == i)
            assert at.size == 1, f"{where}: {i} is not there"
            w = np.exp(d[left] - d[left].max())
            hi = np.cumsum(w)[at[0]] / w.sum()
            lo = hi - w[at[0]] / w.sum()
            assert lo - tol <= u[r, j] < hi + tol, f"{where}: item {i} holds [{lo}, {hi}), drawn with {u[r, j]}"
            lp = d[i] - d[left].max() - math.log(w.sum())
            assert got_lp[r, j] <= 0 and abs(got_lp[r, j] - lp) <= 2.0 ** -24 * abs(lp) + 2 * tol, f"{where}: {got_lp[r, j]} {lp}"
            left = np.delete(left, at[0])


def stepped(seed, n, m, gap, T, dtype="f32", few=3):
    """Scores (in units of T) of standard deviation one around 0, -gap and -2 gap: `few` items on each of the first two steps."""
    g = torch.Generator().manual_seed(seed)
    level = torch.full((n, m), 2.0)
    for r in range(n):
        at = torch.randperm(m, generator=g)
        level[r, at[:few]], level[r, at[few:2 * few]] = 0.0, 1.0
    return ((torch.randn(n, m, generator=g) - gap * level) * T).to(TORCH[dtype])


@gpu
@pytest.mark.parametrize("gap", [10.0, 20.0, 34.0, 36.5, 50.0, 700.0])
@pytest.mark.parametrize("m", [5, 40, 64, 100, 200, 257, 3001, 20000])
@pytest.mark.parametrize("cut", [dict(), dict(top_k=30), dict(top_k=400), dict(min_p=1e-13), dict(T=0.02), dict(top_p=0.75, T=3.0)])
def test_items_far_less_likely_follow_those_that_left(dev, m, gap, cut):
    """Every kept item is drawn before -1, with its probability among those left."""
    T, n = cut.get("T", 1.0), 5
    s = stepped(m, n, m, gap, T).to(dev)
    draws = min(m + 2, 70) if m <= 200 else 10
    u = torch.rand(n, draws, generator=torch.Generator().manual_seed(m + 1)).to(dev)
    kw = {{"T": "temperature"}.get(k, k): v for k, v in cut.items()}
    ids, lp = E.sample_scores(s, u, replacement=False, **kw)
    check_leaving(s, u, ids, lp, **cut)


@gpu
def test_a_step_between_every_two_items(dev):
    """The weights are formed anew at every draw; rows of all kernels, and scores of all types."""
    for m, dtype, cut in ((2, "f32", {}), (64, "f32", {}), (90, "bf16", {}), (256, "f16", {}), (300, "f32", {}), (300, "f32", {"top_k": 100}),
                          (2000, "bf16", {"top_k": 100}), (9000, "f32", {}), (20000, "f32", {"top_p": 0.9})):
        g = torch.Generator().manual_seed(m)
        s = torch.stack([torch.randperm(m, generator=g) for _ in range(3)]).float() * (-250.0 / m if dtype == "f16" else -1.0)
        s = s.to(TORCH[dtype]).to(dev)
        u = torch.rand(3, min(m + 1, 40), generator=g).to(dev)
        T = 250.0 / m / 60 if dtype == "f16" else 1 / 60
        ids, lp = E.sample_scores(s, u, temperature=T, replacement=False, **cut)
        check_leaving(s, u, ids, lp, T=T, **cut)


@gpu
@pytest.mark.parametrize("m,dtype", [(300_007, "f32"), (524_288, "bf16"), (524_288, "f32")])
@pytest.mark.parametrize("cut", [dict(), dict(top_k=60), dict(min_p=1e-12)])
def test_steps_in_rows_of_more_than_1024_chunks(dev, m, dtype, cut):
    s = stepped(m, 2, m, 45.0, 1.0, dtype, few=4).to(dev)
    u = torch.rand(2, 12, generator=torch.Generator().manual_seed(m)).to(dev)
    ids, lp = E.sample_scores(s, u, replacement=False, **cut)
    check_leaving(s, u, ids, lp, **cut)


@gpu
def test_steps_beside_a_filter_and_in_a_replayed_graph(dev):
    """Filtered items stay out of the weights that are formed anew; two captured calls give the eager draws on every replay."""
    for n, m, cut in ((5, 150, {}), (4, 2000, {"top_k": 90}), (4, 5000, {})):
        s = stepped(m, n, m, 50.0, 1.0).to(dev)
        u = torch.rand(n, 10, generator=torch.Generator().manual_seed(m)).to(dev)
        rows, csr = filter_rows(m, n, m, 0.5, dev)
        call = lambda: E.sample_scores(s, u, mask=csr, replacement=False, **cut)
        want = call()
        inside = s.clone()
        for r, out in enumerate(rows):
            inside[r, torch.from_numpy(out).to(dev)] = torch.finfo(torch.float32).min
        check_leaving(inside, u, *want, **cut)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                outs.append(call())
            graphs.append(gr)
        for _ in range(3):
            for gr, o in zip(graphs, outs):
                o[0].fill_(7)
                o[1].fill_(7.0)
                gr.replay()
            again = call()
            torch.cuda.synchronize()
            for o in outs + [again]:
                assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


@gpu
@pytest.mark.parametrize("m", [30, 100, 200])
def test_stepped_lists_that_share_a_wavefront(dev, m):
    """Ranked lists with and without steps side by side: each draws what it draws alone."""
    n = 30011
    g = torch.Generator().manual_seed(m)
    s = torch.randn(n, m, generator=g) - 45.0 * (torch.arange(m) >= torch.randint(1, m + 1, (n, 1), generator=g))
    s = torch.where(torch.rand(n, 1, generator=g) < 0.8, torch.sort(s, dim=1, descending=True).values, s)
    ids = (torch.randint(0, 1 << 20, (n, m), generator=g, dtype=torch.int32) * 1024 + torch.arange(m, dtype=torch.int32)).to(dev)
    ids[::7, ::3] = -1
    s, u = s.to(dev), torch.rand(n, 9, generator=g).to(dev)
    T = (0.3 + torch.rand(n, generator=g)).to(dev)
    got, lp = E.sample_scores(s, u, ids=ids, temperature=T, replacement=False)
    for r in (0, 1, 2, 3, 777, 14976, 14977, n - 2, n - 1):
        one = slice(r, r + 1)
        alone = E.sample_scores(s[one], u[one], ids=ids[one], temperature=T[one], replacement=False)
        assert torch.equal(got[one], alone[0]) and torch.equal(lp[one], alone[1]), r
    at = torch.arange(0, n, 997).to(dev)
    check_leaving(s[at], u[at], got[at], lp[at], ids=ids[at], T=T[at].cpu())


@gpu
def test_a_certain_draw_has_probability_one(dev):
    """What is reported for an item that was sure to be drawn, after others have left and before."""
    for s, T in (([1.0, 0.105], 0.025), ([0.0, -35.0], 1.0), ([1.2, 0.45, 0.44, 0.43, 0.42], 0.02), ([0.0, -36.2, -36.3], 1.0)):
        s = torch.tensor([s], device=dev)
        u = torch.full((1, s.shape[1] + 1), 0.4, device=dev)
        ids, lp = E.sample_scores(s, u, temperature=T, replacement=False)
        check_leaving(s, u, ids, lp, T=T)
        assert lp[0, s.shape[1] - 1] == 0.0 and ids[0, -1] == -1


@gpu
@pytest.mark.parametrize("m", [3, 70, 130, 300])
def test_an_item_listed_twice_has_two_entries(dev, m):
    """Its entries are drawn apart, each with the probability of its own score."""
    g = torch.Generator().manual_seed(m)
    s = torch.randn(4, m, generator=g)
    s[2:] = torch.sort(s[2:], dim=1, descending=True).values
    u = torch.rand(4, m + 1, generator=g)
    one = torch.arange(m, dtype=torch.int32).expand(4, m).contiguous()
    for replacement in (True, False):
        a, la = E.sample_scores(s.to(dev), u.to(dev), ids=one.to(dev), replacement=replacement)
        b, lb = E.sample_scores(s.to(dev), u.to(dev), ids=(one // 2).to(dev), replacement=replacement)
        assert torch.equal(torch.where(a < 0, a, a // 2), b) and torch.equal(la, lb)
        if not replacement:
            assert torch.equal(torch.sort(a[:, :m], dim=1).values.cpu(), one) and torch.all(b[:, m] == -1)


@gpu
@pytest.mark.parametrize("m", [90, 2000])
def test_parameters_per_row(dev, m):
    n = 24
    s, u = make(m, n, m, "f32", 6, dev)
    g = torch.Generator().manual_seed(5)
    T = 0.3 + torch.rand(n, generator=g)
    k = torch.randint(-1, 60, (n,), generator=g, dtype=torch.int32)
    p = torch.rand(n, generator=g)
    q = torch.rand(n, generator=g) * 0.2
    # values only a device array can hold: greedy, no cut, one item
    T[:4] = torch.tensor([0.0, -1.0, float("nan"), 1e-38])
    k[4:6] = torch.tensor([0, -7])
    p[6:10] = torch.tensor([float("nan"), 1.5, 0.0, -1.0])
    q[10:13] = torch.tensor([float("nan"), -1.0, 2.0])
    ids, lp = E.sample_scores(s, u, temperature=T.to(dev), top_k=k.to(dev), top_p=p.to(dev), min_p=q.to(dev))
    pc, qc = p.clone(), q.clone()
    pc[6], qc[10] = 1.0, 0.0
    check(s, u, ids, lp, T=T, top_k=k, top_p=pc, min_p=qc)
    # one at a time beside plain numbers
    ids, lp = E.sample_scores(s, u, temperature=0.7, top_k=k.to(dev), top_p=0.9)
    check(s, u, ids, lp, T=0.7, top_k=k, top_p=0.9)


@gpu
def test_uniforms_at_and_beyond_the_ends(dev):
    s, _ = make(3, 1, 500, "f32", 1, dev)
    u = torch.tensor([[0.0, -1.0, float("nan"), 1.0, 2.0, 1.0 - 2.0 ** -24, float("inf")]], device=dev)
    ids, lp = E.sample_scores(s, u)
    inside = torch.tensor([[0.0, 0.0, 0.0, 1.0 - 1e-16, 1.0 - 1e-16, 1.0 - 2.0 ** -24, 1.0 - 1e-16]], dtype=torch.float64)
    check(s, inside, ids, lp)
    assert ids[0, 0] == ids[0, 1] == ids[0, 2] == 0 and ids[0, 3] == ids[0, 4] == 499


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m", [100, 1001, 40000])
def test_strides_and_alignment(dev, dtype, m):
    """Rows inside a wider matrix, every second row, one row for all, and a first element at every alignment: the
    same draws as from a contiguous copy."""
    wide, u = make(m, 8, m + 13, dtype, 4, dev)
    for view in (wide[:, 1:m + 1], wide[::2, 5:m + 5], wide[:, 13:], wide[3:4, 2:m + 2].expand(8, m)):
        uu = u[:view.shape[0]].contiguous()
        for cut in (dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.9)):
            a = E.sample_scores(view, uu, **cut)
            b = E.sample_scores(view.contiguous(), uu, **cut)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(ValueError):
        E.sample_scores(wide.T, torch.rand(wide.shape[1], 1, device=dev))


@gpu
def test_offsets_beyond_32_bits(dev):
    stride = (1 << 31) + 24
    flat = torch.empty(2 * stride, dtype=torch.bfloat16, device=dev)
    view = flat.as_strided((2, 5000), (stride, 1))
    s, u = make(11, 2, 5000, "bf16", 6, dev)
    view.copy_(s)
    for cut in (dict(), dict(top_p=0.9)):
        a, b = E.sample_scores(view, u, **cut), E.sample_scores(s, u, **cut)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        check(s, u, *a, **cut)


@gpu
def test_empty_shapes_and_outputs_given(dev):
    u = torch.rand(3, 2, device=dev)
    ids, lp = E.sample_scores(torch.empty(3, 0, device=dev), u)
    assert torch.all(ids == -1) and torch.all(lp == -math.inf)
    assert E.sample_scores(torch.empty(0, 5, device=dev), torch.empty(0, 2, device=dev))[0].shape == (0, 2)
    assert E.sample_scores(torch.zeros(3, 5, device=dev), torch.empty(3, 0, device=dev))[0].shape == (3, 0)
    # rows behind the last one stay as they were
    s, _ = make(1, 3, 300, "f32", 2, dev)
    bids = torch.full((5, 2), 77, dtype=torch.int32, device=dev)
    blp = torch.full((5, 2), 7.5, device=dev)
    out = E.sample_scores(s, u, out=(bids[:3], blp[:3]))
    check(s, u, *out)
    assert torch.all(bids[3:] == 77) and torch.all(blp[3:] == 7.5)


@gpu
def test_wrapper_refusals(dev):
    s, u = make(1, 4, 50, "f32", 2, dev)
    ids = torch.zeros(4, 50, dtype=torch.int32, device=dev)
    _, csr = filter_rows(1, 4, 50, 0.2, dev)
    bad = [dict(uniforms=u[:3]), dict(uniforms=u.double()), dict(uniforms=u.cpu()), dict(uniforms=torch.rand(2, 4, device=dev).T),
           dict(ids=ids, mask=csr), dict(ids=ids[:, :40]), dict(ids=ids.long()), dict(mask=csr.rows(0, 3)),
           dict(temperature=torch.ones(3, device=dev)), dict(temperature=torch.ones(4)), dict(top_k=torch.ones(4, device=dev)),
           dict(top_p=torch.ones(4, 1, device=dev)), dict(min_p=torch.ones(8, device=dev)[::2]),
           dict(out=(ids, torch.zeros(4, 2, device=dev)))]
    for kw in bad:
        with pytest.raises(ValueError):
            E.sample_scores(s, kw.pop("uniforms", u), **kw)
    for kw in (dict(temperature=-1.0), dict(top_p=1.5), dict(min_p=-0.5), dict(top_k=-2), dict(temperature=float("nan"))):
        with pytest.raises(_lib.MirecError):
            E.sample_scores(s, u, **kw)
    with pytest.raises(_lib.MirecError):
        E.sample_scores(s, torch.rand(4, 1025, device=dev))


@gpu
def test_many_rows_streams_and_repeated_calls(dev):
    """More rows than workgroups of a small launch, on a stream of its own beside another call: same bits."""
    n, m = 5000, 700
    s, u = make(9, n, m, "f32", 2, dev)
    first = E.sample_scores(s, u, top_p=0.9, temperature=0.8)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(3):
                outs.append(E.sample_scores(s, u, top_p=0.9, temperature=0.8))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
    pick = torch.randperm(n, generator=torch.Generator().manual_seed(1))[:40].to(dev)
    check(s[pick], u[pick], first[0][pick], first[1][pick], T=0.8, top_p=0.9)


@gpu
@pytest.mark.parametrize("n,m,cut", [(3, 40000, dict(top_p=0.9)), (300, 100, dict(top_k=20, min_p=0.05)), (2, 27000, dict())])
def test_captured_calls_replay(dev, n, m, cut):
    """Two captured calls of the same inputs' buffers, replayed between eager calls, against eager results."""
    s, u = make(n + m, n, m, "f32", 3, dev)
    static_s, static_u = s.clone(), u.clone()
    E.sample_scores(static_s, static_u, **cut)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(E.sample_scores(static_s, static_u, **cut))
        graphs.append(gr)
    for rep in range(3):
        s2, u2 = make(1000 + rep, n, m, "f32", 3, dev)
        static_s.copy_(s2)
        static_u.copy_(u2)
        want = E.sample_scores(s2, u2, **cut)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


@gpu
def test_draw_frequencies(dev):
    """Draws of evenly spaced numbers: an item's count is its probability times their number, to one at each of its
    two borders."""
    m, draws = 37, 1024
    s, _ = make(4, 1, m, "f32", 1, dev, spread=1.0)
    u = ((torch.arange(draws, device=dev) + 0.5) / draws)[None].float()
    ids, _ = E.sample_scores(s, u)
    p = torch.softmax(s[0].double(), 0).cpu()
    count = torch.bincount(ids[0].long().cpu(), minlength=m)
    assert torch.all((count - p * draws).abs() <= 2)
