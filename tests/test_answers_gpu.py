"""dosma_amd.models.answers on the GPU against the 64-bit definitions (oracle/answers_oracle.py).

Tolerances (u = 2^-24, half a step of float32; all derived, per element).  A row of C categories is summed by at least 64 lanes
or, where one lane owns a row, one by one: at most ``n = min(C, C / 64 + 64) + 16`` roundings of the running sums, each relative,
as all terms of a sum have one sign.  exp2 of an argument x carries the rounding of x: 3 u |x| log2(e), and 2 u of its own.
  log_prob     d = (z - M) / T: 3 u |d|; ln s: n u + 3 u E|d| + 4 u (1 + |ln s|)                             -> _tol_lp
  entropy      ln s as above; t / s: relative n u + 8 u, and 3 u E[d^2]                                       -> _tol_h
  gradients    p: relative 4 u |log p| + error of ln s + 4 u; then half a step of the stored type             -> _tol_g
"""
import numpy as np
import pytest

from dosma_amd.models import answers as A
from oracle import answers_oracle as ao

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -126}  # (float16: half a subnormal step is 2^-25)
DTYPES = ["float32", "float16", "bfloat16"]
SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 13, 16, 17, 31, 32, 33, 63, 64, 65, 100, 117, 127, 128, 129, 255, 256, 257, 511, 1000, 1023, 1024,
         1025, 2048, 2049, 4097, 8191, 8200, 16385, 50021]


def torch_():
    import torch

    return torch


def _n(cats):
    return min(cats, cats / 64 + 64) + 16


def _moments(lp):
    """E|d|, E d^2 of a row, d = log p - max log p."""
    with np.errstate(all="ignore"):
        m = lp.max(-1, keepdims=True)
        d = np.where(np.isneginf(lp), 0.0, lp - np.where(np.isfinite(m), m, 0.0))
        p = np.exp(lp)
        return np.sum(p * np.abs(d), -1), np.sum(p * d * d, -1)


def _tol_ls(lp, ls):
    e1, _ = _moments(lp)
    return U * (_n(lp.shape[-1]) + 3 * e1 + 4 * (1 + np.abs(np.where(np.isfinite(ls), ls, 0.0))))


def _tol_lp(lp, ls, value):
    return _tol_ls(lp, ls) + U * 4 * (np.abs(np.where(np.isfinite(value), value, 0.0)) + np.abs(np.where(np.isfinite(ls), ls, 0.0)) + 1)


def _tol_h(lp, ls):
    e1, e2 = _moments(lp)
    return _tol_ls(lp, ls) + U * ((_n(lp.shape[-1]) + 8) * e1 + 4 * e2 + 4 * (np.abs(np.where(np.isfinite(ls), ls, 0.0)) + 1))


def _same(got, want, tol, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), what
    err = np.abs(got[fin] - want[fin])
    lim = np.nan_to_num(np.broadcast_to(tol, want.shape)[fin], nan=0.0)  # (the bound of a NaN row, where a 0 of an ignored label stands)
    if err.size:
        worst = np.argmax(err - lim)
        assert np.all(err <= lim), (what, "off by", err[worst], "allowed", lim[worst], "at", want[fin][worst])


def _scores(rng, rows, C, kind="plain"):
    z = rng.standard_normal((rows, C)) * 2.5
    if kind == "peaked":
        z[np.arange(rows), rng.integers(0, C, rows)] += 25.0
    elif kind == "masked":
        z[rng.uniform(size=z.shape) < 0.3] = -np.inf
    elif kind == "ties":
        z = np.round(z)
    elif kind == "far":
        z = z + 3000.0
    return z


def _tensor(z, dtype, layout, rng):
    """z (rows, C) -> (GPU tensor, dim, the values it holds as float64 (rows, C), function: result rows -> (rows, ...))."""
    torch = torch_()
    t = torch.from_numpy(z.astype(np.float32)).to(getattr(torch, dtype))
    if dtype == "float16":
        t = t.clamp(min=-65504.0).masked_fill(torch.from_numpy(np.isneginf(z)), float("-inf"))
    held = t.double().numpy()
    rows, C = z.shape
    t = t.cuda()
    if layout == "rows":
        return t, -1, held
    if layout == "padded":  # rows further apart than C, not aligned to anything
        wide = torch.full((rows, C + 5), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, 3:3 + C] = t
        return wide[:, 3:3 + C], 1, held
    if layout == "strided":  # every third class of a wider row
        wide = torch.full((rows, 3 * C), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, ::3] = t
        return wide[:, ::3], 1, held
    if layout == "planes":  # (C, rows): class planes
        return t.t().contiguous(), 0, held
    if layout == "nchw":  # (B, C, P) with the rows split over batch and pixel
        b = next(d for d in (3, 2, 5, 7, 1) if rows % d == 0)
        return t.reshape(b, rows // b, C).permute(0, 2, 1).contiguous(), 1, held
    raise AssertionError(layout)


def _rowshape(t, dim):
    s = list(t.shape)
    del s[dim]
    return s


def _host(t):
    return t.detach().double().cpu().numpy()


def _back(t, dim, C):
    """A gradient tensor in the logits' layout -> (rows, C) float64."""
    return np.moveaxis(_host(t), dim, -1).reshape(-1, C)


def _check_scores(z, dtype, layout, rng, T=1.0, top=0, bg=False, label_type="int32", ignore=-1, labels=None):
    torch = torch_()
    t, dim, held = _tensor(z, dtype, layout, rng)
    rows, C = z.shape
    cats = C + bg
    full = ao.with_background(held) if bg else held
    if labels is None:
        labels = rng.integers(0, cats, rows)
        labels[rng.uniform(size=rows) < 0.1] = ignore
        if cats < 250 and rows > 3:
            labels[3] = cats + 1  # out of range
    lab = torch.from_numpy(labels.astype(label_type)).reshape(_rowshape(t, dim)).cuda()
    r = A.label_scores(t, lab, dim=dim, top=top, norm=True, temperature=T, background=bg, ignore_label=ignore)
    want = ao.scores(full, T, labels, top, ignore)
    ls = want["norm"][:, 1]
    _same(_host(r.log_prob).reshape(-1), want["log_prob"], _tol_lp(want["lp"], ls, want["log_prob"]), "log_prob")
    _same(_host(r.entropy).reshape(-1), want["entropy"], _tol_h(want["lp"], ls), "entropy")
    _same(_host(r.norm).reshape(-1, 2)[:, 0], want["norm"][:, 0], 0.0, "row maximum")
    _same(_host(r.norm).reshape(-1, 2)[:, 1], ls, _tol_ls(want["lp"], ls), "ln s")
    if top:
        assert np.array_equal(_host(r.top_label).reshape(rows, top), want["top_label"]), "top_label"
        _same(_host(r.top_log_prob).reshape(rows, top), want["top_log_prob"],
              _tol_lp(want["lp"], ls, 0.0)[:, None] + 4 * U * np.abs(np.where(np.isfinite(want["top_log_prob"]), want["top_log_prob"], 0)),
              "top_log_prob")
    return t, dim, full, labels, lab, r


def _tol_g(want, lp, ls, scale, T, dtype, cats):
    """scale: sum of |coefficients| in front of p, per element."""
    p = np.exp(lp)
    tl = np.abs(np.where(np.isfinite(lp), lp, 0.0))
    rel = 8 * U * (tl + np.abs(np.where(np.isfinite(ls), ls, 0.0))[:, None] + 2) + _tol_ls(lp, ls)[:, None]
    return HALF[dtype] * np.abs(np.where(np.isfinite(want), want, 0)) * (1 + 8 * U) + TINY[dtype] + scale * p * rel / T + 8 * U * scale * p / T


def _check_scores_grad(z, dtype, layout, rng, T=1.0, bg=False, with_a=True, with_b=True, ignore=-1):
    torch = torch_()
    t, dim, full, labels, lab, r = _check_scores(z, dtype, layout, rng, T=T, bg=bg, ignore=ignore)
    rows, C = z.shape
    a = rng.standard_normal(rows).astype(np.float32) if with_a else None
    b = rng.standard_normal(rows).astype(np.float32) if with_b else None
    dev = lambda v: None if v is None else torch.from_numpy(v).reshape(_rowshape(t, dim)).cuda()  # noqa: E731
    g = A.label_scores_grad(t, lab if with_a else None, r.norm, grad_log_prob=dev(a), entropy=r.entropy if with_b else None,
                            grad_entropy=dev(b), dim=dim, temperature=T, background=bg, ignore_label=ignore)
    assert g.dtype == t.dtype and g.shape == t.shape
    want = ao.scores_grad(full, T, labels if with_a else None, None if a is None else a.astype(float), None if b is None else b.astype(float), ignore)
    lp, M, ls = ao.log_softmax(full, T)
    aa = 0.0 if a is None else np.abs(a)[:, None]
    H = np.abs(ao.scores(full, T)["entropy"])[:, None]
    tl = np.abs(np.where(np.isfinite(lp), lp, 0.0))
    # the entropy the kernel is given carries the forward's error
    bb = 0.0 if b is None else np.abs(b)[:, None] * (1 + H + tl)
    tol = _tol_g(want, lp, ls, aa + bb, T, dtype, full.shape[1])
    if b is not None:
        tol = tol + np.abs(b)[:, None] * np.exp(lp) * (_tol_h(lp, ls)[:, None] + 8 * U * tl) / T
    # the label's own element adds its coefficient and -a p: one rounding of their sum
    tol = tol + 4 * U * aa / T
    _same(_back(g, dim, C), want[:, 1:] if bg else want, (tol + np.zeros_like(lp))[:, 1:] if bg else tol, "grad")


def _teacher(rng, rows, cats, K, tail, T, v_dtype="float32"):
    """Entries of a perturbed teacher: distinct labels, some slots empty, one row all empty, one label twice."""
    torch = torch_()
    zt = rng.standard_normal((rows, cats)) * 3
    lp = ao.log_softmax(zt, T if tail else 1.0)[0]
    idx = np.argsort(-zt, axis=-1, kind="stable")[:, :K]
    if idx.shape[1] < K:
        idx = np.concatenate([idx, np.full((rows, K - idx.shape[1]), -1)], 1)
    val = np.where(idx >= 0, np.take_along_axis(lp if tail else zt, np.maximum(idx, 0), -1), 7.0)
    if K > 1 and rows > 2:
        idx[1, K - 1] = -1
        idx[2, :] = -1
        if rows > 4 and not tail:
            idx[4, 1] = idx[4, 0]
        if rows > 5:
            idx[5, 0] = cats + 3
    val = torch.from_numpy(val.astype(np.float32)).to(getattr(torch, v_dtype))
    return idx.astype(np.int64), val


def _check_distill(z, dtype, layout, rng, K, T=1.0, tail=False, bg=False, index_type="int32", v_dtype="float32"):
    torch = torch_()
    t, dim, held = _tensor(z, dtype, layout, rng)
    rows, C = z.shape
    cats = C + bg
    full = ao.with_background(held) if bg else held
    idx, val = _teacher(rng, rows, cats, K, tail, T, v_dtype)
    shp = _rowshape(t, dim) + [K]
    ti = torch.from_numpy(idx.astype(index_type)).reshape(shp).cuda()
    tv = val.reshape(shp).cuda()
    w = rng.uniform(-2, 2, rows).astype(np.float32)
    r = A.distill_loss(t, ti, tv, dim=dim, norm=True, temperature=T, tail=tail, background=bg)
    want = ao.distill(full, idx, val.double().numpy(), T, tail, w.astype(float))
    lp, M, ls = ao.log_softmax(full, T)
    base = _tol_ls(lp, ls)
    tlsum = np.zeros(rows)
    for k in range(K):
        ok = (idx[:, k] >= 0) & (idx[:, k] < cats)
        v = np.take_along_axis(lp, np.where(ok, idx[:, k], 0)[:, None], -1)[:, 0]
        q = want["q"][:, k]
        with np.errstate(all="ignore"):
            lq = np.where(q > 0, np.log(q), 0.0)
        # q: relative 8 u (1 + |log q|) + the sum over K; log q, log p: 4 u of their sizes and of the values they come from
        tlsum += np.where(q > 0, q * ((8 + K) * U * (1 + np.abs(lq)) * (1 + np.abs(lq - np.where(np.isfinite(v), v, 0))) +
                                      8 * U * (1 + np.abs(lq) + np.abs(np.where(np.isfinite(v), v, 0)) + np.abs(ls))) , 0.0)
    tol = base + tlsum + K * U * (1 + np.abs(np.where(np.isfinite(want["loss"]), want["loss"], 0)))
    if tail:
        # q_t = (1 - e^{v_max}) - others: K + 4 roundings of numbers <= 1; p_t: as ln s
        dr = (K + 8) * U
        lt = want["log_tail"]
        with np.errstate(all="ignore"):
            lr = np.where(want["rest"] > 0, np.log(want["rest"]), 0.0)
        ltf = np.where(np.isfinite(lt), lt, 0.0)
        tol = tol + dr * (2 + np.abs(lr) + np.abs(ltf)) + 8 * U * want["rest"] * (1 + np.abs(lr) + np.abs(ltf))
        tol = tol + 2 * want["rest"] * _tol_ls(lp, ls) + 4 * U * want["rest"] * np.abs(ltf)
        _same(np.where(np.isneginf(_host(r.log_tail).reshape(-1)), -1e9, _host(r.log_tail).reshape(-1)),
              np.where(np.isneginf(lt), -1e9, lt), 2 * base + 8 * U * (1 + np.abs(ltf)) * 2 + 3 * U * np.abs(ltf), "log_tail")
    else:
        assert r.log_tail is None
    _same(_host(r.loss).reshape(-1), want["loss"], tol, "loss")
    _same(_host(r.norm).reshape(-1, 2)[:, 1], ls, base, "ln s")
    g = A.distill_loss_grad(t, ti, tv, r.norm, grad_loss=torch.from_numpy(w).reshape(shp[:-1]).cuda(), log_tail=r.log_tail,
                            dim=dim, temperature=T, tail=tail, background=bg)
    assert g.dtype == t.dtype and g.shape == t.shape
    aw = np.abs(w)[:, None]
    tot = (want["q"].sum(-1) + want["rest"])[:, None]
    p = np.exp(lp)
    tolg = _tol_g(want["grad"], lp, ls, aw * (1 + tot), T, dtype, cats) + aw / T * (K + 16) * U * (p + 1.0 * (np.abs(want["grad"]) > 0) * _inside(idx, cats, want["q"]))
    if tail:
        with np.errstate(all="ignore"):
            share = np.where((want["rest"] > 0)[:, None] & (p > 0), np.exp(lp - want["log_tail"][:, None]), 0.0)
        tl = np.abs(np.where(np.isfinite(lp), lp, 0.0))
        ltf = np.abs(np.where(np.isfinite(want["log_tail"]), want["log_tail"], 0.0))[:, None]
        tolg = tolg + aw / T * share * (dr + want["rest"][:, None] * (8 * U * (2 + tl + ltf) + 3 * _tol_ls(lp, ls)[:, None] + 24 * U * (1 + ltf)))
    _same(_back(g, dim, C), want["grad"][:, 1:] if bg else want["grad"], (tolg + np.zeros_like(p))[:, 1:] if bg else tolg, "grad")


def _inside(idx, cats, q):
    """Sum of |q| (1 + |log q|) over the entries of a category: what rounding of q a member's gradient sees."""
    out = np.zeros((idx.shape[0], cats))
    with np.errstate(all="ignore"):
        s = np.where(q > 0, q * (1 + np.abs(np.log(q))), 0.0)
    for k in range(idx.shape[1]):
        ok = (idx[:, k] >= 0) & (idx[:, k] < cats)
        np.add.at(out, (np.flatnonzero(ok), idx[ok, k]), s[ok, k])
    return out


# ---- sizes, types, layouts ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", SIZES)
def test_label_scores_sizes(C):
    rng = np.random.default_rng(C)
    for dtype in DTYPES:
        for layout, rows in (("rows", 7), ("padded", 5)) if C > 300 else (("rows", 130), ("padded", 67), ("nchw", 66), ("strided", 9)):
            top = min(C, int(rng.choice([0, 1, 2, 5, 20, 64])))
            _check_scores(_scores(rng, rows, C, rng.choice(["plain", "peaked", "masked", "ties"])), dtype, layout, rng,
                          T=float(rng.choice([1.0, 0.7, 3.0])), top=top, bg=bool(C < 300 and rng.integers(2)))


@pytest.mark.parametrize("C", SIZES)
def test_label_scores_grad_sizes(C):
    rng = np.random.default_rng(1000 + C)
    for i, dtype in enumerate(DTYPES):
        for layout, rows in (("rows", 6), ("padded", 5)) if C > 300 else (("rows", 67), ("padded", 66), ("planes", 65), ("strided", 9)):
            _check_scores_grad(_scores(rng, rows, C, rng.choice(["plain", "peaked", "masked"])), dtype, layout, rng,
                               T=float(rng.choice([1.0, 0.7, 3.0])), bg=bool(C < 300 and rng.integers(2)),
                               with_a=i != 1, with_b=i != 2)


@pytest.mark.parametrize("C", SIZES)
def test_distill_sizes(C):
    rng = np.random.default_rng(2000 + C)
    for i, dtype in enumerate(DTYPES):
        for layout, rows in (("rows", 7), ("padded", 6)) if C > 300 else (("rows", 66), ("padded", 67), ("nchw", 66), ("strided", 9)):
            for tail in (False, True):
                K = int(rng.choice([1, 2, 3, 8, 17, 64]))
                _check_distill(_scores(rng, rows, C, rng.choice(["plain", "masked"])), dtype, layout, rng, K,
                               T=float(rng.choice([1.0, 0.7, 3.0])), tail=tail, bg=bool(C < 300 and rng.integers(2)),
                               index_type=("int32", "int64")[i % 2], v_dtype="float32" if tail else dtype)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 255, 256, 257, 1000, 70001])
@pytest.mark.parametrize("C", [4, 40, 3000])
def test_row_counts(rows, C):
    if rows * C > 10 ** 7:
        rows = 3001
    rng = np.random.default_rng(rows * 7 + C)
    _check_scores_grad(_scores(rng, rows, C), "float32", "rows", rng, bg=C == 4)
    _check_distill(_scores(rng, rows, C), "bfloat16", "rows", rng, 3, tail=True, bg=C == 4)
    _check_scores(_scores(rng, rows, C), "float16", "planes", rng, top=min(C, 6), bg=C == 4)


@pytest.mark.parametrize("top", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 63, 64])
def test_top_counts(top):
    rng = np.random.default_rng(top)
    for C in (64, 65, 200, 900, 1500, 20000):
        for kind in ("plain", "ties", "masked"):
            _check_scores(_scores(rng, 5, C, kind), "float32", "rows", rng, top=top, bg=C == 65)
    # the orders that a running list of the best finds hardest: rising, falling, all equal, the best at the very end
    for C in (70, 777, 9000):
        z = np.stack([np.arange(C) / C, -np.arange(C) / C, np.zeros(C), np.r_[np.zeros(C - 1), 1.0], np.r_[1.0, np.zeros(C - 1)]])
        for dtype in DTYPES:
            _check_scores(z, dtype, "rows", rng, top=top)
            _check_scores(z, dtype, "planes", rng, top=top)


@pytest.mark.parametrize("top", [5, 9, 19, 31, 33, 64])
def test_long_lists_of_the_best_in_planes(top):
    rng = np.random.default_rng(3000 + top)
    for i, dtype in enumerate(DTYPES):
        for rows in (63, 1000):
            _check_scores(_scores(rng, rows, 70, ("plain", "ties", "masked")[i]), dtype, ("planes", "nchw")[rows == 1000], rng, top=top)


@pytest.mark.parametrize("top", [5, 20, 33, 64])
@pytest.mark.parametrize("C", [60011, 131071])
def test_best_of_a_long_row_that_offers_few_categories(C, top):
    """A row cut into segments, most of which offer nothing or less than the list is long: their empty slots are no answers."""
    rng = np.random.default_rng(C + top)
    offers = {"a late one": [C - 1071], "three far apart": [1000, C // 2, C - 1071], "the end": range(C - C // 8, C), "nothing": [],
              "the beginning": range(0, 50), "two segments": range(8192 - 10, 8192 + 10), "one in 997": range(3, C, 997)}
    for i, (what, those) in enumerate(offers.items()):
        for rows in (1, 3):
            z = np.full((rows, C), -np.inf)
            z[:, list(those)] = rng.standard_normal((rows, len(those))) * 2.5
            if rows == 3:
                z[1] = np.where(np.isfinite(z[1]), 1.0, -np.inf)  # all alike: the lowest labels
            _check_scores(z, DTYPES[(i + rows) % 3], "rows", rng, top=top, bg=(i + rows // 3) % 2 == 1)


@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 33, 64])
def test_entry_counts(K):
    """Numbers of teacher's answers around which the kernels hold them elsewhere, in rows that end inside a vector and in whole ones."""
    rng = np.random.default_rng(4000 + K)
    for i, C in enumerate((5, 9, 16, 23, 32, 33, 60, 64, 117, 200, 400, 700, 1024, 1300)):
        for tail in (False, True):
            for layout, rows in (("rows", 70), ("planes", 67)) if C <= 200 else (("padded", 9),):
                _check_distill(_scores(rng, rows, C, ("plain", "masked")[i % 2]), DTYPES[(i + K) % 3], layout, rng, K, tail=tail,
                               bg=bool(i % 4 == 1), index_type=("int32", "int64")[(i + tail) % 2])


@pytest.mark.parametrize("C", [1100, 2051])
def test_many_rows_of_some_thousand_classes(C):
    """Enough rows for a wave each."""
    rng = np.random.default_rng(5000 + C)
    z = _scores(rng, 4099, C)
    _check_scores(z, "bfloat16", "rows", rng, top=5)
    for dtype in ("float32", "bfloat16"):
        _check_scores_grad(z, dtype, "rows", rng)
        _check_distill(z, dtype, "padded", rng, 5, tail=dtype == "float32")


@pytest.mark.parametrize("kind, ignore", [("int32", -1), ("uint8", 255), ("int16", -7), ("int64", -1), ("int64", 2)])
def test_label_types_and_the_ignored_label(kind, ignore):
    rng = np.random.default_rng(5)
    for C, layout in ((4, "rows"), (5, "nchw"), (300, "rows"), (2000, "rows")):
        z = _scores(rng, 60, C)
        labels = rng.integers(0, min(C, 200), 60)
        labels[::5] = ignore
        if kind == "int64":
            labels[1], labels[2] = 2 ** 32, -2 ** 40  # must not wrap into a category
        elif kind != "uint8":
            labels[1], labels[2] = -2, C
        _check_scores(z, "float32", layout, rng, labels=labels, label_type=kind, ignore=ignore)


# ---- special scores -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", [1, 3, 4, 24, 130, 1500, 9000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_special_rows(C, dtype):
    rng = np.random.default_rng(C)
    lowest = {"float32": -3.4e38, "float16": -65504.0, "bfloat16": -3.38e38}[dtype]
    z = _scores(rng, 12, C)
    z[0] = -np.inf                      # empty
    z[1] = lowest                       # the type's lowest value everywhere: uniform
    z[2, : C // 2] = lowest             # ... as a mask
    z[3, C // 2] = np.nan
    z[4, C - 1] = np.inf
    z[5] = -np.inf
    z[5, C // 3] = 2.0                  # one category offered
    z[6, :] = -lowest / 2               # far up, all equal
    z[7] = 0.0
    z[8, 0] = lowest
    for layout in ("rows", "planes", "padded"):
        for T in (1.0, 2.0):
            t, dim, full, labels, lab, r = _check_scores(z, dtype, layout, rng, T=T)
            _check_scores_grad(z, dtype, layout, rng, T=T)
            top = min(C, 5)
            r = A.label_scores(t, dim=dim, top=top, temperature=T)
            want = ao.scores(full, T, top=top)
            ok = ~np.isnan(want["norm"][:, 1])
            got = _host(r.top_label).reshape(12, top)
            assert np.array_equal(got[ok], want["top_label"][ok])
            assert np.isnan(_host(r.top_log_prob).reshape(12, top)[~ok]).all()
            assert r.log_prob is None
    # with the background an otherwise empty row has one category
    _check_scores(z, dtype, "rows", rng, bg=True)


def test_far_from_zero_and_extreme_temperatures():
    rng = np.random.default_rng(3)
    for C in (5, 200, 3000):
        for T in (0.01, 1.0, 50.0):
            _check_scores_grad(_scores(rng, 20, C, "far"), "float32", "rows", rng, T=T)
            _check_scores_grad(_scores(rng, 21, C, "far"), "float32", "planes", rng, T=T)


@pytest.mark.parametrize("C", [4, 90, 5000])
def test_distill_special(C):
    torch = torch_()
    rng = np.random.default_rng(C)
    z = _scores(rng, 8, C)
    z[0] = -np.inf                       # empty student: loss 0, gradient 0
    z[1, 1] = -np.inf                    # the student does not offer what the teacher says: inf
    z[2, 0] = np.nan
    z[3, 3:] = -np.inf                   # nothing outside the entries below
    idx = np.tile(np.array([1, 0, 2]), (8, 1))
    idx[4] = -1
    idx[5] = [2, 2, 2]
    val = np.log(np.tile(np.array([0.5, 0.3, 0.1]), (8, 1)))
    val[6, 0] = -np.inf                  # an entry of no weight
    val[7] = -np.inf
    for tail in (False, True):
        for layout in ("rows", "planes"):
            t, dim, held = _tensor(z, "float32", layout, rng)
            ti, tv = torch.from_numpy(idx).cuda(), torch.from_numpy(val.astype(np.float32)).cuda()
            r = A.distill_loss(t, ti, tv, dim=dim, norm=True, tail=tail)
            want = ao.distill(held, idx, val.astype(np.float32).astype(float), 1.0, tail, np.ones(8))
            got = _host(r.loss)
            assert np.isnan(got[2]) and got[0] == 0 and got[4] == 0 and np.isposinf(got[1])
            if tail:
                assert np.isposinf(got[3]) == np.isposinf(want["loss"][3])
            else:
                assert got[7] == 0  # (no weight anywhere: no teacher)
            ok = np.isfinite(want["loss"])
            assert np.allclose(got[ok], want["loss"][ok], rtol=0, atol=(C / 64 + 100) * U * 8)
            g = _back(A.distill_loss_grad(t, ti, tv, r.norm, grad_loss=torch.ones(8, device="cuda"), log_tail=r.log_tail, dim=dim,
                                          tail=tail), dim, C)
            assert np.all(g[0] == 0) and np.all(g[4] == 0) and np.isnan(g[2]).all()
            fin = np.isfinite(want["grad"]).all(-1)
            fin[2] = False
            assert np.allclose(g[fin], want["grad"][fin], rtol=0, atol=(C / 64 + 100) * U * 8)


def test_a_sure_student_keeps_its_small_tail():
    """The student leaves e^-150 outside the entries: the sum out there is taken relative to its own largest term."""
    torch = torch_()
    for C, layout in ((6, "rows"), (5, "planes"), (100, "rows"), (40, "planes"), (3000, "rows"), (200000, "rows"), (3000, "planes")):
        rng = np.random.default_rng(C)
        z = rng.standard_normal((3, C))
        z[:, 2] += 150.0
        t, dim, held = _tensor(z, "float32", layout, rng)
        idx = np.tile(np.array([[2]]), (3, 1))
        val = np.log(np.full((3, 1), 0.75)).astype(np.float32)
        ti, tv = torch.from_numpy(idx).cuda(), torch.from_numpy(val).cuda()
        r = A.distill_loss(t, ti, tv, dim=dim, norm=True, tail=True)
        want = ao.distill(held, idx, val.astype(float), 1.0, True, np.ones(3))
        # log p_t ~ -150: 3 u 150 of the distance to the maximum, and the sum of the outside
        tol = U * (3 * 160 + _n(C) + 100)
        assert np.all(np.abs(_host(r.log_tail) - want["log_tail"]) < tol)
        assert np.all(np.abs(_host(r.loss) - want["loss"]) < tol)
        g = _back(A.distill_loss_grad(t, ti, tv, r.norm, grad_loss=torch.ones(3, device="cuda"), log_tail=r.log_tail, dim=dim, tail=True), dim, C)
        assert np.all(np.abs(g - want["grad"]) < 2 * tol * (np.abs(want["grad"]) + 1e-3))


def test_a_sure_student_of_a_certain_teacher():
    """The teacher leaves nothing outside its entries: the loss does not look there, ``log_tail`` still says what the student does."""
    torch = torch_()
    for C, layout in ((6, "rows"), (5, "planes"), (33, "planes"), (64, "rows"), (100, "rows"), (117, "planes"), (3000, "rows"), (3000, "planes")):
        rng = np.random.default_rng(7 * C)
        z = rng.standard_normal((5, C))
        z[:, 2] += 150.0
        z[1, 4:] = -np.inf
        z[2, np.arange(C) != 2] = -np.inf  # nothing else is offered
        t, dim, held = _tensor(z, "float32", layout, rng)
        idx = np.tile(np.array([[2, 0]]), (5, 1))
        val = np.tile(np.array([[0.0, -200.0]], np.float32), (5, 1))
        ti, tv = torch.from_numpy(idx).cuda(), torch.from_numpy(val).cuda()
        r = A.distill_loss(t, ti, tv, dim=dim, norm=True, tail=True)
        want = ao.distill(held, idx, val.astype(float), 1.0, True, np.ones(5))
        assert np.all(want["rest"] == 0.0) and np.isneginf(want["log_tail"][2])
        fin = np.isfinite(want["log_tail"])
        got = _host(r.log_tail)
        assert np.all(np.isneginf(got[~fin]))
        assert np.all(np.abs(got[fin] - want["log_tail"][fin]) < U * (3 * 160 + _n(C) + 100))  # (as above)
    # every category an entry
    r = A.distill_loss(torch.zeros(4, 12, device="cuda"), torch.arange(12, device="cuda").repeat(4, 1), torch.full((4, 12), np.log(1 / 12), device="cuda"),
                       norm=True, tail=True)
    assert np.all(np.isneginf(_host(r.log_tail))) and np.all(np.abs(_host(r.loss)) < 100 * U)


def test_a_sure_teacher_keeps_its_small_rest():
    """1 - sum q of a teacher that is all but certain: taken as 1 - e^{v_max} without the cancellation."""
    torch = torch_()
    for C in (6, 400, 4000):
        z = np.zeros((1, C))
        v = np.array([[np.log1p(-3e-4), np.log(1e-4)]]).astype(np.float32)
        i = np.array([[1, 0]])
        r = A.distill_loss(torch.from_numpy(z.astype(np.float32)).cuda(), torch.from_numpy(i).cuda(), torch.from_numpy(v).cuda(), tail=True)
        want = ao.distill(z, i, v.astype(float), 1.0, True)
        # rest = 2e-4: its error 4 u 3e-4 times |log rest| ~ 8; the other terms as everywhere
        assert abs(float(r.loss[0]) - want["loss"][0]) < U * (C / 64 + 100) + 4 * U * (1 + abs(want["loss"][0]))


# ---- layouts, offsets, streams, graphs ------------------------------------------------------------------------------------
def test_broadcast_and_many_stride_inputs():
    torch = torch_()
    rng = np.random.default_rng(8)
    base = torch.from_numpy(rng.standard_normal((5, 1)).astype(np.float32)).cuda().requires_grad_()
    wide = base.expand(5, 40)            # one row for every pixel: class stride 1, row stride 0
    lab = torch.arange(40, device="cuda") % 5
    r = A.label_scores(wide, lab, dim=0)
    want = ao.scores(np.repeat(_host(base).T, 40, 0), 1.0, np.arange(40) % 5)
    _same(_host(r.log_prob), want["log_prob"], 100 * U)
    (g,) = torch.autograd.grad(r.log_prob.sum(), base)
    ref = ao.scores_grad(np.repeat(_host(base).T, 40, 0), 1.0, np.arange(40) % 5, np.ones(40)).sum(0)
    assert np.allclose(_host(g)[:, 0], ref, rtol=0, atol=40 * 20 * U)
    # rows that need three strides: one dense copy, the same answers
    t = torch.from_numpy(rng.standard_normal((6, 7, 8, 9)).astype(np.float32)).cuda()[::2, ::3, ::2]
    a, b = A.label_scores(t, top=3, norm=True), A.label_scores(t.contiguous(), top=3, norm=True)
    assert all(torch.equal(x, y) for x, y in zip(a[1:], b[1:]))
    # the same scores in every layout give the same labels and nearly the same numbers
    t = torch.from_numpy(rng.standard_normal((4, 10, 6, 6)).astype(np.float32)).cuda()
    c = A.label_scores(t, dim=1, top=4)
    d = A.label_scores(t.to(memory_format=torch.channels_last), dim=1, top=4)
    assert torch.equal(c.top_label, d.top_label) and torch.allclose(c.entropy, d.entropy, rtol=0, atol=100 * U)


def _check_gradients_of(t, dim, rng):
    """The gradients of both operators for a tensor as it lies, against the definitions on the values it holds."""
    torch = torch_()
    dim = dim % t.ndim
    C = t.shape[dim]
    z = _back(t, dim, C)
    rows, shp = z.shape[0], _rowshape(t, dim)
    dev = lambda v: torch.from_numpy(v).reshape(shp + list(v.shape[1:])).cuda()  # noqa: E731
    lab = rng.integers(0, C, rows)
    a, b = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    r = A.label_scores(t, dev(lab), dim=dim, norm=True)
    g = A.label_scores_grad(t, dev(lab), r.norm, grad_log_prob=dev(a), entropy=r.entropy, grad_entropy=dev(b), dim=dim)
    assert g.shape == t.shape and g.dtype == t.dtype
    lp, _, ls = ao.log_softmax(z, 1.0)
    name = str(t.dtype)[6:]
    want = ao.scores_grad(z, 1.0, lab, a.astype(float), b.astype(float))
    H, aa, bb = np.abs(ao.scores(z)["entropy"])[:, None], np.abs(a)[:, None], np.abs(b)[:, None]
    # (as _check_scores_grad)
    tol = _tol_g(want, lp, ls, aa + bb * (1 + H + np.abs(lp)), 1.0, name, C) + bb * np.exp(lp) * (_tol_h(lp, ls)[:, None] + 8 * U * np.abs(lp)) + 4 * U * aa
    _same(_back(g, dim, C), want, tol, ("label_scores_grad", tuple(t.shape), t.stride(), dim))
    K = min(3, C)
    idx, val = _teacher(rng, rows, C, K, False, 1.0)
    d = A.distill_loss(t, dev(idx), dev(val.numpy()), dim=dim, norm=True)
    g = A.distill_loss_grad(t, dev(idx), dev(val.numpy()), d.norm, grad_loss=dev(a), dim=dim)
    want = ao.distill(z, idx, val.double().numpy(), 1.0, False, a.astype(float))
    # (as _check_distill without the tail)
    tol = _tol_g(want["grad"], lp, ls, aa * 2, 1.0, name, C) + aa * (K + 16) * U * (np.exp(lp) + _inside(idx, C, want["q"]))
    _same(_back(g, dim, C), want["grad"], tol, ("distill_loss_grad", tuple(t.shape), t.stride(), dim))


@pytest.mark.parametrize("C", [4, 13, 100, 1500])
def test_gradients_of_crops_repeats_and_orders_of_the_axes(C):
    torch = torch_()
    rng = np.random.default_rng(C + 77)
    make = lambda s: torch.from_numpy(rng.standard_normal(s).astype(np.float32) * 2).cuda()  # noqa: E731
    for t, dim in ((make((2, 9, C))[:, :-1], -1), (make((2, 9, C))[:, 1:], -1), (make((3, 7, 6, C)).permute(0, 3, 1, 2)[:, :, 1:-1, 2:], 1),
                   (make((8, 7, 3, C))[2:-2, 1:-1], -1), (make((1, C, 1)).expand(3, C, 5), 1), (make((4, 1, C)).expand(4, 5, C), -1),
                   (make((5, C)).expand(3, 5, C), -1), (make((2, C, 8, 9))[:, :, ::2, ::3], 1), (make((C, 3, 8)).permute(1, 0, 2)[:, :, 1:6], 1)):
        _check_gradients_of(t, dim, rng)
        _check_gradients_of(t.to(torch.bfloat16) if t.is_contiguous() else t.bfloat16(), dim, rng)


def test_gradients_of_random_layouts():
    from test_answers import random_layout

    torch = torch_()
    rng = np.random.default_rng(99)
    for turn in range(60):
        nd = int(rng.integers(2, 5))
        shape = [int(v) for v in rng.integers(1, 7, nd)]
        dim = int(rng.integers(0, nd))
        shape[dim] = int(rng.choice([3, 8, 9, 40, 130]))
        t = random_layout(rng, tuple(shape), lambda s: torch.from_numpy(rng.standard_normal(s).astype(np.float32) * 2).cuda())
        _check_gradients_of(t, dim, rng)


def test_backward_through_views():
    """A next-token loss on ``logits[:, :-1]`` and a class prior repeated over the voxels."""
    torch = torch_()
    rng = np.random.default_rng(17)
    z = torch.from_numpy(rng.standard_normal((2, 6, 50)).astype(np.float32)).cuda().requires_grad_()
    tok = torch.from_numpy(rng.integers(0, 50, (2, 6))).cuda()
    (-A.label_scores(z[:, :-1], tok[:, 1:]).log_prob.sum()).backward()
    want = -ao.scores_grad(_host(z)[:, :-1].reshape(10, 50), 1.0, tok[:, 1:].cpu().numpy().reshape(-1), np.ones(10)).reshape(2, 5, 50)
    assert np.all(_host(z.grad)[:, -1] == 0) and np.all(np.abs(_host(z.grad)[:, :-1] - want) < 200 * U)
    bias = torch.from_numpy(rng.standard_normal(4).astype(np.float32)).cuda().requires_grad_()
    lab = torch.from_numpy(rng.integers(0, 4, (3, 70))).cuda()
    A.label_scores(bias.view(1, 4, 1).expand(3, 4, 70), lab, dim=1).log_prob.sum().backward()
    want = ao.scores_grad(np.tile(_host(bias), (210, 1)), 1.0, lab.cpu().numpy().reshape(-1), np.ones(210)).sum(0)
    assert np.all(np.abs(_host(bias.grad) - want) < 210 * 40 * U)  # (210 gradients, each within 40 u, summed in 32 bits)


def test_nothing_is_written_outside_the_results():
    """The scores lie inside a larger array; the gradient's neighbours and the rows behind the last one stay as they were."""
    torch = torch_()
    from dosma_amd import _lib as L

    rng = np.random.default_rng(11)
    for rows, C in ((3, 5), (65, 4), (9, 33), (5, 700), (3, 9001)):
        for dtype in DTYPES:
            td = getattr(torch, dtype)
            z = torch.from_numpy(rng.standard_normal((rows, C + 9)).astype(np.float32)).cuda().to(td)
            geo = L.Rows(rows, C, None, 0, C + 9, 1)
            guard = 64
            outs = {k: torch.full((rows * w + 2 * guard,), 12345, dtype=d, device="cuda")
                    for k, w, d in (("log_prob", 1, torch.float32), ("entropy", 1, torch.float32), ("norm", 2, torch.float32),
                                    ("top_log_prob", 3, torch.float32), ("top_label", 3, torch.int32))}
            grad = torch.full((rows * (C + 9) + 2 * guard,), 77.0, dtype=td, device="cuda")
            lab = torch.zeros(rows, dtype=torch.int32, device="cuda")
            p = {k: v.data_ptr() + guard * 4 for k, v in outs.items()}
            e = z.element_size()
            st = torch.cuda.current_stream().cuda_stream
            kw = dict(labels_ptr=lab.data_ptr(), l_dtype="int32", device=0, stream=st)
            L.label_scores(z.data_ptr() + 4 * e, dtype, geo, top=3, workspace=None, **p, **kw)
            one = torch.ones(rows, device="cuda")
            L.label_scores_grad(z.data_ptr() + 4 * e, dtype, geo, grad.data_ptr() + guard * e, geo, p["norm"], entropy=p["entropy"],
                                grad_log_prob=one.data_ptr(), grad_entropy=one.data_ptr(), **kw)
            torch.cuda.synchronize()
            for k, v in outs.items():
                assert bool((v[:guard] == 12345).all()) and bool((v[-guard:] == 12345).all()), k
                assert not bool((v[guard:-guard] == 12345).any()), k
            assert bool((grad[:guard] == 77).all()) and bool((grad[guard + rows * (C + 9) - 9:] == 77).all())
            inner = grad[guard:guard + rows * (C + 9)].view(rows, C + 9)
            assert bool((inner[:, C:] == 77).all()) and not bool((inner[:, :C] == 77).any())
            grad.fill_(77.0)
            idx = torch.zeros((rows, 2), dtype=torch.int32, device="cuda")
            val = torch.zeros((rows, 2), device="cuda")
            L.distill_grad(z.data_ptr() + 4 * e, dtype, geo, grad.data_ptr() + guard * e, geo, idx.data_ptr(), "int32",
                           val.data_ptr(), "float32", 2, p["norm"], one.data_ptr(), device=0, stream=st)
            torch.cuda.synchronize()
            inner = grad[guard:guard + rows * (C + 9)].view(rows, C + 9)
            assert bool((grad[:guard] == 77).all()) and bool((inner[:, C:] == 77).all()) and not bool((inner[:, :C] == 77).any())


def test_offsets_beyond_32_bits():
    """Scores behind the 2^31st element and the 2^32nd byte, in both layouts: the last rows against the 64-bit definitions."""
    torch = torch_()
    for layout, shape in (("rows", (2 ** 22 + 3, 520)), ("planes", (9, 2 ** 28 + 5)), ("long", (17, 2 ** 27 + 1))):
        z = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        z.normal_(generator=torch.Generator(device="cuda").manual_seed(3))
        dim = 0 if layout == "planes" else 1
        rows, C = (shape[1], shape[0]) if layout == "planes" else shape
        lab = torch.full((rows,), C - 1, dtype=torch.int32, device="cuda")
        r = A.label_scores(z, lab, dim=dim, top=2, norm=True)
        for n in (0, rows - 1):
            row = (z[:, n] if layout == "planes" else z[n]).double()
            m = row.max()
            ls = torch.log(torch.exp(row - m).sum())
            lp = row - m - ls
            tol = U * (_n(C) + 60)
            assert abs(float(r.log_prob[n]) - float(lp[C - 1])) < tol
            v, i = torch.sort(row, descending=True, stable=True)
            assert r.top_label[n].tolist() == i[:2].tolist()
            assert abs(float(r.entropy[n]) + float((lp.exp() * lp).sum())) < tol * 30
        g = A.label_scores_grad(z, lab, r.norm, grad_log_prob=torch.ones(rows, device="cuda"), dim=dim)
        row = (z[:, rows - 1] if layout == "planes" else z[rows - 1]).double()
        lp = torch.log_softmax(row, 0)
        got = (g[:, rows - 1] if layout == "planes" else g[rows - 1]).double()
        want = -lp.exp()
        want[C - 1] += 1.0
        assert float((got - want).abs().max()) < 2.0 ** -8 * float(want.abs().max()) + 1e-5
        idx = torch.tensor([[0, C - 1]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
        d = A.distill_loss(z, idx, torch.zeros(rows, 2, device="cuda"), dim=dim)
        ref = float(-0.6931471805599453 - 0.5 * (lp[0] + lp[C - 1]))
        assert abs(float(d.loss[rows - 1]) - ref) < U * (_n(C) + 100)
        del z, g, r, d, lab, idx
        torch.cuda.empty_cache()


def _step(z, lab, ti, tv, wts):
    """A training step's use of all four: likelihood of labels, an entropy term, a distillation term, one gradient."""
    torch = torch_()
    s = A.label_scores(z, lab, background=True, dim=1)
    d = A.distill_loss(z, ti, tv, tail=True, background=True, dim=1)
    total = (wts * (d.loss - s.log_prob - 0.1 * s.entropy)).sum()
    return total, torch.autograd.grad(total, z)[0]


def test_a_training_step_against_differences():
    torch = torch_()
    rng = np.random.default_rng(21)
    z = torch.from_numpy(rng.standard_normal((2, 4, 6, 5)).astype(np.float32)).cuda().requires_grad_()
    teacher = torch.from_numpy(rng.standard_normal((2, 4, 6, 5)).astype(np.float32)).cuda()
    t = A.label_scores(teacher, background=True, dim=1, top=2)
    lab = torch.from_numpy(rng.integers(0, 5, (2, 6, 5))).cuda()
    wts = torch.from_numpy(rng.uniform(0.5, 1.5, (2, 6, 5)).astype(np.float32)).cuda()
    total, g = _step(z, lab, t.top_label, t.top_log_prob, wts)
    assert g.shape == z.shape and g.stride() == z.stride()

    def exact(x):
        rows = ao.with_background(np.moveaxis(x, 1, -1).reshape(-1, 4))
        w = _host(wts).reshape(-1)
        s = ao.scores(rows, 1.0, lab.cpu().numpy().reshape(-1))
        d = ao.distill(rows, t.top_label.cpu().numpy().reshape(-1, 2), _host(t.top_log_prob).reshape(-1, 2), 1.0, True)
        return np.sum(w * (d["loss"] - s["log_prob"] - 0.1 * s["entropy"]))

    x = _host(z)
    assert abs(float(total) - exact(x)) < 60 * 100 * U * 4
    for i in [(0, 0, 0, 0), (1, 3, 5, 4), (0, 2, 3, 1), (1, 1, 2, 2)]:
        up, dn = x.copy(), x.copy()
        up[i] += 1e-5
        dn[i] -= 1e-5
        assert abs((exact(up) - exact(dn)) / 2e-5 - float(g[i])) < 1e-8 + 400 * U


def test_gradients_reach_only_what_asks_for_them():
    torch = torch_()
    z = torch.randn(6, 9, device="cuda", requires_grad=True)
    lab = torch.zeros(6, dtype=torch.int64, device="cuda")
    r = A.label_scores(z, lab, top=2)
    assert r.log_prob.requires_grad and r.entropy.requires_grad and not r.norm.requires_grad and not r.top_log_prob.requires_grad
    (g,) = torch.autograd.grad(r.log_prob.sum(), z)
    ref = ao.scores_grad(_host(z), 1.0, np.zeros(6, int), np.ones(6))
    assert np.allclose(_host(g), ref, rtol=0, atol=64 * U)
    (g,) = torch.autograd.grad(A.label_scores(z).entropy.sum(), z)
    assert np.allclose(_host(g), ao.scores_grad(_host(z), 1.0, b=np.ones(6)), rtol=0, atol=200 * U)
    with torch.no_grad():
        assert not A.label_scores(z, lab).log_prob.requires_grad
    # a non-dense incoming gradient
    (g,) = torch.autograd.grad(A.label_scores(z, lab).log_prob, z, torch.ones((), device="cuda").expand(6))
    assert np.allclose(_host(g), ref, rtol=0, atol=64 * U)


def test_another_stream_and_two_calls_at_once():
    torch = torch_()
    rng = np.random.default_rng(2)
    data = [torch.from_numpy(rng.standard_normal((3, 70001)).astype(np.float32)).cuda() for _ in range(4)]
    data += [torch.from_numpy(rng.standard_normal((20000, 6)).astype(np.float32)).cuda() for _ in range(4)]
    want = [A.label_scores(d, top=5, norm=True) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [None] * len(data)
    for _ in range(5):
        for i, d in enumerate(data):
            with torch.cuda.stream(streams[i % 4]):
                got[i] = A.label_scores(d, top=5, norm=True)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w[1:], g[1:]))


@pytest.mark.parametrize("shape, K", [((2, 60011), 20), ((3000, 5), 3), ((40, 700), 8)])
def test_captured_and_replayed(shape, K):
    """Forward and gradients of both operators in one graph, replayed with other inputs between eager work; two graphs that
    are replayed in turn do not disturb each other."""
    torch = torch_()
    rows, C = shape
    gen = torch.Generator(device="cuda").manual_seed(5)
    sets = []
    for _ in range(2):
        z = torch.empty(shape, device="cuda")
        lab = torch.zeros(rows, dtype=torch.int32, device="cuda")
        idx = torch.zeros((rows, K), dtype=torch.int32, device="cuda")
        val = torch.zeros((rows, K), device="cuda")
        one = torch.ones(rows, device="cuda")

        def work(z=z, lab=lab, idx=idx, val=val, one=one):
            s = A.label_scores(z, lab, top=min(K, C), norm=True)
            g = A.label_scores_grad(z, lab, s.norm, grad_log_prob=one, entropy=s.entropy, grad_entropy=one)
            d = A.distill_loss(z, idx, val, norm=True, tail=True)
            h = A.distill_loss_grad(z, idx, val, d.norm, grad_loss=one, log_tail=d.log_tail, tail=True)
            return [*s, g, d.loss, h]

        def fill(z=z, lab=lab, idx=idx, val=val):
            z.normal_(generator=gen)
            lab.copy_(torch.randint(0, C, (rows,), generator=gen, device="cuda"))
            t = A.label_scores(torch.randn(shape, generator=gen, device="cuda"), top=min(K, C))
            idx[:, :min(K, C)].copy_(t.top_label)
            val[:, :min(K, C)].copy_(t.top_log_prob)

        fill()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        sets.append((graph, out, work, fill))
    for turn in range(4):
        for graph, out, work, fill in (sets if turn % 2 else sets[::-1]):
            fill()
            want = work()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_training_step_captured_and_replayed():
    """Forward and backward by autograd in one graph, replayed with other inputs between eager steps."""
    torch = torch_()
    rng = np.random.default_rng(31)
    z = torch.empty((3, 12, 70), device="cuda", requires_grad=True)  # (B, C, P)
    lab = torch.empty((3, 70), dtype=torch.int64, device="cuda")
    t_lab = torch.empty((3, 70, 4), dtype=torch.int32, device="cuda")
    t_val = torch.empty((3, 70, 4), device="cuda")
    w = torch.ones((3, 70), device="cuda")

    def fill():
        with torch.no_grad():
            z.copy_(torch.from_numpy(rng.standard_normal((3, 12, 70)).astype(np.float32)))
            t = A.label_scores(torch.from_numpy(rng.standard_normal((3, 12, 70)).astype(np.float32)).cuda(), dim=1, top=4)
        lab.copy_(torch.from_numpy(rng.integers(0, 12, (3, 70))))
        t_lab.copy_(t.top_label)
        t_val.copy_(t.top_log_prob)

    def step():
        s = A.label_scores(z, lab, dim=1)
        d = A.distill_loss(z, t_lab, t_val, dim=1, tail=True)
        return torch.autograd.grad([d.loss, s.log_prob, s.entropy], z, [w, -w, w])[0], d.loss.detach()

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        fill()
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        del want


@pytest.mark.parametrize("layout", ["rows", "planes"])
def test_many_answers_captured_and_replayed(layout):
    """More answers than registers are given to: memory beyond a kernel's usual share is asked for while capturing."""
    torch = torch_()
    C, rows, K, dim = 20, 700, 64, -1 if layout == "rows" else 0
    z = torch.empty((rows, C) if layout == "rows" else (C, rows), device="cuda")
    idx = torch.full((rows, K), -1, dtype=torch.int32, device="cuda")
    val = torch.zeros((rows, K), device="cuda")
    one = torch.ones(rows, device="cuda")

    def fill():
        z.normal_()
        t = A.label_scores(torch.randn(rows, C, device="cuda"), top=C)
        idx[:, :C].copy_(t.top_label)
        idx[:, C:2 * C].copy_(t.top_label)  # every label twice
        val[:, :2 * C].copy_(torch.randn(rows, 2 * C, device="cuda"))

    def work():
        d = A.distill_loss(z, idx, val, dim=dim, norm=True)
        return d.loss, A.distill_loss_grad(z, idx, val, d.norm, grad_loss=one, dim=dim)

    fill()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for _ in range(3):
        fill()
        want = work()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    full = _host(z) if layout == "rows" else _host(z).T
    ref = ao.distill(full, idx.cpu().numpy(), _host(val), 1.0, False, np.ones(rows))
    # K + 16 roundings of terms whose weights sum to 1, and of log q, log p below 20
    assert np.all(np.abs(_host(out[0]) - ref["loss"]) < (K + 16) * U * 40)
    g = _host(out[1]) if layout == "rows" else _host(out[1]).T
    assert np.all(np.abs(g - ref["grad"]) < (K + 16) * U * 4)


def test_threads_with_few_and_many_answers():
    """Calls of one kernel from several threads at once, with different amounts of LDS: the limit is the kernel's, not the call's."""
    import threading

    torch = torch_()
    C, rows = 20, 900
    z = torch.randn(rows, C, device="cuda")
    sets = []
    for K in (9, 17, 33, 64):
        idx = torch.randint(0, C, (rows, K), device="cuda", dtype=torch.int32)
        val = torch.randn(rows, K, device="cuda")
        d = A.distill_loss(z, idx, val, norm=True)
        g = A.distill_loss_grad(z, idx, val, d.norm, grad_loss=torch.ones(rows, device="cuda"))
        sets.append((idx, val, d, g))
    torch.cuda.synchronize()
    failed = []

    def work(idx, val, d, g):
        try:
            one = torch.ones(rows, device="cuda")
            for _ in range(100):
                now = A.distill_loss(z, idx, val, norm=True)
                grad = A.distill_loss_grad(z, idx, val, now.norm, grad_loss=one)
            torch.cuda.synchronize()
            assert torch.equal(now.loss, d.loss) and torch.equal(grad, g)
        except Exception as e:  # (a thread's own exceptions reach nobody)
            failed.append(e)

    threads = [threading.Thread(target=work, args=s) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_the_same_bits_every_time():
    torch = torch_()
    for shape, bg in (((5, 100003), False), ((30000, 4), True), ((900, 900), False)):
        z = torch.randn(shape, device="cuda").bfloat16()
        idx = torch.randint(0, shape[1], (shape[0], 4), device="cuda", dtype=torch.int32)
        val = torch.zeros(shape[0], 4, device="cuda")
        first = None
        for _ in range(4):
            s = A.label_scores(z, top=3, norm=True, background=bg)
            d = A.distill_loss(z, idx, val, norm=True, background=bg)
            g = A.distill_loss_grad(z, idx, val, d.norm, grad_loss=torch.ones(shape[0], device="cuda"), background=bg)
            now = [*s[1:], d.loss, g]
            first = first or now
            assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_numpy_arrays():
    rng = np.random.default_rng(4)
    z = rng.standard_normal((3, 4, 6, 5)).astype(np.float32)
    lab = rng.integers(0, 5, (3, 6, 5)).astype(np.uint8)
    r = A.label_scores(z, lab, dim=1, background=True, top=2, norm=True, temperature=1.5)
    rows = ao.with_background(np.moveaxis(z, 1, -1).reshape(-1, 4).astype(float))
    want = ao.scores(rows, 1.5, lab.reshape(-1), 2)
    assert r.log_prob.shape == (3, 6, 5) and r.top_label.shape == (3, 6, 5, 2) and r.top_label.dtype == np.int32
    _same(r.log_prob.reshape(-1), want["log_prob"], 100 * U)
    assert np.array_equal(r.top_label.reshape(-1, 2), want["top_label"])
    a = np.ones((3, 6, 5), np.float32)
    g = A.label_scores_grad(z, lab, r.norm, grad_log_prob=a, entropy=r.entropy, grad_entropy=a, dim=1, background=True, temperature=1.5)
    ref = ao.scores_grad(rows, 1.5, lab.reshape(-1), np.ones(90), np.ones(90))[:, 1:]
    assert g.shape == z.shape and np.allclose(np.moveaxis(g, 1, -1).reshape(-1, 4), ref, rtol=0, atol=200 * U)
    d = A.distill_loss(z, r.top_label, r.top_log_prob, dim=1, norm=True, background=True, tail=True, temperature=1.5)
    # a network against its own answers: zero up to the rounding of the stored log probabilities
    assert np.abs(d.loss).max() < 100 * U
    h = A.distill_loss_grad(z, r.top_label, r.top_log_prob, d.norm, grad_loss=a, log_tail=d.log_tail, dim=1, tail=True,
                            background=True, temperature=1.5)
    assert h.shape == z.shape and np.abs(h).max() < 200 * U  # ... and its gradient
    half = A.label_scores(z.astype(np.float16), dim=1)
    assert half.entropy.dtype == np.float32
    empty = A.label_scores(np.zeros((0, 4), np.float32), np.zeros(0, np.int32), top=2)
    assert empty.log_prob.shape == (0,) and empty.top_label.shape == (0, 2)


def test_one_row_without_an_axis():
    """(C,) scores: the row's arguments and results have no axis, as tensors and as arrays."""
    torch = torch_()
    rng = np.random.default_rng(6)
    for C in (4, 700):
        z = rng.standard_normal(C).astype(np.float32)
        idx, val = np.array([1, 0], np.int32), np.zeros(2, np.float32)
        want, wd = ao.scores(z[None].astype(float), 1.0, np.array([2]), 3), ao.distill(z[None].astype(float), idx[None], val[None], w=np.ones(1))
        g_want = ao.scores_grad(z[None].astype(float), 1.0, np.array([2]), np.ones(1))[0]
        one = np.float32(1.0)
        for conv in (lambda v: v, lambda v: torch.from_numpy(np.asarray(v)).cuda()):
            back = lambda v: v if isinstance(v, np.ndarray) else _host(v)  # noqa: E731
            r = A.label_scores(conv(z), conv(np.int64(2)), top=3, norm=True)
            assert r.log_prob.shape == () and r.entropy.shape == () and r.norm.shape == (2,) and r.top_label.shape == (3,)
            _same(back(r.log_prob), want["log_prob"][0], 100 * U)
            assert np.array_equal(back(r.top_label), want["top_label"][0])
            g = A.label_scores_grad(conv(z), conv(np.int64(2)), r.norm, grad_log_prob=conv(one))
            _same(back(g), g_want, 100 * U)
            d = A.distill_loss(conv(z), conv(idx), conv(val), norm=True)
            assert d.loss.shape == ()
            _same(back(d.loss), wd["loss"][0], 100 * U)
            _same(back(A.distill_loss_grad(conv(z), conv(idx), conv(val), d.norm, grad_loss=conv(one))), wd["grad"][0], 100 * U)


def test_empty_tensors():
    torch = torch_()
    z = torch.zeros((0, 4), device="cuda", requires_grad=True)
    r = A.label_scores(z, torch.zeros(0, dtype=torch.int32, device="cuda"), top=1)
    assert r.entropy.shape == (0,) and r.top_label.shape == (0, 1)
    (g,) = torch.autograd.grad(r.entropy.sum(), z)
    assert g.shape == (0, 4)
    d = A.distill_loss(z, torch.zeros((0, 2), dtype=torch.int32, device="cuda"), torch.zeros((0, 2), device="cuda"))
    assert d.loss.shape == (0,)


def test_views_whose_memory_has_the_other_sign():
    """The imaginary part of a conjugate is a view that torch negates when it is read."""
    torch = torch_()
    neg = lambda *s: torch.view_as_complex(torch.randn(*s, 2, device="cuda")).conj().imag  # noqa: E731
    for shape, dim in (((5, 6), -1), ((2, 40, 3), 1), ((3, 2000), -1)):
        z = neg(*shape)
        plain = z.resolve_neg().contiguous()
        assert z.is_neg() and not plain.is_neg()
        d = dim % len(shape)
        rows = list(shape[:d] + shape[d + 1:])
        lab = torch.zeros(rows, dtype=torch.int64, device="cuda")
        a, b = A.label_scores(z, lab, dim=dim, top=2, norm=True), A.label_scores(plain, lab, dim=dim, top=2, norm=True)
        assert torch.equal(a.top_label, b.top_label) and torch.allclose(a.log_prob, b.log_prob, rtol=0, atol=100 * U)
        w = neg(*rows)
        kw = dict(entropy=b.entropy, dim=dim)
        g = A.label_scores_grad(z, lab, b.norm, grad_log_prob=w, grad_entropy=w, **kw)
        h = A.label_scores_grad(plain, lab, b.norm, grad_log_prob=w.resolve_neg(), grad_entropy=w.resolve_neg(), **kw)
        assert not g.is_neg() and torch.allclose(g, h, rtol=0, atol=100 * U)
        idx, val = torch.zeros(rows + [2], dtype=torch.int32, device="cuda"), neg(*rows, 2)
        idx[..., 1] = 1
        assert torch.allclose(A.distill_loss(z, idx, val, dim=dim).loss, A.distill_loss(plain, idx, val.resolve_neg(), dim=dim).loss,
                              rtol=0, atol=200 * U)
        c = torch.view_as_complex(torch.randn(*shape, 2, device="cuda")).requires_grad_()
        A.label_scores(c.conj().imag, lab, dim=dim).entropy.sum().backward()
        x = (-c.detach().imag).contiguous().requires_grad_()
        A.label_scores(x, lab, dim=dim).entropy.sum().backward()
        assert torch.allclose(c.grad.imag, -x.grad, rtol=0, atol=100 * U)


def test_forward_mode_is_refused():
    """A dual tensor does not require gradients: without the refusal its tangent would be lost without a word."""
    torch = torch_()
    fw = torch.autograd.forward_ad
    z, one = torch.randn(3, 4, device="cuda"), torch.ones(3, device="cuda")
    lab, idx, val = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, device="cuda")
    s, d = A.label_scores(z, lab, norm=True), A.distill_loss(z, idx, val, norm=True)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: A.label_scores(dual(z), lab), lambda: A.label_scores(dual(z)), lambda: A.distill_loss(dual(z), idx, val),
                     lambda: A.distill_loss(z, idx, dual(val)), lambda: A.label_scores_grad(dual(z), lab, s.norm, grad_log_prob=one),
                     lambda: A.label_scores_grad(z, lab, dual(s.norm), grad_log_prob=one),
                     lambda: A.label_scores_grad(z, lab, s.norm, grad_log_prob=dual(one)),
                     lambda: A.distill_loss_grad(z, idx, val, d.norm, grad_loss=dual(one))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        # a primal inside the level is an ordinary tensor
        assert torch.equal(A.label_scores(z, lab).log_prob, s.log_prob)


def test_refusals_on_tensors():
    torch = torch_()
    z = torch.zeros(3, 4, device="cuda")
    i2 = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for call, says in (
            (lambda: A.label_scores(z.double()), "float32, float16 or bfloat16"),
            (lambda: A.label_scores(z, torch.zeros(3, dtype=torch.int32)), "is on cpu"),
            (lambda: A.label_scores(z, np.zeros(3, np.int32)), "tensor like the logits"),
            (lambda: A.label_scores(z, torch.zeros(3, device="cuda")), "labels must be one of"),
            (lambda: A.label_scores(z, top=5), "categories"),
            (lambda: A.label_scores(z, temperature=0.0), "temperature"),
            (lambda: A.distill_loss(z, i2, torch.zeros(3, 2, device="cuda").half(), tail=True), "float32 log"),
            (lambda: A.distill_loss(z, i2[:, :0], torch.zeros(3, 0, device="cuda")), "entries"),
            (lambda: A.label_scores_grad(z, None, torch.zeros(3, 2, device="cuda"), grad_log_prob=torch.zeros(3, device="cuda")), "needs labels"),
            (lambda: A.label_scores_grad(z, None, torch.zeros(3, 2, device="cuda"), grad_entropy=torch.zeros(3, device="cuda")), "needs entropy"),
            (lambda: A.distill_loss_grad(z, i2, torch.zeros(3, 2, device="cuda"), torch.zeros(3, 2, device="cuda"),
                                         grad_loss=torch.zeros(3, device="cuda"), tail=True), "log_tail")):
        with pytest.raises(ValueError, match=says):
            call()
