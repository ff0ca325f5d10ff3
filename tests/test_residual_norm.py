"""snb200_residual_norm_fwd / _bwd against float64.

Tolerances, with u = 2^-24 and D the row's width.  A sum over a row goes through at most L = D / 256 + 40 additions on its
longest path (a thread adds every 256th element, or fewer; the rest is a tree), so it is off by at most L u times the sum
of the magnitudes.
  r:     four rounded operations on its two terms and those of u behind a norm: 4 u (|a x| + |b gate u|) + |b gate| E(u).
  E(y):  of a norm of t with statistics m, s: m is off by (L + 1) u mean|t|, s by (L / 2 + 4) u of itself plus the effect
         of m's error, which is smaller; so |gamma| (s (2 u (|t| + |m|) + (L + 1) u mean|t|) + (L / 2 + 8) u |xhat|) + 2 u |y|.
  dR:    s ((L + 8) u (|g| + mean|g| + |xhat| mean|g xhat|)) + 4 u |dR|, from the statistics given.
  column sums: at most `rows` additions of terms that are off by what dR and xhat are: (rows + 8) u sum|term| + sum E(term).
         The gate's gradient may be taken as post_gamma sum(b dR hhat) + post_beta sum(b dR): its terms count as two each.
y is checked on the r that the call returned, the backward pass on the statistics that it is given, so that each bound
covers one call.  Bounds are multiplied by 1.1 for higher orders."""
import ctypes
import itertools

import numpy as np
import pytest

from oracle import sharpnet_oracle as orc
from tests.guarded import Guarded, pointer

U = 2.0 ** -24
KINDS = {"none": 0, "layer": 1, "rms": 2}
NAMES = ("gamma", "beta", "post_gamma", "post_beta", "gate")
EPS = 1e-5


def _desc(rows, dim, norm, post, gate_rows, a, b, eps=EPS):
    from sharpnet_b200 import _capi
    return _capi.NormDesc(rows, dim, KINDS[norm], KINDS[post], gate_rows, a, b, eps)


def _path(dim):
    return dim / 256 + 40


def _norm_error(t, stats, gamma, y, dim):
    L, s, m = _path(dim), stats[:, 1:], stats[:, :1]
    xhat = np.abs((t - m) * s)
    e = s * (2 * U * (np.abs(t) + np.abs(m)) + (L + 1) * U * np.abs(t).mean(1, keepdims=True)) + (L / 2 + 8) * U * xhat
    return (1 if gamma is None else np.abs(gamma)) * e + 2 * U * np.abs(y)


# -------------------------------------------------------------------------------------------- no device needed
@pytest.mark.parametrize("norm, post, gate_rows", list(itertools.product(("none", "layer", "rms"), ("none", "layer", "rms"), (0, 1, 2, 6))))
def test_oracle_gradient_by_differences(norm, post, gate_rows):
    rng = np.random.default_rng(1)
    rows, dim, a, b = 6, 5, 0.7, 1.3
    x, h, dy, dr = (rng.normal(size=(rows, dim)) for _ in range(4))
    p = {"gamma": rng.normal(size=dim), "beta": rng.normal(size=dim), "post_gamma": rng.normal(size=dim), "post_beta": rng.normal(size=dim),
         "gate": rng.normal(size=(max(1, gate_rows), dim))}
    used = [n for n in NAMES if (norm != "none" or n not in ("gamma", "beta")) and (post != "none" or "post" not in n) and (gate_rows or n != "gate")]

    def loss():
        r = orc.residual_norm_sum(x, h, None if post == "none" else orc.norm_statistics(h, post, EPS), p, gate_rows, a, b)
        total = (r * dr).sum()
        if norm != "none":
            total += (orc.norm_apply(r, orc.norm_statistics(r, norm, EPS), p["gamma"], p["beta"]) * dy).sum()
        return total

    r = orc.residual_norm_sum(x, h, None if post == "none" else orc.norm_statistics(h, post, EPS), p, gate_rows, a, b)
    got = orc.residual_norm_backward(r, h, dy, dr, None if norm == "none" else orc.norm_statistics(r, norm, EPS),
                                     None if post == "none" else orc.norm_statistics(h, post, EPS), p, norm, post, gate_rows, a, b)
    for name, t in [("dx", x), ("dblock", h)] + [(n, p[n]) for n in used]:
        for i in np.ndindex(t.shape):
            old, e = t[i], 1e-5
            t[i] = old + e
            up = loss()
            t[i] = old - e
            down = loss()
            t[i] = old
            # central differences: truncation ~ e^2, cancellation ~ 1e-15 / e, against values of order 1 to 100
            assert abs(got[name].reshape(t.shape)[i] - (up - down) / (2 * e)) < 1e-6, (name, i)


def test_scratch_size(built_library):
    from sharpnet_b200 import _capi
    size = _capi.load().snb200_residual_norm_scratch_floats
    assert size(None) == -1 and size(_desc(-1, 4, "layer", "none", 0, 1, 1)) == -1 and size(_desc(1, -4, "layer", "none", 0, 1, 1)) == -1
    assert size(_desc(0, 4, "layer", "none", 0, 1, 1)) >= 0
    assert size(_desc(1 << 40, 16384, "layer", "rms", 1, 1, 1)) > 0
    assert size(_desc(10, 8, "layer", "none", 0, 1, 1)) >= 2 * 8


def test_null_handle_is_refused(built_library):
    from sharpnet_b200 import _capi
    lib = _capi.load()
    assert lib.snb200_residual_norm_fwd(None, _desc(1, 1, "rms", "none", 0, 1, 1), _capi.NormParams(), *[None] * 6) == 1
    assert lib.snb200_residual_norm_bwd(None, _desc(1, 1, "rms", "none", 0, 1, 1), _capi.NormParams(), *[None] * 9, None) == 1


# -------------------------------------------------------------------------------------------- on the device
def _inputs(rows, dim, norm, post, gate_rows, affine, seed):
    rng = np.random.default_rng(seed)
    f = lambda *s, m=0.0, k=1.0: (rng.normal(size=s) * k + m).astype(np.float32)  # noqa: E731
    p = {"gamma": f(dim, m=1, k=0.3) if affine and norm != "none" else None, "beta": f(dim) if affine and norm != "none" else None,
         "post_gamma": f(dim, m=1, k=0.3) if affine and post != "none" else None, "post_beta": f(dim) if affine and post != "none" else None,
         "gate": f(gate_rows, dim, m=0.5) if gate_rows else None}
    return p, f(rows, dim, m=0.7, k=2), f(rows, dim, m=-0.4), f(rows, dim, k=0.1), f(rows, dim, k=0.1)


def _params(p, w, shift=0):
    from sharpnet_b200 import _capi
    up = {n: None if p[n] is None else Guarded(p[n], w.device, shift) for n in NAMES}
    return up, _capi.NormParams(*[pointer(up[n]) for n in NAMES])


def _run_forward(w, rows, dim, norm, post, gate_rows, a, b, p, x, h, shift=0, in_place=False, want_r=True, want_stats=True):
    up, params = _params(p, w, shift)
    X, H = Guarded(x, w.device, shift), None if h is None else Guarded(h, w.device, shift)
    R = X if in_place else Guarded(np.zeros_like(x), w.device, shift) if want_r else None
    Y = Guarded(np.zeros_like(x), w.device, shift) if norm != "none" else None
    S = Guarded(np.zeros((rows, 2), np.float32), w.device) if want_stats and norm != "none" else None
    P = Guarded(np.zeros((rows, 2), np.float32), w.device) if want_stats and post != "none" else None
    st = w.lib.snb200_residual_norm_fwd(w.handle, _desc(rows, dim, norm, post, gate_rows, a, b), params, X.pointer, pointer(H), pointer(R),
                                        pointer(Y), pointer(S), pointer(P))
    assert st == 0, w.lib.snb200_last_error_string(w.handle)
    return [None if t is None else t.numpy() for t in (R, Y, S, P)]


def _check_forward(w, rows, dim, norm, post, gate_rows, a, b, affine=True, block=True, shift=0, in_place=False, want_r=True, want_stats=True):
    p, x, h, _, _ = _inputs(rows, dim, norm, post, gate_rows, affine, rows + dim)
    h = h if block else None
    a, b = float(np.float32(a)), float(np.float32(b))
    r, y, s, ps = _run_forward(w, rows, dim, norm, post, gate_rows, a, b, p, x, h, shift, in_place, want_r, want_stats)
    hstats = orc.norm_statistics(h, post, EPS) if post != "none" else None
    if r is not None:
        want = orc.residual_norm_sum(x, h, hstats, p, gate_rows, a, b)
        bound = 4 * U * np.abs(a * x.astype(np.float64))
        if block:
            g = np.abs(b * (np.repeat(p["gate"], rows // gate_rows, 0).astype(np.float64) if gate_rows else 1.0))
            u = h.astype(np.float64) if post == "none" else orc.norm_apply(h, hstats, p["post_gamma"], p["post_beta"])
            e = 0 if post == "none" else _norm_error(h.astype(np.float64), hstats, p["post_gamma"], np.abs(u) + (0 if p["post_beta"] is None else np.abs(p["post_beta"])), dim)
            bound = bound + 4 * U * g * np.abs(u) + g * e
        assert (np.abs(r - want) <= 1.1 * bound).all(), float((np.abs(r - want) / bound).max())
    else:
        r = (np.float32(a) * x).astype(np.float32)
    if ps is not None:
        np.testing.assert_allclose(ps[:, 1], hstats[:, 1], rtol=1.1 * (_path(dim) / 2 + 8) * U)
        assert (np.abs(ps[:, 0] - hstats[:, 0]) <= 1.1 * (_path(dim) + 1) * U * np.abs(h).mean(1)).all()
    if norm == "none":
        return
    stats = orc.norm_statistics(r, norm, EPS)
    want = orc.norm_apply(r, stats, p["gamma"], p["beta"])
    bound = _norm_error(r.astype(np.float64), stats, p["gamma"], np.abs(want) + (0 if p["beta"] is None else np.abs(p["beta"])), dim)
    assert (np.abs(y - want) <= 1.1 * bound).all(), float((np.abs(y - want) / bound).max())
    if s is not None:
        # rstd: off by L / 2 + 8 of u, and by the error of m against the deviation, at most (m's error * rstd)^2 / 2
        np.testing.assert_allclose(s[:, 1], stats[:, 1], rtol=1.1 * (_path(dim) / 2 + 8) * U)
        assert (np.abs(s[:, 0] - stats[:, 0]) <= 1.1 * (_path(dim) + 1) * U * np.abs(r).mean(1)).all()


COMBINATIONS = [("layer", "none", 0), ("rms", "none", 0), ("layer", "rms", 1), ("rms", "layer", 1), ("none", "rms", 1), ("none", "none", 1),
                ("rms", "rms", "groups"), ("layer", "layer", "rows"), ("none", "none", 0)]
SHAPES = [(1, 1), (1, 4), (3, 7), (6, 64), (10, 128), (33, 100), (7, 333), (600, 48), (30, 512), (12, 516), (301, 777), (9, 1024),
          (5, 2048), (310, 2050), (4, 4096), (3, 5001), (2, 8192), (2, 8196), (3, 12288), (2, 20001), (6, 16384)]


def _groups(gate, rows):
    if gate == "rows":
        return rows
    if gate == "groups":
        return next(k for k in (7, 6, 5, 4, 3, 2, 1) if rows % k == 0)
    return gate


@pytest.mark.gpu
@pytest.mark.parametrize("rows, dim", SHAPES)
def test_forward(wrapper, rows, dim):
    for i, (norm, post, gate) in enumerate(COMBINATIONS):
        _check_forward(wrapper, rows, dim, norm, post, _groups(gate, rows), 0.8, 1.25, affine=i % 3 != 2, shift=i % 2, in_place=i % 4 == 1)
    _check_forward(wrapper, rows, dim, "layer", "none", 0, 1.0, 1.0, block=False, want_r=False)
    _check_forward(wrapper, rows, dim, "rms", "none", 0, 1.5, 1.0, block=False, want_r=False, want_stats=False)
    _check_forward(wrapper, rows, dim, "rms", "none", 0, 1.5, 1.0, block=False, shift=3)
    wrapper.check_device_status()


def _run_backward(w, rows, dim, norm, post, gate_rows, a, b, p, r, h, dy, dr, stats, hstats, shift=0, in_place=False, wanted=None):
    import torch
    from sharpnet_b200 import _capi
    up, params = _params(p, w, shift)
    guard = lambda t, s=shift: None if t is None else Guarded(t, w.device, s)  # noqa: E731
    R, H, DY, DR, S, P = guard(r), guard(h), guard(dy), guard(dr), guard(stats, shift % 2), guard(hstats, shift % 2)
    wanted = ("dx", "dblock") + NAMES if wanted is None else wanted
    DX = (DR if in_place else guard(np.ones_like(r))) if "dx" in wanted else None
    DH = guard(np.ones_like(r)) if "dblock" in wanted else None
    G = {n: guard(np.ones_like(p[n])) if p[n] is not None and n in wanted else None for n in NAMES}
    desc = _desc(rows, dim, norm, post, gate_rows, a, b)
    need = w.lib.snb200_residual_norm_scratch_floats(desc)
    scratch = torch.full((need + 256,), 77.0, device=w.device)                       # never cleared by the caller
    st = w.lib.snb200_residual_norm_bwd(w.handle, desc, params, pointer(R), pointer(H), pointer(DY), pointer(DR), pointer(S), pointer(P),
                                        scratch.data_ptr(), pointer(DX), pointer(DH), _capi.NormParams(*[pointer(G[n]) for n in NAMES]))
    assert st == 0, w.lib.snb200_last_error_string(w.handle)
    assert bool((scratch[need:] == 77).all()), "written behind the scratch memory"
    out = {"dx": DX, "dblock": DH, **G}
    return {k: t.numpy() for k, t in out.items() if t is not None}


def _check_backward(w, rows, dim, norm, post, gate_rows, a, b, affine=True, block=True, shift=0, in_place=False, with_dr=True, wanted=None):
    p, r, h, dy, dr = _inputs(rows, dim, norm, post, gate_rows, affine, rows * 3 + dim)
    h = h if block else None
    dr = dr if with_dr or norm == "none" else None
    dy = dy if norm != "none" else None
    a, b = float(np.float32(a)), float(np.float32(b))
    stats = orc.norm_statistics(r, norm, EPS).astype(np.float32) if norm != "none" else None
    hstats = orc.norm_statistics(h, post, EPS).astype(np.float32) if post != "none" else None
    got = _run_backward(w, rows, dim, norm, post, gate_rows, a, b, p, r, h, dy, dr, stats, hstats, shift, in_place, wanted)
    d64 = {k: None if v is None else v.astype(np.float64) for k, v in p.items()}
    want = orc.residual_norm_backward(r, h, dy, dr, None if stats is None else stats.astype(np.float64),
                                      None if hstats is None else hstats.astype(np.float64), d64, norm, post, gate_rows, a, b)
    # how far dR and what follows from it may be off
    L, e = _path(dim), np.zeros((rows, dim))
    dR = want["dx"] / a
    magnitude = np.abs(dR) + (0 if dr is None else np.abs(dr))
    terms = {}

    def through(g, xhat, s, e_g):
        """Error of s (g - mean g - xhat mean(g xhat)) for g off by e_g: by the errors that come in and by its own arithmetic."""
        ag = np.abs(g)
        own = (L + 8) * U * (ag + ag.mean(1, keepdims=True) + np.abs(xhat) * (ag * np.abs(xhat)).mean(1, keepdims=True))
        # xhat itself is off by 2 u (|t| + |m|) s, which is at most 2 u (|xhat| + 2 |m| s); it enters times mean(g xhat) and in the mean
        return s * (own + e_g + e_g.mean(1, keepdims=True) + np.abs(xhat) * (e_g * np.abs(xhat)).mean(1, keepdims=True))

    def xhat_error(t, st):
        return 2 * U * (np.abs(t) + np.abs(st[:, :1])) * st[:, 1:]

    if norm != "none":
        xhat = orc.norm_apply(r, stats.astype(np.float64), None, None)
        ex = xhat_error(r.astype(np.float64), stats.astype(np.float64))
        g = dy.astype(np.float64) * (1 if p["gamma"] is None else d64["gamma"])
        e = through(g, xhat, stats[:, 1:].astype(np.float64), U * np.abs(g))
        mean_gx = np.abs((g * xhat).mean(1, keepdims=True))
        e = e + stats[:, 1:] * (ex * mean_gx + np.abs(xhat) * (np.abs(g) * ex).mean(1, keepdims=True)) + 4 * U * magnitude
        terms["gamma"] = (dy * xhat, np.abs(dy) * ex)
        terms["beta"] = (dy, 0 * e)
    bounds = {"dx": abs(a) * e + 2 * U * np.abs(want["dx"])}
    gate = np.repeat(d64["gate"], rows // gate_rows, 0) if gate_rows else 1.0
    du, e_du = b * gate * dR, np.abs(b * gate) * e + 3 * U * np.abs(b * gate * dR)
    bounds["dblock"] = e_du
    if block:
        hhat, eh = h.astype(np.float64), 0 * e
        if post != "none":
            hs = hstats.astype(np.float64)
            hhat, eh = orc.norm_apply(h, hs, None, None), xhat_error(h.astype(np.float64), hs)
            g = du * (1 if p["post_gamma"] is None else d64["post_gamma"])
            e_g = e_du * (1 if p["post_gamma"] is None else np.abs(d64["post_gamma"])) + U * np.abs(g)
            bounds["dblock"] = through(g, hhat, hs[:, 1:], e_g) + hs[:, 1:] * (
                eh * np.abs((g * hhat).mean(1, keepdims=True)) + np.abs(hhat) * (np.abs(g) * eh).mean(1, keepdims=True)) + 2 * U * np.abs(want["dblock"])
            terms["post_gamma"] = (du * hhat, e_du * np.abs(hhat) + np.abs(du) * eh)
            terms["post_beta"] = (du, e_du)
        if gate_rows:
            pg = 1 if p["post_gamma"] is None else d64["post_gamma"]
            pb = 0 if p["post_beta"] is None else d64["post_beta"]
            u_size = np.abs(hhat * pg) + np.abs(pb)
            terms["gate"] = (np.abs(b * dR) * u_size, abs(b) * (e * u_size + np.abs(dR) * (eh * np.abs(pg) + 4 * U * u_size)))
    for name, (t, et) in terms.items():
        shape = (gate_rows, rows // gate_rows, dim) if name == "gate" else (1, rows, dim)
        n = shape[1]
        bounds[name] = ((n + 8) * U * np.abs(t).reshape(shape).sum(1) + et.reshape(shape).sum(1)).reshape(want[name].shape)
    for name, t in got.items():
        off = np.abs(t.astype(np.float64) - want[name].reshape(t.shape))
        assert (off <= 1.1 * bounds[name].reshape(t.shape) + 1e-30).all(), (name, float((off / (bounds[name].reshape(t.shape) + 1e-30)).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows, dim", SHAPES)
def test_backward(wrapper, rows, dim):
    for i, (norm, post, gate) in enumerate(COMBINATIONS):
        _check_backward(wrapper, rows, dim, norm, post, _groups(gate, rows), 0.8, 1.25, affine=i % 3 != 2, shift=i % 2, in_place=i % 4 == 1)
    _check_backward(wrapper, rows, dim, "layer", "none", 0, 1.0, 1.0, block=False, with_dr=False)
    _check_backward(wrapper, rows, dim, "rms", "rms", 1, 1.0, 1.0, wanted=("gamma", "gate"))
    _check_backward(wrapper, rows, dim, "layer", "layer", 1, 1.0, 1.0, wanted=("dblock",))
    _check_backward(wrapper, rows, dim, "layer", "layer", _groups("groups", rows), 1.0, 1.0, wanted=("post_beta", "dx"))
    wrapper.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("rows, groups", [(1000, 250), (1000, 500), (1000, 1000), (777, 7), (777, 259), (2400, 600), (999, 3), (5000, 2)])
def test_gates_of_every_grouping(wrapper, rows, groups):
    for dim in (20, 333, 640):
        _check_forward(wrapper, rows, dim, "rms", "none", groups, 1.0, 1.0)
        _check_backward(wrapper, rows, dim, "rms", "none", groups, 1.0, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, dim", [(40000, 32), (20000, 129), (3000, 1000)])
def test_many_rows(wrapper, rows, dim):
    _check_forward(wrapper, rows, dim, "layer", "rms", 1, 1.0, 0.5)
    _check_backward(wrapper, rows, dim, "layer", "rms", 1, 1.0, 0.5)


@pytest.mark.gpu
def test_the_same_every_time(wrapper):
    p, r, h, dy, dr = _inputs(700, 260, "rms", "layer", 7, True, 3)
    stats, hstats = orc.norm_statistics(r, "rms", EPS).astype(np.float32), orc.norm_statistics(h, "layer", EPS).astype(np.float32)
    runs = [_run_backward(wrapper, 700, 260, "rms", "layer", 7, 1.0, 1.0, p, r, h, dy, dr, stats, hstats) for _ in range(3)]
    for other in runs[1:]:
        for k in runs[0]:
            np.testing.assert_array_equal(runs[0][k], other[k])


@pytest.mark.gpu
def test_rows_without_spread_and_infinities(wrapper):
    rows, dim = 6, 100
    x = np.random.default_rng(0).normal(size=(rows, dim)).astype(np.float32)
    x[0], x[1], x[2, 5], x[3, 7] = 0, 3.25, np.nan, np.inf
    none = {n: None for n in NAMES}
    for norm in ("layer", "rms"):
        r, y, s, _ = _run_forward(wrapper, rows, dim, norm, "none", 0, 1.0, 1.0, none, x, None)
        assert (y[0] == 0).all()                                        # a row of zeros: nothing over sqrt(epsilon)
        np.testing.assert_allclose(s[0, 1], 1 / np.sqrt(np.float32(EPS)), rtol=1e-6)
        if norm == "layer":
            assert (y[1] == 0).all()                                    # a constant that sums without rounding
        assert np.isnan(y[2]).all() and not np.isfinite(y[3, 7])
        np.testing.assert_array_equal(y[4:], _run_forward(wrapper, 2, dim, norm, "none", 0, 1.0, 1.0, none, x[4:], None)[1])


@pytest.mark.gpu
def test_a_large_mean_does_not_cancel(wrapper):
    # deviation 1 around 4096: squares would need 24 + 24 bits; the deviations from the mean do not
    x = (np.random.default_rng(1).normal(size=(8, 4096)) + 4096).astype(np.float32)
    none = {n: None for n in NAMES}
    _, y, s, _ = _run_forward(wrapper, 8, 4096, "layer", "none", 0, 1.0, 1.0, none, x, None)
    stats = orc.norm_statistics(x, "layer", EPS)
    # the mean is off by at most (L + 1) u 4096 = 0.014; the variance by that squared and L u
    e = 1.1 * (_path(4096) + 1) * U * 4096
    assert (np.abs(s[:, 0] - stats[:, 0]) <= e).all()
    np.testing.assert_allclose(s[:, 1], stats[:, 1], rtol=e * e + (_path(4096) + 8) * U)
    assert np.abs(y - orc.norm_apply(x, stats, None, None)).max() <= 1.1 * (e + 5 * e * e + 1e-4)


@pytest.mark.gpu
def test_no_rows(wrapper):
    import torch
    from sharpnet_b200 import _capi
    lib, h = wrapper.lib, wrapper.handle
    g = torch.ones(5, 8, device=wrapper.device)
    at = [g[i].data_ptr() for i in range(5)]
    params = _capi.NormParams(at[0], at[0], at[0], at[0], at[0])
    desc = _desc(0, 8, "layer", "rms", 1, 1, 1)
    assert lib.snb200_residual_norm_fwd(h, desc, params, *[None] * 6) == 0
    assert lib.snb200_residual_norm_bwd(h, desc, params, *[None] * 9, _capi.NormParams(*at)) == 0
    assert not g.cpu().numpy().any()                                       # sums over no rows


@pytest.mark.gpu
def test_refusals(wrapper):
    import torch
    from sharpnet_b200 import _capi
    lib, h = wrapper.lib, wrapper.handle
    t = torch.zeros(4096, device=wrapper.device)
    q = t.data_ptr()

    def fwd(desc, params=None, x=q, block=q, r=q, y=q, s=q, ps=q):
        return lib.snb200_residual_norm_fwd(h, desc, params or _capi.NormParams(), x, block, r, y, s, ps)

    def bwd(desc, params=None, r=q, block=q, dy=q, dr=q, s=q, ps=q, scratch=q, dx=q, dh=q, grads=None):
        return lib.snb200_residual_norm_bwd(h, desc, params or _capi.NormParams(), r, block, dy, dr, s, ps, scratch, dx, dh, grads)

    P = _capi.NormParams
    for call in (fwd, bwd):
        for bad in (_desc(-1, 4, "layer", "none", 0, 1, 1), _desc(4, -1, "layer", "none", 0, 1, 1), _desc(4, 4, "layer", "none", -1, 1, 1),
                    _desc(4, 4, "layer", "none", 0, 1, 1, 0.0), _desc(4, 4, "layer", "none", 0, 1, 1, -1.0), _desc(4, 4, "layer", "none", 0, 1, 1, float("nan")),
                    _capi.NormDesc(4, 4, 3, 0, 0, 1, 1, EPS), _capi.NormDesc(4, 4, 1, -1, 0, 1, 1, EPS)):
            assert call(bad) == 7
        assert call(_desc(4, 4, "layer", "none", 3, 1, 1), P(gate=q)) == 7 and call(_desc(4, 4, "layer", "none", 8, 1, 1), P(gate=q)) == 7
        assert call(_desc(4, 4, "layer", "none", 1, 1, 1)) == 7 and call(_desc(4, 4, "layer", "none", 0, 1, 1), P(gate=q)) == 7
        assert call(_desc(4, 4, "none", "rms", 0, 1, 1), P(gamma=q)) == 7 and call(_desc(4, 4, "rms", "none", 0, 1, 1), P(post_beta=q)) == 7
        assert call(_desc(4, (1 << 24) + 1, "layer", "none", 0, 1, 1)) == 15
        assert call(_desc(1 << 31, 4, "layer", "none", (1 << 30) + 1, 1, 1), P(gate=q)) == 15
        assert lib.snb200_last_error_string(h)
    layer = _desc(4, 4, "layer", "none", 0, 1, 1)
    assert fwd(layer, x=None) == 7 and fwd(layer, y=None) == 7 and fwd(layer, r=None) == 7
    assert fwd(_desc(4, 4, "layer", "rms", 0, 1, 1), block=None) == 7 and fwd(_desc(4, 4, "layer", "none", 1, 1, 1), P(gate=q), block=None) == 7
    assert fwd(_desc(4, 4, "none", "none", 0, 1, 1), block=None, r=None) == 7
    assert lib.snb200_residual_norm_fwd(h, None, P(), *[None] * 6) == 7
    assert bwd(layer, r=None) == 7 and bwd(layer, dy=None) == 7 and bwd(layer, s=None) == 7
    assert bwd(_desc(4, 4, "none", "none", 0, 1, 1), dr=None) == 7
    post = _desc(4, 4, "layer", "rms", 1, 1, 1)
    assert bwd(post, P(gate=q), block=None) == 7 and bwd(post, P(gate=q), ps=None) == 7
    assert bwd(layer, dx=None, dh=None) == 7
    assert bwd(layer, grads=P(gamma=q)) == 7                                # a gradient without its parameter
    assert bwd(layer, P(gamma=q), scratch=None, grads=P(gamma=q)) == 7
    assert bwd(layer, P(gamma=q), scratch=q + 4, grads=P(gamma=q)) == 7
    assert bwd(_desc(4, 4, "layer", "none", 1, 1, 1), P(gate=q), block=None, grads=P(gate=q)) == 7
    assert not t.cpu().numpy().any()


@pytest.mark.gpu
def test_layer(wrapper):
    from sharpnet_b200.normalization import ResidualNorm
    from sharpnet_b200.tensor import GPUTensor
    rng = np.random.default_rng(9)
    B, T, D = 3, 4, 24
    T_ = lambda a: GPUTensor(a.shape, a, wrapper)  # noqa: E731
    x, h, dy, dr = (rng.normal(size=(B, T, D)).astype(np.float32) for _ in range(4))
    layer = ResidualNorm(D, wrapper, norm="layer", post_norm="rms", gate_rows=B, residual_scale=0.5)
    layer.Parameters["gate"].storage.copy_(T_(rng.normal(size=(B, D))).storage)
    r, y, dx, dh = (GPUTensor((B, T, D), None, wrapper) for _ in range(4))
    layer.ForwardPropagation(T_(x), T_(h), r, y)
    layer.BackwardPropagation(r, T_(h), T_(dy), T_(dr), dx, dh)
    p = {n: None if t is None else t.ContentAsFloatArray().astype(np.float64) for n, t in layer.Parameters.items()}
    p = {n: None if v is None else v if n == "gate" else v.reshape(-1) for n, v in p.items()}
    x2, h2, dy2, dr2 = (v.reshape(-1, D) for v in (x, h, dy, dr))
    hs = orc.norm_statistics(h2, "rms", EPS)
    r64 = orc.residual_norm_sum(x2, h2, hs, p, B, 0.5, 1.0)
    rs = orc.norm_statistics(r64, "layer", EPS)
    # values of order one through about forty rounded operations each way; the backward pass divides by deviations near one
    tol = dict(rtol=0, atol=200 * U)
    np.testing.assert_allclose(r.ContentAsFloatArray().reshape(-1, D), r64, **tol)
    np.testing.assert_allclose(y.ContentAsFloatArray().reshape(-1, D), orc.norm_apply(r64, rs, p["gamma"], p["beta"]), **tol)
    want = orc.residual_norm_backward(r64, h2, dy2, dr2, rs, hs, p, "layer", "rms", B, 0.5, 1.0)
    np.testing.assert_allclose(dx.ContentAsFloatArray().reshape(-1, D), want["dx"], **tol)
    np.testing.assert_allclose(dh.ContentAsFloatArray().reshape(-1, D), want["dblock"], **tol)
    for n, t in layer.Gradients.items():
        if t is not None:
            np.testing.assert_allclose(t.ContentAsFloatArray().reshape(want[n].shape), want[n], rtol=0, atol=200 * U * B * T)
    assert layer.Gradients["post_beta"] is None
    with pytest.raises(ValueError):
        ResidualNorm(D, wrapper, norm="batch")
    with pytest.raises(ValueError):
        layer.ForwardPropagation(T_(x), T_(h[:2]), r, y)
    with pytest.raises(ValueError):
        ResidualNorm(D, wrapper, parameters={"gamma": GPUTensor((D + 1,), None, wrapper)})
    with pytest.raises(ValueError):
        ResidualNorm(D, wrapper).BackwardPropagation(r, None, T_(dy), None, dx, None)       # no forward pass yet
    assert ctypes.sizeof(type(layer._desc)) == 40
