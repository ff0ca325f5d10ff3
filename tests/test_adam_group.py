"""snb200_adam_group_update: many tensors in one launch, moments in 32 or 8 bits.

32 bits: the formula of snb200_adam_update.  With u = 2^-24, each of the two calls is off by at most
  v: 3 u (|b1 v| + |(1 - b1) g|), two products and a sum;  s: 4 u s, three products and a sum of positive terms;
  W: factor E(v) / (sqrt(s) + eps) + 8 u |step| + 4 u |W|, E(s) / 2 and six more rounded operations on the step,
and what earlier steps left is carried on by factors below one, so that t steps add up to t times that at most; the two
calls may differ by twice as much.  (They round differently: the compiler chooses which product it fuses into a sum.)
The same tensors at other alignments give the same bits.  8 bits: codes and scales bit for bit against the oracle's 32-bit
arithmetic; the weight within u (9 |step| + 4 |W|): in the step factor v / (root + eps) the factor, its product with v, eps
and the sum are off by u each and the quotient, taken as a product with an approximate reciprocal, by 2 ulp or 4 u;
wd W is off by u, and the two sums by u each."""
import numpy as np
import pytest

from oracle import sharpnet_oracle as orc
from tests.guarded import Guarded

RATE, B1, B2, EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 0.01


# -------------------------------------------------------------------------------------------- no device needed
def test_oracle_codes():
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    np.testing.assert_array_equal(orc.e4m3_encode(orc.e4m3_decode(codes)), codes)      # every code, both zeros among them
    assert orc.e4m3_decode(np.uint8(0x7e)) == 448 and orc.e4m3_decode(np.uint8(1)) == 2.0 ** -9
    assert orc.e4m3_encode(np.array([17.0]))[0] == orc.e4m3_encode(np.array([16.0]))[0]      # a tie goes to the even code
    assert orc.e4m3_encode(np.array([19.0]))[0] == orc.e4m3_encode(np.array([20.0]))[0]
    np.testing.assert_array_equal(orc.adam8_scale(np.array([0, 1.0, 255, 256, 2.0 ** -101, np.inf], np.float32)),
                                  np.array([0, 2.0 ** -7, 1, 2, 0, np.nan], np.float32))


def test_oracle_rounds_the_root_without_bias():
    # over many seeds the mean of the rounded root is the root: its deviation is at most half a step (2^-4 of the value)
    # over the square root of the number of draws, five times that is allowed
    seeds, n = 400, 512
    root = np.linspace(0.02, 1.0, n).astype(np.float32)
    total = np.zeros(n)
    for seed in range(seeds):
        s, sc, v, vc = np.zeros(n, np.uint8), np.zeros(2, np.float32), np.zeros(n, np.uint8), np.zeros(2, np.float32)
        g = (root / np.float32(np.sqrt(1 - 0.999))).astype(np.float32)
        orc.update_adam8_optimizer(np.zeros(n, np.float32), RATE, B1, B2, EPS, 0.0, g, v, s, vc, sc, 1, seed, 3)
        total += orc.e4m3_decode(s) * np.repeat(sc, 256)
    assert (np.abs(total / seeds / root - 1) < 5 * 2.0 ** -4 / np.sqrt(seeds)).all()


def test_null_handle_is_refused(built_library):
    from sharpnet_b200 import _capi
    assert _capi.load().snb200_adam_group_update(None, 0, None, 32, RATE, B1, B2, EPS, WD, 1, 0) == 1


# -------------------------------------------------------------------------------------------- on the device
def _tensors(rng, sizes, bits, history=True):
    """Host copies: (W, dW, v, s[, v_scale, s_scale]) per tensor."""
    out = []
    for n in sizes:
        W, g = (rng.normal(size=n).astype(np.float32) for _ in range(2))
        g *= np.exp(rng.normal(size=n)).astype(np.float32)
        v, r = rng.normal(size=n).astype(np.float32), np.abs(rng.normal(size=n)).astype(np.float32)
        if not history:
            v[:], r[:] = 0, 0
        if bits == 32:
            out.append([W, g, v, r * r])
            continue
        blocks = -(-n // 256)
        pad = lambda a: np.pad(a, (0, blocks * 256 - n)).reshape(blocks, 256)  # noqa: E731
        vs, ss = orc.adam8_scale(np.abs(pad(v)).max(1) if n else []), orc.adam8_scale(pad(r).max(1) if n else [])
        inverse = lambda c: np.repeat(np.where(c == 0, 0, 1 / np.where(c == 0, 1, c)), 256)[:n]  # noqa: E731
        out.append([W, g, orc.e4m3_encode(v * inverse(vs)), orc.e4m3_encode(r * inverse(ss)), vs, ss])
    return out


def _upload(w, tensors, shifts):
    return [[Guarded(a, w.device, s) for a, s in zip(t, shifts[i % len(shifts)])] for i, t in enumerate(tensors)]


def _table(uploaded, decays):
    from sharpnet_b200 import _capi
    rows = []
    for t, d in zip(uploaded, decays):
        at = [a.pointer for a in t] + [None] * (6 - len(t))
        rows.append(_capi.AdamTensor(t[0].n, at[1], at[0], at[2], at[3], at[4], at[5], d))
    return (_capi.AdamTensor * len(rows))(*rows)


def _step(w, uploaded, decays, bits, t, seed=0):
    st = w.lib.snb200_adam_group_update(w.handle, len(uploaded), _table(uploaded, decays), bits, RATE, B1, B2, EPS, WD, t, seed)
    assert st == 0, w.lib.snb200_last_error_string(w.handle)


SIZES = [[1], [2, 0, 3], [255, 256, 257], [1023, 4096, 4097, 1, 12345], [100003], [77] * 33, [300, 5] * 230]
SHIFTS = {32: [(0, 0, 0, 0), (1, 0, 0, 0), (1, 1, 1, 1), (0, 0, 2, 3)],
          8: [(0, 0, 0, 0, 0, 0), (1, 0, 0, 0, 1, 0), (0, 3, 4, 8, 0, 1), (0, 0, 1, 2, 0, 0)]}


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_32_bits(wrapper, sizes):
    rng = np.random.default_rng(len(sizes))
    tensors, decays = _tensors(rng, sizes, 32), rng.integers(0, 3, len(sizes)) / 2.0
    many, one = _upload(wrapper, tensors, SHIFTS[32]), _upload(wrapper, tensors, SHIFTS[32])
    aligned = _upload(wrapper, tensors, [(0, 0, 0, 0)])
    u = 2.0 ** -24
    slack = [[0.0, None, 0.0, 0.0] for _ in sizes]
    for t in (1, 2, 50):
        factor = RATE * np.sqrt(1 - B2 ** t) / (1 - B1 ** t)
        for k, (up, d) in enumerate(zip(one, decays)):
            (W0, g, v0, _), at = [a.numpy().astype(np.float64) for a in up], [a.pointer for a in up]
            assert wrapper.lib.snb200_adam_update(wrapper.handle, up[0].n, RATE, B1, B2, EPS, WD * d, t, at[1], at[0], at[2], at[3]) == 0
            s1, root = up[3].numpy().astype(np.float64), np.sqrt(up[3].numpy().astype(np.float64)) + EPS
            ev = 3 * u * (np.abs(B1 * v0) + np.abs((1 - B1) * g))
            step = factor * np.abs(up[2].numpy()) / root + WD * d * np.abs(W0)
            slack[k][2] = slack[k][2] + ev
            slack[k][3] = slack[k][3] + 4 * u * s1
            slack[k][0] = slack[k][0] + factor * slack[k][2] / root + 8 * u * step + factor * np.abs(up[2].numpy()) / root * slack[k][3] / (2 * s1) + 4 * u * np.abs(W0)
        _step(wrapper, many, decays, 32, t)
        _step(wrapper, aligned, decays, 32, t)
    for m, o, a, host, e in zip(many, one, aligned, tensors, slack):
        for k in (0, 2, 3):
            assert (np.abs(m[k].numpy().astype(np.float64) - o[k].numpy()) <= 2 * e[k]).all()
            np.testing.assert_array_equal(m[k].numpy(), a[k].numpy())
        np.testing.assert_array_equal(m[1].numpy(), host[1])           # the gradient is read only


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("history", [True, False])
def test_8_bits(wrapper, sizes, history):
    rng = np.random.default_rng(len(sizes))
    tensors, decays = _tensors(rng, sizes, 8, history), rng.integers(0, 3, len(sizes)) / 2.0
    up = _upload(wrapper, tensors, SHIFTS[8])
    for t, seed in ((1, 0), (2, 1), (1000, 0xFFFFFFFF)):
        before = [u[0].numpy().copy() for u in up]
        _step(wrapper, up, decays, 8, t, seed)
        for i, (u, host) in enumerate(zip(up, tensors)):
            if not u[0].n:
                continue
            want = orc.update_adam8_optimizer(before[i], RATE, B1, B2, EPS, WD * decays[i], host[1], *host[2:], t, seed, i)
            for k in (2, 3, 4, 5):
                np.testing.assert_array_equal(u[k].numpy(), host[k])
            still = np.abs(want - before[i])
            bound = 2.0 ** -24 * (9 * (still + WD * decays[i] * np.abs(before[i])) + 4 * np.abs(before[i]))
            assert (np.abs(u[0].numpy() - want) <= bound).all()


@pytest.mark.gpu
def test_8_bits_extremes(wrapper):
    # a block of zeros, of the smallest and largest numbers, one with a NaN and one with an infinity; each its own block
    n = 256 * 7
    g = np.ones(n, np.float32)
    g[:256] = 0
    g[256:512] = 1e-38
    g[512:768] = np.linspace(0, 3e18, 256)
    g[800], g[1030] = np.nan, np.inf
    g[1280:1536] = np.where(np.arange(256) % 2, 1.0, 1e-12)
    host = [np.ones(n, np.float32), g, np.zeros(n, np.uint8), np.zeros(n, np.uint8), np.zeros(7, np.float32), np.zeros(7, np.float32)]
    up = _upload(wrapper, [host], SHIFTS[8][:1])[0]
    _step(wrapper, [up], [0.0], 8, 1, 5)
    orc.update_adam8_optimizer(host[0], RATE, B1, B2, EPS, 0.0, g, *host[2:], 1, 5, 0)
    finite = np.repeat(~np.isnan(host[4]), 256)        # what a block with a NaN scale holds besides does not matter
    for k in (2, 3):
        np.testing.assert_array_equal(up[k].numpy()[finite], host[k][finite])
    for k in (4, 5):
        np.testing.assert_array_equal(up[k].numpy(), host[k])
    W, vs, ss = up[0].numpy(), up[4].numpy(), up[5].numpy()
    assert (W[:256] == 1).all() and vs[0] == 0 and ss[0] == 0
    assert np.isnan(vs[3]) and np.isnan(ss[3]) and np.isnan(vs[4]) and np.isnan(ss[4])
    assert np.isnan(W[[800, 1030]]).all() and np.isfinite(np.delete(W, [800, 1030])).all()
    # an element with a history keeps a denominator: its root is held as the smallest code at least
    assert (up[3].numpy()[1280:1536] > 0).all()


@pytest.mark.gpu
def test_8_bits_track_32_bits(wrapper):
    # gradients of constant size: sqrt(s) / |g| of the 32-bit moments after t steps is sqrt(1 - B2^t), whatever the
    # element; under nearest rounding the 8-bit root would stop growing after about eight steps.  The rounded root makes
    # steps of at most 2^-3 of itself up or down with a mean of what is right; s forgets with a time of 1000 steps, so
    # about t steps add up, each an independent error of at most 2^-3 times its share 2 (1 - B2): the mean over 4096
    # elements is off by far less than the 5 % that are allowed
    from sharpnet_b200.optimizers import AdamGroup
    from sharpnet_b200.tensor import GPUTensor
    rng = np.random.default_rng(2)
    g = (rng.choice([-1.0, 1.0], 4096) * np.exp(rng.normal(size=4096))).astype(np.float32)
    W, dW = GPUTensor((4096,), None, wrapper), GPUTensor((4096,), g, wrapper)
    group = AdamGroup(wrapper, B1, B2, EPS, 0.0, [W], [dW], state_bits=8)
    for _ in range(300):
        group.UpdateWeights(RATE, RATE)
    v, s, vs, ss = (a.cpu().numpy() for a in group.states[0])
    root = orc.e4m3_decode(s) * np.repeat(ss, 256)
    assert abs(np.mean(root / np.abs(g)) / np.sqrt(1 - B2 ** 300) - 1) < 0.05


@pytest.mark.gpu
def test_refusals(wrapper):
    from sharpnet_b200 import _capi
    rng = np.random.default_rng(4)
    host = _tensors(rng, [300, 200], 8)
    up = _upload(wrapper, host, SHIFTS[8][:1])
    call = lambda table, n=None, bits=8, t=1: wrapper.lib.snb200_adam_group_update(  # noqa: E731
        wrapper.handle, len(table) if n is None else n, table, bits, RATE, B1, B2, EPS, WD, t, 0)
    good = _table(up, [1, 1])
    assert call(good, n=-1) == 7 and call(good, t=0) == 7 and call(good, bits=16) == 7 and call(good, bits=4) == 7
    assert call(good, n=0) == 0
    assert wrapper.lib.snb200_adam_group_update(wrapper.handle, 1, None, 8, RATE, B1, B2, EPS, WD, 1, 0) == 7
    for field in ("dW", "W", "adam_vW", "adam_sW", "v_scale", "s_scale"):
        table = _table(up, [1, 1])
        setattr(table[1], field, None)
        assert call(table) == 7 and b"tensor 1" in wrapper.lib.snb200_last_error_string(wrapper.handle), field
    table = _table(up, [1, 1])
    table[0].count = -1
    assert call(table) == 7
    table = _table(up, [1, 1])
    table[0].count = 1 << 62
    assert call(table) == 15
    for field in ("W", "adam_vW", "adam_sW", "v_scale", "s_scale"):           # the same memory twice, and a partial overlap
        for offset in (0, 4):
            table = _table(up, [1, 1])
            setattr(table[1], field, getattr(table[0], field) + offset)
            assert call(table) == 7 and b"share memory" in wrapper.lib.snb200_last_error_string(wrapper.handle), field
    for field, other in (("adam_sW", "adam_vW"), ("adam_vW", "W"), ("adam_sW", "W"), ("W", "dW")):
        table = _table(up, [1, 1])
        setattr(table[0], field, getattr(table[0], other))
        assert call(table) == 7, (field, other)
    table = (_capi.AdamTensor * 2)(good[1], good[0])                            # descending order is no overlap
    assert call(table) == 0
    for u, h in zip(up, host):
        np.testing.assert_array_equal(u[1].numpy(), h[1])


@pytest.mark.gpu
def test_group_object(wrapper):
    import torch
    from sharpnet_b200.optimizers import Adam, AdamGroup
    from sharpnet_b200.tensor import GPUTensor
    rng = np.random.default_rng(6)
    host = [(rng.normal(size=s).astype(np.float32), rng.normal(size=s).astype(np.float32)) for s in ((8, 5), (5,), (3, 3))]
    make = lambda: [[GPUTensor(h[k].shape, h[k], wrapper) for h in host] for k in (0, 1)]  # noqa: E731
    W, dW = make()
    W1, dW1 = make()
    group = AdamGroup(wrapper, B1, B2, EPS, WD, W, dW)
    ones = [Adam(wrapper, B1, B2, EPS, WD, t.Shape, None) for t in W1]
    for rate in (1e-3, 5e-4, 5e-4):
        group.UpdateWeights(rate, 1e-3)
        for o, a, b in zip(ones, W1, dW1):
            o.UpdateWeights(rate, 1e-3, 1, a, b, None, None)
    for a, b in zip(W, W1):                 # three steps of at most 3 RATE, each off by 2^-24 times a few of that and of W
        np.testing.assert_allclose(a.ContentAsFloatArray(), b.ContentAsFloatArray(), rtol=24 * 2.0 ** -24, atol=3 * 3 * RATE * 32 * 2.0 ** -24)
        b.storage.copy_(a.storage)
    # going on from copied states is the same as going on
    resumed = AdamGroup(wrapper, B1, B2, EPS, WD, W1, dW1, states=[tuple(p.clone() for p in s) for s in group.states], timestep=group.timestep)
    group.UpdateWeights(1e-3, 1e-3)
    resumed.UpdateWeights(1e-3, 1e-3)
    for a, b in zip(W, W1):
        np.testing.assert_array_equal(a.ContentAsFloatArray(), b.ContentAsFloatArray())
    for bad in (dict(state_bits=16), dict(decays=[1.0]), dict(states=[]), dict(states=[(torch.zeros(1), torch.zeros(1))] * 3)):
        with pytest.raises(ValueError):
            AdamGroup(wrapper, B1, B2, EPS, WD, W, dW, **bad)
    with pytest.raises(ValueError):
        AdamGroup(wrapper, B1, B2, EPS, WD, W, dW[:2])
    with pytest.raises(ValueError):
        AdamGroup(wrapper, B1, B2, EPS, WD, W, dW, state_bits=8, states=group.states)


@pytest.mark.gpu
def test_more_than_2_31_elements(wrapper):
    import torch
    n = (1 << 31) + 1000
    from sharpnet_b200 import _capi
    W, g = torch.zeros(n, device=wrapper.device), torch.ones(n, device=wrapper.device)
    v, s = (torch.zeros(n, dtype=torch.uint8, device=wrapper.device) for _ in range(2))
    vs, ss = (torch.zeros(-(-n // 256), device=wrapper.device) for _ in range(2))
    table = (_capi.AdamTensor * 1)(_capi.AdamTensor(n, g.data_ptr(), W.data_ptr(), v.data_ptr(), s.data_ptr(), vs.data_ptr(), ss.data_ptr(), 1.0))
    assert wrapper.lib.snb200_adam_group_update(wrapper.handle, 1, table, 8, 1.0, B1, B2, EPS, 0.0, 1, 0) == 0
    # every element takes the same first step, by -1 up to the rounding of factor, v and the root
    assert bool((W == W[0]).all()) and abs(float(W[0]) + 1) < 1e-5
    assert bool((vs == vs[0]).all()) and bool((v == v[0]).all()) and bool((ss == ss[0]).all())
