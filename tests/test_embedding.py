"""snb200_embedding_fwd / _bwd against float64 sums.

Tolerances.  Forward: one product per element, rounded once: equal to numpy's float32 product.  Backward: an element of
word v is a sum of c_v terms in some order, one product with the scale and, with accumulate, one more sum: by the usual
bound for a floating sum, |error| <= (c_v + 2) 2^-24 S, S the sum of the magnitudes of what is added (higher orders of
2^-24 are below a thousandth of that for the sizes here; the factor 1.01 covers them), and an exact zero for other words."""
import ctypes

import numpy as np
import pytest

from oracle import sharpnet_oracle as orc
from tests.guarded import Guarded

INT32, INT64, FP32 = 0, 1, 2
DTYPES = {INT32: np.int32, INT64: np.int64, FP32: np.float32}


def _zipf(rng, n, vocab):
    return np.minimum((np.exp(rng.random(n) * np.log(vocab + 1)) - 1).astype(np.int64), vocab - 1)


# -------------------------------------------------------------------------------------------- no device needed
def test_oracle_gradient_is_the_transpose_of_the_lookup():
    rng = np.random.default_rng(0)
    table, dy, ids = rng.normal(size=(7, 5)), rng.normal(size=(20, 5)), rng.integers(-1, 8, 20)
    grad, _, _ = orc.embedding_backward(ids, 1.5, 3, dy, np.zeros((7, 5)), False)
    one = np.zeros((7, 5))
    for v in range(7):                                  # <dy, lookup(table)> is linear in the table
        for c in range(5):
            unit = np.zeros((7, 5))
            unit[v, c] = 1
            one[v, c] = (dy * orc.embedding_forward(ids, 1.5, unit)).sum() if v != 3 else 0.0
    np.testing.assert_allclose(grad, one, atol=1e-13)


def test_scratch_size(built_library):
    from sharpnet_b200 import _capi
    lib = _capi.load()
    size = lib.snb200_embedding_scratch_bytes
    assert size(0, 10, 10) >= 0
    assert size(-1, 10, 10) == -1 and size(10, 0, 10) == -1 and size(10, 10, -1) == -1 and size((1 << 30) + 1, 10, 10) == -1
    assert size(1000, 10, 64) >= 4 * 4 * 1000           # keys and places, two of each
    assert size(1 << 30, (1 << 31) - 1, 4) > 1 << 34    # counts that pass 32 bits
    for n in (1, 31, 4096, 4097, 1 << 20):
        assert size(n + 1, 50000, 256) >= size(n, 50000, 256) - 16 * 2 * 256 * 4 * (n // 8)   # sane growth, never negative


def test_null_handle_is_refused(built_library):
    from sharpnet_b200 import _capi
    lib = _capi.load()
    assert lib.snb200_embedding_fwd(None, 0, 1, 1, 1, None, 1.0, None, None) == 1
    assert lib.snb200_embedding_bwd(None, 0, 1, 1, 1, None, 1.0, -1, 0, None, None, None) == 1


# -------------------------------------------------------------------------------------------- on the device
def _forward(w, kind, ids, scale, table, shift=0):
    n, (vocab, dim) = len(ids), table.shape
    i, t, y = (Guarded(a, w.device, s) for a, s in ((ids.astype(DTYPES[kind]), 0), (table, shift), (np.full((n, dim), 9, np.float32), shift)))
    st = w.lib.snb200_embedding_fwd(w.handle, kind, n, vocab, dim, i.pointer, scale, t.pointer, y.pointer)
    assert st == 0, w.lib.snb200_last_error_string(w.handle)
    return y.numpy()


def _backward(w, kind, ids, scale, padding, accumulate, dy, dtable, shift=0):
    import torch
    n, (vocab, dim) = len(ids), dtable.shape
    i, g, d = (Guarded(a, w.device, s) for a, s in ((ids.astype(DTYPES[kind]), 0), (dy, shift), (dtable, shift)))
    need = w.lib.snb200_embedding_scratch_bytes(n, vocab, dim)
    scratch = torch.full((need + 1024,), 77, dtype=torch.uint8, device=w.device)       # never cleared by the caller
    st = w.lib.snb200_embedding_bwd(w.handle, kind, n, vocab, dim, i.pointer, scale, padding, int(accumulate), g.pointer,
                                    scratch.data_ptr(), d.pointer)
    assert st == 0, w.lib.snb200_last_error_string(w.handle)
    assert bool((scratch[need:] == 77).all()), "written behind the scratch memory"
    return d.numpy()


def _check_backward(w, kind, ids, scale, padding, accumulate, dim, vocab, seed, shift=0):
    rng = np.random.default_rng(seed)
    dy = rng.normal(size=(len(ids), dim)).astype(np.float32)
    dtable = rng.normal(size=(vocab, dim)).astype(np.float32)
    got = _backward(w, kind, ids, scale, padding, accumulate, dy, dtable, shift)
    scale = float(np.float32(scale))
    want, size, terms = orc.embedding_backward(ids, scale, padding, dy, dtable, accumulate)
    bound = 1.01 * (terms[:, None] + 2) * 2.0 ** -24 * size
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
    if accumulate:
        assert (got[terms == 0] == dtable[terms == 0]).all()
    else:
        assert (got[terms == 0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [INT32, INT64, FP32])
@pytest.mark.parametrize("dim", [1, 3, 4, 50, 128, 333, 1024, 2500])
def test_forward(wrapper, kind, dim):
    rng = np.random.default_rng(dim)
    for n, vocab in ((1, 1), (2, 50), (31, 7), (1000, 300), (20011 if dim <= 128 else 2011, 5000)):
        table, ids = rng.normal(size=(vocab, dim)).astype(np.float32), _zipf(rng, n, vocab)
        for shift in (0, 1):
            got = _forward(wrapper, kind, ids, 1.7, table, shift)
            assert (got == np.float32(1.7) * table[ids]).all()
    wrapper.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [INT32, INT64, FP32])
def test_indices_outside_the_table(wrapper, kind):
    from sharpnet_b200 import SharpNetB200Error
    rng = np.random.default_rng(5)
    table = rng.normal(size=(10, 12)).astype(np.float32)
    bad = {INT32: [-1, 10, 2 ** 31 - 1, -2 ** 31], INT64: [-1, 10, 2 ** 32, 2 ** 63 - 1, -2 ** 63, 2 ** 32 + 3],
           FP32: [-1.0, 10.0, np.nan, np.inf, -np.inf, 3e9]}[kind]
    ids = np.array([0, 9, 3] + bad + [5, 9], DTYPES[kind])
    good = np.array([0, 9, 3] + [-1] * len(bad) + [5, 9])
    got = _forward(wrapper, kind, ids, 2.0, table)
    np.testing.assert_array_equal(got, orc.embedding_forward(good, 2.0, table).astype(np.float32))
    with pytest.raises(SharpNetB200Error, match="token index"):
        wrapper.check_device_status()
    wrapper.check_device_status()                         # reported once
    dy = rng.normal(size=(len(ids), 12)).astype(np.float32)
    got = _backward(wrapper, kind, ids, 1.0, -1, False, dy, np.ones((10, 12), np.float32))
    want, _, _ = orc.embedding_backward(good, 1.0, -1, dy, np.zeros((10, 12)), False)
    np.testing.assert_allclose(got, want, rtol=0, atol=4 * 2.0 ** -24 * 2 * np.abs(dy).max())
    with pytest.raises(SharpNetB200Error, match="token index") as e:
        wrapper.check_device_status()
    assert e.value.status == 7


@pytest.mark.gpu
def test_float_indices_are_rounded(wrapper):
    table = np.arange(40, dtype=np.float32).reshape(10, 4)
    ids = np.array([2.9999, 3.0001, 0.2, -0.3, 8.75], np.float32)
    np.testing.assert_array_equal(_forward(wrapper, FP32, ids, 1.0, table), table[[3, 3, 0, 0, 9]])
    wrapper.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [INT32, INT64, FP32])
@pytest.mark.parametrize("n, vocab, dim", [(1, 1, 1), (1, 5, 4), (2, 3, 7), (31, 4, 33), (32, 40, 32), (33, 1, 130), (100, 7, 12),
                                           (513, 300, 129), (2049, 511, 64), (5000, 512, 20), (4100, 70000, 8), (3000, 600001, 3),
                                           (70000, 1000, 16), (20000, 32768, 100)])
def test_backward(wrapper, kind, n, vocab, dim):
    rng = np.random.default_rng(n + dim)
    ids = _zipf(rng, n, vocab)
    for padding, accumulate, shift in ((-1, False, 0), (0, True, 0), (min(1, vocab - 1), False, 1)):
        _check_backward(wrapper, kind, ids, 0.37, padding, accumulate, dim, vocab, n, shift)
    wrapper.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("n, dim", [(1000, 64), (66000, 40), (300000, 4)])
def test_backward_of_one_word(wrapper, n, dim):
    for ids in (np.full(n, 6), np.where(np.arange(n) % 2, 6, 2), np.where(np.arange(n) < n // 2 + 1, 9, 0)):
        _check_backward(wrapper, INT32, ids, 1.0, -1, False, dim, 10, n)
    _check_backward(wrapper, INT32, np.full(n, 6), 1.0, 6, False, dim, 10, n)      # nothing but padding
    _check_backward(wrapper, INT32, np.full(n, 6), 1.0, 6, True, dim, 10, n)


@pytest.mark.gpu
def test_backward_orders(wrapper):
    # sorted, reversed and once-each orders; every length around the cuts of the sums
    for n in (7, 8, 9, 15, 16, 17, 127, 128, 129, 255, 257, 1025, 2047, 2048, 4097, 8200):
        for ids in (np.arange(n), np.arange(n)[::-1].copy(), np.repeat(np.arange((n + 4) // 5), 5)[:n]):
            _check_backward(wrapper, INT32, ids, 1.0, -1, False, 36, n, n)


@pytest.mark.gpu
def test_backward_is_the_same_every_time(wrapper):
    rng = np.random.default_rng(8)
    ids, dy = _zipf(rng, 30000, 700), rng.normal(size=(30000, 72)).astype(np.float32)
    first = _backward(wrapper, INT64, ids, 1.0, -1, False, dy, np.zeros((700, 72), np.float32))
    for _ in range(3):
        np.testing.assert_array_equal(first, _backward(wrapper, INT64, ids, 1.0, -1, False, dy, np.ones((700, 72), np.float32)))


@pytest.mark.gpu
def test_backward_without_tokens_and_infinities(wrapper):
    got = _backward(wrapper, INT32, np.zeros(0, np.int64), 1.0, -1, False, np.zeros((0, 6), np.float32), np.ones((5, 6), np.float32))
    assert (got == 0).all()
    got = _backward(wrapper, INT32, np.zeros(0, np.int64), 1.0, -1, True, np.zeros((0, 6), np.float32), np.ones((5, 6), np.float32))
    assert (got == 1).all()
    # what a padded token holds does not matter, and other words do not see a NaN
    dy = np.ones((64, 8), np.float32)
    dy[5], dy[6, 3], dy[7, 0] = np.nan, np.inf, np.nan
    ids = np.arange(64) % 8
    ids[5] = 0
    ids[6] = 3
    ids[7] = 4
    got = _backward(wrapper, INT32, ids, 1.0, 0, False, dy, np.ones((8, 8), np.float32))
    assert (got[0] == 0).all() and np.isinf(got[3, 3]) and np.isnan(got[4, 0])
    rest = got.copy()
    rest[3, 3] = rest[4, 0] = 0
    assert np.isfinite(rest).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(wrapper):
    # 2.3 G elements of gradient rows and a table of 2.2 G elements; ones add up exactly
    import torch
    n, vocab, dim = 1100000, 1050000, 2080
    dy = torch.ones(n, dim, device=wrapper.device)
    dtable = torch.empty(vocab, dim, device=wrapper.device)
    ids = torch.arange(n, device=wrapper.device).remainder_(vocab)
    need = wrapper.lib.snb200_embedding_scratch_bytes(n, vocab, dim)
    scratch = torch.empty(need, dtype=torch.uint8, device=wrapper.device)
    assert wrapper.lib.snb200_embedding_bwd(wrapper.handle, INT64, n, vocab, dim, ids.data_ptr(), 0.5, -1, 0, dy.data_ptr(),
                                            scratch.data_ptr(), dtable.data_ptr()) == 0
    assert bool((dtable[:n - vocab] == 1.0).all()) and bool((dtable[n - vocab:] == 0.5).all())
    dtable[vocab - 1] = 3
    assert wrapper.lib.snb200_embedding_fwd(wrapper.handle, INT64, n, vocab, dim, ids.data_ptr(), 2.0, dtable.data_ptr(), dy.data_ptr()) == 0
    assert bool((dy[vocab - 1] == 6.0).all()) and bool((dy[vocab:] == 2.0).all()) and bool((dy[n - vocab:vocab - 1] == 1.0).all())
    wrapper.check_device_status()


@pytest.mark.gpu
def test_refusals(wrapper):
    import torch
    lib, h = wrapper.lib, wrapper.handle
    t = torch.zeros(4096, device=wrapper.device)
    p = t.data_ptr()
    fwd, bwd = lib.snb200_embedding_fwd, lib.snb200_embedding_bwd
    for args in ((0, -1, 4, 4, p), (0, 4, 0, 4, p), (0, 4, 4, -1, p), (3, 4, 4, 4, p), (-1, 4, 4, 4, p), (0, 4, 4, 4, None),
                 (1, 4, 4, 4, p + 4), (0, 4, 4, 4, p + 2)):
        kind, n, vocab, dim, at = args
        assert fwd(h, kind, n, vocab, dim, at, 1.0, p, p) == 7, args
        assert lib.snb200_last_error_string(h)
        assert bwd(h, kind, n, vocab, dim, at, 1.0, -1, 0, p, p, p) == 7, args
    assert fwd(h, 0, 4, 4, 4, p, 1.0, None, p) == 7 and fwd(h, 0, 4, 4, 4, p, 1.0, p, None) == 7
    assert bwd(h, 0, 4, 4, 4, p, 1.0, -1, 0, None, p, p) == 7 and bwd(h, 0, 4, 4, 4, p, 1.0, -1, 0, p, None, p) == 7
    assert bwd(h, 0, 4, 4, 4, p, 1.0, -1, 0, p, p, None) == 7
    assert bwd(h, 0, 4, 4, 4, p, 1.0, -1, 0, p, p + 4, p) == 7                     # scratch alignment
    assert bwd(h, 0, (1 << 30) + 1, 4, 4, p, 1.0, -1, 0, p, p, p) == 15
    assert fwd(h, 0, 4, 4, (1 << 24) + 1, p, 1.0, p, p) == 15 and fwd(h, 0, 1 << 62, 4, 4, p, 1.0, p, p) == 15
    assert bwd(h, 0, 4, 4, (1 << 24) + 1, p, 1.0, -1, 0, p, p, p) == 15 and lib.snb200_embedding_scratch_bytes(4, 4, (1 << 24) + 1) == -1
    assert fwd(h, 0, 0, 4, 4, None, 1.0, None, None) == 0 and fwd(h, 0, 4, 4, 0, None, 1.0, None, None) == 0
    assert not t.cpu().numpy().any()


@pytest.mark.gpu
def test_layer(wrapper):
    import torch
    from sharpnet_b200.embedding import EmbeddingLayer
    from sharpnet_b200.tensor import GPUTensor
    rng = np.random.default_rng(3)
    table = rng.normal(size=(20, 6)).astype(np.float32)
    layer = EmbeddingLayer(20, 6, wrapper, scale=2.0, paddingIndex=0, weights=GPUTensor((20, 6), table, wrapper))
    ids = rng.integers(0, 20, (3, 5))
    y = GPUTensor((3, 5, 6), None, wrapper)
    dy = rng.normal(size=(3, 5, 6)).astype(np.float32)
    for x in (GPUTensor((3, 5), ids, wrapper), torch.from_numpy(ids).to(wrapper.device), torch.from_numpy(ids).int().to(wrapper.device)):
        layer.ForwardPropagation(x, y)
        np.testing.assert_array_equal(y.ContentAsFloatArray(), 2 * table[ids])
        layer.BackwardPropagation(x, GPUTensor((3, 5, 6), dy, wrapper))
        layer.BackwardPropagation(x, GPUTensor((3, 5, 6), dy, wrapper), accumulate=True)
        want, size, terms = orc.embedding_backward(ids.reshape(-1), 4.0, 0, dy.reshape(-1, 6), np.zeros((20, 6)), False)
        assert (np.abs(layer.WeightGradients.ContentAsFloatArray() - want) <= (2 * terms[:, None] + 3) * 2.0 ** -24 * size).all()
    with pytest.raises(ValueError):
        layer.ForwardPropagation(torch.zeros(4, dtype=torch.int16, device=wrapper.device), y)
    with pytest.raises(ValueError):
        layer.ForwardPropagation(torch.zeros(15, dtype=torch.int32), y)             # on the host
    with pytest.raises(ValueError):
        layer.ForwardPropagation(torch.zeros(14, dtype=torch.int32, device=wrapper.device), y)
    with pytest.raises(ValueError):
        EmbeddingLayer(21, 6, wrapper, weights=layer.Weights)
    assert ctypes.c_int(layer.paddingIndex).value == 0
