"""Cache attention where its work is divided otherwise than the sizes of small
calls have it: two blocks of rows to an operand, long ranges in one piece,
lengths announced wrongly; and scales, shared pages, graphs side by side."""

import contextlib
import ctypes

import numpy as np
import pytest

import cache_oracle
from cache_cases import HALF_STEP, Batch, OnDevice, pages_of, rounded

pytestmark = pytest.mark.gpu

P = ctypes.c_void_p
TYPES = ["fp32", "fp16", "bf16"]
TWO_BLOCKS = [("fp16", 768), ("bf16", 768), ("fp32", 128)]


def _run(cw, batch, k, v, q, precision, scale, causal):
    """The launch's output; out starts as all 3."""
    heads, dim = q.shape[1:]
    with contextlib.ExitStack() as owned:
        dev = OnDevice(cw, owned, batch, k, v, precision)
        dq = dev.put(cw._encode(q, precision))
        out = dev.put(cw._encode(np.full_like(q, 3.0), precision))
        dev.attend(dq, heads * dim, out, heads * dim, heads, scale, causal, dev.scratch(heads))
        assert cw.cudart.hipDeviceSynchronize() == 0
        return cw._decode(out.download(q.shape, cw._bits_type(precision)), precision)


def _off(got, batch, k, v, q, precision, scale, causal):
    """How far got is from the oracle, in tolerances."""
    prefix = (batch.prefix_pages, batch.prefix_len) if batch.prefix_len else (None, 0)
    want, size = cache_oracle.attend(q, k, v, *batch.where, scale, causal, *prefix)
    tol = cache_oracle.attend_tolerance(want, size, q.shape[2],
                                        batch.prefix_len + int(max(batch.kv_lens)),
                                        HALF_STEP[precision])
    return np.abs(got - want) / tol


def _check(cw, rng, batch, kv_heads, heads, dim, precision, causal=True, scale=None):
    k, v = pages_of(rng, cw, batch, kv_heads, dim, precision)
    q = rounded(cw, 1.5 * rng.standard_normal((batch.tokens, heads, dim)), precision)
    scale = dim ** -0.5 if scale is None else scale
    got = _run(cw, batch, k, v, q, precision, scale, causal)
    rows = batch.rows()
    others = np.setdiff1d(np.arange(batch.tokens), rows)
    np.testing.assert_array_equal(got[others], np.full_like(got[others], 3.0))
    off = _off(got, batch, k, v, q, precision, scale, causal)[rows]
    assert np.all(off <= 1), off.max()


@pytest.mark.parametrize("precision, dim", TWO_BLOCKS)
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("prefix", [0, 130])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("keys", [13000, 60000])
def test_two_row_blocks(cw, precision, dim, page, prefix, causal, keys):
    rng = np.random.default_rng(page + prefix)
    batch = Batch(rng, [40, 3, 0, 17], [1000, 3, 5, 300], page, before=1, behind=2,
                  prefix_len=prefix)
    batch.widen(keys)
    _check(cw, rng, batch, 2, 4, dim, precision, causal)


@pytest.mark.parametrize("precision, dim", TWO_BLOCKS)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_keys_that_are_not_seen_by_two_blocks(cw, precision, dim, bad):
    rng = np.random.default_rng(20)
    m = 150
    batch = Batch(rng, [m], [m + 3], 16)
    batch.widen(60000)
    k, v = pages_of(rng, cw, batch, 1, dim, precision)
    q = rounded(cw, np.abs(rng.standard_normal((m, 2, dim))), precision)
    clean_k, clean_v = k.copy(), v.copy()
    for c in range(3 + m // 2, m + 3, 2):
        page, slot = batch.page_table[0, c // 16], c % 16
        v[page, 0, slot] = bad
        if c % 4 < 2:
            k[page, 0, slot] = bad
    got = _run(cw, batch, k, v, q, precision, dim ** -0.5, True)
    off = _off(got, batch, clean_k, clean_v, q, precision, dim ** -0.5, True)
    assert np.all(off[:m // 2] <= 1), off[:m // 2].max()
    assert not np.any(np.isfinite(got[m // 2:]))


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256, 768])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("keys", [0, 1, 60000])
def test_lengths_announced_wrongly(cw, precision, dim, page, keys):
    """The work is divided by max_kv_len: far too small, every range is whole
    (hundreds of tiles to a wavefront); far too large, ranges go empty."""
    rng = np.random.default_rng(dim + page)
    for q_lens, kv_lens in (([1, 1], [5000, 70]), ([9, 40], [4200, 1500])):
        batch = Batch(rng, q_lens, kv_lens, page)
        batch.widen(keys)
        _check(cw, rng, batch, 1, 2, dim, precision)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 768])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30])
def test_scales(cw, precision, dim, scale):
    """Negative ones, zero and next to it (a mean of what is seen); keys that
    are not seen stay out of it."""
    rng = np.random.default_rng(21)
    for prefix in (0, 37):
        batch = Batch(rng, [1, 50, 2], [300, 90, 0], 16, prefix_len=prefix)
        _check(cw, rng, batch, 1, 4, dim, precision, True, scale)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 768])
def test_more_new_tokens_than_announced(cw, precision, dim):
    """Those of that sequence are unspecified; everything else is as ever."""
    rng = np.random.default_rng(22)
    batch = Batch(rng, [1, 40, 1], [700, 60, 33], 16, before=1, behind=1)
    batch.max_q_len = lambda: 1
    k, v = pages_of(rng, cw, batch, 1, dim, precision)
    q = rounded(cw, rng.standard_normal((batch.tokens, 2, dim)), precision)
    got = _run(cw, batch, k, v, q, precision, dim ** -0.5, True)
    np.testing.assert_array_equal(got[[0, -1]], np.full_like(got[[0, -1]], 3.0))
    off = _off(got, batch, k, v, q, precision, dim ** -0.5, True)
    assert np.all(off[[1, -2]] <= 1)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 768])
def test_pages_that_are_listed_twice(cw, precision, dim):
    """Sequences that share pages, and one page twice in a sequence."""
    rng = np.random.default_rng(23)
    batch = Batch(rng, [1, 20], [200, 200], 16)
    batch.page_table[1, :6] = batch.page_table[0, :6]
    batch.page_table[1, 3] = batch.page_table[1, 2]
    _check(cw, rng, batch, 1, 2, dim, precision)


@pytest.mark.parametrize("precision, dim", [("bf16", 128), ("fp32", 768)])
def test_two_graphs_side_by_side(cw, precision, dim):
    """Two captured calls on scratch of their own, replayed at once on two
    streams, with eager calls in between: every replay is the eager result."""
    hip = cw._load_hip()
    rng = np.random.default_rng(24)
    batch = Batch(rng, [1, 2], [2500, 900], 16)
    k, v = pages_of(rng, cw, batch, 2, dim, precision)
    row = 4 * dim
    with contextlib.ExitStack() as owned:
        runs = []
        for seed in range(2):
            q = rounded(cw, np.random.default_rng(seed).standard_normal((3, 4, dim)), precision)
            dev = OnDevice(cw, owned, batch, k, v, precision)
            dq, out = dev.put(cw._encode(q, precision)), dev.put(cw._encode(q, precision))
            scratch, stream, graph, run = dev.scratch(4), P(), P(), P()
            assert scratch[1] > 0
            assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
            owned.callback(hip.hipStreamDestroy, stream)
            assert hip.hipStreamBeginCapture(stream, 0) == 0
            dev.attend(dq, row, out, row, 4, 0.1, True, scratch, stream)
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            owned.callback(hip.hipGraphDestroy, graph)
            assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, P(0)) == 0
            owned.callback(hip.hipGraphExecDestroy, run)
            eager = dev.put(cw._encode(np.zeros_like(q), precision))
            runs.append((dev, dq, out, stream, run, eager, dev.scratch(4), q.shape))
        for _ in range(4):
            for dev, dq, out, stream, run, eager, mine, shape in runs:
                assert hip.hipGraphLaunch(run, stream) == 0
            for dev, dq, out, stream, run, eager, mine, shape in runs:
                assert hip.hipStreamSynchronize(stream) == 0
                dev.attend(dq, row, eager, row, 4, 0.1, True, mine)
                assert cw.cudart.hipDeviceSynchronize() == 0
                got, want = (x.download(shape, cw._bits_type(precision)) for x in (out, eager))
                np.testing.assert_array_equal(got, want)
                assert np.any(got != 0)
                out.upload(np.zeros(shape, cw._bits_type(precision)))
