"""The cache operators on the GPU against their oracle in 64 bits: rotary
positions and their gradient, appending to a paged cache, attention over it
and over a prefix that a batch shares, and a run of them together.  Inputs are
rounded to the type first, so the tolerances count the kernels' own roundings."""

import contextlib
import ctypes
import threading

import numpy as np
import pytest

import cache_oracle
from cache_cases import HALF_STEP, Batch, OnDevice, pages_of, rounded

pytestmark = pytest.mark.gpu

P = ctypes.c_void_p
TYPES = ["fp32", "fp16", "bf16"]
U = 2.0 ** -24


def _wait(cw):
    assert cw.cudart.hipDeviceSynchronize() == 0


# --------------------------------------------------------------------------
# Rotary positions
# --------------------------------------------------------------------------

def _rope_tolerance(x, y, precision, amplitude, rot, interleaved):
    """An angle is off by up to 2^-25 turns (its rounding to 32 bits) or 2 pi
    2^-25 < 4 half steps, sine and cosine by two steps (four half steps), the
    amplitude, the products and their sum by one half step each; the result is
    rounded to the type.  All relative to amplitude (|a| + |b|) of the pair."""
    x = np.abs(np.asarray(x, np.float64))
    both = x.copy()
    if interleaved:
        both[..., 0:rot:2] = both[..., 1:rot:2] = x[..., 0:rot:2] + x[..., 1:rot:2]
    else:
        both[..., :rot // 2] = both[..., rot // 2:rot] = x[..., :rot // 2] + x[..., rot // 2:rot]
    return 12 * U * max(amplitude, 1.0) * both + HALF_STEP[precision] * np.abs(y) + 1e-30


ROPE = [  # tokens, heads, dim, rot, amplitude
    (1, 12, 64, 64, 1.0), (5, 3, 128, 64, 1.2), (33, 2, 768, 768, 1.0), (7, 5, 80, 40, 1.0),
    (4, 3, 10, 6, 0.7), (3, 1, 7, 2, 1.0), (2, 2, 64, 0, 1.0), (1500, 4, 64, 32, 1.0)]


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, dim, rot, amplitude", ROPE)
def test_rope(cw, tokens, heads, dim, rot, amplitude, interleaved, precision):
    rng = np.random.default_rng(tokens + dim)
    x = rounded(cw, rng.standard_normal((tokens, heads, dim)), precision)
    positions = rng.integers(0, 100000, tokens).astype(np.int32)
    positions[:2] = [2 ** 31 - 1, -2 ** 31][:tokens]
    freqs = cw.rope_frequencies(rot)
    with cw.Rope(freqs, amplitude, interleaved) as rope:
        for inverse in (False, True):
            y = cw.run_rope(x, positions, rope, inverse, precision)
            want = cache_oracle.rope(x, positions, freqs, amplitude, interleaved, inverse)
            off = np.abs(y - want)
            assert np.all(off <= _rope_tolerance(x, want, precision, amplitude, rot, interleaved)), \
                (inverse, off.max())
            np.testing.assert_array_equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(cw, interleaved):
    """The inverse is the gradient: against the formula's (above) and against
    differences.  The map is linear, so a central difference has no error but
    rounding: <w, y(x + d) - y(x - d)> / 2 = <gradient, d>."""
    rng = np.random.default_rng(3)
    x, d, w = (rng.standard_normal((9, 4, 64)).astype(np.float32) for _ in range(3))
    positions = rng.integers(0, 5000, 9)
    with cw.Rope(cw.rope_frequencies(48), 1.1, interleaved) as rope:
        up, down = (cw.run_rope(x + s * d, positions, rope).astype(np.float64) for s in (1, -1))
        gradient = cw.run_rope(w, positions, rope, inverse=True).astype(np.float64)
    # each of the three results is off by at most 12 half steps of its pair's
    # magnitude (below 2 * 1.1 * 5 + 1), x + d by one half step more
    bound = 3 * 13 * U * 12 * np.abs(w).sum()
    assert abs((w * (up - down)).sum() / 2 - (gradient * d).sum()) < bound


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("gap", [0, 5, 128])
def test_rope_strides_and_in_place(cw, precision, interleaved, gap):
    """Heads that are columns of a wider tensor; what lies beside them stays."""
    rng = np.random.default_rng(4)
    tokens, heads, dim = 6, 3, 64
    row = heads * dim + gap
    host = rounded(cw, rng.standard_normal((tokens, row)), precision)
    x = host[:, :heads * dim].reshape(tokens, heads, dim)
    positions = np.arange(tokens, dtype=np.int32) * 31
    freqs = cw.rope_frequencies(dim)
    want = cw.run_rope  # the contiguous call's result, bit for bit
    with cw.Rope(freqs, 1.0, interleaved) as rope, \
            cw.DeviceBuffer.holding(cw._encode(host, precision)) as buf, \
            cw.DeviceBuffer.holding(positions) as pos:
        want = want(x, positions, rope, False, precision)
        cw.lib.launch_rope_kernel(buf.ptr, buf.ptr, pos.ptr, ctypes.byref(rope.args),
                                  cw.PRECISIONS[precision], tokens, heads, dim, row, row, 0, None)
        cw._lib_error_check("rope")
        _wait(cw)
        got = cw._decode(buf.download(host.shape, cw._bits_type(precision)), precision)
    np.testing.assert_array_equal(got[:, :heads * dim].reshape(x.shape), want)
    np.testing.assert_array_equal(got[:, heads * dim:], host[:, heads * dim:])


# --------------------------------------------------------------------------
# Append
# --------------------------------------------------------------------------

APPEND = [  # q_lens, kv_lens, page, kv heads, heads, dim, rot
    ([1], [1], 16, 1, 1, 64, 64),
    ([1] * 70, list(range(1, 71)), 16, 2, 4, 128, 64),
    ([5, 0, 1, 40], [17, 9, 1, 40], 3, 3, 6, 64, 32),
    ([300, 2], [777, 2], 64, 1, 2, 768, 768),
    ([4, 3], [2, 3], 1, 2, 2, 30, 10),      # more new tokens than keys; scalar pieces
    ([3, 0], [8, 0], 20, 1, 0, 256, 0)]     # no queries, no rotation


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("q_lens, kv_lens, page, kv_heads, heads, dim, rot", APPEND)
@pytest.mark.parametrize("given", [False, True])
def test_append(cw, q_lens, kv_lens, page, kv_heads, heads, dim, rot, interleaved, precision,
                given):
    rng = np.random.default_rng(sum(kv_lens) + dim)
    batch = Batch(rng, q_lens, kv_lens, page, before=2, behind=3)
    k, v = (rounded(cw, rng.standard_normal((batch.tokens, kv_heads, dim)), precision)
            for _ in range(2))
    q = rounded(cw, rng.standard_normal((batch.tokens, max(heads, 1), dim)), precision)
    positions = rng.integers(0, 9000, batch.tokens) if given else None
    freqs = cw.rope_frequencies(rot)
    with cw.PagedCache(batch.num_pages, page, kv_heads, dim, precision) as cache, \
            cw.Rope(freqs, 1.0, interleaved) as rope:
        turned = cache.append(k, v, *batch.where, q=q if heads else None, rope=rope,
                              positions=positions)
        got_k, got_v = cache.pages()
    zero = np.zeros(got_k.shape)
    want_k, want_v = cache_oracle.append(zero, zero, k, v, *batch.where, freqs, 1.0, interleaved,
                                         positions)
    # the same slots through the same map of |k|, for the tolerance
    reach = _rope_tolerance(k, cache_oracle.rope(k, np.zeros(len(k)), freqs), precision, 1.0, rot,
                            interleaved)
    reach += HALF_STEP[precision] * 2 * np.abs(k).max()
    far, _ = cache_oracle.append(zero, zero, reach, v, *batch.where)
    assert np.all(np.abs(got_k - want_k) <= far)  # exact where nothing was put: far is 0 there
    np.testing.assert_array_equal(got_v, want_v)
    if heads:
        at = {t: pos for t, _, pos in cache_oracle.places(batch.q_starts, batch.kv_lens)}
        rows = sorted(at)
        where = [at[t] if positions is None else positions[t] for t in rows]
        want = cache_oracle.rope(q[rows], where, freqs, 1.0, interleaved)
        assert np.all(np.abs(turned[rows] - want)
                      <= _rope_tolerance(q[rows], want, precision, 1.0, rot, interleaved))
        others = [t for t in range(batch.tokens) if t not in at]
        np.testing.assert_array_equal(turned[others], q[others])  # in place: as they were


def test_append_into_bad_pages(cw):
    """A page number outside the cache, a length beyond the table, a negative
    one and starts that run backwards: those tokens go nowhere, the others
    where they belong."""
    rng = np.random.default_rng(5)
    q_starts = np.array([0, 2, 4, 6, 8, 5], np.int32)   # the last runs backwards
    kv_lens = np.array([4, 4, 9, -3, 4], np.int32)      # the third is beyond its row
    table = np.array([[0, 1], [2, 99], [3, 4], [5, 6], [-1, 7]], np.int32)
    k, v = (rng.standard_normal((8, 1, 64)).astype(np.float32) for _ in range(2))
    with cw.PagedCache(8, 2, 1, 64) as cache:
        cache.append(k, v, q_starts, kv_lens, table)
        got_k, got_v = cache.pages()
    want = np.zeros_like(got_k)
    want[1, 0, :2] = k[0:2, 0]   # sequence 0: positions 2, 3 on page 1
    np.testing.assert_array_equal(got_k, want)
    want[1, 0, :2] = v[0:2, 0]
    np.testing.assert_array_equal(got_v, want)


# --------------------------------------------------------------------------
# Attention
# --------------------------------------------------------------------------

def _check_attend(cw, rng, batch, kv_heads, heads, dim, precision, causal, garbage=np.nan,
                  gap=0, scale=None, q_scale=1.5, k_scale=1.0):
    """One launch against the oracle; token rows of no sequence and the gaps
    between rows stay as they were.  Returns the output."""
    k, v = pages_of(rng, cw, batch, kv_heads, dim, precision, garbage, k_scale)
    row = heads * dim + gap
    q = rounded(cw, q_scale * rng.standard_normal((batch.tokens, row)), precision)
    scale = dim ** -0.5 if scale is None else scale
    before = np.full((batch.tokens, row), 3.0, np.float32)
    with contextlib.ExitStack() as owned:
        dev = OnDevice(cw, owned, batch, k, v, precision)
        dq, out = dev.put(cw._encode(q, precision)), dev.put(cw._encode(before, precision))
        dev.attend(dq, row, out, row, heads, scale, causal, dev.scratch(heads))
        _wait(cw)
        got = cw._decode(out.download(before.shape, cw._bits_type(precision)), precision)
    np.testing.assert_array_equal(got[:, heads * dim:], before[:, heads * dim:])
    rows = batch.rows()
    others = np.setdiff1d(np.arange(batch.tokens), rows)
    np.testing.assert_array_equal(got[others], before[others])
    qh = q[:, :heads * dim].reshape(-1, heads, dim)
    prefix = (batch.prefix_pages, batch.prefix_len) if batch.prefix_len else (None, 0)
    want, size = cache_oracle.attend(qh, k, v, *batch.where, scale, causal, *prefix)
    got = got[:, :heads * dim].reshape(qh.shape)
    tol = cache_oracle.attend_tolerance(want, size, dim,
                                        batch.prefix_len + int(max(batch.kv_lens, default=0)),
                                        HALF_STEP[precision])
    off = np.abs(got - want)[rows]
    assert np.all(np.isfinite(got[rows]))
    assert np.all(off <= tol[rows]), (off.max(), (off / tol[rows]).max())
    return got


ATTEND = [  # q_lens, kv_lens, page, (kv heads, heads)
    ([1], [1], 16, (1, 1)),
    ([1], [784], 16, (3, 3)),
    ([1, 1, 1], [33, 1, 700], 20, (2, 8)),
    ([1] * 5, [5, 0, 64, 31, 1], 16, (1, 7)),             # an empty sequence
    ([7, 0, 130, 1], [7, 12, 190, 65], 16, (2, 6)),       # prompts, pieces, nothing new
    ([5, 40], [3, 33], 8, (1, 2)),                        # tokens that see no key
    ([65], [65], 1, (1, 1)),                              # pages of one slot
    ([33, 17], [500, 257], 128, (1, 16)),
    ([257], [300], 48, (1, 4)),
]


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256, 768])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens, kv_lens, page, kvh", ATTEND)
def test_attention(cw, q_lens, kv_lens, page, kvh, dim, causal, precision):
    rng = np.random.default_rng(sum(kv_lens) + dim)
    batch = Batch(rng, q_lens, kv_lens, page, before=1, behind=2)
    _check_attend(cw, rng, batch, kvh[0], kvh[1], dim, precision, causal, gap=8)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim, kvh", [(64, (2, 2)), (128, (2, 8)), (768, (1, 1))])
def test_attention_of_long_ragged_batches(cw, dim, kvh, precision):
    """Sequences that are divided over workgroups, unlike ones at once."""
    rng = np.random.default_rng(7)
    batch = Batch(rng, [1, 1, 2, 1, 1], [5000, 1, 3011, 128, 1025], 16)
    _check_attend(cw, rng, batch, kvh[0], kvh[1], dim, precision, True)


@pytest.mark.parametrize("precision", TYPES)
def test_attention_of_many_sequences(cw, precision):
    """More sequences than a wavefront has lanes, some without tokens."""
    rng = np.random.default_rng(8)
    q_lens = [int(n) for n in rng.integers(0, 4, 150)]
    kv_lens = [n + int(m) for n, m in zip(q_lens, rng.integers(0, 60, 150))]
    batch = Batch(rng, q_lens, kv_lens, 16, before=3)
    _check_attend(cw, rng, batch, 2, 4, 64, precision, True)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 768])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_large_scores(cw, dim, precision, sign):
    """Scores of several hundred, so that one key takes all, growing along
    the keys and falling (every rescaling, and none)."""
    rng = np.random.default_rng(9)
    batch = Batch(rng, [40, 1], [600, 300], 16)
    k, v = pages_of(rng, cw, batch, 1, dim, precision)
    for b in range(2):
        n = int(batch.kv_lens[b])
        ramp = np.linspace(-1, 1, n) * sign
        for c in range(n):
            k[batch.page_table[b, c // 16], 0, c % 16] = rounded(
                cw, np.full(dim, 4 * ramp[c]), precision)
    q = rounded(cw, np.full((batch.tokens, 2, dim), 8.0), precision)
    where = batch.where
    with contextlib.ExitStack() as owned:
        dev = OnDevice(cw, owned, batch, k, v, precision)
        dq, out = dev.put(cw._encode(q, precision)), dev.put(cw._encode(q, precision))
        dev.attend(dq, 2 * dim, out, 2 * dim, 2, dim ** -0.5, True, dev.scratch(2))
        _wait(cw)
        got = cw._decode(out.download(q.shape, cw._bits_type(precision)), precision)
    want, size = cache_oracle.attend(q, k, v, *where, dim ** -0.5)
    tol = cache_oracle.attend_tolerance(want, size, dim, 600, HALF_STEP[precision])
    assert np.all(np.abs(got - want) <= tol)


def _attend_raw(cw, batch, k, v, q, precision, causal=True, q_starts=None, kv_lens=None,
                table=None):
    heads, dim = q.shape[1:]
    with contextlib.ExitStack() as owned:
        dev = OnDevice(cw, owned, batch, k, v, precision)
        if q_starts is not None:
            dev.q_starts.upload(np.asarray(q_starts, np.int32))
        if kv_lens is not None:
            dev.kv_lens.upload(np.asarray(kv_lens, np.int32))
        if table is not None:
            dev.table.upload(np.asarray(table, np.int32))
        dq, out = dev.put(cw._encode(q, precision)), dev.put(cw._encode(np.full_like(q, 3.0), precision))
        dev.attend(dq, heads * dim, out, heads * dim, heads, dim ** -0.5, causal,
                   dev.scratch(heads))
        _wait(cw)
        return cw._decode(out.download(q.shape, cw._bits_type(precision)), precision)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256, 768])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("m", [6, 150])
def test_keys_that_are_not_seen_do_not_count(cw, precision, dim, bad, m):
    """NaN and infinities in the keys and values of a prompt's later tokens:
    the earlier tokens come out as without them, those that see them do not."""
    rng = np.random.default_rng(10)
    batch = Batch(rng, [m], [m + 3], 16)
    k, v = pages_of(rng, cw, batch, 1, dim, precision)
    q = rounded(cw, np.abs(rng.standard_normal((m, 2, dim))), precision)
    want, size = cache_oracle.attend(q, k, v, *batch.where, dim ** -0.5)
    tol = cache_oracle.attend_tolerance(want, size, dim, m + 3, HALF_STEP[precision])
    first = 3 + m // 2  # cache position of the first bad key
    for c in range(first, m + 3, 2):
        page, slot = batch.page_table[0, c // 16], c % 16
        v[page, 0, slot] = bad
        if c % 4 < 2:
            k[page, 0, slot] = bad
    got = _attend_raw(cw, batch, k, v, q, precision)
    assert np.all(np.abs(got - want)[:m // 2] <= tol[:m // 2])
    if np.isnan(bad):
        assert np.all(np.isnan(got[m // 2:]))
    else:
        assert not np.any(np.isfinite(got[m // 2:]))


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 768])
@pytest.mark.parametrize("n", [40, 2000])
@pytest.mark.parametrize("m", [1, 37])
def test_bad_sequences_come_out_as_nan(cw, precision, dim, n, m):
    """A bad page number, a length beyond the table, a negative one: NaN for
    that sequence; the others as ever.  A bad page that no key lies on is none."""
    rng = np.random.default_rng(11)
    batch = Batch(rng, [m] * 5, [n] * 5, 16)
    k, v = pages_of(rng, cw, batch, 2, dim, precision)
    q = rounded(cw, rng.standard_normal((batch.tokens, 2, dim)), precision)
    clean = _attend_raw(cw, batch, k, v, q, precision, causal=False)
    wide = batch.page_table.shape[1] * 16
    lens = [n, n, wide + 1, -1, n]
    for page in (batch.num_pages, -1, 2 ** 31 - 1):
        table = batch.page_table.copy()
        table[1, n // 32] = page
        table[2] = page
        got = _attend_raw(cw, batch, k, v, q, precision, False, kv_lens=lens, table=table)
        for b, nan in enumerate([False, True, True, True, False]):
            rows = slice(b * m, (b + 1) * m)
            if nan:
                assert np.all(np.isnan(got[rows])), b
            else:
                np.testing.assert_array_equal(got[rows], clean[rows])


def test_starts_out_of_range(cw):
    """q_starts below zero, beyond the tokens and running backwards: nothing
    is read or written out of the tensors, rows of no sequence stay."""
    rng = np.random.default_rng(12)
    batch = Batch(rng, [4, 4, 4], [40, 40, 40], 16)
    k, v = pages_of(rng, cw, batch, 1, 64, "bf16")
    q = rounded(cw, rng.standard_normal((12, 2, 64)), "bf16")
    clean = _attend_raw(cw, batch, k, v, q, "bf16", causal=False)
    got = _attend_raw(cw, batch, k, v, q, "bf16", False, q_starts=[0, 4, 2, 4000])
    np.testing.assert_array_equal(got[:2], clean[:2])
    got = _attend_raw(cw, batch, k, v, q, "bf16", False, q_starts=[-50, 4, 8, 8])
    np.testing.assert_array_equal(got[4:8], clean[4:8])
    np.testing.assert_array_equal(got[8:], np.full_like(got[8:], 3.0))


@pytest.mark.parametrize("precision", TYPES)
def test_attention_is_reproducible(cw, precision):
    rng = np.random.default_rng(13)
    batch = Batch(rng, [1, 1, 70], [4000, 900, 70], 16)
    k, v = pages_of(rng, cw, batch, 2, 128, precision)
    q = rounded(cw, rng.standard_normal((72, 8, 128)), precision)
    first = _attend_raw(cw, batch, k, v, q, precision)
    for _ in range(4):
        np.testing.assert_array_equal(_attend_raw(cw, batch, k, v, q, precision), first)


@pytest.mark.parametrize("precision, dim, pages", [("bf16", 64, 2_200_000), ("fp32", 128, 560_000)])
def test_pages_beyond_four_gigabytes(cw, precision, dim, pages):
    """A cache of over 4 GiB of keys (and over 2^31 elements in 16 bits) whose
    last pages are in use: append, then attend."""
    rng = np.random.default_rng(14)
    size, n = 16, 40
    table = np.array([[pages - 1, pages - 3, pages - 2]], np.int32)
    k, v = (rounded(cw, rng.standard_normal((n, 1, dim)), precision) for _ in range(2))
    q = rounded(cw, rng.standard_normal((n, 2, dim)), precision)
    bytes_ = pages * size * dim * (4 if precision == "fp32" else 2)
    assert bytes_ > 2 ** 32
    with contextlib.ExitStack() as owned:
        new = lambda a: owned.enter_context(cw.DeviceBuffer.holding(a))  # noqa: E731
        kp, vp = (owned.enter_context(cw.DeviceBuffer(bytes_)) for _ in range(2))
        cache = cw.CacheArgs(kp.ptr.value, vp.ptr.value, cw.PRECISIONS[precision], pages, 1, size,
                             dim)
        ints = [new(np.array(a, np.int32)) for a in ([0, n], [n], table)]
        batch = cw.BatchArgs(*(b.ptr.value for b in ints), 1, 3, n, n, n)
        dk, dv, dq = (new(cw._encode(a, precision)) for a in (k, v, q))
        out = owned.enter_context(cw.DeviceBuffer(dq.nbytes))
        ref = ctypes.byref
        cw.lib.launch_cache_append_kernel(ref(cache), ref(batch), dk.ptr, dim, dv.ptr, dim, None,
                                          0, None, 0, 0, None, None, None)
        cw._lib_error_check("append")
        need = cw.lib.xattn_cache_attention_scratch(ref(cache), ref(batch), None, 2)
        scratch = owned.enter_context(cw.DeviceBuffer(need))
        cw.lib.launch_cache_attention_kernel(ref(cache), ref(batch), dq.ptr, 2 * dim, out.ptr,
                                             2 * dim, 2, dim ** -0.5, 1, scratch.ptr, need, None)
        cw._lib_error_check("attend")
        _wait(cw)
        got = cw._decode(out.download(q.shape, cw._bits_type(precision)), precision)
    small = np.zeros((3, 1, size, dim), np.float32)
    ks, vs = small.copy(), small.copy()
    for c in range(n):
        ks[[0, 1, 2][c // size], 0, c % size], vs[[0, 1, 2][c // size], 0, c % size] = k[c], v[c]
    where = (np.array([0, n]), np.array([n]), np.array([[0, 1, 2]]))
    want, size_ = cache_oracle.attend(q, ks, vs, *where, dim ** -0.5)
    assert np.all(np.abs(got - want) <= cache_oracle.attend_tolerance(
        want, size_, dim, n, HALF_STEP[precision]))


# --------------------------------------------------------------------------
# A shared prefix
# --------------------------------------------------------------------------

PREFIX = [  # q_lens, kv_lens, prefix, page, (kv heads, heads)
    ([1], [1], 1, 16, (1, 1)),
    ([1] * 6, [9, 0, 33, 1, 200, 64], 1025, 16, (2, 8)),  # one has no keys of its own
    ([17] * 4, [230, 17, 40, 100], 300, 20, (1, 3)),
    ([1, 0, 140], [70, 8, 140], 95, 32, (2, 2)),
    ([3, 5], [1, 0], 7, 1, (1, 4)),                       # tokens that see the prefix alone
    ([1] * 40, [16] * 40, 2500, 64, (1, 4)),
]


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256, 768])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens, kv_lens, prefix, page, kvh", PREFIX)
def test_prefix_attention(cw, q_lens, kv_lens, prefix, page, kvh, dim, causal, precision):
    rng = np.random.default_rng(prefix + dim)
    batch = Batch(rng, q_lens, kv_lens, page, before=1, behind=2, prefix_len=prefix)
    _check_attend(cw, rng, batch, kvh[0], kvh[1], dim, precision, causal, gap=8)


@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("prefix", [0, 40])
def test_prefix_of_nothing_and_bad_prefix(cw, precision, prefix):
    rng = np.random.default_rng(15)
    batch = Batch(rng, [1, 3], [5, 30], 16, prefix_len=prefix)
    k, v = pages_of(rng, cw, batch, 1, 64, precision)
    q = rounded(cw, rng.standard_normal((4, 2, 64)), precision)
    with cw.PagedCache(batch.num_pages, 16, 1, 64, precision) as cache:
        cache._k.upload(cw._encode(k, precision))
        cache._v.upload(cw._encode(v, precision))
        if not prefix:
            np.testing.assert_array_equal(
                cache.attend(q, *batch.where, prefix_pages=[], prefix_len=0),
                cache.attend(q, *batch.where))
            return
        for bad in (-1, batch.num_pages):
            pages = batch.prefix_pages.copy()
            pages[1] = bad
            assert np.all(np.isnan(cache.attend(q, *batch.where, prefix_pages=pages,
                                                prefix_len=prefix)))


# --------------------------------------------------------------------------
# Together, as they are used
# --------------------------------------------------------------------------

@pytest.mark.parametrize("precision", TYPES)
@pytest.mark.parametrize("dim, kvh", [(64, (2, 4)), (768, (1, 1))])
def test_prompt_then_token_by_token(cw, precision, dim, kvh):
    """A prompt is put into the cache and answered, then five tokens one by
    one, two sequences at a time: every token's output is that of causal
    attention over the rotated keys of its whole sequence."""
    rng = np.random.default_rng(16)
    kv_heads, heads = kvh
    prompt, more, page = [37, 5], 5, 16
    total = [n + more for n in prompt]
    k, v = ([rounded(cw, rng.standard_normal((n, kv_heads, dim)), precision) for n in total]
            for _ in range(2))
    q = [rounded(cw, rng.standard_normal((n, heads, dim)), precision) for n in total]
    table = np.array([[4, 1, 5], [0, -1, -1]], np.int32)
    freqs = cw.rope_frequencies(dim)
    outs = [[], []]
    with cw.PagedCache(6, page, kv_heads, dim, precision) as cache, cw.Rope(freqs) as rope:
        done = [0, 0]
        for step in range(more + 1):
            take = prompt if step == 0 else [1, 1]
            rows = [slice(d, d + n) for d, n in zip(done, take)]
            done = [d + n for d, n in zip(done, take)]
            where = (np.array([0, take[0], sum(take)]), np.array(done), table)
            pick = lambda x: np.concatenate([x[b][rows[b]] for b in range(2)])  # noqa: E731
            turned = cache.append(pick(k), pick(v), *where, q=pick(q), rope=rope)
            out = cache.attend(turned, *where)
            for b, part in enumerate(np.split(out, [take[0]])):
                outs[b].append(part)
        k_pages, v_pages = cache.pages()
    for b in range(2):
        n = total[b]
        at = np.arange(n)
        turned = rounded(cw, cache_oracle.rope(q[b], at, freqs), precision)
        where = (np.array([0, n]), np.array([n]), table[b:b + 1])
        stored = cache_oracle.gather(k_pages, table[b], n)
        want_k = cache_oracle.rope(k[b], at, freqs)
        assert np.all(np.abs(stored - want_k) <= _rope_tolerance(k[b], want_k, precision, 1.0, dim,
                                                                 False))
        want, size = cache_oracle.attend(turned, k_pages, v_pages, *where, dim ** -0.5)
        tol = cache_oracle.attend_tolerance(want, size, dim, n, HALF_STEP[precision])
        # a query's own rounding may fall on the other side: a whole step of each
        # of its elements moves a score by up to two half steps of its terms
        step_ = 2 * max(HALF_STEP[precision], 16 * U)
        tol = tol + 2 * step_ * size["terms"][..., None] * size["mass"]
        assert np.all(np.abs(np.concatenate(outs[b]) - want) <= tol)


@pytest.mark.parametrize("precision", TYPES)
def test_captured_step_is_replayed(cw, precision):
    """Append and attention recorded into a graph once; the lengths on the
    device then grow token by token between its replays, with eager calls of
    another batch (on scratch of their own) in between.  Every replay is the
    eager result."""
    hip = cw._load_hip()
    rng = np.random.default_rng(17)
    dim, heads, kv_heads, n0 = 64, 4, 2, 300
    batch = Batch(rng, [1, 1], [n0, 40], 16)
    table = np.arange(2 * 24, dtype=np.int32).reshape(2, 24)
    batch.page_table, batch.num_pages = table, 48
    k, v = pages_of(rng, cw, batch, kv_heads, dim, precision, garbage=0.0)
    new = rounded(cw, rng.standard_normal((3, 2, heads, dim)), precision)
    row = heads * dim
    with contextlib.ExitStack() as owned:
        dev = OnDevice(cw, owned, batch, k, v, precision)
        other = OnDevice(cw, owned, batch, k, v, precision)
        dev.batch.max_kv_len = other.batch.max_kv_len = 24 * 16  # as long as they grow
        rope = owned.enter_context(cw.Rope(cw.rope_frequencies(dim)))
        q, turned, out, out2 = (dev.put(cw._encode(new[0], precision)) for _ in range(4))
        scratch, mine = dev.scratch(heads), other.scratch(heads)
        ref, stream, graph, run = ctypes.byref, P(), P(), P()
        assert hip.hipStreamCreate(ctypes.byref(stream)) == 0

        def step(d, out, scratch, stream):
            cw.lib.launch_cache_append_kernel(
                ref(d.cache), ref(d.batch), q.ptr, row, q.ptr, row, q.ptr, row, turned.ptr, row,
                heads, None, ref(rope.args), stream)
            d.attend(turned, row, out, row, heads, 0.125, True, scratch, stream)
            cw._lib_error_check("step")

        try:
            assert hip.hipStreamBeginCapture(stream, 0) == 0
            step(dev, out, scratch, stream)
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, P(0)) == 0
            for i in range(4):
                q.upload(cw._encode(new[i % 3], precision))
                lens = batch.kv_lens + i
                for d in (dev, other):
                    d.kv_lens.upload(lens)
                assert hip.hipGraphLaunch(run, stream) == 0
                assert hip.hipStreamSynchronize(stream) == 0
                got = out.download(new[0].shape, cw._bits_type(precision))
                step(other, out2, mine, None)
                _wait(cw)
                want = out2.download(new[0].shape, cw._bits_type(precision))
                np.testing.assert_array_equal(got, want)
                assert np.any(got != 0)
        finally:
            _wait(cw)
            hip.hipGraphExecDestroy(run)
            hip.hipGraphDestroy(graph)
            hip.hipStreamDestroy(stream)


def test_two_threads_on_their_own_streams(cw):
    """Two host threads launch at once, each on its own stream and scratch."""
    hip = cw._load_hip()
    rng = np.random.default_rng(18)
    jobs = []
    with contextlib.ExitStack() as owned:
        for precision, lens in (("bf16", [3000, 50]), ("fp32", [70, 2000])):
            batch = Batch(rng, [1, 2], lens, 16)
            k, v = pages_of(rng, cw, batch, 2, 128, precision)
            q = rounded(cw, rng.standard_normal((3, 4, 128)), precision)
            dev = OnDevice(cw, owned, batch, k, v, precision)
            stream = P()
            assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
            jobs.append((dev, dev.put(cw._encode(q, precision)), dev.put(cw._encode(q, precision)),
                         dev.scratch(4), stream, precision, batch, k, v, q))
        failures = []

        def work(dev, dq, out, scratch, stream, *rest):
            try:
                for _ in range(20):
                    dev.attend(dq, 512, out, 512, 4, 0.1, True, scratch, stream)
            except Exception as e:  # reported after the join
                failures.append(repr(e))

        threads = [threading.Thread(target=work, args=job) for job in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        _wait(cw)
        assert not failures, failures
        for dev, dq, out, scratch, stream, precision, batch, k, v, q in jobs:
            got = cw._decode(out.download(q.shape, cw._bits_type(precision)), precision)
            want, size = cache_oracle.attend(q, k, v, *batch.where, 0.1)
            tol = cache_oracle.attend_tolerance(want, size, 128, 3000, HALF_STEP[precision])
            assert np.all(np.abs(got - want) <= tol)
            hip.hipStreamDestroy(stream)
