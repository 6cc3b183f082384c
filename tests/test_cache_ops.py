"""CPU tests of the cache operators: their oracle against closed forms, the
rotary frequencies, and every refusal (decided before any HIP call, so no
GPU is needed to see it)."""

import ctypes

import numpy as np
import pytest

import cache_oracle
from cache_cases import Batch

P = ctypes.c_void_p
OK, INVALID, UNSUPPORTED = 0, 1, 2


# --------------------------------------------------------------------------
# The oracle
# --------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rope_is_a_rotation(interleaved):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 10))
    freqs = np.array([0.25, 1 / 3])
    y = cache_oracle.rope(x, [0, 1, 3], freqs, interleaved=interleaved)
    np.testing.assert_array_equal(y[0], x[0])                # position 0
    np.testing.assert_array_equal(y[..., 4:], x[..., 4:])    # behind rot_dim
    a, b = (0, 1) if interleaved else (0, 2)                 # first pair: a quarter turn
    np.testing.assert_allclose(y[1, :, a], -x[1, :, b], atol=1e-15)
    np.testing.assert_allclose(y[1, :, b], x[1, :, a], atol=1e-15)
    a, b = (2, 3) if interleaved else (1, 3)                 # second pair: a whole turn
    np.testing.assert_allclose(y[2, :, [a, b]], x[2, :, [a, b]], atol=1e-15)
    back = cache_oracle.rope(y, [0, 1, 3], freqs, interleaved=interleaved, inverse=True)
    np.testing.assert_allclose(back, x, atol=1e-15)


def test_oracle_attend_closed_forms():
    rng = np.random.default_rng(1)
    batch = Batch(rng, [2, 1, 3], [5, 0, 3], 2, before=1, behind=1)
    k = np.zeros((batch.num_pages, 1, 2, 4))
    v = rng.standard_normal(k.shape)
    q = rng.standard_normal((batch.tokens, 2, 4))
    out, _ = cache_oracle.attend(q, k, v, *batch.where, 1.0)
    rows = cache_oracle.gather(v, batch.page_table[0], 5)[:, 0]
    np.testing.assert_allclose(out[1], [rows[:4].mean(0)] * 2)  # K = 0: the mean of what is seen
    np.testing.assert_allclose(out[2], [rows.mean(0)] * 2)
    assert not out[3].any() and not out[0].any() and not out[7].any()
    rows = cache_oracle.gather(v, batch.page_table[2], 3)[:, 0]
    np.testing.assert_allclose(out[4, 0], rows[0])              # one key
    out, _ = cache_oracle.attend(q, k, v, *batch.where, 1.0, causal=False)
    np.testing.assert_allclose(out[4, 1], rows.mean(0))


# --------------------------------------------------------------------------
# Frequencies
# --------------------------------------------------------------------------

def test_rope_frequencies(cw):
    i = np.arange(32)
    plain = 10000.0 ** (-i / 32) / (2 * np.pi)
    np.testing.assert_allclose(cw.rope_frequencies(64), plain, rtol=1e-14)
    np.testing.assert_allclose(cw.rope_frequencies(64, scaling="linear", factor=8.0), plain / 8,
                               rtol=1e-14)
    base = cw.rope_frequencies(64, scaling="base", factor=8.0)
    np.testing.assert_allclose([base[0], base[-1]], [plain[0], plain[-1] / 8], rtol=1e-13)
    parts = cw.rope_frequencies(64, scaling="parts", factor=8.0, trained_len=4096)
    turns = plain * 4096
    assert (turns >= 32).any() and (turns <= 1).any()
    np.testing.assert_allclose(parts[turns >= 32], plain[turns >= 32], rtol=1e-14)
    np.testing.assert_allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14)
    keep = (turns - 1) / 31
    mid = (turns > 1) & (turns < 32)
    np.testing.assert_allclose(parts[mid], (plain * keep + plain / 8 * (1 - keep))[mid],
                               rtol=1e-14)
    assert cw.rope_frequencies(0).size == 0


@pytest.mark.parametrize("kw", [
    dict(rot_dim=7), dict(rot_dim=-2), dict(rot_dim=8, base=0.0), dict(rot_dim=8, base=np.inf),
    dict(rot_dim=8, factor=-1.0), dict(rot_dim=2, scaling="base", factor=2.0),
    dict(rot_dim=8, scaling="parts", factor=2.0),
    dict(rot_dim=8, scaling="parts", factor=2.0, trained_len=64, slow_turns=4, fast_turns=4)])
def test_rope_frequencies_refusals(cw, kw):
    with pytest.raises(RuntimeError, match="code 1"):
        cw.rope_frequencies(**kw)
    assert cw.lib.xattn_get_last_error() == OK
    with pytest.raises(ValueError):
        cw.rope_frequencies(8, scaling="cubic")


# --------------------------------------------------------------------------
# Refusals.  The addresses are never followed: every call below is refused, or
# has nothing to do.
# --------------------------------------------------------------------------

def _said(cw):
    code = cw.lib.xattn_get_last_error()
    return code, cw.lib.xattn_get_last_error_string().decode() if code else ""


def _rope(cw, **kw):
    a = dict(x=0x1000, y=0x2000, positions=0x3000, freqs=0x4000, amplitude=1.0, rot=64,
             interleaved=0, dtype=2, tokens=3, heads=2, dim=64, xs=128, ys=128, inverse=0,
             rope=True)
    a.update(kw)
    rope = cw.RopeArgs(a["freqs"], a["amplitude"], a["rot"], a["interleaved"])
    cw.lib.launch_rope_kernel(a["x"], a["y"], a["positions"],
                              ctypes.byref(rope) if a["rope"] else None, a["dtype"], a["tokens"],
                              a["heads"], a["dim"], a["xs"], a["ys"], a["inverse"], None)
    return _said(cw)


@pytest.mark.parametrize("kw, code, word", [
    (dict(dtype=3), INVALID, "type"), (dict(dtype=-1), INVALID, "type"),
    (dict(tokens=-1), INVALID, "tokens=-1"), (dict(heads=-1), INVALID, "heads=-1"),
    (dict(dim=0), INVALID, "dim=0"), (dict(rot=63), INVALID, "rot_dim"),
    (dict(rot=66), INVALID, "rot_dim"), (dict(rot=-2), INVALID, "rot_dim"),
    (dict(rot=2050, dim=4096, xs=8192, ys=8192), UNSUPPORTED, "rot_dim"),
    (dict(freqs=None), INVALID, "frequencies"), (dict(freqs=0x4004), INVALID, "frequencies"),
    (dict(amplitude=np.nan), INVALID, "amplitude"), (dict(rope=False), INVALID, "rotation"),
    (dict(x=None), INVALID, "x"), (dict(y=None), INVALID, "y"),
    (dict(x=0x1001), INVALID, "aligned"), (dict(xs=127), INVALID, "rows"),
    (dict(ys=100), INVALID, "rows"), (dict(y=0x1000, ys=256), INVALID, "in place"),
    (dict(positions=None), INVALID, "positions"), (dict(positions=0x3002), INVALID, "positions"),
    (dict(heads=1 << 20, dim=256, xs=1 << 28, ys=1 << 28), UNSUPPORTED, "elements"),
    (dict(tokens=0, x=None), OK, ""), (dict(heads=0, x=None), OK, "")])
def test_rope_refusals(cw, kw, code, word):
    got, msg = _rope(cw, **kw)
    assert got == code and word in msg, (got, msg)


def _args(cw, **kw):
    c = dict(k=0x10000, v=0x20000, dtype=2, num_pages=9, kv_heads=2, page_size=16, dim=64)
    b = dict(q_starts=0x3000, kv_lens=0x4000, page_table=0x5000, batch=2, table_width=4,
             tokens=5, max_q_len=3, max_kv_len=60)
    c.update({n: kw[n] for n in c if n in kw})
    b.update({n: kw[n] for n in b if n in kw})
    return cw.CacheArgs(*c.values()), cw.BatchArgs(*b.values())


CACHE_REFUSALS = [
    (dict(dtype=5), INVALID, "type"), (dict(num_pages=-1), INVALID, "num_pages=-1"),
    (dict(kv_heads=0), INVALID, "kv_heads=0"), (dict(page_size=0), INVALID, "page_size=0"),
    (dict(dim=0), INVALID, "dim=0"), (dict(k=None), INVALID, "NULL pages"),
    (dict(v=None), INVALID, "NULL pages"), (dict(k=0x10008), INVALID, "16-byte"),
    (dict(num_pages=1 << 30), UNSUPPORTED, "2^32"),
    (dict(kv_heads=1 << 20, page_size=1 << 12, num_pages=1), UNSUPPORTED, "rows"),
    (dict(batch=-1), INVALID, "batch=-1"), (dict(table_width=-1), INVALID, "table_width=-1"),
    (dict(tokens=-5), INVALID, "tokens=-5"), (dict(max_q_len=-1), INVALID, "max_q_len"),
    (dict(max_kv_len=-1), INVALID, "max_kv_len"), (dict(q_starts=None), INVALID, "q_starts"),
    (dict(kv_lens=None), INVALID, "kv_lens"), (dict(page_table=None), INVALID, "page_table"),
    (dict(kv_lens=0x4001), INVALID, "4-byte")]


def _append(cw, **kw):
    cache, batch = _args(cw, **kw)
    a = dict(tk=0x60000, ks=128, tv=0x70000, vs=128, q=0x80000, qs=256, q_out=0x90000, qos=256,
             heads=4, positions=None, freqs=0xa000, rot=64)
    a.update({n: kw[n] for n in a if n in kw})
    rope = cw.RopeArgs(a["freqs"], 1.0, a["rot"], 0)
    cw.lib.launch_cache_append_kernel(
        ctypes.byref(cache), ctypes.byref(batch), a["tk"], a["ks"], a["tv"], a["vs"], a["q"],
        a["qs"], a["q_out"], a["qos"], a["heads"], a["positions"], ctypes.byref(rope), None)
    return _said(cw)


@pytest.mark.parametrize("kw, code, word", CACHE_REFUSALS + [
    (dict(tk=None), INVALID, "NULL k"), (dict(tv=None), INVALID, "NULL v"),
    (dict(ks=127), INVALID, "k rows"), (dict(vs=0), INVALID, "v rows"),
    (dict(tk=0x60001), INVALID, "aligned"), (dict(q_out=None), INVALID, "q_out"),
    (dict(qs=255), INVALID, "q rows"), (dict(qos=0), INVALID, "q_out rows"),
    (dict(heads=0), INVALID, "query heads"), (dict(rot=65), INVALID, "rot_dim"),
    (dict(q_out=0x80000, qos=512), INVALID, "in place"),
    (dict(freqs=None), INVALID, "frequencies"), (dict(positions=0x3), INVALID, "positions"),
    (dict(tokens=0, tk=None), OK, ""), (dict(batch=0, q_starts=None), OK, "")])
def test_append_refusals(cw, kw, code, word):
    got, msg = _append(cw, **kw)
    assert got == code and word in msg, (got, msg)


def _attend(cw, **kw):
    cache, batch = _args(cw, **kw)
    a = dict(q=0x60000, qs=256, out=0x70000, os=256, heads=4, scale=0.125, causal=1,
             scratch=0x80000, scratch_bytes=1 << 40, pages=0x9000, listed=3, len=40, with_prefix=False)
    a.update({n: kw[n] for n in a if n in kw})
    args, fn = [ctypes.byref(cache), ctypes.byref(batch)], cw.lib.launch_cache_attention_kernel
    if a["with_prefix"] is not False:
        prefix = cw.PrefixArgs(a["pages"], a["listed"], a["len"])
        args.append(ctypes.byref(prefix) if a["with_prefix"] else None)
        fn = cw.lib.launch_prefix_attention_kernel
    fn(*args, a["q"], a["qs"], a["out"], a["os"], a["heads"], a["scale"], a["causal"],
       a["scratch"], a["scratch_bytes"], None)
    return _said(cw)


ATTEND_REFUSALS = CACHE_REFUSALS + [
    (dict(dim=96, qs=384, os=384), UNSUPPORTED, "dim=96"), (dict(heads=3), INVALID, "3 heads"),
    (dict(heads=0), INVALID, "0 heads"), (dict(scale=np.inf), INVALID, "scale"),
    (dict(q=None), INVALID, "NULL q"), (dict(out=None), INVALID, "NULL out"),
    (dict(qs=255), INVALID, "q rows"), (dict(qs=260), INVALID, "16-byte"),
    (dict(os=252), INVALID, "out rows"), (dict(out=0x70004), INVALID, "16-byte"),
    (dict(out=0x60000), INVALID, "may not be q"),
    (dict(tokens=1 << 30, max_q_len=1), UNSUPPORTED, "tokens"),
    (dict(tokens=0, q=None), OK, ""), (dict(max_q_len=0, q=None), OK, ""),
    (dict(batch=0, q_starts=None), OK, "")]


@pytest.mark.parametrize("kw, code, word", ATTEND_REFUSALS)
@pytest.mark.parametrize("with_prefix", [False, True])
def test_attention_refusals(cw, kw, code, word, with_prefix):
    got, msg = _attend(cw, with_prefix=with_prefix, **kw)
    assert got == code and word in msg, (got, msg)


@pytest.mark.parametrize("kw, code, word", [
    (dict(with_prefix=None), INVALID, "NULL prefix"), (dict(len=-1), INVALID, "prefix of -1"),
    (dict(listed=-1), INVALID, "on -1 pages"), (dict(len=49), INVALID, "49 keys on 3 pages"),
    (dict(pages=None), INVALID, "prefix pages"), (dict(pages=0x9002), INVALID, "4-byte")])
def test_prefix_refusals(cw, kw, code, word):
    got, msg = _attend(cw, **{"with_prefix": True, **kw})
    assert got == code and word in msg, (got, msg)


def test_host_api_refusals(cw):
    """Shapes that do not fit are refused before anything is allocated."""
    cache = object.__new__(cw.PagedCache)  # no device memory behind it
    cache.shape, cache.precision, cache.code = (4, 2, 16, 96), "fp32", 0
    q = np.zeros((1, 4, 96), np.float32)
    with pytest.raises(cw.DesignLimited):
        cache.attend(q, [0, 1], [1], [[0]])
    for bad in (q[..., :64], q[0]):
        with pytest.raises(ValueError):
            cache.append(bad, bad, [0, 1], [1], [[0]])
    with pytest.raises(ValueError):
        cw.PagedCache(0, 16, 1, 64)
    with pytest.raises(ValueError):
        cw.PagedCache(1, 16, 1, 64, "fp8")


# --------------------------------------------------------------------------
# Sizes past a launch's grid, and positions past an int's sums
# --------------------------------------------------------------------------

WIDE = dict(dim=2048, rot=2048)


def test_more_workgroups_than_a_grid_has(cw):
    many = 1 << 26
    got, msg = _rope(cw, tokens=many, heads=1, xs=2048, ys=2048, **WIDE)
    assert got == UNSUPPORTED and "workgroups" in msg, (got, msg)
    got, msg = _append(cw, tokens=many, kv_heads=1, heads=1, ks=2048, vs=2048, qs=2048, qos=2048,
                       **WIDE)
    assert got == UNSUPPORTED and "workgroups" in msg, (got, msg)
    for with_prefix in (False, True):
        got, msg = _attend(cw, with_prefix=with_prefix, tokens=many, batch=many, max_q_len=1,
                           kv_heads=1, heads=1, qs=64, os=64)
        assert got == UNSUPPORTED and "workgroups" in msg, (got, msg)


def test_more_keys_than_positions_go_to(cw):
    for call in (_append, _attend):
        got, msg = call(cw, table_width=(1 << 26) + 1)
        assert got == UNSUPPORTED and "2^30" in msg, (got, msg)
    got, msg = _attend(cw, with_prefix=True, listed=1 << 27, len=(1 << 30) + 1)
    assert got == UNSUPPORTED and "2^30" in msg, (got, msg)


def test_work_is_not_divided_without_need(cw):
    """Short sequences, and as many as the device has room for, need no scratch."""
    def need(**kw):
        cache, batch = _args(cw, **kw)
        return cw.lib.xattn_cache_attention_scratch(ctypes.byref(cache), ctypes.byref(batch), None,
                                                    4)
    assert need(tokens=1, batch=1, max_q_len=1, max_kv_len=60) == 0
    assert need(tokens=1, batch=1, max_q_len=1, max_kv_len=60000, table_width=10000) > 0
    assert need(tokens=4096, batch=4096, max_q_len=1, max_kv_len=60000, table_width=10000) == 0
    assert need(tokens=1 << 27, batch=1 << 27, max_q_len=1, max_kv_len=60000) == 0  # refused
    assert cw.HAS_CACHE


@pytest.mark.parametrize("q_starts, kv_lens, table", [
    ([0, 1], [2 ** 32 + 1], [[0]]), ([0, 1], [1], [[2 ** 31]]), ([0, 1], [1.5], [[0]]),
    ([0, -2 ** 31 - 1], [1], [[0]])])
def test_host_api_takes_no_other_integers(cw, q_starts, kv_lens, table):
    """Numbers that 32 bits would change are refused, not wrapped."""
    cache = object.__new__(cw.PagedCache)  # no device memory behind it
    cache.shape, cache.precision, cache.code = (4, 2, 16, 64), "fp32", 0
    x = np.zeros((1, 2, 64), np.float32)
    with pytest.raises(ValueError, match="32-bit"):
        cache.append(x, x, q_starts, kv_lens, table)
    with pytest.raises(ValueError, match="32-bit"):
        cache.append(x, x, [0, 1], [1], [[0]], positions=[2 ** 31])
    with pytest.raises(ValueError, match="32-bit"):
        cw.run_rope(x, [2 ** 31], object.__new__(cw.Rope))
    with pytest.raises(ValueError, match="tokens, heads, dim"):
        cw.run_rope(x[0], [0], object.__new__(cw.Rope))
