"""CPU oracle of the cache operators, in 64 bits and straight from their
definitions: rotary positions, append to a paged cache, attention over one,
with or without a shared prefix.  Test infrastructure only, like
xattn_oracle.py; test_cache_ops.py pins it against closed forms.

Pages are [num_pages, kv_heads, page_size, dim]; sequence b owns token rows
q_starts[b] .. q_starts[b + 1] - 1 and kv_lens[b] keys, its new tokens' last.
"""

from __future__ import annotations

import numpy as np


def rope(x, positions, freqs, amplitude=1.0, interleaved=False, inverse=False):
    """x [tokens, heads, dim] with its first 2 len(freqs) elements rotated by
    2 pi position freqs[i] (inverse: the transposed map)."""
    y = np.array(x, np.float64)
    rot = 2 * len(freqs)
    turns = np.asarray(positions, np.float64)[:, None] * np.asarray(freqs, np.float64)
    angle = 2 * np.pi * (turns - np.rint(turns)) * (-1 if inverse else 1)
    c, s = amplitude * np.cos(angle)[:, None], amplitude * np.sin(angle)[:, None]
    first = np.s_[..., 0:rot:2] if interleaved else np.s_[..., :rot // 2]
    second = np.s_[..., 1:rot:2] if interleaved else np.s_[..., rot // 2:rot]
    a, b = y[first].copy(), y[second].copy()
    y[first], y[second] = a * c - b * s, b * c + a * s
    return y


def places(q_starts, kv_lens):
    """(token row, sequence, cache position) of every token that has a sequence."""
    return [(t, b, int(kv_lens[b]) - (int(q_starts[b + 1]) - t))
            for b in range(len(kv_lens)) for t in range(q_starts[b], q_starts[b + 1])]


def append(k_pages, v_pages, k, v, q_starts, kv_lens, page_table, freqs=(), amplitude=1.0,
           interleaved=False, positions=None):
    """New (k_pages, v_pages) in 64 bits."""
    k_pages, v_pages = np.array(k_pages, np.float64), np.array(v_pages, np.float64)
    size = k_pages.shape[2]
    for t, b, pos in places(q_starts, kv_lens):
        if not 0 <= pos < page_table.shape[1] * size:
            continue
        page = page_table[b, pos // size]
        if not 0 <= page < len(k_pages):
            continue
        at = pos if positions is None else positions[t]
        k_pages[page, :, pos % size] = rope(k[t:t + 1], [at], freqs, amplitude, interleaved)[0]
        v_pages[page, :, pos % size] = v[t]
    return k_pages, v_pages


def gather(pages, numbers, length):
    """[length, kv_heads, dim]: the first rows on the pages listed."""
    size = pages.shape[2]
    at = np.arange(length)
    return pages[np.asarray(numbers, np.int64)[at // size], :, at % size]


def attend(q, k_pages, v_pages, q_starts, kv_lens, page_table, scale, causal=True,
           prefix_pages=None, prefix_len=0):
    """(out [tokens, heads, dim], how far the sum of |weight v| and the largest
    |score| and sum of |score terms| go: dict) in 64 bits; rows of no sequence
    and rows that see no key are zero."""
    q = np.asarray(q, np.float64)
    tokens, heads, dim = q.shape
    group = heads // k_pages.shape[1]
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    top, terms = np.zeros((tokens, heads)), np.zeros((tokens, heads))
    for t, b, pos in places(q_starts, kv_lens):
        n = int(np.clip(pos + 1, 0, kv_lens[b])) if causal else int(kv_lens[b])
        k, v = gather(k_pages, page_table[b], n), gather(v_pages, page_table[b], n)
        if prefix_pages is not None:
            k = np.concatenate([gather(k_pages, prefix_pages, prefix_len), k])
            v = np.concatenate([gather(v_pages, prefix_pages, prefix_len), v])
        if not len(k):
            continue
        k, v = k.astype(np.float64), v.astype(np.float64)
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            s = scale * (kh @ q[t, h])
            w = np.exp(s - s.max())
            w /= w.sum()
            out[t, h], mass[t, h] = w @ vh, w @ np.abs(vh)
            top[t, h] = np.abs(s).max()
            terms[t, h] = abs(scale) * (np.abs(kh) @ np.abs(q[t, h])).max()
    return out, {"mass": mass, "top": top, "terms": terms}


def attend_tolerance(out, size, dim, keys, step):
    """How far an evaluation in 32 bits, with weights and results rounded to a
    type whose half step is `step` (0 for 32 bits), may be from attend()'s
    (out, size): element by element.

    A score is a sum of dim products: rounding errors of dim half steps 2^-24 of
    its terms' sum, growing as their square root; four times that.  Its
    exponent is formed from numbers of up to `top` with three more roundings,
    and exp2 is good to two steps.  A weight of relative error e moves the
    quotient by up to 2 e of the mass.  Numerator and denominator are sums of
    `keys` terms in 32 bits (square root again), each weight of the numerator
    rounded to the type by up to `step`, and the quotient once more."""
    u = 2.0 ** -24
    score = 4 * np.sqrt(dim) * u * size["terms"] + 6 * u * size["top"] + 4 * u
    wide = 2 * score + 4 * np.sqrt(max(keys, 1)) * u + 8 * u
    return (wide[..., None] + step) * size["mass"] + (step + 2 * u) * np.abs(out) + 1e-30
