"""Ragged batches over a paged cache, for the tests of the cache operators."""

import ctypes

import numpy as np

HALF_STEP = {"fp32": 0.0, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rounded(cw, x, precision):
    """The values of x in the type, as float32."""
    return cw._decode(cw._encode(np.asarray(x, np.float32), precision), precision)


class Batch:
    """New tokens and cache lengths of a few sequences, their pages handed out
    in random order, with token rows before the first and behind the last."""

    def __init__(self, rng, q_lens, kv_lens, page_size, before=0, behind=0, spare=2,
                 prefix_len=0):
        self.q_lens, self.kv_lens = list(q_lens), np.array(kv_lens, np.int32)
        self.page_size, self.prefix_len = page_size, prefix_len
        self.q_starts = (before + np.concatenate([[0], np.cumsum(q_lens)])).astype(np.int32)
        self.tokens = int(self.q_starts[-1]) + behind
        counts = [-(-int(n) // page_size) for n in kv_lens]
        first = -(-prefix_len // page_size)
        self.num_pages = sum(counts) + first + spare
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.prefix_pages, order = order[:first], order[first:]
        width = max(counts + [1])
        # entries behind a sequence's pages are never looked at
        self.page_table = np.full((len(counts), width), -7, np.int32)
        for b, n in enumerate(counts):
            self.page_table[b, :n], order = order[:n], order[n:]

    def widen(self, keys):
        """Rows of page_table for `keys` keys, and as many announced."""
        more = -(-keys // self.page_size) - self.page_table.shape[1]
        self.page_table = np.pad(self.page_table, ((0, 0), (0, max(more, 0))), constant_values=-7)
        self.max_kv_len = lambda: keys

    def max_q_len(self):
        return max(self.q_lens, default=0)

    def max_kv_len(self):
        return int(max(self.kv_lens, default=0))

    @property
    def where(self):
        return self.q_starts, self.kv_lens, self.page_table

    def rows(self):
        return np.arange(self.q_starts[0], self.q_starts[-1])


def pages_of(rng, cw, batch, kv_heads, dim, precision, garbage=np.nan, k_scale=1.0):
    """(k, v) pages in the type's values; every slot that holds no key of the
    batch or its prefix is `garbage`."""
    shape = (batch.num_pages, kv_heads, batch.page_size, dim)
    k, v = (np.full(shape, garbage, np.float32) for _ in range(2))
    lists = [(batch.page_table[b], int(n)) for b, n in enumerate(batch.kv_lens)]
    lists.append((batch.prefix_pages, batch.prefix_len))
    for numbers, n in lists:
        for p in range(-(-n // batch.page_size)):
            m = min(batch.page_size, n - p * batch.page_size)
            k[numbers[p], :, :m] = k_scale * rng.standard_normal((kv_heads, m, dim))
            v[numbers[p], :, :m] = rng.standard_normal((kv_heads, m, dim))
    return rounded(cw, k, precision), rounded(cw, v, precision)


class OnDevice:
    """A cache, a batch and token tensors on the device, for direct calls of
    the launchers."""

    def __init__(self, cw, owned, batch, k_pages, v_pages, precision):
        self.cw, self.owned, self.precision = cw, owned, precision
        self.k, self.v = (self.put(cw._encode(a, precision)) for a in (k_pages, v_pages))
        n, kv_heads, size, dim = k_pages.shape
        self.cache = cw.CacheArgs(self.k.ptr.value, self.v.ptr.value, cw.PRECISIONS[precision],
                                  n, kv_heads, size, dim)
        self.q_starts, self.kv_lens, self.table = (self.put(a) for a in batch.where)
        self.batch = cw.BatchArgs(self.q_starts.ptr.value, self.kv_lens.ptr.value,
                                  self.table.ptr.value, len(batch.kv_lens),
                                  batch.page_table.shape[1], batch.tokens,
                                  batch.max_q_len(), batch.max_kv_len())
        self.prefix = None
        if batch.prefix_len:
            self.listed = self.put(batch.prefix_pages)
            self.prefix = cw.PrefixArgs(self.listed.ptr.value, len(batch.prefix_pages),
                                        batch.prefix_len)

    def put(self, host):
        return self.owned.enter_context(self.cw.DeviceBuffer.holding(np.ascontiguousarray(host)))

    def scratch(self, heads):
        prefix = self.prefix and ctypes.byref(self.prefix)
        need = self.cw.lib.xattn_cache_attention_scratch(
            ctypes.byref(self.cache), ctypes.byref(self.batch), prefix, heads)
        return self.owned.enter_context(self.cw.DeviceBuffer(need)), need

    def attend(self, q, q_stride, out, out_stride, heads, scale, causal, scratch, stream=None):
        ref = ctypes.byref
        args = [ref(self.cache), ref(self.batch)]
        fn = self.cw.lib.launch_cache_attention_kernel
        if self.prefix is not None:
            args.append(ref(self.prefix))
            fn = self.cw.lib.launch_prefix_attention_kernel
        fn(*args, q.ptr, q_stride, out.ptr, out_stride, heads, scale, int(causal),
           scratch[0].ptr, scratch[1], stream)
        self.cw._lib_error_check(fn.__name__)
