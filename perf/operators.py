"""The operators of a key/value cache that the library's speed is measured on:
rotary positions and their gradient, appending to a paged cache with the
rotation on the way, the attention that reads the cache, and the attention of a
batch that shares a long prefix.

A pass is one call on tensors that are resident on the GPU, on torch's current
stream.  With ``own`` it is the library's launcher; without, the same
operator in elementary torch operations, in 32 bits (angles in 64) and rounded
once at the end.  A batch is ragged: sequence b owns the token rows q_starts[b]
to q_starts[b + 1], and kv_lens[b] keys, those of its new tokens last, on the
pages that row b of page_table lists.  Pages are [page, kv head, slot, dim].
"""

import ctypes
import math
import os
import random
import sys

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
CODE = {"fp32": 0, "fp16": 1, "bf16": 2}
TURN = 2.0 * math.pi


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _rope(name, dtype, tokens, heads, dim, rot, interleaved=False, inverse=False, scaling="none",
          far=4096):
    return {"name": name, "op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads,
            "dim": dim, "rot": rot, "interleaved": interleaved, "inverse": inverse,
            "scaling": scaling, "far": far}


def _cache(name, op, dtype, batch, max_q, max_kv, heads, kv_heads, dim, page, lens, rot=0,
           interleaved=False, scaling="none", queries=False, causal=True, prefix=0):
    """lens 0: every sequence has max_q new tokens and max_kv keys; else the
    seed of its lengths, which then lie between one and those."""
    case = {"name": name, "op": op, "dtype": dtype, "batch": batch, "max_q": max_q,
            "max_kv": max_kv, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "lens": lens}
    if op == "append":
        case.update(rot=rot, interleaved=interleaved, scaling=scaling, queries=queries)
    else:
        case["causal"] = causal
    if op == "prefix":
        case["prefix"] = prefix
    return case


def listed():
    return [
        # The queries of one new token, far into a long context: launch latency.
        _rope("rope-token", "bf16", 1, 12, 64, 64, far=50176),
        # The queries of a long prompt; half of each head, pairs side by side,
        # frequencies blended for a context longer than the trained one.
        _rope("rope-prompt", "bf16", 8192, 32, 128, 64, interleaved=True, scaling="parts",
              far=65536),
        # The gradient of the same on the way back, in full precision, odd length.
        _rope("rope-gradient", "fp32", 4111, 8, 128, 128, inverse=True, scaling="linear"),
        # One new token of each of 64 sequences, its queries in the same launch.
        _cache("append-tokens", "append", "fp16", 64, 1, 700, 32, 8, 128, 16, 1, rot=128,
               queries=True),
        # The keys and values of five prompts of unlike lengths.
        _cache("append-prompts", "append", "bf16", 5, 4096, 4800, 8, 8, 128, 48, 2, rot=64,
               interleaved=True, scaling="base"),
        # One new token over a short cache: the smallest call, latency.
        _cache("attend-token", "attend", "fp16", 1, 1, 784, 12, 12, 64, 16, 0),
        # Serving: 64 sequences of unlike lengths, one new token each, grouped heads.
        _cache("attend-tokens", "attend", "bf16", 64, 1, 8192, 32, 8, 128, 16, 3),
        # This library's own shape over a cache: 64 latents, one head of 768, a
        # pixel array of 224 x 224.
        _cache("attend-latents", "attend", "fp32", 1, 64, 50176, 1, 1, 768, 64, 0, causal=False),
        # A prompt from nothing: the arithmetic counts.
        _cache("attend-prompt", "attend", "bf16", 1, 4096, 4096, 32, 8, 128, 16, 0),
        # Pieces of prompts behind what is cached already; pages of no power of two.
        _cache("attend-pieces", "attend", "fp16", 6, 700, 6000, 12, 4, 64, 20, 4),
        # One new token of each of 32 sequences that share a long prompt.
        _cache("prefix-tokens", "prefix", "bf16", 32, 1, 512, 32, 8, 128, 16, 5, prefix=16384),
        # A few latents of each of nine sequences behind a short prefix of odd length.
        _cache("prefix-latents", "prefix", "fp16", 9, 17, 230, 1, 1, 768, 32, 6, prefix=1025),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    dim = rng.choice([64, 64, 128, 128, 256, 768])
    op = rng.choice(["rope", "append", "attend", "attend", "prefix"])
    scaling = rng.choice(["none", "linear", "base", "parts"])
    if op == "rope":
        return _rope(None, dtype, _log_int(rng, 1, 8192), rng.randint(1, 32), dim,
                     dim // rng.choice([1, 1, 2, 4]), rng.random() < 0.5, rng.random() < 0.5,
                     scaling, _log_int(rng, 64, 131072))
    if dim == 768:
        kv_heads, group = 1, rng.choice([1, 1, 2])
    else:
        kv_heads, group = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4, 7, 8])
    batch, page = _log_int(rng, 1, 64), rng.choice([16, 16, 32, 64, rng.randint(1, 128)])
    lens = rng.randint(1, 1 << 20) if rng.random() < 0.8 else 0
    max_kv = _log_int(rng, 1, 50176)
    max_q = 1 if rng.random() < 0.5 else min(_log_int(rng, 1, 4096), max_kv)
    if op == "append":
        return _cache(None, op, dtype, batch, max_q, max_kv, kv_heads * group, kv_heads, dim,
                      page, lens, rot=dim // rng.choice([1, 1, 2, 4]),
                      interleaved=rng.random() < 0.5, scaling=scaling,
                      queries=rng.random() < 0.5)
    return _cache(None, op, dtype, batch, max_q, max_kv, kv_heads * group, kv_heads, dim, page,
                  lens, causal=rng.random() < 0.75,
                  prefix=_log_int(rng, 1, 32768) if op == "prefix" else 0)


# What a drawn case may cost at most: the floating operations of the listed prompt,
# about the bytes of the listed serving batch, and room for the plain form's scores
# and padded keys, and for the pages that an append returns.
MOST = {"flops": 1.38e11, "bytes": 1.12e9, "scores": 6e8, "pool": 1.2e9, "appended": 2e8}


def draw(rng):
    """One of the operators, in any of the types: 1 to 64 sequences, 1 to 4,096
    new tokens each (one in half of the cases), caches of 1 to 50,176 keys, pages
    of 1 to 128 slots, prefixes of 1 to 32,768 keys, heads of 64 to 768 in groups of 1 to 8."""
    while True:
        case = _drawn(rng)
        cost = work(case)
        if cost["flops"] > MOST["flops"] or cost["bytes"] > MOST["bytes"]:
            continue
        if case["op"] != "rope":
            keys = case["batch"] * (case["max_kv"] + case.get("prefix", 0))
            pool = case["batch"] * case["max_kv"] * case["kv_heads"] * case["dim"]
            if pool > MOST["pool"] or (case["op"] == "append" and pool > MOST["appended"]):
                continue
            if case["op"] != "append" and keys * case["heads"] * case["max_q"] > MOST["scores"]:
                continue
        del case["name"]
        return case


def _lengths(case):
    """(new tokens, keys) of each sequence; the keys of the new tokens count
    among the keys."""
    batch, max_q, max_kv = case["batch"], case["max_q"], case["max_kv"]
    if not case["lens"]:
        return [max_q] * batch, [max_kv] * batch
    rng = random.Random(case["lens"])
    q = [rng.randint(1, max_q) for _ in range(batch)]
    kv = [rng.randint(min(n, max_kv), max_kv) for n in q]
    at = rng.randrange(batch)  # one sequence is as long as the case says
    q[at], kv[at] = max_q, max_kv
    return q, kv


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    q, kv = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        moved = sum(q) * dim * (2 * kv_heads + (heads if case["queries"] else 0))
        turned = sum(q) * case["rot"] * (kv_heads + (heads if case["queries"] else 0))
        return {"bytes": 2 * moved * size, "flops": 3 * turned}
    prefix = case.get("prefix", 0)
    if case["causal"]:
        seen = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(q, kv))
    else:
        seen = sum(n * k for n, k in zip(q, kv))
    seen += sum(q) * prefix
    return {"bytes": size * dim * (2 * heads * sum(q) + 2 * kv_heads * (sum(kv) + prefix)),
            "flops": 4 * dim * heads * seen}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _frequencies(rot, scaling):
    """Turns per position of each rotated pair, and the factor on cos and sin:
    the usual base 10,000, stretched by 8 from a trained length of 4,096."""
    base, factor, trained, slow, fast = 10000.0, 8.0, 4096, 1.0, 32.0
    if scaling == "base" and rot > 2:
        base *= factor ** (rot / (rot - 2))
    f = torch.tensor([base ** (-2.0 * i / rot) / TURN for i in range(rot // 2)],
                     dtype=torch.float64)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = ((f * trained - slow) / (fast - slow)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    state = {"case": case}
    if case["op"] in ("rope", "append"):
        freqs, amplitude = _frequencies(case["rot"], case["scaling"])
        state.update(freqs=freqs.cuda(), amplitude=amplitude)
    if case["op"] == "rope":
        state["x"] = normal(case["tokens"], case["heads"], case["dim"])
        state["y"] = torch.empty_like(state["x"])
        state["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=gen,
                                           device="cuda", dtype=torch.int32)
        return state

    q_lens, kv_lens = _lengths(case)
    heads, kv_heads, dim, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    tokens = sum(q_lens)
    counts = [-(-n // page) for n in kv_lens]
    prefix = case.get("prefix", 0)
    prefix_pages = -(-prefix // page)
    pages = sum(counts) + prefix_pages
    # Pages are handed out in the order in which a running server frees them: none.
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    width = max(counts)
    table = torch.zeros(case["batch"], width, dtype=torch.int32)
    at, shuffled = 0, order.cpu()
    for b, n in enumerate(counts):
        table[b, :n] = shuffled[at:at + n]
        at += n
    starts = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    state.update(
        q_starts=starts.cuda(), kv_lens=torch.tensor(kv_lens, dtype=torch.int32).cuda(),
        page_table=table.cuda(), prefix_pages=order[at:].contiguous(), tokens=tokens,
        width=width, pages=pages, max_q=max(q_lens), max_kv=max(kv_lens))
    # q, k and v are the columns of one projection's output, as a model makes them.
    if case["op"] == "append":
        qkv = normal(tokens, heads + 2 * kv_heads, dim)
        state.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv_heads],
                     v=qkv[:, heads + kv_heads:],
                     q_out=torch.empty(tokens, heads, dim, dtype=dtype, device="cuda"))
        state["k_pages"] = torch.zeros(pages, kv_heads, page, dim, dtype=dtype, device="cuda")
        state["v_pages"] = torch.zeros_like(state["k_pages"])
        return state
    state["q"] = normal(tokens, heads, dim, scale=1.5)
    state["k_pages"] = normal(pages, kv_heads, page, dim)
    state["v_pages"] = normal(pages, kv_heads, page, dim)
    state["out"] = torch.empty_like(state["q"])
    state["scale"] = dim ** -0.5
    return state


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------

def _arguments(state):
    """The launcher of a state and its arguments but the stream: the handles,
    strides and scratch that a program makes once and keeps."""
    sys.path.insert(0, os.path.join(os.getcwd(), "fast-cuda-cross-attention_amd"))
    import cuda_wrappers as cw

    case, ref, lib = state["case"], ctypes.byref, cw.lib
    dim, code = case["dim"], CODE[case["dtype"]]
    if case["op"] in ("rope", "append"):
        rope = cw.RopeArgs(state["freqs"].data_ptr(), state["amplitude"], case["rot"],
                           int(case["interleaved"]))
    if case["op"] == "rope":
        row = case["heads"] * dim
        return lib.launch_rope_kernel, [
            state["x"].data_ptr(), state["y"].data_ptr(), state["positions"].data_ptr(),
            ref(rope), code, case["tokens"], case["heads"], dim, row, row, int(case["inverse"])]
    cache = cw.CacheArgs(state["k_pages"].data_ptr(), state["v_pages"].data_ptr(), code,
                         state["pages"], case["kv_heads"], case["page"], dim)
    batch = cw.BatchArgs(state["q_starts"].data_ptr(), state["kv_lens"].data_ptr(),
                         state["page_table"].data_ptr(), case["batch"], state["width"],
                         state["tokens"], state["max_q"], state["max_kv"])
    heads = case["heads"]
    if case["op"] == "append":
        q = state["q"].data_ptr() if case["queries"] else None
        q_out = state["q_out"].data_ptr() if case["queries"] else None
        return lib.launch_cache_append_kernel, [
            ref(cache), ref(batch), state["k"].data_ptr(), state["k"].stride(0),
            state["v"].data_ptr(), state["v"].stride(0), q, state["q"].stride(0), q_out,
            heads * dim, heads, None, ref(rope)]
    prefix = None
    if case["op"] == "prefix":
        prefix = ref(cw.PrefixArgs(state["prefix_pages"].data_ptr(),
                                   state["prefix_pages"].numel(), case["prefix"]))
    need = lib.xattn_cache_attention_scratch(ref(cache), ref(batch), prefix, heads)
    state["scratch"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    rest = [state["q"].data_ptr(), heads * dim, state["out"].data_ptr(), heads * dim, heads,
            state["scale"], int(case["causal"]), state["scratch"].data_ptr(), need]
    if prefix is None:
        return lib.launch_cache_attention_kernel, [ref(cache), ref(batch)] + rest
    return lib.launch_prefix_attention_kernel, [ref(cache), ref(batch), prefix] + rest


def _outputs(state):
    op = state["case"]["op"]
    if op == "rope":
        return state["y"]
    if op == "append":
        out = {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}
        if state["case"]["queries"]:
            out["q"] = state["q_out"]
        return out
    return state["out"]


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _turned(x, positions, state, inverse=False):
    """x [tokens, heads, dim] with its leading elements rotated, in 32 bits."""
    case = state["case"]
    rot, half = case["rot"], case["rot"] // 2
    angle = positions.double()[:, None] * state["freqs"] * TURN
    cos = (angle.cos() * state["amplitude"]).float()[:, None]
    sin = (angle.sin() * (-state["amplitude"] if inverse else state["amplitude"])).float()[:, None]
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1)


def _places(state):
    """(sequence, place among the sequence's new tokens, cache position) of every token."""
    starts = state["q_starts"].long()
    token = torch.arange(state["tokens"], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    at = token - starts[seq]
    return seq, at, state["kv_lens"].long()[seq] - (starts[1:] - starts[:-1])[seq] + at


def _plain_append(state):
    case, page = state["case"], state["case"]["page"]
    dtype = TYPES[case["dtype"]]
    seq, _, position = _places(state)
    where = state["page_table"].long()[seq, position // page]
    slot = position % page
    state["k_pages"][where, :, slot] = _turned(state["k"], position, state).to(dtype)
    state["v_pages"][where, :, slot] = state["v"]
    if case["queries"]:
        state["q_out"].copy_(_turned(state["q"], position, state))
    return _outputs(state)


def _plain_attend(state):
    """Sequences padded to the longest; the shared prefix's scores are one
    product over the queries of all of them."""
    case = state["case"]
    batch, heads, kv_heads, dim = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    page, max_q, max_kv = case["page"], state["max_q"], state["max_kv"]
    group, prefix = heads // kv_heads, case.get("prefix", 0)
    seq, at, position = _places(state)
    q = torch.zeros(batch, max_q, heads, dim, device="cuda")
    q[seq, at] = state["q"].float() * state["scale"]
    q = q.view(batch, max_q, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    q = q.reshape(batch, kv_heads, max_q * group, dim)
    key = torch.arange(max_kv, device="cuda")
    where = state["page_table"].long()[:, key // page]
    slot = (key % page).expand_as(where)
    k = state["k_pages"][where, :, slot].permute(0, 2, 1, 3).float()
    v = state["v_pages"][where, :, slot].permute(0, 2, 1, 3).float()
    last = torch.full((batch, max_q), -1, device="cuda", dtype=torch.long)
    last[seq, at] = position if case["causal"] else state["kv_lens"].long()[seq] - 1
    seen = key <= last.repeat_interleave(group, dim=1)[:, None, :, None]
    scores = (q @ k.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    if prefix:
        key = torch.arange(prefix, device="cuda")
        where, slot = state["prefix_pages"].long()[key // page], key % page
        pk = state["k_pages"][where, :, slot].transpose(0, 1).float()
        pv = state["v_pages"][where, :, slot].transpose(0, 1).float()
        flat = q.transpose(0, 1).reshape(kv_heads, batch * max_q * group, dim)
        first = (flat @ pk.transpose(-1, -2)).view(kv_heads, batch, max_q * group, prefix)
        scores = torch.cat((first.transpose(0, 1), scores), dim=-1)
    top = scores.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = (scores - top).exp()
    total = weights.sum(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    out = weights[..., prefix:] @ v
    if prefix:
        flat = weights[..., :prefix].transpose(0, 1).reshape(kv_heads, -1, prefix)
        out = out + (flat @ pv).view(kv_heads, batch, max_q * group, dim).transpose(0, 1)
    out = (out / total).view(batch, kv_heads, max_q, group, dim).permute(0, 2, 1, 3, 4)
    state["out"].copy_(out.reshape(batch, max_q, heads, dim)[seq, at])
    return state["out"]


def run(state):
    if own:
        call = state.get("call")
        if call is None:
            call = state["call"] = _arguments(state)
        call[0](*call[1], torch.cuda.current_stream().cuda_stream)
        return _outputs(state)
    op = state["case"]["op"]
    if op == "rope":
        state["y"].copy_(_turned(state["x"], state["positions"], state, state["case"]["inverse"]))
        return state["y"]
    return _plain_append(state) if op == "append" else _plain_attend(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_rotation(x, positions, state, inverse=False):
    """Pairs as complex numbers times A e^(i angle)."""
    case = state["case"]
    rot = case["rot"]
    x = x.double()
    pairs = x[..., :rot].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
    axis = -1 if case["interleaved"] else -2
    z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1))
    turns = torch.outer(positions.double(), state["freqs"])
    turns = (turns - turns.round()) * (-TURN if inverse else TURN)
    z = z * torch.polar(torch.full_like(turns, state["amplitude"]), turns)[:, None, :]
    return torch.cat((torch.stack((z.real, z.imag), dim=axis).flatten(-2), x[..., rot:]), dim=-1)


def _rows(pages, listed_pages, page, length, head):
    """The first `length` rows of one head on the pages listed, in 64 bits."""
    count = -(-length // page)
    return pages[listed_pages[:count].long(), head].reshape(-1, pages.shape[-1])[:length].double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rotation(state["x"], state["positions"], state, case["inverse"])
    q_lens, kv_lens = _lengths(case)
    page, heads, group = case["page"], case["heads"], case["heads"] // case["kv_heads"]
    if case["op"] == "append":
        position = torch.cat([torch.arange(n - m, n) for m, n in zip(q_lens, kv_lens)]).cuda()
        k, v = _exact_rotation(state["k"], position, state), state["v"].double()
        out = {"k_pages": state["k_pages"].double(), "v_pages": state["v_pages"].double()}
        row = 0
        for b, (m, n) in enumerate(zip(q_lens, kv_lens)):
            count = -(-n // page)
            listed_pages = state["page_table"][b, :count].long()
            for name, new in (("k_pages", k), ("v_pages", v)):
                whole = out[name][listed_pages].transpose(1, 2).flatten(0, 1)
                whole[n - m:n] = new[row:row + m]
                out[name][listed_pages] = whole.unflatten(0, (count, page)).transpose(1, 2)
            row += m
        if case["queries"]:
            out["q"] = _exact_rotation(state["q"], position, state)
        return out
    out = torch.zeros(state["tokens"], heads, case["dim"], dtype=torch.float64, device="cuda")
    row, prefix = 0, case.get("prefix", 0)
    shared = [[_rows(p, state["prefix_pages"], page, prefix, h) for p in
               (state["k_pages"], state["v_pages"])] for h in range(case["kv_heads"])]
    for b, (m, n) in enumerate(zip(q_lens, kv_lens)):
        hidden = None
        if case["causal"]:
            reach = torch.arange(n - m, n, device="cuda")[:, None] + prefix
            hidden = torch.arange(prefix + n, device="cuda")[None, :] > reach
        for h in range(case["kv_heads"]):
            k, v = (torch.cat((shared[h][i], _rows(p, state["page_table"][b], page, n, h)))
                    for i, p in enumerate((state["k_pages"], state["v_pages"])))
            for j in range(h * group, (h + 1) * group):
                s = state["q"][row:row + m, j].double() @ k.t() * state["scale"]
                if hidden is not None:
                    s = s.masked_fill(hidden, -math.inf)
                out[row:row + m, j] = torch.softmax(s, dim=-1) @ v
        row += m
    return out
