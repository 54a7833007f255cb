"""Operators of language models that answer about images, as cases to time.

A network of this framework turns an image into a map of features.  A language model
takes the map's cells as tokens beside those of the text, and four operators carry its
attention while it serves requests:

  reserve   the cache's bookkeeping on the GPU: block tables, slots and positions of new
            tokens from the lengths of the requests
  rotary    rotary positions with several axes (time, height, width) on queries and keys,
            the keys and values stored in the paged cache
  prompt    attention of packed sequences of different lengths, causal or, for the cells
            of images, over all of a sequence, with grouped heads
  paged     attention of new tokens, one per request or a chunk of a prompt, over the
            paged cache

The plain forms compute in 32 bits with elementary operations of torch, on sequences padded
to the longest, and round once.  Lengths belong to the case, their order and all values to
the seed.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One step of text for 32 requests: each gets one slot, now and then a block.
        {"name": "reserve_decode_32", "op": "reserve", "requests": 32, "longest_new": 1, "longest_cached": 2000, "block": 16},
        # 500 prompts of all lengths arrive together at an empty server.
        {"name": "reserve_prompts_500", "op": "reserve", "requests": 500, "longest_new": 250, "longest_cached": 0, "block": 16},
        # One step of text for 64 requests, three axes that hold the same position.
        {"name": "rotary_decode_64", "op": "rotary", "type": "bf16", "tokens": 64, "heads": 32, "heads_kv": 8, "dim": 128,
         "rotary": 128, "axes": 3, "adjacent": False, "cycled": False, "first": 30000, "block": 16},
        # A long prompt with images, all its keys and values stored.
        {"name": "rotary_images_16384", "op": "rotary", "type": "bf16", "tokens": 16384, "heads": 32, "heads_kv": 8, "dim": 128,
         "rotary": 128, "axes": 3, "adjacent": False, "cycled": True, "first": 0, "block": 16},
        # The cells of an image in 32 bits, height and width as axes, neighbours as pairs.
        {"name": "rotary_f32_2049", "op": "rotary", "type": "f32", "tokens": 2049, "heads": 12, "heads_kv": 12, "dim": 64,
         "rotary": 64, "axes": 2, "adjacent": True, "cycled": False, "first": 0, "block": 32},
        # One short question: what a call costs.
        {"name": "prompt_1x77", "op": "prompt", "type": "f16", "sequences": 1, "longest": 77, "heads": 8, "heads_kv": 8, "dim": 64,
         "causal": True},
        # Two dozen prompts of different lengths packed behind each other.
        {"name": "prompt_24x1500", "op": "prompt", "type": "bf16", "sequences": 24, "longest": 1500, "heads": 32, "heads_kv": 8,
         "dim": 128, "causal": True},
        # One long document.
        {"name": "prompt_1x8192", "op": "prompt", "type": "bf16", "sequences": 1, "longest": 8192, "heads": 32, "heads_kv": 8,
         "dim": 128, "causal": True},
        # The cells of five images of different sizes among themselves, in this framework's own type.
        {"name": "prompt_f32_images_5x1369", "op": "prompt", "type": "f32", "sequences": 5, "longest": 1369, "heads": 12,
         "heads_kv": 12, "dim": 64, "causal": False},
        # The next token of one interactive request.
        {"name": "paged_decode_1x513", "op": "paged", "type": "f16", "requests": 1, "longest_new": 1, "longest": 513, "heads": 16,
         "heads_kv": 4, "dim": 80, "block": 16},
        # The next token of 64 requests with long and short histories.
        {"name": "paged_decode_64x8192", "op": "paged", "type": "bf16", "requests": 64, "longest_new": 1, "longest": 8192,
         "heads": 32, "heads_kv": 8, "dim": 128, "block": 16},
        # A chunk of a very long prompt beside what the cache already holds of it.
        {"name": "paged_chunk_512x32768", "op": "paged", "type": "bf16", "requests": 1, "longest_new": 512, "longest": 32768,
         "heads": 32, "heads_kv": 8, "dim": 128, "block": 64},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng, most):
    heads_kv = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if g * heads_kv <= most])
    return {"heads": group * heads_kv, "heads_kv": heads_kv, "dim": rng.choice([64, 64, 80, 96, 128, 128, 128, 256])}


def draw(rng):
    op = rng.choice(["reserve", "rotary", "prompt", "prompt", "paged", "paged", "paged"])
    case = {"op": op}
    block = rng.choice([16, 16, 32, 64, 24])
    if op == "reserve":
        requests = _log_int(rng, 1, 1024)
        prompts = rng.random() < 0.5
        case.update(requests=requests, longest_new=_log_int(rng, 1, max(1, min(8192, 120000 // requests))) if prompts else 1,
                    longest_cached=rng.choice([0, _log_int(rng, 1, 32768)]), block=block)
        return case
    case.update(_heads(rng, 32), type=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if op == "rotary":
        half = rng.random() < 0.25
        case.update(tokens=_log_int(rng, 1, 12000 * 48 * 128 // ((case["heads"] + 2 * case["heads_kv"]) * case["dim"])
                                    // (2 if case["type"] == "f32" else 1)),
                    rotary=case["dim"] // 2 if half else case["dim"], axes=rng.choice([1, 2, 3, 3]), adjacent=rng.random() < 0.3,
                    cycled=rng.random() < 0.5, first=0 if case["type"] == "f32" else rng.choice([0, _log_int(rng, 100, 100000)]),
                    block=block)
    elif op == "prompt":
        # the products and sums of the largest listed case; the plain form pads, and in 32 bits
        # every product costs more
        causal = rng.random() < 0.7
        sequences = _log_int(rng, 1, 32)
        cells = (8192 ** 2 * 32 * 128) // (case["heads"] * case["dim"] * sequences * (1 if causal else 2))
        cells = cells // 16 if case["type"] == "f32" else cells
        case.update(sequences=sequences, causal=causal, longest=_log_int(rng, 1, min(8192, math.isqrt(cells))))
    else:
        requests = _log_int(rng, 1, 96)
        new = rng.choice([1, 1, _log_int(rng, 1, 512)])
        most = min(32768, 200000 // requests * 1024 // (case["heads_kv"] * case["dim"]), 512 * 32768 * 32 * 128 //
                   (new * requests * case["heads"] * case["dim"] * (16 if case["type"] == "f32" else 1)))
        new = max(1, min(new, most))
        case.update(requests=requests, longest_new=new, longest=_log_int(rng, new, max(new, most)), block=block)
    return case


# ---- lengths, which belong to the case ----------------------------------------------

def _spread(count, low, high):
    """`count` lengths from low to high, the longest among them: steps of the golden ratio, as even as can be."""
    part = (np.arange(count) * 0.6180339887498949 + 1.0) % 1.0     # the first is 0
    return np.maximum(low, np.round(high - part * (high - low))).astype(np.int64)


def _news(case):
    """New tokens of each request (a step of text: one each)."""
    return _spread(case["requests"], 1, case["longest_new"])


def _contexts(case):
    """Tokens that each request holds with its new ones: between an eighth of the longest and the longest."""
    new = _news(case)
    return np.maximum(new, _spread(case["requests"], max(1, case["longest"] // 8), case["longest"]))


def _lengths(case):
    return _spread(case["sequences"], 1 + case["longest"] // 16, case["longest"])


def _ceil(a, b):
    return -(-a // b)


# ---- inputs -------------------------------------------------------------------------

def _cumulated(lengths):
    return np.concatenate([[0], np.cumsum(lengths)])


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()


def _values(g, shape, dtype, spread=1.0):
    """Normal values; over the heads, the last axis but one, their size falls from 2 to 1 times `spread`: heads with sharp and with even weights."""
    size = torch.linspace(2.0, 1.0, shape[-2], device="cuda")[:, None] * spread
    return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)


def _tables(r, lengths, block, spare=1.25):
    """Block tables of requests of these lengths: blocks of one pool in no order, and `spare` times as many there as are used."""
    need = _ceil(lengths, block)
    blocks = int(need.sum() * spare) + 1
    order = r.permutation(blocks)
    table = np.zeros((len(lengths), max(1, int(need.max()))), np.int64)
    at = _cumulated(need)
    for i, n in enumerate(need):
        table[i, :n] = order[at[i]:at[i + 1]]
    return table, blocks, order[at[-1]:]


def prepare(case, seed):
    r = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case, "seed": seed}
    if case["op"] == "reserve":
        return _prepare_reserve(case, r, s)
    dtype = TYPES[case["type"]]
    heads, kv, dim = case["heads"], case["heads_kv"], case["dim"]
    if case["op"] == "rotary":
        tokens = case["tokens"]
        s["qkv"] = _values(g, (tokens, heads + 2 * kv, dim), dtype)      # as one projection leaves them
        pairs = case["rotary"] // 2
        s["frequencies"] = (1e6 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().cuda()
        s["axis"] = _int(_axis_of(case))
        s["positions"] = _int(_image_positions(r, case))
        # tokens of a few requests: their slots are scattered by blocks
        table, blocks, _ = _tables(r, np.array([tokens]), case["block"], 1.1)
        t = np.arange(tokens)
        s["slots"] = torch.from_numpy(table[0, t // case["block"]] * case["block"] + t % case["block"]).cuda().int()
        s["keys"], s["cached_values"] = (torch.zeros((blocks, case["block"], kv, dim), dtype=dtype, device="cuda") for _ in range(2))
        s["out"] = torch.empty((tokens, heads, dim), dtype=dtype, device="cuda")
    elif case["op"] == "prompt":
        lengths = r.permutation(_lengths(case))
        s["starts"], s["longest"], s["total"] = _int(_cumulated(lengths)), int(lengths.max()), int(lengths.sum())
        s["qkv"] = _values(g, (s["total"], heads + 2 * kv, dim), dtype)
        s["out"] = torch.empty((s["total"], heads, dim), dtype=dtype, device="cuda")
        s["lse"] = torch.empty((heads, s["total"]), device="cuda")
    else:
        order = r.permutation(case["requests"])
        new, contexts = _news(case)[order], _contexts(case)[order]
        s["starts"], s["contexts"], s["total"] = _int(_cumulated(new)), _int(contexts), int(new.sum())
        s["longest_new"], s["longest"] = int(new.max()), int(contexts.max())
        table, blocks, _ = _tables(r, contexts, case["block"])
        s["table"] = _int(table)
        s["q"] = _values(g, (s["total"], heads, dim), dtype)
        s["keys"], s["cached_values"] = (_values(g, (blocks, case["block"], kv, dim), dtype) for _ in range(2))
        s["out"] = torch.empty((s["total"], heads, dim), dtype=dtype, device="cuda")
        s["lse"] = torch.empty((heads, s["total"]), device="cuda")
    return s


def _prepare_reserve(case, r, s):
    requests, block = case["requests"], case["block"]
    order = r.permutation(requests)
    new = _news(case)[order]
    cached = _spread(requests, 0, case["longest_cached"])[order]
    table, blocks, rest = _tables(r, cached, block, 1.0)
    need = int((_ceil(cached + new, block) - _ceil(cached, block)).sum())
    width = int(_ceil(cached + new, block).max())
    wide = np.full((requests, width), -1, np.int64)
    wide[:, :min(width, table.shape[1])] = table[:, :width]
    free = np.concatenate([r.permutation(need + need // 4 + 8) + blocks, rest])    # more blocks than are asked for
    s.update(cached=_int(cached), new=_int(new), table=_int(wide), free=_int(free), free_count=_int([len(free)]),
             total=int(new.sum()))
    s["contexts"], s["starts"] = _int(np.zeros(requests)), _int(np.zeros(requests + 1))
    s["slots"], s["positions"] = _int(np.zeros(s["total"])), _int(np.zeros(s["total"]))
    s["free_left"], s["denied"] = _int([0]), _int([0])
    return s


def _axis_of(case):
    """The axis whose position turns each pair: sections in a row, or dealt out in turn (time, height, width, time, ...)."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    sections = _sections(case)
    if not case["cycled"]:
        return np.repeat(np.arange(axes), sections)
    axis, left = [], list(sections)
    while len(axis) < pairs:
        for a in range(axes):
            if left[a]:
                axis.append(a)
                left[a] -= 1
    return np.array(axis)


def _sections(case):
    pairs, axes = case["rotary"] // 2, case["axes"]
    if axes == 3:                              # time has the smaller share
        part = pairs * 3 // 8
        return [pairs - 2 * part, part, part]
    return [pairs // axes + (pairs % axes if a == 0 else 0) for a in range(axes)]


def _image_positions(r, case):
    """Positions on every axis: text counts on all of them together, an image counts its rows and columns."""
    tokens, axes = case["tokens"], case["axes"]
    at = np.zeros((axes, tokens), np.int64)
    t, p = 0, case["first"]
    while t < tokens:
        n = min(tokens - t, int(r.integers(1, 200)))
        at[:, t:t + n] = p + np.arange(n)
        t, p = t + n, p + n
        h, w = int(r.integers(4, 32)), int(r.integers(4, 32))
        n = min(tokens - t, h * w)
        cell = np.arange(n)
        for a in range(axes):
            at[a, t:t + n] = p + (cell // w if a == axes - 2 else cell % w if a == axes - 1 and axes > 1 else 0)
        t, p = t + n, p + max(h, w)
    return at


# ---- a pass -------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _split(s):
    heads, kv = s["case"]["heads"], s["case"]["heads_kv"]
    return s["qkv"][:, :heads], s["qkv"][:, heads:heads + kv], s["qkv"][:, heads + kv:]


def _plain_reserve(s):
    block, cached, new = s["case"]["block"], s["cached"], s["new"]
    starts = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0, dtype=torch.int32)])
    contexts = cached + new
    have, need = (cached + block - 1) // block, (contexts + block - 1) // block
    more = need - have
    taken = torch.cumsum(more, 0) - more                                  # blocks that earlier requests take
    column = torch.arange(s["table"].shape[1], device="cuda")[None]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    at = s["free_count"] - 1 - (taken[:, None] + column - have[:, None])  # from the end of the list of free blocks
    table = torch.where(fresh, s["free"][at.clamp(0, len(s["free"]) - 1)], s["table"])
    token = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    of = torch.searchsorted(starts, token, right=True) - 1
    positions = cached[of] + token - starts[of]
    slots = table[of, positions // block] * block + positions % block
    return {"table": table, "contexts": contexts, "starts": starts, "slots": slots, "positions": positions,
            "free_left": s["free_count"] - more.sum(dtype=torch.int32), "denied": torch.zeros_like(s["denied"])}


def _turned(x, cos, sin, rotary, adjacent):
    """The first `rotary` values of each head, turned by pairs; the others as they are."""
    if adjacent:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _plain_rotary(s):
    case, dtype = s["case"], s["qkv"].dtype
    q, k, v = _split(s)
    angle = s["positions"][s["axis"]].t().float() * s["frequencies"]
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    out = _turned(q.float(), cos, sin, case["rotary"], case["adjacent"]).to(dtype)
    s["keys"].view(-1, *k.shape[1:])[s["slots"]] = _turned(k.float(), cos, sin, case["rotary"], case["adjacent"]).to(dtype)
    s["cached_values"].view(-1, *v.shape[1:])[s["slots"]] = v
    return out, s["keys"], s["cached_values"]


def _weights(scores, allowed):
    """exp(scores - largest) where allowed, the sums and the largest; nothing allowed: zeros."""
    scores = scores.masked_fill(~allowed, -math.inf)
    largest = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(scores.dtype).min)
    weights = torch.exp(scores - largest)
    return weights, weights.sum(-1, keepdim=True), largest


def _plain_attention(q, k, v, starts, rows_max, lengths, causal):
    """q [tokens, heads, dim] packed by `starts`; k, v [sequences, keys, heads_kv, dim] of which `lengths` count."""
    tokens, heads, dim = q.shape
    n, keys, kv = k.shape[:3]
    count = starts[1:] - starts[:-1]
    row = torch.arange(rows_max, device="cuda")
    at = (starts[:-1, None] + row).clamp(max=tokens - 1)                    # [n, rows]
    qs = q[at].float().view(n, rows_max, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, dim)
    ks, vs = k.float().transpose(1, 2), v.float().transpose(1, 2)
    scores = torch.matmul(qs, ks.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(dim)).view(n, kv, -1, rows_max, keys)
    key = torch.arange(keys, device="cuda")
    allowed = key < lengths[:, None, None]                                  # [n, 1, keys]
    if causal:
        allowed = allowed & (key <= (lengths - count)[:, None, None] + row[:, None])
    weights, sums, largest = _weights(scores, allowed[:, None, None])
    out = torch.matmul(weights.view(n, kv, -1, keys), vs).view(n, kv, -1, rows_max, dim) / sums
    lse = (torch.log(sums) + largest)[..., 0]                               # [n, kv, group, rows]
    token = torch.arange(tokens, device="cuda", dtype=starts.dtype)
    of = torch.searchsorted(starts, token, right=True) - 1
    at = token - starts[of]
    return out[of, :, :, at].reshape(tokens, heads, dim).to(q.dtype), lse[of, :, :, at].reshape(tokens, heads).t().contiguous()


def _plain_prompt(s):
    q, k, v = _split(s)
    lengths = s["starts"][1:] - s["starts"][:-1]
    at = (s["starts"][:-1, None] + torch.arange(s["longest"], device="cuda")).clamp(max=s["total"] - 1)
    return _plain_attention(q, k[at], v[at], s["starts"], s["longest"], lengths, s["case"]["causal"])


def _plain_paged(s):
    block = s["case"]["block"]
    t = torch.arange(s["longest"], device="cuda")
    slots = s["table"][:, t // block].long() * block + t % block             # [requests, keys]
    k, v = (c.view(-1, *c.shape[2:])[slots] for c in (s["keys"], s["cached_values"]))
    return _plain_attention(s["q"], k, v, s["starts"], s["longest_new"], s["contexts"], True)


_plain = {"reserve": _plain_reserve, "rotary": _plain_rotary, "prompt": _plain_prompt, "paged": _plain_paged}


def _attention():
    root = os.path.join(os.getcwd(), "mini-caffe_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from minicaffe import attention
    return attention


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _kept(s, make):
    """The descriptors of a call, which a program makes once for its buffers."""
    if "call" not in s:
        s["call"] = make(_attention(), s)
    return s["call"]


def _own_reserve(s):
    def make(A, s):
        return A, [len(s["cached"]), s["case"]["block"], s["table"].shape[1], s["total"], len(s["free"])] + [s[n].data_ptr() for n in (
            "cached", "new", "free", "free_count", "table", "contexts", "starts", "slots", "positions", "free_left", "denied")]
    A, args = _kept(s, make)
    A.cache_reserve(*args, stream=_stream())
    return {n: s[n] for n in ("table", "contexts", "starts", "slots", "positions", "free_left", "denied")}


def _cache(A, s):
    c = s["keys"]
    return A.PagedCache(c.data_ptr(), s["cached_values"].data_ptr(), c.shape[0], c.shape[1], c.stride(0), c.stride(1), c.stride(2))


def _own_rotary(s):
    def make(A, s):
        c = s["case"]
        geom = A.rotary_geom(A.TYPES[c["type"]], c["heads"], c["heads_kv"], c["dim"], c["rotary"], _sections(c), adjacent=c["adjacent"],
                             cycled=c["cycled"])
        q, k, v = _split(s)
        return A, geom, A.heads_of(q), A.heads_of(k), A.heads_of(v), A.heads_of(s["out"]), _cache(A, s)
    A, geom, q, k, v, out, cache = _kept(s, make)
    A.rotary(geom, s["frequencies"].data_ptr(), s["positions"].data_ptr(), s["positions"].stride(0), s["case"]["tokens"],
             q, out, k=k, v=v, cache=cache, slots=s["slots"].data_ptr(), stream=_stream())
    return s["out"], s["keys"], s["cached_values"]


def _geom(A, c, causal):
    return A.AttentionGeom(A.TYPES[c["type"]], c["heads"], c["heads_kv"], c["dim"], int(causal), 1 / math.sqrt(c["dim"]))


def _own_prompt(s):
    def make(A, s):
        q, k, v = _split(s)
        return A, _geom(A, s["case"], s["case"]["causal"]), A.heads_of(q), A.heads_of(k), A.heads_of(v), A.heads_of(s["out"])
    A, geom, q, k, v, out = _kept(s, make)
    starts = s["starts"].data_ptr()
    A.attention_packed(geom, q, k, v, starts, starts, s["case"]["sequences"], s["total"], s["total"], out, lse=s["lse"].data_ptr(),
                       stream=_stream())
    return s["out"], s["lse"]


def _own_paged(s):
    def make(A, s):
        return A, _geom(A, s["case"], True), A.heads_of(s["q"]), _cache(A, s), A.heads_of(s["out"])
    A, geom, q, cache, out = _kept(s, make)
    A.attention_paged(geom, q, cache, s["table"].data_ptr(), s["table"].shape[1], s["starts"].data_ptr(), s["contexts"].data_ptr(),
                      s["case"]["requests"], s["total"], s["longest_new"], s["longest"], out, lse=s["lse"].data_ptr(),
                      stream=_stream())
    return s["out"], s["lse"]


_own = {"reserve": _own_reserve, "rotary": _own_rotary, "prompt": _own_prompt, "paged": _own_paged}


# ---- what cannot be done without ----------------------------------------------------

def work(case):
    if case["op"] == "reserve":
        new = _news(case)
        cached = _spread(case["requests"], 0, case["longest_cached"])
        fresh = int((_ceil(cached + new, case["block"]) - _ceil(cached, case["block"])).sum())
        tokens = int(new.sum())
        # lengths in and out, starts; fresh blocks out of the list into the table; a slot and a
        # position per token, and the table's entry where the token's block is an old one
        return {"bytes": 4 * (4 * case["requests"] + 2 * fresh + 2 * tokens), "flops": 0}
    size, dim = 4 if case["type"] == "f32" else 2, case["dim"]
    if case["op"] == "rotary":
        values = case["tokens"] * (case["heads"] + 2 * case["heads_kv"]) * dim
        turned = case["tokens"] * (case["heads"] + case["heads_kv"]) * case["rotary"]
        return {"bytes": 2 * size * values + 4 * case["tokens"] * (case["axes"] + 1), "flops": 3 * turned}
    if case["op"] == "prompt":
        keys = rows = _lengths(case)
        cells = rows * (rows + 1) // 2 if case["causal"] else rows * rows
        extra = 0
    else:
        rows, keys = _news(case), _contexts(case)
        cells = rows * keys - rows * (rows - 1) // 2
        extra = 4 * int(_ceil(keys, case["block"]).sum())
    return {"bytes": size * dim * (2 * case["heads"] * int(rows.sum()) + 2 * case["heads_kv"] * int(keys.sum()))
            + 4 * case["heads"] * int(rows.sum()) + extra,
            "flops": 4 * dim * case["heads"] * int(cells.sum())}


# ---- the definitions, in 64 bits ----------------------------------------------------

def exact(case, seed):
    if case["op"] == "reserve":
        return None                    # whole numbers
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "prompt": _exact_prompt, "paged": _exact_paged}[case["op"]](s)


def _exact_rotary(s):
    c = s["case"]
    q, k, v = _split(s)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[s["axis"].long()].t() * s["frequencies"].double())[:, None]

    def turned(x):
        """A pair is a complex number, and its turn a product."""
        x = x.double()
        y = x.clone()
        first, second = (slice(0, c["rotary"], 2), slice(1, c["rotary"], 2)) if c["adjacent"] else (
            slice(0, c["rotary"] // 2), slice(c["rotary"] // 2, c["rotary"]))
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y
    keys, values = s["keys"].double(), s["cached_values"].double()
    block = c["block"]
    at = s["slots"].long()
    keys[at // block, at % block] = turned(k)
    values[at // block, at % block] = v.double()
    return turned(q), keys, values


def _exact_one(q, k, v, causal):
    """One head: rows of q that end where the keys end."""
    rows, keys = len(q), len(k)
    scores = q.double() @ k.double().t().contiguous() / math.sqrt(q.shape[1])
    if causal:
        scores.masked_fill_(torch.ones((rows, keys), dtype=torch.bool, device="cuda").triu(keys - rows + 1), -math.inf)
    lse = torch.logsumexp(scores, -1)
    return torch.exp(scores - lse[:, None]) @ v.double(), lse


def _exact_prompt(s):
    c = s["case"]
    q, k, v = _split(s)
    out = torch.zeros((s["total"], c["heads"], c["dim"]), dtype=torch.float64, device="cuda")
    lse = torch.zeros((c["heads"], s["total"]), dtype=torch.float64, device="cuda")
    ends = s["starts"].tolist()
    for a, b in zip(ends[:-1], ends[1:]):
        for h in range(c["heads"]):
            j = h // (c["heads"] // c["heads_kv"])
            out[a:b, h], lse[h, a:b] = _exact_one(q[a:b, h], k[a:b, j], v[a:b, j], c["causal"])
    return out, lse


def _exact_paged(s):
    c = s["case"]
    out = torch.zeros((s["total"], c["heads"], c["dim"]), dtype=torch.float64, device="cuda")
    lse = torch.zeros((c["heads"], s["total"]), dtype=torch.float64, device="cuda")
    ends = s["starts"].tolist()
    for i, n in enumerate(s["contexts"].tolist()):
        blocks = s["table"][i, :_ceil(n, c["block"])].long()
        k, v = (x[blocks].flatten(0, 1)[:n] for x in (s["keys"], s["cached_values"]))
        a, b = ends[i], ends[i + 1]
        for h in range(c["heads"]):
            j = h // (c["heads"] // c["heads_kv"])
            out[a:b, h], lse[h, a:b] = _exact_one(s["q"][a:b, h], k[:, j], v[:, j], True)
    return out, lse
