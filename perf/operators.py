"""The four-bit operators of serving: products with 4-bit weights, tokens into a 4-bit cache and back, attention over that cache.

One format for all: a row of values lies in groups of 32, 64 or 128 neighbours, each group with two fp16 numbers (scale, low); a code
0..15 stands for low + scale * code; byte b of a row holds code 2b in its low and code 2b + 1 in its high four bits.

`own` False: each operator in its plain form, elementary torch operations in fp32.  `own` True: the calls of darknet_b200.fourbit.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
PRODUCT_WEIGHTS = 16384 * 16384           # most weights of one product
CACHE_VALUES = 131072 * 8 * 128           # most values of the keys (and of the values) that one call goes over, padding included
SCORES = 16 * 8192 * 4 * 24             # most scores of one attention call (batch * positions * tokens * heads)
APPEND_VALUES = 4 * 2048 * 8 * 128        # most values of the keys that one call writes


def _product(name, n, k, group, rows, dtype, bias, leaky):
    return {"name": name, "kind": "product", "n": n, "k": k, "group": group, "rows": rows, "dtype": dtype, "bias": bias, "leaky": leaky}


def _attend(name, batch, longest, tokens, heads, kv_heads, dim, group, page, window, dtype):
    return {"name": name, "kind": "attend", "batch": batch, "longest": longest, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "group": group, "page": page, "window": window, "dtype": dtype}


def _append(name, batch, tokens, held, kv_heads, dim, group, page, dtype):
    return {"name": name, "kind": "append", "batch": batch, "tokens": tokens, "held": held, "kv_heads": kv_heads, "dim": dim,
            "group": group, "page": page, "dtype": dtype}


def listed():
    return [
        # a classifier behind 1024 averaged channels, one picture: the smallest product
        _product("product 1024-1000 r1 fp32", 1000, 1024, 64, 1, "fp32", True, False),
        # one token through a square projection
        _product("product 4096-4096 r1 fp16", 4096, 4096, 128, 1, "fp16", False, False),
        # odd sizes everywhere, the smallest group, Darknet's activation
        _product("product 2305-5003 r3 fp32", 5003, 2305, 32, 3, "fp32", True, True),
        # sixteen sequences decoded at once through a matrix that does not fit the L2
        _product("product 16384-16384 r16 bf16", 16384, 16384, 128, 16, "bf16", False, False),
        # one user, a short conversation: latency
        _attend("attend b1 1000 fp16", 1, 1000, 1, 32, 8, 128, 128, 64, 0, "fp16"),
        # a served batch, lengths all over the place
        _attend("attend b64 to 2048 bf16", 64, 2048, 1, 32, 8, 128, 64, 64, 0, "bf16"),
        # one long document
        _attend("attend b1 131072 bf16", 1, 131072, 1, 64, 8, 128, 128, 256, 0, "bf16"),
        # a head of keys for every head of queries, small heads, all in fp32
        _attend("attend b8 to 4001 fp32", 8, 4001, 1, 16, 16, 64, 32, 16, 0, "fp32"),
        # four drafted tokens checked at once, behind a sliding window
        _attend("attend b16 t4 window bf16", 16, 8192, 4, 24, 4, 128, 64, 32, 4096, "bf16"),
        # the new token of every sequence of a batch
        _append("append b64 t1 bf16", 64, 1, 2047, 8, 128, 64, 64, "bf16"),
        # a few tokens of a few sequences, heads that are no power of two
        _append("append b5 t7 fp32", 5, 7, 100, 3, 96, 32, 16, "fp32"),
        # prompts
        _append("append b4 t2048 fp16", 4, 2048, 0, 8, 128, 128, 64, "fp16"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("product", "product", "attend", "attend", "append"))
    dtype = rng.choice(sorted(DTYPES))
    while True:
        if kind == "product":
            case = _product("", _log(rng, 64, 16384), _log(rng, 64, 16384), rng.choice((32, 64, 128)), rng.choice((1, _log(rng, 1, 16))),
                            dtype, rng.random() < 0.3, rng.random() < 0.2)
            fits = True
        elif kind == "attend":
            kv_heads, dim = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((32, 64, 96, 128, 128, 192, 256))
            case = _attend("", _log(rng, 1, 64), _log(rng, 1, 131072), rng.choice((1, 1, rng.randint(2, 8))),
                           kv_heads * rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 16)), kv_heads, dim, _group(rng, dim),
                           rng.choice((16, 32, 64, 128, 256)), rng.choice((0, 0, 0, _log(rng, 1, 8192))), dtype)
            seen = case["batch"] * case["longest"]
            fits = seen * kv_heads * dim <= CACHE_VALUES and seen * case["tokens"] * case["heads"] <= SCORES
        else:
            kv_heads, dim = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((32, 64, 96, 128, 128, 192, 256))
            case = _append("", _log(rng, 1, 64), _log(rng, 1, 2048), rng.choice((0, _log(rng, 1, 4096))), kv_heads, dim, _group(rng, dim),
                           rng.choice((16, 32, 64, 128, 256)), dtype)
            fits = (case["batch"] * case["tokens"] * kv_heads * dim <= APPEND_VALUES
                    and case["batch"] * (case["held"] + case["tokens"]) * kv_heads * dim <= 4 * APPEND_VALUES)
        if fits:
            del case["name"]
            return case


def _group(rng, dim):
    return rng.choice([g for g in (32, 64, 128) if dim % g == 0])


def _lengths(case):
    """Tokens that each sequence holds: all the way down from the longest to a quarter of it, in no order.  Part of the case: what a call
    has to read depends on it."""
    b = case["batch"]
    return [max(1, case["longest"] - (i * 5 % b) * case["longest"] * 3 // (4 * b)) for i in range(b)]


def _counts(case):
    """New tokens of each sequence: all there is room for in the first, down to half of it."""
    b = case["batch"]
    return [max(1, case["tokens"] - i * case["tokens"] // (2 * b)) for i in range(b)]


# ---- the format, in plain operations ----------------------------------------------------------------------------------------


def _half_down(v):
    h = v.half()
    bits = h.view(torch.int16)
    below = torch.where(h > 0, bits - 1, torch.where(h == 0, torch.full_like(bits, -32767), bits + 1))
    return torch.where(h.to(v.dtype) > v, below, bits).view(torch.float16)


def _half_up(v):
    return -_half_down(-v)


def _quantize(v, group):
    """codes (one a byte), and (scale, low) of each group of the last dimension, whose length is a multiple of the group's."""
    g = v.double().reshape(*v.shape[:-1], -1, group)          # a scale next to one of fp16's values, a value half way between two codes
    low = _half_down(g.amin(-1))
    scale = _half_up((g.amax(-1) - low.double()) / g.new_full((), 15.0))
    step = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    codes = ((g - low.double()[..., None]) / step[..., None]).round().clamp(0, 15).to(torch.uint8)
    return codes.reshape(v.shape), torch.stack((scale, low), -1)


def _pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _values(codes, scales, group, to=torch.float32):
    """What packed rows stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).to(to)
    c = c.reshape(*codes.shape[:-1], -1, group)
    return (scales[..., 1, None].to(to) + scales[..., 0, None].to(to) * c).reshape(*codes.shape[:-1], -1)


# ---- what a program has in hand before the call -----------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return {"product": _prepare_product, "attend": _prepare_attend, "append": _prepare_append}[case["kind"]](case, gen)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _prepare_product(case, gen):
    n, k, group = case["n"], case["k"], case["group"]
    held = -(-k // group) * group
    weights = _normal(gen, n, held) * k ** -0.5
    if held > k:
        weights[:, k:] = weights[:, k - 1:k]                 # the last group is filled up with values of its own
    packed, scales = zip(*((_pack(codes)[:, :-(-k // 32) * 16], scales) for codes, scales in (_quantize(w, group) for w in weights.split(4096))))
    state = {"kind": "product", "codes": torch.cat(packed), "scales": torch.cat(scales), "n": n, "k": k, "group": group,
             "leaky": case["leaky"], "biases": _normal(gen, n) * 0.1 if case["bias"] else None}
    # activations: a few channels are much larger than the others
    loud = torch.where(torch.rand(k, generator=gen, device=DEVICE) < 0.01, 10.0, 1.0)
    state["x"] = (_normal(gen, case["rows"], k) * loud).to(DTYPES[case["dtype"]])
    return state


def _tables(case, lengths, gen):
    """Pages in no order, some of them nobody's."""
    per = [-(-n // case["page"]) for n in lengths]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((case["batch"], max(per)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for row, n in zip(table, per):
        row[:n] = order[at:at + n]
        at += n
    return pages, table


def _prepare_attend(case, gen):
    lengths = _lengths(case)
    pages, table = _tables(case, lengths, gen)
    state = {"kind": "attend", "group": case["group"], "window": case["window"], "table": table, "longest": max(lengths),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE)}
    for name in ("k", "v"):
        # keys have channels that stand out, with a mean of their own
        loud = 1 + 4 * (torch.rand(case["kv_heads"], 1, case["dim"], generator=gen, device=DEVICE) < 0.03) if name == "k" else 1
        values = _normal(gen, pages, case["kv_heads"], case["page"], case["dim"]) * loud + (0.5 * loud if name == "k" else 0)
        codes, state[name + "_scales"] = _quantize(values, case["group"])
        state[name + "_codes"] = _pack(codes)
    state["q"] = _normal(gen, case["batch"], case["tokens"], case["heads"], case["dim"]).to(DTYPES[case["dtype"]])
    return state


def _prepare_append(case, gen):
    counts = _counts(case)
    lengths = [case["held"] + n for n in counts]
    pages, table = _tables(case, lengths, gen)
    kv, d, group = case["kv_heads"], case["dim"], case["group"]
    state = {"kind": "append", "group": group, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
             "counts": torch.tensor(counts, dtype=torch.int32, device=DEVICE)}
    for name in ("k", "v"):
        state[name + "_codes"] = torch.zeros(pages, kv, case["page"], d // 2, dtype=torch.uint8, device=DEVICE)
        state[name + "_scales"] = torch.zeros(pages, kv, case["page"], d // group, 2, dtype=torch.float16, device=DEVICE)
        state[name] = _normal(gen, case["batch"], case["tokens"], kv, d).to(DTYPES[case["dtype"]])
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return {"product": _plain_product, "attend": _plain_attend, "append": _plain_append}[state["kind"]](state)


def _own(state):
    from darknet_b200 import capi, fourbit
    handle = state.get("handle")
    if state["kind"] == "product":
        if handle is None:
            handle = state["handle"] = fourbit.Matrix4(state["codes"], state["scales"], state["k"], state["group"])
        return fourbit.forward_connected4(handle, state["x"], state["biases"], capi.LEAKY if state["leaky"] else capi.LINEAR)
    if handle is None:
        handle = state["handle"] = fourbit.Cache4(state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"], state["group"])
    if state["kind"] == "attend":
        return fourbit.attend4(handle, state["q"], state["table"], state["lengths"], window=state["window"])
    fourbit.append4(handle, state["k"], state["v"], state["table"], state["lengths"], state["counts"])
    return fourbit.read4(handle, state["table"], state["lengths"], state["k"].shape[1], state["counts"], state["k"].dtype)


def _plain_product(state):
    k, group = state["k"], state["group"]
    codes = state["codes"]
    short = state["scales"].shape[1] * group // 2 - codes.shape[1]
    if short:
        codes = torch.nn.functional.pad(codes, (0, short))
    y = state["x"].float() @ _values(codes, state["scales"], group)[:, :k].T
    if state["biases"] is not None:
        y = y + state["biases"]
    if state["leaky"]:
        y = torch.where(y > 0, y, 0.1 * y)
    return y.to(state["x"].dtype)


def _plain_attend(state):
    q, lengths, group = state["q"], state["lengths"], state["group"]
    b, t, heads, d = q.shape
    kv = state["k_codes"].shape[1]
    table = state["table"].clamp(min=0).long()

    def of_sequences(name):
        v = _values(state[name + "_codes"][table], state[name + "_scales"][table], group)        # [b][pages][kv][page][d]
        return v.transpose(1, 2).reshape(b, kv, -1, d)[:, :, :state["longest"]]

    keys = of_sequences("k")
    at = torch.arange(keys.shape[2], device=q.device)
    own_at = lengths[:, None] - t + torch.arange(t, device=q.device)                              # [b][t]
    seen = (at <= own_at[..., None]) & (at < lengths[:, None, None])
    if state["window"]:
        seen = seen & (at > own_at[..., None] - state["window"])
    seen = seen[:, None, :, None]                                                                 # [b][1][t][1][position]
    rows = q.float().reshape(b, t, kv, heads // kv, d).transpose(1, 2)                            # [b][kv][t][group of heads][d]
    scores = (rows.reshape(b, kv, -1, d) @ keys.transpose(2, 3) * d ** -0.5).reshape(b, kv, t, heads // kv, -1)
    del keys
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total > 0, total, 1.0)
    out = weights.reshape(b, kv, -1, weights.shape[-1]) @ of_sequences("v")
    return out.reshape(b, kv, t, heads // kv, d).transpose(1, 2).reshape(b, t, heads, d).to(q.dtype)


def _plain_append(state):
    lengths, counts = state["lengths"].long(), state["counts"].long()
    b, t = state["k"].shape[:2]
    page = state["k_codes"].shape[2]
    row = torch.arange(t, device=lengths.device)
    new = row < counts[:, None]
    row, sequence = torch.where(new, row, 0), torch.arange(b, device=lengths.device)[:, None]    # a row that is not new: row 0 once more
    at = (lengths - counts)[:, None] + row
    pages, places = state["table"].long().gather(1, at // page), at % page
    out = []
    for name in ("k", "v"):
        codes, scales = _quantize(state[name][sequence, row], state["group"])
        state[name + "_codes"][pages, :, places] = _pack(codes)
        state[name + "_scales"][pages, :, places] = scales
        stored = _values(_pack(codes), scales, state["group"])
        out.append(torch.where(new[..., None, None], stored, 0.0).to(state[name].dtype))
    return out


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"product": _exact_product, "attend": _exact_attend, "append": _exact_append}[case["kind"]](case, state)


def _exact_rows(codes, scales, group):
    both = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    both[..., 0::2], both[..., 1::2] = codes % 16, codes // 16
    spread = scales.double().repeat_interleave(group, dim=-2)[..., :both.shape[-1], :]
    return both.mul_(spread[..., 0]).add_(spread[..., 1])


def _exact_product(case, state):
    y, x = [], state["x"].double()
    for part, scales in zip(state["codes"].split(2048), state["scales"].split(2048)):
        y.append(torch.einsum("ni,ri->rn", _exact_rows(part, scales, case["group"])[:, :case["k"]], x))
    y = torch.cat(y, 1)
    if case["bias"]:
        y += state["biases"].double()
    return torch.maximum(y, y / 10) if case["leaky"] else y


def _exact_attend(case, state):
    heads, kv, d, t = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    out = torch.zeros(case["batch"], t, heads, d, dtype=torch.float64, device=DEVICE)
    for b, length in enumerate(_lengths(case)):
        pages = state["table"][b, :-(-length // case["page"])].long()
        for h in range(kv):
            k, v = (_exact_rows(state[x + "_codes"][pages, h].flatten(0, 1)[:length], state[x + "_scales"][pages, h].flatten(0, 1)[:length],
                                case["group"]) for x in "kv")
            for i in range(t):
                end = length - t + i + 1
                first = max(0, end - case["window"]) if case["window"] else 0
                if end > first:
                    mine = slice(h * heads // kv, (h + 1) * heads // kv)
                    p = torch.softmax(state["q"][b, i, mine].double() @ k[first:end].T / math.sqrt(d), -1)
                    out[b, i, mine] = p @ v[first:end]
    return out


def _exact_append(case, state):
    out = []
    for name in ("k", "v"):
        v = state[name].double()
        groups = v.unflatten(-1, (-1, case["group"]))
        low, top = groups.min(-1).values, groups.max(-1).values
        low = _exact_half(low, -1)
        scale = _exact_half((top - low) / torch.full_like(top, 15.0), 1)
        codes = torch.round((groups - low[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None])
        v = (low[..., None] + scale[..., None] * codes.clamp(0, 15)).flatten(-2)
        for row, n in zip(v, _counts(case)):
            row[n:] = 0
        out.append(v)
    return out


def _exact_half(v, way):
    """To fp16's grid, downwards (-1) or upwards (1)."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -14))) - 10)
    return torch.ceil(v / step) * step if way > 0 else torch.floor(v / step) * step


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "product":
        n, k, rows = case["n"], case["k"], case["rows"]
        nbytes = n * (k / 2 + 4 * -(-k // case["group"])) + size * rows * (n + k) + (4 * n if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 2.0 * rows * n * k}
    kv, d = case["kv_heads"], case["dim"]
    row = d / 2 + 4 * d // case["group"]                       # bytes of one packed key, or value, of one head
    if case["kind"] == "append":
        new = sum(_counts(case))
        # read once, written packed; read packed, written again
        return {"bytes": new * kv * 2 * (size * d + row) + new * kv * 2 * (size * d + row), "flops": 8.0 * new * kv * d}
    seen = scores = 0
    for length in _lengths(case):
        first = max(0, length - case["tokens"] - case["window"] + 1) if case["window"] else 0
        seen += length - first
        for i in range(case["tokens"]):
            end = max(0, length - case["tokens"] + i + 1)
            scores += min(end, case["window"]) if case["window"] else end
    return {"bytes": seen * kv * 2 * row + 2 * size * case["batch"] * case["tokens"] * case["heads"] * d, "flops": 4.0 * scores * case["heads"] * d}
