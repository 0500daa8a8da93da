"""The operators that take prompts into a small key/value cache and decode from it, as cases to be timed: attention over packed prompts,
the cache of 4 bits (rows into it and out of it), attention of new tokens over it, and its reduction to the positions that got the most
weight.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call, made from the seed
    run(state)          one pass: the operators' plain form, or (own) the framework's entry points
    work(case)          bytes and floating-point operations one pass cannot do without
    exact(case, seed)   the pass's outputs in 64 bits

A case is a dict: "kind" (below), "heads", "kv_heads", "head_size" and the kind's own sizes.

    prompt  causal attention over `sequences` prompts of ragged lengths up to `longest`, packed             type
    store   `tokens` new rows a sequence (ragged up to it where `packed`) into a cache that holds `start`   type
    attend  `rows` new rows a sequence over a 4-bit cache of ragged lengths up to `longest`                  mass
    evict   a cache of lengths up to `longest` reduced to `keep` positions, the last `recent` among them

A cache is one buffer: codes of K, codes of V, scales of K, scales of V, each [sequence][KV head][position] and then, of 32 values
each, 16 bytes of codes or two binary16 numbers (scale, lowest).  A word of 32 bits holds the codes of eight values: value 2 i at bit
4 i, value 2 i + 1 at bit 16 + 4 i.  A code stands for lowest + code * scale, rounded to binary16.
"""
import math
import random

import torch

own = False

GROUP = 32
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


def listed():
    return [
        # Four short questions that arrived together, read at once: latency.
        {"name": "prompt_questions", "kind": "prompt", "heads": 32, "kv_heads": 4, "head_size": 64, "sequences": 4, "longest": 45, "type": "f32"},
        # Several pages of different lengths, packed, with fp32 activations as the prefill has them.
        {"name": "prompt_pages_f32", "kind": "prompt", "heads": 32, "kv_heads": 8, "head_size": 64, "sequences": 7, "longest": 1500, "type": "f32"},
        # Many short requests packed, binary16 activations.
        {"name": "prompt_requests_f16", "kind": "prompt", "heads": 32, "kv_heads": 4, "head_size": 64, "sequences": 24, "longest": 250, "type": "f16"},
        # A long document through a larger model, binary16 activations.
        {"name": "prompt_document_f16", "kind": "prompt", "heads": 32, "kv_heads": 8, "head_size": 128, "sequences": 1, "longest": 8191, "type": "f16"},
        # One token of each conversation into the cache: the store of a decode step.
        {"name": "store_tokens", "kind": "store", "heads": 32, "kv_heads": 8, "head_size": 64, "sequences": 16, "tokens": 1, "start": 1000, "packed": False, "type": "f32"},
        # Packed prompts into the cache.
        {"name": "store_prompts", "kind": "store", "heads": 32, "kv_heads": 8, "head_size": 128, "sequences": 6, "tokens": 4000, "start": 0, "packed": True, "type": "f16"},
        # The next token of one short chat: latency.
        {"name": "attend_chat", "kind": "attend", "heads": 32, "kv_heads": 8, "head_size": 64, "sequences": 1, "rows": 1, "longest": 500, "mass": False},
        # The next token behind a long document.
        {"name": "attend_document", "kind": "attend", "heads": 32, "kv_heads": 8, "head_size": 64, "sequences": 1, "rows": 1, "longest": 16001, "mass": False},
        # A serving batch of a larger model, counting what each position is worth.
        {"name": "attend_batch_mass", "kind": "attend", "heads": 32, "kv_heads": 8, "head_size": 128, "sequences": 32, "rows": 1, "longest": 8000, "mass": True},
        # The last rows of some prompts asked once more, for the weights by which the cache is to be reduced.
        {"name": "attend_window_mass", "kind": "attend", "heads": 32, "kv_heads": 4, "head_size": 64, "sequences": 4, "rows": 16, "longest": 3000, "mass": True},
        # One conversation reduced to its budget.
        {"name": "evict_chat", "kind": "evict", "heads": 32, "kv_heads": 8, "head_size": 64, "sequences": 1, "longest": 2048, "keep": 512, "recent": 64},
        # A batch of long conversations reduced, larger heads.
        {"name": "evict_batch", "kind": "evict", "heads": 32, "kv_heads": 8, "head_size": 128, "sequences": 16, "longest": 8100, "keep": 2000, "recent": 256},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads, kv_heads, head_size = rng.choice(((32, 4, 64), (32, 8, 64), (32, 8, 128), (8, 8, 64), (12, 4, 128), (16, 1, 64), (6, 6, 128)))
    kind = rng.choice(("prompt", "prompt", "store", "attend", "attend", "attend", "evict"))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_size": head_size}
    if kind == "prompt":
        # (the plain form has the scores of all tokens with all tokens: no more than about 6000 in all)
        sequences = _log_uniform(rng, 1, 24)
        return case | {"sequences": sequences, "longest": _log_uniform(rng, 1, 6000 // sequences), "type": rng.choice(("f32", "f16"))}
    sequences = _log_uniform(rng, 1, 32)
    if kind == "store":
        packed = rng.random() < 0.5
        tokens = _log_uniform(rng, 1, 20000 // sequences) if packed else _log_uniform(rng, 1, 8)
        return case | {"sequences": sequences, "tokens": tokens, "start": 0 if rng.random() < 0.4 else _log_uniform(rng, 1, 2000), "packed": packed,
                       "type": rng.choice(("f32", "f16"))}
    longest = _log_uniform(rng, 1, min(20000, 160000 // sequences))
    if kind == "attend":
        rows = min(longest, rng.choice((1, 1, 1, rng.randint(2, 20))))
        return case | {"sequences": sequences, "rows": rows, "longest": longest, "mass": rng.random() < 0.5}
    keep = _log_uniform(rng, 1, longest)
    return case | {"sequences": sequences, "longest": longest, "keep": keep, "recent": rng.randint(0, keep)}


def _lengths(case):
    """The sequences' lengths: `longest`, and others from a sixth of it up, always the same for a case."""
    longest = case["tokens"] if case["kind"] == "store" else case["longest"]
    rng = random.Random(longest * 1009 + case["sequences"])
    if case["kind"] == "store" and not case["packed"]:
        return [longest] * case["sequences"]
    least = max(1, longest // 6, case.get("rows", 1))
    return [longest] + [rng.randint(least, longest) for _ in range(case["sequences"] - 1)]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _planes(buffer, sequences, kv_heads, room, head_size):
    """The four parts of a cache buffer as tensors of words: codes of K and V, scales of K and V."""
    rows = sequences * kv_heads * room
    parts = buffer.view(torch.int32).split([rows * head_size // 8] * 2 + [rows * head_size // GROUP] * 2)
    return [p.view(sequences, kv_heads, room, -1) for p in parts]


def _new_cache(sequences, kv_heads, room, head_size):
    return torch.zeros(sequences * kv_heads * room * head_size * 5 // 4, dtype=torch.uint8, device="cuda")


def _fill_cache(buffer, planes, gen):
    """A cache with something in it: codes of any value, groups between about -2.5 and 2.5."""
    codes = planes[0].numel() + planes[1].numel()
    buffer.view(torch.int32)[:codes].random_(-(2 ** 31), 2 ** 31 - 1, generator=gen)
    for p in planes[2:]:
        scale = torch.rand(p.shape, device="cuda", generator=gen) * 0.3 + 0.15
        low = scale * (torch.rand(p.shape, device="cuda", generator=gen) * 2.0 - 8.5)
        p.copy_(torch.stack((scale.half(), low.half()), -1).view(torch.int32).squeeze(-1))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    heads, kv_heads, hs, sequences = case["heads"], case["kv_heads"], case["head_size"], case["sequences"]
    lengths = _lengths(case)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    state = {"case": case, "lengths": lengths}
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    tokens = offsets[-1]
    if case["kind"] == "prompt":
        dtype = torch.float32 if case["type"] == "f32" else torch.float16
        state |= {"q": normal(tokens, heads * hs, dtype=dtype), "k": normal(tokens, kv_heads * hs, dtype=torch.float16),
                  "v": normal(tokens, kv_heads * hs, dtype=torch.float16), "offsets": whole(offsets),
                  "out": torch.zeros(tokens, heads * hs, dtype=dtype, device="cuda")}
    elif case["kind"] == "store":
        dtype = torch.float32 if case["type"] == "f32" else torch.float16
        room, count = case["start"] + max(lengths), max(lengths)
        cache = _new_cache(sequences, kv_heads, room, hs)
        state |= {"k": normal(tokens, kv_heads * hs, dtype=dtype), "v": normal(tokens, kv_heads * hs, dtype=dtype), "cache": cache, "room": room,
                  "offsets": whole(offsets) if case["packed"] else None, "starts": whole([case["start"]] * sequences),
                  "values": torch.zeros(2, sequences, kv_heads, count, hs, dtype=torch.float16, device="cuda")}
    elif case["kind"] == "attend":
        room = -(-max(lengths) // 64) * 64
        cache = _new_cache(sequences, kv_heads, room, hs)
        _fill_cache(cache, _planes(cache, sequences, kv_heads, room, hs), gen)
        rows = case["rows"]
        state |= {"cache": cache, "room": room, "q": normal(sequences, rows, heads * hs), "starts": whole([n - rows for n in lengths]),
                  "out": torch.zeros(sequences, rows, heads * hs, device="cuda"),
                  "mass": torch.zeros(sequences, kv_heads, room, device="cuda") if case["mass"] else None}
    else:
        room, keep = max(lengths), case["keep"]
        cache = _new_cache(sequences, kv_heads, room, hs)
        _fill_cache(cache, _planes(cache, sequences, kv_heads, room, hs), gen)
        # (weights as many steps leave them: a few positions with most of it, equal ones among the small)
        mass = torch.exp(2.0 * normal(sequences, kv_heads, room)).mul_(64.0).round_().div_(64.0)
        state |= {"cache": cache, "room": room, "mass": mass, "starts": whole(lengths), "less": _new_cache(sequences, kv_heads, keep, hs),
                  "less_mass": torch.zeros(sequences, kv_heads, keep, device="cuda"), "less_lengths": whole([0] * sequences),
                  "kept": torch.zeros(sequences, kv_heads, keep, dtype=torch.int32, device="cuda"),
                  "values": torch.zeros(2, sequences, kv_heads, keep, hs, dtype=torch.float16, device="cuda")}
    if case["kind"] == "attend":
        # what lpp_kv4_attention_workspace asks for at most: partial results of 64 ranges for every 16 rows of a KV head
        tiles = -(-case["rows"] // max(1, 16 // (heads // kv_heads)))
        state["workspace"] = torch.zeros(sequences * kv_heads * tiles * 64 * 16 * (hs + 2) * 4, dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return OWN[case["kind"]](state, case)
    return PLAIN[case["kind"]](state, case)


def _plain_prompt(state, case):
    heads, kv_heads, hs = case["heads"], case["kv_heads"], case["head_size"]
    tokens, shared = state["q"].shape[0], heads // kv_heads
    q = state["q"].float().view(tokens, kv_heads, shared, hs).permute(1, 2, 0, 3).reshape(kv_heads, shared * tokens, hs)
    k = state["k"].float().view(tokens, kv_heads, hs).permute(1, 2, 0).contiguous()
    v = state["v"].float().view(tokens, kv_heads, hs).permute(1, 0, 2).contiguous()
    at = torch.arange(tokens, device="cuda")
    sequence = torch.bucketize(at, state["offsets"][1:].long(), right=True)
    hidden = (sequence[:, None] != sequence[None, :]) | (at[:, None] < at[None, :])
    scores = torch.matmul(q, k).view(kv_heads, shared, tokens, tokens)
    scores = scores.mul_(1.0 / math.sqrt(hs)).masked_fill_(hidden, -math.inf)
    weights = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(kv_heads, shared * tokens, tokens), v).view(kv_heads, shared, tokens, hs) / total
    return out.permute(2, 0, 1, 3).reshape(tokens, heads * hs).to(state["q"].dtype)


def _codes(x):
    """Rows in groups of 32: (codes, scale, lowest), the last two binary16."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1, keepdim=True)
    scale = ((x.amax(-1, keepdim=True) - low) / 15.0).half()
    low = low.half()
    codes = torch.round((x.double() - low.double()) / scale.double()).nan_to_num_(0.0).clamp_(0, 15)
    return codes, scale, low


def _stands_for(codes, scale, low):
    return (low.float() + codes.float() * scale.float()).half().flatten(-2)


def _values(codes, scales):
    """What the words of a cache stand for, in binary16."""
    shifts = torch.tensor(SHIFTS, dtype=torch.int32, device="cuda")
    unpacked = ((codes.unsqueeze(-1) >> shifts) & 15).flatten(-2).unflatten(-1, (-1, GROUP))
    pair = scales.unsqueeze(-1).view(torch.float16)
    return _stands_for(unpacked, pair[..., 0:1], pair[..., 1:2])


def _plain_store(state, case):
    kv_heads, hs, sequences = case["kv_heads"], case["head_size"], case["sequences"]
    values, count = state["values"], state["values"].shape[3]
    tokens = state["k"].shape[0]
    at = torch.arange(tokens, device="cuda")
    if state["offsets"] is None:
        sequence, row = at // count, at % count
    else:
        sequence = torch.bucketize(at, state["offsets"][1:].long(), right=True)
        row = at - state["offsets"].long()[sequence]
    for i, x in enumerate((state["k"], state["v"])):
        values[i, sequence, :, row] = _stands_for(*_codes(x.view(tokens, kv_heads, hs)))
    return {"k": values[0], "v": values[1]}


def _plain_attend(state, case):
    heads, kv_heads, hs, rows, sequences = case["heads"], case["kv_heads"], case["head_size"], case["rows"], case["sequences"]
    shared, room = heads // kv_heads, state["room"]
    kc, vc, ks, vs = _planes(state["cache"], sequences, kv_heads, room, hs)
    k = _values(kc, ks).float().transpose(-1, -2).contiguous()
    q = state["q"].view(sequences, rows, kv_heads, shared, hs).permute(0, 2, 1, 3, 4).reshape(sequences, kv_heads, rows * shared, hs)
    end = state["starts"].long()[:, None] + 1 + torch.arange(rows, device="cuda")
    hidden = torch.arange(room, device="cuda") >= end[:, None, :, None, None]
    scores = (torch.matmul(q, k) * (1.0 / math.sqrt(hs))).view(sequences, kv_heads, rows, shared, room).masked_fill_(hidden, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    v = _values(vc, vs).float()
    v = v.masked_fill_((torch.arange(room, device="cuda") >= end[:, -1:]).view(sequences, 1, room, 1), 0.0)
    out = torch.matmul(weights.view(sequences, kv_heads, rows * shared, room), v)
    out = out.view(sequences, kv_heads, rows, shared, hs).permute(0, 2, 1, 3, 4).reshape(sequences, rows, heads * hs)
    if state["mass"] is None:
        return out
    state["mass"] += weights.sum((2, 3))
    return {"out": out, "mass": state["mass"]}


def _plain_evict(state, case):
    kv_heads, hs, sequences, keep, recent = case["kv_heads"], case["head_size"], case["sequences"], case["keep"], case["recent"]
    room, lengths = state["room"], state["starts"].long()[:, None, None]
    at = torch.arange(room, device="cuda")
    # recent positions before all others, positions behind the end after all others; equal weights in the order of the positions
    worth = state["mass"].double().masked_fill(at >= lengths - recent, math.inf).masked_fill(at >= lengths, -math.inf)
    best = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :keep]
    held = torch.arange(keep, device="cuda") < lengths
    kept = torch.where(held, best, room).sort(-1).values
    source = kept.clamp(max=room - 1)
    kc, vc, ks, vs = _planes(state["cache"], sequences, kv_heads, room, hs)
    moved = [torch.gather(p, 2, source.unsqueeze(-1).expand(-1, -1, -1, p.shape[-1])) for p in (kc, vc, ks, vs)]
    values = [_values(moved[i], moved[i + 2]).masked_fill(~held.unsqueeze(-1), 0.0) for i in (0, 1)]
    return {"k": values[0], "v": values[1], "mass": torch.gather(state["mass"], 2, source).masked_fill(~held, 0.0),
            "kept": torch.where(held, kept, -1).int(), "lengths": state["starts"].clamp(max=keep)}


PLAIN = {"prompt": _plain_prompt, "store": _plain_store, "attend": _plain_attend, "evict": _plain_evict}


_library = []


def _framework():
    """(the binding's module, the library), looked up once."""
    if not _library:
        from lighterpp_amd import capi
        _library.extend((capi, capi.load()))
    return _library


def _ptr(x):
    return None if x is None else x.data_ptr()


def _shape(capi, case, room):
    return capi.LppKv4Shape(1, case["sequences"], case["kv_heads"], room, case["head_size"])


def _own_prompt(state, case):
    capi, lib = _framework()
    q, k, v, out = state["q"], state["k"], state["v"], state["out"]
    capi.check(lib.lpp_prompt_attention(_ptr(out), _ptr(q), _ptr(k), _ptr(v), capi.F32 if case["type"] == "f32" else capi.F16,
                                        _ptr(state["offsets"]), case["sequences"], q.shape[0], case["heads"], case["kv_heads"],
                                        case["head_size"], q.shape[1], k.shape[1], out.shape[1]))
    return out


def _own_store(state, case):
    capi, lib = _framework()
    shape, k, v, values = _shape(capi, case, state["room"]), state["k"], state["v"], state["values"]
    capi.check(lib.lpp_kv4_store(_ptr(state["cache"]), shape, 0, _ptr(k), _ptr(v), capi.F32 if case["type"] == "f32" else capi.F16, k.shape[1],
                                 _ptr(state["offsets"]), k.shape[0], _ptr(state["starts"])))
    capi.check(lib.lpp_kv4_load(_ptr(values[0]), _ptr(values[1]), _ptr(state["cache"]), shape, 0, case["start"], values.shape[3]))
    return {"k": values[0], "v": values[1]}


def _own_attend(state, case):
    capi, lib = _framework()
    capi.check(lib.lpp_kv4_attention(_ptr(state["out"]), _ptr(state["q"]), _ptr(state["cache"]), _shape(capi, case, state["room"]), 0, case["heads"],
                                     case["rows"], _ptr(state["starts"]), _ptr(state["mass"]), _ptr(state["workspace"]), state["workspace"].numel()))
    return state["out"] if state["mass"] is None else {"out": state["out"], "mass": state["mass"]}


def _own_evict(state, case):
    capi, lib = _framework()
    keep, less, values = case["keep"], state["less"], state["values"]
    shape = _shape(capi, case, keep)
    capi.check(lib.lpp_kv4_evict(_ptr(less), shape, 0, _ptr(state["less_mass"]), _ptr(state["less_lengths"]), _ptr(state["kept"]), _ptr(state["cache"]),
                                 _shape(capi, case, state["room"]), 0, _ptr(state["mass"]), _ptr(state["starts"]), keep, case["recent"]))
    capi.check(lib.lpp_kv4_load(_ptr(values[0]), _ptr(values[1]), _ptr(less), shape, 0, 0, keep))
    return {"k": values[0], "v": values[1], "mass": state["less_mass"], "kept": state["kept"], "lengths": state["less_lengths"]}


OWN = {"prompt": _own_prompt, "store": _own_store, "attend": _own_attend, "evict": _own_evict}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    heads, kv_heads, hs = case["heads"], case["kv_heads"], case["head_size"]
    lengths = _lengths(case)
    tokens, row = sum(lengths), 2 * kv_heads * hs  # values of a position's K and V
    if case["kind"] == "prompt":
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": 2.0 * size * tokens * heads * hs + 2.0 * tokens * row, "flops": 4.0 * hs * heads * sum(n * (n + 1) / 2 for n in lengths)}
    if case["kind"] == "store":
        # rows read, codes and scales written; codes and scales read, values written
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": float(tokens * row * size + 1.25 * tokens * row + 2 * case["sequences"] * max(lengths) * row), "flops": 6.0 * tokens * row}
    if case["kind"] == "attend":
        rows = case["rows"]
        attended = sum(rows * n - rows * (rows - 1) // 2 for n in lengths)
        size = 0.625 * tokens * row + 8.0 * case["sequences"] * rows * heads * hs + (8.0 * kv_heads * tokens if case["mass"] else 0.0)
        return {"bytes": size, "flops": 4.0 * hs * heads * attended}
    kept = sum(min(n, case["keep"]) for n in lengths)
    # weights read; kept rows read, written, read again and written as values; the list and the weights kept
    return {"bytes": 4.0 * kv_heads * tokens + 3 * 0.625 * kept * row + 2.0 * kept * row + 8.0 * kv_heads * kept, "flops": 2.0 * kv_heads * tokens}


def _wide(codes, scales):
    """A cache's words as the binary16 numbers they stand for, in 64 bits."""
    parts = []
    for j in range(8):
        parts.append((codes >> ((j // 2) * 4 + (j % 2) * 16)) % 16)
    n = torch.stack(parts, -1).reshape(*codes.shape[:-1], scales.shape[-1], GROUP).to(torch.float64)
    halves = scales.contiguous().view(torch.float16).reshape(*scales.shape, 2).to(torch.float64)
    x = halves[..., 1].unsqueeze(-1) + n * halves[..., 0].unsqueeze(-1)
    return x.to(torch.float16).to(torch.float64).reshape(*codes.shape[:-1], -1)


def exact(case, seed):
    state = prepare(case, seed)
    heads, kv_heads, hs, sequences = case["heads"], case["kv_heads"], case["head_size"], case["sequences"]
    lengths, shared = state["lengths"], heads // kv_heads
    if case["kind"] == "prompt":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        begin = 0
        for n in lengths:
            upper = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            for h in range(heads):
                g = h // shared
                q = state["q"][begin:begin + n, h * hs:(h + 1) * hs].to(torch.float64)
                k = state["k"][begin:begin + n, g * hs:(g + 1) * hs].to(torch.float64)
                v = state["v"][begin:begin + n, g * hs:(g + 1) * hs].to(torch.float64)
                s = (q @ k.t().contiguous()) / math.sqrt(hs)
                s[upper] = -math.inf
                out[begin:begin + n, h * hs:(h + 1) * hs] = torch.softmax(s, -1) @ v
            begin += n
        return out
    if case["kind"] == "store":
        result = torch.zeros(state["values"].shape, dtype=torch.float64, device="cuda")
        begin = 0
        for s, n in enumerate(lengths):
            for i, x in enumerate((state["k"], state["v"])):
                x = x[begin:begin + n].reshape(n, kv_heads, hs // GROUP, GROUP).to(torch.float64)
                least, most = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
                scale = ((most.float() - least.float()) / 15.0).half().to(torch.float64)
                least = least.half().to(torch.float64)
                code = torch.clamp(torch.round((x - least) / scale), 0, 15)
                result[i, s, :, :n] = (least + code * scale).half().to(torch.float64).reshape(n, kv_heads, hs).transpose(0, 1)
            begin += n
        return {"k": result[0], "v": result[1]}
    planes = _planes(state["cache"], sequences, kv_heads, state["room"], hs)
    if case["kind"] == "attend":
        rows = case["rows"]
        out = torch.zeros(sequences, rows, heads * hs, dtype=torch.float64, device="cuda")
        mass = torch.zeros(sequences, kv_heads, state["room"], dtype=torch.float64, device="cuda")
        for s, n in enumerate(lengths):
            k, v = (_wide(planes[i][s, :, :n], planes[i + 2][s, :, :n]) for i in (0, 1))
            for j in range(rows):
                end = n - rows + j + 1
                q = state["q"][s, j].to(torch.float64).view(kv_heads, shared, hs)
                w = torch.softmax((q @ k[:, :end].transpose(1, 2).contiguous()) / math.sqrt(hs), -1)
                out[s, j] = (w @ v[:, :end]).reshape(-1)
                mass[s, :, :end] += w.sum(1)
        return out if not case["mass"] else {"out": out, "mass": mass}
    keep, recent = case["keep"], case["recent"]
    values = torch.zeros(2, sequences, kv_heads, keep, hs, dtype=torch.float64, device="cuda")
    mass = torch.zeros(sequences, kv_heads, keep, dtype=torch.float64, device="cuda")
    kept = torch.full((sequences, kv_heads, keep), -1, dtype=torch.int32, device="cuda")
    for s, n in enumerate(lengths):
        last, most = min(recent, n), min(keep, n)
        for h in range(kv_heads):
            weight = state["mass"][s, h, :n - last].to(torch.float64)
            order = torch.sort(weight, dim=0, descending=True, stable=True).indices[:most - last]
            at = torch.cat((order.sort().values, torch.arange(n - last, n, device="cuda")))
            kept[s, h, :most] = at.to(torch.int32)
            mass[s, h, :most] = state["mass"][s, h, at].to(torch.float64)
            for i in (0, 1):
                values[i, s, h, :most] = _wide(planes[i][s, h, at], planes[i + 2][s, h, at])
    return {"k": values[0], "v": values[1], "mass": mass, "kept": kept, "lengths": torch.tensor([min(keep, n) for n in lengths], dtype=torch.int32)}
