"""The operators of a paged cache in 4 bits, each through the call that a user's program makes.

  append  `paged.rope_append`: rotary embedding in either layout, a Hadamard transform of queries and keys, keys and values into an e2m1 cache
          with one scale per token and head
  attend  `paged.attention`: attention over that cache, from single tokens to prompts
  unpack  `paged.unpack`: pages of it as 16-bit keys and values
  angles  `rotary.angles`: cosines and sines of the positions of a long context

The plain form computes the same in elementary torch operations: 32 bits, 64 for the angles, whose positions go far.
What the cache holds in 4 bits is compared as the values that it stands for: an append returns the pages it wrote unpacked.
"""
import math

import torch

own = False

DEV = torch.device("cuda:0")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FLOOR = 2.0 ** -100                                               # smallest scale
LARGEST = 6.0 * 2.0 ** 119                                        # largest magnitude that is held
THETA = 1.0e6


def listed():
    return [
        # the keys and values of a decode step of 8 sequences: all latency
        {"name": "append_decode_8", "kind": "append", "R": 8, "ctx": 1500, "new": 1, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16", "layout": "interleaved", "rot": 128},
        # those of a prompt of 4096 tokens
        {"name": "append_prompt_4096", "kind": "append", "R": 1, "ctx": 0, "new": 4096, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16", "layout": "half", "rot": 128},
        # ragged pieces of prompts that begin and end inside pages, smaller heads of which half is rotated, fp16
        {"name": "append_ragged_13", "kind": "append", "R": 13, "ctx": 333, "new": 57, "hq": 15, "hkv": 5, "D": 64, "page": 16, "dtype": "fp16", "layout": "half", "rot": 32},
        # one sequence, a token: the step of a single user
        {"name": "attend_token_1", "kind": "attend", "R": 1, "ctx": 1000, "new": 1, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # a decode step of 64 sequences of 10 to 16384 tokens
        {"name": "attend_decode_64", "kind": "attend", "R": 64, "ctx": 16383, "new": 1, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # a few tokens at a time on one shared key and value head of 64, small pages, fp16
        {"name": "attend_shared_9", "kind": "attend", "R": 9, "ctx": 5003, "new": 3, "hq": 24, "hkv": 1, "D": 64, "page": 16, "dtype": "fp16"},
        # the second half of a prompt of 4096 tokens
        {"name": "attend_prompt_2048", "kind": "attend", "R": 1, "ctx": 2048, "new": 2048, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # odd pieces of three prompts, fp16
        {"name": "attend_pieces_3", "kind": "attend", "R": 3, "ctx": 1777, "new": 601, "hq": 16, "hkv": 4, "D": 128, "page": 32, "dtype": "fp16"},
        # the pages of one sequence, handed on to another cache
        {"name": "unpack_24", "kind": "unpack", "pages": 24, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # those of all sequences of a server that moves them
        {"name": "unpack_901", "kind": "unpack", "pages": 901, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # the positions of a context of 4096 tokens
        {"name": "angles_4096", "kind": "angles", "rows": 4096, "dim": 128, "factor": 1.0, "original": 0},
        # those of one of 262144 tokens for a model that learned 32768, slow dimensions stretched
        {"name": "angles_long", "kind": "angles", "rows": 262144, "dim": 128, "factor": 8.0, "original": 32768},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "append", "attend", "attend", "attend", "unpack", "angles"))
    if kind == "angles":
        return {"kind": kind, "rows": _log(rng, 1, 262144), "dim": rng.choice((32, 64, 96, 128)), "factor": rng.choice((1.0, 2.5, 4.0, 16.0)),
                "original": rng.choice((0, 2048, 8192, 32768))}
    hkv = rng.choice((1, 2, 4, 5, 8))
    D, page, dtype = rng.choice((64, 128, 128)), rng.choice((16, 32, 64, 128)), rng.choice(("bf16", "bf16", "fp16"))
    if kind == "unpack":
        return {"kind": kind, "pages": _log(rng, 1, 50 * 2 ** 20 // (hkv * page * D)), "hkv": hkv, "D": D, "page": page, "dtype": dtype}
    c = {"hq": hkv * rng.choice((1, 2, 3, 4, 6, 8, 16)), "hkv": hkv, "D": D, "page": page, "dtype": dtype}
    if kind == "append":
        R = _log(rng, 1, 64)
        most = max(1, 4096 * 6144 // (R * (c["hq"] + 2 * hkv) * D))
        return {"kind": kind, "R": R, "ctx": _log(rng, 1, 4000) - 1, "new": _log(rng, 1, min(4096, most)) if rng.random() < 0.6 else 1, **c,
                "layout": rng.choice(("interleaved", "half")), "rot": rng.choice((D, D, D, D // 2, 16, 48))}
    if rng.random() < 0.6:                                        # decoding, one token or a few of each request
        R = _log(rng, 1, 96)
        most = max(2, 64 * 16384 * 1024 // (R * hkv * D))
        return {"kind": kind, "R": R, "ctx": _log(rng, 1, min(16384, most)), "new": rng.choice((1, 1, 1, 2, 5)), **c}
    R = _log(rng, 1, 8)
    while True:                                                   # pieces of prompts
        new, ctx = _log(rng, 2, 2048), _log(rng, 1, 4096) - 1
        if R * new * (ctx + new) * c["hq"] <= 2048 * 4096 * 32:
            return {"kind": kind, "R": R, "ctx": ctx, "new": new, **c}


def _lengths(case):
    """What every request of the case has in the cache, and what it adds: spread from next to nothing to `ctx` and `new`."""
    R, ctx, new = case["R"], case["ctx"], case["new"]
    spread = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(R)]
    full = R // 2                                                 # one request has all of both
    have = [ctx if i == full else int(ctx * s * s) for i, s in enumerate(spread)]
    adds = [new if i == full or new == 1 else 1 + int((new - 1) * ((s * 7) % 1.0)) for i, s in enumerate(spread)]
    return have, adds


def _pages(tokens, page):
    return -(-tokens // page)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _quantised(x):
    """e2m1 codes, two in a byte, and the scale of every row of x (float32 [..., D])."""
    most = x.abs().amax(-1).clamp(max=LARGEST)                    # (a NaN stays one)
    scale = (most / 6.0).clamp(min=FLOOR).to(torch.bfloat16)
    y = x / scale.float()[..., None]
    a = y.abs()
    # to the nearest of the eight, ties to the even code
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0) + 8 * torch.signbit(y).to(torch.uint8)
    return code[..., ::2] + 16 * code[..., 1::2], scale


def _values(codes, scale):
    """The float32 values that codes and scales stand for."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=DEV)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return table[code.int()] * scale.float()[..., None]


def _cache(pages, case, g):
    """Keys and values of earlier steps: e2m1 under scales that differ by token and head."""
    shape = (pages, case["hkv"], case["page"])
    out = []
    for size in (2.0, 0.7):
        codes = torch.empty(*shape, case["D"] // 2, dtype=torch.uint8, device=DEV)
        scale = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        for at in range(0, pages, 1024):
            n = min(1024, pages - at)
            x = torch.randn(n, *shape[1:], case["D"], device=DEV, generator=g)
            x *= size * torch.exp(0.4 * torch.randn(n, *shape[1:], 1, device=DEV, generator=g))
            codes[at:at + n], scale[at:at + n] = _quantised(x)
        out += [codes, scale]
    return {"k": out[0], "k_scale": out[1], "v": out[2], "v_scale": out[3]}


def _hadamard(D):
    i = torch.arange(D, device=DEV)
    b = i[:, None] & i
    b = b ^ (b >> 4)
    b = b ^ (b >> 2)
    return (1 - 2 * ((b ^ (b >> 1)) & 1)).float()


def _frequencies(case):
    """Radians per position of every pair; those that turn less than `high` times within `original` positions are slowed, by up to `factor`."""
    inv = THETA ** -(torch.arange(0, case["dim"], 2, device=DEV).double() / case["dim"])
    if not case["original"]:
        return inv / case["factor"]
    keep = ((case["original"] * inv / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return inv * (keep + (1 - keep) / case["factor"])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    if kind == "angles":                                          # positions begin where the seed says: a step's table goes on where another ended
        return {"kind": kind, "case": case, "first": seed * 7919 % 100003, "magnitude": 1.0 + 0.01 * (seed % 17)}
    if kind == "unpack":
        total = case["pages"] + 5
        ids = torch.randperm(total, device=DEV, generator=g).to(torch.int32)[:case["pages"]].clone()
        return {"kind": kind, "pages": ids, "dtype": DTYPES[case["dtype"]], "H": _hadamard(case["D"]), **_cache(total, case, g)}
    have, n = _lengths(case)
    page = case["page"]
    starts = [0]
    for a in n:
        starts.append(starts[-1] + a)
    width = _pages(case["ctx"] + case["new"], page) + 1
    seen = [h + a for h, a in zip(have, n)]
    used = [_pages(h, page) for h in seen]
    total = sum(used) + 3
    ids = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    tables = torch.full((len(have), width), -1, dtype=torch.int32, device=DEV)
    mask = torch.arange(width, device=DEV)[None, :] < _ints(used)[:, None]
    tables[mask] = ids[:sum(used)]
    state = {"kind": kind, "hq": case["hq"], "page": page, "tables": tables, "starts": _ints(starts), "seen": _ints(seen), "most": max(n), "longest": max(seen),
             **_cache(total, case, g)}
    dt, T, D = DTYPES[case["dtype"]], starts[-1], case["D"]
    if kind == "attend":
        state["q"] = (1.5 * torch.randn(T, case["hq"], D, device=DEV, generator=g)).to(dt)
        return state
    row = torch.repeat_interleave(torch.arange(len(n), device=DEV), _ints(n).long())
    pos = torch.arange(T, device=DEV) - state["starts"][row] + _ints(have)[row]
    state["positions"] = pos.to(torch.int32)
    state["slots"] = (tables[row, pos // page] * page + pos % page).to(torch.int32)
    state["written"] = torch.unique(state["slots"] // page)       # the pages of this step
    x = torch.randn(T, (case["hq"] + 2 * case["hkv"]) * D, device=DEV, generator=g)
    x *= torch.where(torch.rand(x.shape[1], device=DEV, generator=g) < 0.02, 8.0, 1.0)             # channels that stand out
    state["qkv"] = x.to(dt)
    inv = THETA ** -(torch.arange(0, case["rot"], 2, device=DEV).double() / case["rot"])
    angle = torch.arange(state["longest"], device=DEV).double()[:, None] * inv
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    state["layout"], state["H"] = case["layout"], _hadamard(D)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _rotated(x, cos, sin, layout):
    r = 2 * cos.shape[-1]
    y, rest = x[..., :r], x[..., r:]
    if layout == "half":
        a, b = y[..., :r // 2], y[..., r // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
    a, b = y[..., ::2], y[..., 1::2]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)


def _append(s):
    hq, page, slots = s["hq"], s["page"], s["slots"].long()
    hkv, D = s["k"].shape[1], 2 * s["k"].shape[3]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, D)
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]
    y = _rotated(x[:, :hq + hkv], cos, sin, s["layout"]) @ s["H"]
    where, off = slots // page, slots % page
    for name, z in (("k", y[:, hq:] / 8), ("v", x[:, hq + hkv:])):
        s[name][where, :, off], s[name + "_scale"][where, :, off] = _quantised(z)
    return {"q": (y[:, :hq] / (D // 8)).to(s["qkv"].dtype), **_unpack(s, s["written"], s["qkv"].dtype)}


def _unpack(s, pages, dtype):
    at = pages.long()
    D = 2 * s["k"].shape[3]
    return {"k": (_values(s["k"][at], s["k_scale"][at]) @ s["H"] / (D // 8)).to(dtype), "v": _values(s["v"][at], s["v_scale"][at]).to(dtype)}


def _attend(s):
    q, starts, seen = s["q"].float(), s["starts"].long(), s["seen"].long()
    hq, D = q.shape[1:]
    hkv, R, L, N = s["k"].shape[1], seen.numel(), s["longest"], s["most"]
    ids = s["tables"][:, :-(-L // s["page"])].long().clamp(min=0)

    def whole(name):                                              # [R, hkv, L, D], requests padded to the longest
        return _values(s[name][ids], s[name + "_scale"][ids]).transpose(1, 2).reshape(R, hkv, -1, D)[:, :, :L]

    n = starts[1:] - starts[:-1]
    i = torch.arange(N, device=DEV)
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qq = q[rows].view(R, N, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(R, hkv, -1, D)
    pos = seen[:, None] - n[:, None] + i
    score = (qq @ whole("k").transpose(2, 3)).view(R, hkv, -1, N, L) * D ** -0.5
    hidden = torch.arange(L, device=DEV) > pos[:, :, None]
    score = score.masked_fill(hidden[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = (p.view(R, hkv, -1, L) @ whole("v")).view(R, hkv, -1, N, D) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(R, N, hq, D)[i < n[:, None]].to(s["q"].dtype)


def _angles(s):
    angle = torch.arange(s["first"], s["first"] + s["case"]["rows"], device=DEV).double()[:, None] * _frequencies(s["case"])
    return {"cos": (angle.cos() * s["magnitude"]).float(), "sin": (angle.sin() * s["magnitude"]).float()}


def run(state):
    kind = state["kind"]
    if not own:
        if kind == "unpack":
            return _unpack(state, state["pages"], state["dtype"])
        return {"append": _append, "attend": _attend, "angles": _angles}[kind](state)
    from htr_b200 import paged, rotary

    if kind == "angles":
        c = state["case"]
        cos, sin = rotary.angles(c["rows"], c["dim"], THETA, first=state["first"], factor=c["factor"], original=c["original"] or None,
                                 magnitude=state["magnitude"], device=DEV)
        return {"cos": cos, "sin": sin}
    cache = paged.LayerCache4(state["k"], state["v"], state["k_scale"], state["v_scale"])
    if kind == "unpack":
        k, v = paged.unpack(cache, state["pages"], state["dtype"])
        return {"k": k, "v": v}
    if kind == "attend":
        return paged.attention(state["q"], state["starts"], state["seen"], state["tables"], cache, state["most"])
    q = paged.rope_append(state["qkv"], state["positions"], state["slots"], state["cos"], state["sin"], cache, state["hq"], layout=state["layout"])
    k, v = paged.unpack(cache, state["written"], state["qkv"].dtype)
    return {"q": q, "k": k, "v": v}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def _sylvester(D):
    h = torch.ones(1, 1, dtype=torch.double, device=DEV)
    while h.shape[0] < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h


def _held(codes, scale):
    low, high = codes.long() % 16, codes.long() // 16
    c = torch.stack((low, high), -1).flatten(-2)
    e, m = c % 8 // 2, c % 2
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
    return torch.where(c >= 8, -size, size) * scale.double()[..., None]


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "angles":
        turns = torch.arange(s["first"], s["first"] + case["rows"], device=DEV).double()[:, None] * (_frequencies(case) / (2 * math.pi))
        z = torch.polar(torch.full_like(turns, s["magnitude"]), 2 * math.pi * (turns - turns.round()))
        return {"cos": z.real, "sin": z.imag}
    H = _sylvester(case["D"])
    if kind == "unpack":
        at = s["pages"].long()
        return {"k": _held(s["k"][at], s["k_scale"][at]) @ H * 8 / case["D"], "v": _held(s["v"][at], s["v_scale"][at])}
    if kind == "append":
        return _exact_append(case, s, H)
    out, rep = [], case["hq"] // case["hkv"]
    starts = s["starts"].tolist()
    for r, seen in enumerate(s["seen"].tolist()):                 # one request and head after the other
        q = s["q"][starts[r]:starts[r + 1]].double()
        pages = s["tables"][r, :_pages(seen, case["page"])].long()
        heads = []
        for h in range(case["hq"]):
            k, v = (_held(s[c][pages, h // rep], s[c + "_scale"][pages, h // rep]).reshape(-1, case["D"])[:seen] for c in ("k", "v"))
            a = q[:, h] @ k.T / math.sqrt(case["D"])
            a = a.masked_fill(torch.ones_like(a, dtype=torch.bool).triu(seen - q.shape[0] + 1), -math.inf)
            heads.append(a.softmax(-1) @ v)
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _exact_append(case, s, H):
    hq, hkv, D, page, half = case["hq"], case["hkv"], case["D"], case["page"], case["rot"] // 2
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    # the angles' sines and cosines are inputs
    first = torch.arange(half, device=DEV) * (2 if case["layout"] == "interleaved" else 1)
    second = first + (1 if case["layout"] == "interleaved" else half)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
    z = torch.complex(x[..., first], x[..., second])[:, :hq + hkv] * turn
    y = x[:, :hq + hkv].clone()
    y[..., first], y[..., second] = z.real, z.imag
    y = y @ H
    found = {"q": y[:, :hq] * 8 / D}
    at = s["written"].long()
    levels = torch.tensor(E2M1, dtype=torch.double, device=DEV)
    slots = s["slots"].long()
    for name, new in (("k", y[:, hq:] / 8), ("v", x[:, hq + hkv:])):
        scale = (new.abs().amax(-1, keepdim=True) / 6).to(torch.bfloat16).double()
        below, above = (torch.bucketize((new / scale).abs(), (levels[1:] + levels[:-1]) / 2, right=right) for right in (False, True))
        size = levels[torch.where(below % 2 == 0, below, above)]  # (they differ at a tie, which goes to the even code)
        held = _held(s[name], s[name + "_scale"])
        held[slots // page, :, slots % page] = torch.copysign(size, new) * scale
        found[name] = held[at] @ H * 8 / D if name == "k" else held[at]
    return found


def work(case):
    kind = case["kind"]
    if kind == "angles":
        return {"bytes": 4 * case["rows"] * case["dim"], "flops": 20 * case["rows"] * case["dim"]}
    hkv, D, page = case["hkv"], case["D"], case["page"]
    held, wide = D + 4, 4 * D                                     # bytes of a token and head, keys and values: in the cache, and unpacked
    turn = D * D.bit_length()                                     # additions of a transform
    if kind == "unpack":
        return {"bytes": case["pages"] * hkv * page * (held + wide), "flops": case["pages"] * hkv * page * turn}
    have, n = _lengths(case)
    T, hq = sum(n), case["hq"]
    if kind == "append":
        pages = sum(_pages(h + a, page) - h // page for h, a in zip(have, n))
        return {"bytes": 2 * T * (2 * hq + 2 * hkv) * D + T * hkv * held + 8 * T + 4 * T * case["rot"] + pages * hkv * page * (held + wide),
                "flops": T * (hq + hkv) * (3 * case["rot"] + turn) + pages * hkv * page * turn}
    seen = sum(h + a for h, a in zip(have, n))
    pairs = sum(a * h + a * (a + 1) // 2 for h, a in zip(have, n))
    return {"bytes": seen * hkv * held + 4 * T * hq * D, "flops": 4 * hq * D * pairs}
