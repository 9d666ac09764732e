"""The operators of serving many sequences from a paged 8-bit cache, each through the call that a user's program makes.

  plan    `paged.plan_step`: page tables, positions and slots of a step, built on the GPU from the requests' lengths
  append  `paged.rope_append`: rotary embedding, keys and values into an e4m3 cache with one scale per page and head
  attend  `paged.attention`: attention over that cache, from single tokens to prompts
  sample  `sampling.sample`: temperature, top-k, top-p and min-p from one given random number per row

The plain form computes the same in elementary torch operations: 32 bits, 64 for the sampler, whose borders decide about tokens.
Inputs are made on the GPU from the seed; the lengths of the requests follow from the case, so that its work is known.
"""
import math

import torch

own = False

DEV = torch.device("cuda:0")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
TOP = 448.0                                                       # largest value of e4m3
FLOOR = -100                                                      # smallest exponent of a scale
THETA = 1.0e6


def listed():
    return [
        # a decode step of 32 sequences: each adds a token, one in 64 needs a page
        {"name": "plan_decode_32", "kind": "plan", "R": 32, "ctx": 4000, "new": 1, "page": 64, "mixed": False},
        # a step of a large server: prompts admitted beside decoding sequences, others over and their pages back
        {"name": "plan_admit_1024", "kind": "plan", "R": 1024, "ctx": 2000, "new": 200, "page": 16, "mixed": True},
        # the keys and values of a decode step of 8 sequences: all latency
        {"name": "append_decode_8", "kind": "append", "R": 8, "ctx": 1500, "new": 1, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # those of a prompt of 4096 tokens
        {"name": "append_prompt_4096", "kind": "append", "R": 1, "ctx": 0, "new": 4096, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # ragged pieces of prompts that begin and end inside pages, smaller heads, fp16
        {"name": "append_ragged_13", "kind": "append", "R": 13, "ctx": 333, "new": 57, "hq": 15, "hkv": 5, "D": 64, "page": 16, "dtype": "fp16"},
        # one sequence, a token: the step of a single user
        {"name": "attend_token_1", "kind": "attend", "R": 1, "ctx": 1000, "new": 1, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # a decode step of 64 sequences of 10 to 16384 tokens
        {"name": "attend_decode_64", "kind": "attend", "R": 64, "ctx": 16383, "new": 1, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # a few tokens at a time on one shared key and value head of 64, small pages, fp16
        {"name": "attend_shared_9", "kind": "attend", "R": 9, "ctx": 5003, "new": 3, "hq": 24, "hkv": 1, "D": 64, "page": 16, "dtype": "fp16"},
        # the second half of a prompt of 4096 tokens
        {"name": "attend_prompt_2048", "kind": "attend", "R": 1, "ctx": 2048, "new": 2048, "hq": 32, "hkv": 8, "D": 128, "page": 64, "dtype": "bf16"},
        # the logits of one sequence, nucleus sampling
        {"name": "sample_1", "kind": "sample", "R": 1, "V": 151936, "pad": 0, "dtype": "bf16", "mode": "nucleus"},
        # 64 sequences, each with settings of its own
        {"name": "sample_64", "kind": "sample", "R": 64, "V": 151936, "pad": 0, "dtype": "bf16", "mode": "mixed"},
        # an odd vocabulary in float32 behind which the head is padded, no filter
        {"name": "sample_odd_7", "kind": "sample", "R": 7, "V": 32003, "pad": 125, "dtype": "fp32", "mode": "plain"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "append", "attend", "attend", "sample"))
    if kind == "plan":
        R = _log(rng, 1, 1024)
        return {"kind": kind, "R": R, "ctx": _log(rng, 1, 8000), "new": _log(rng, 1, max(1, 200000 // R)) if rng.random() < 0.7 else 1,
                "page": rng.choice((16, 32, 64, 128)), "mixed": rng.random() < 0.6}
    if kind == "sample":
        R = _log(rng, 1, 64)
        return {"kind": kind, "R": R, "V": _log(rng, 100, 151936), "pad": rng.choice((0, 0, 1, 37, 128)), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                "mode": rng.choice(("nucleus", "mixed", "plain", "top_k"))}
    hkv = rng.choice((1, 2, 4, 5, 8))
    c = {"hq": hkv * rng.choice((1, 2, 3, 4, 6, 8, 16)), "hkv": hkv, "D": rng.choice((64, 128, 128)), "page": rng.choice((16, 32, 64, 128)),
         "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    if kind == "append":
        R = _log(rng, 1, 64)
        most = max(1, 4096 * 6144 // (R * (c["hq"] + 2 * hkv) * c["D"]))
        return {"kind": kind, "R": R, "ctx": _log(rng, 1, 4000) - 1, "new": _log(rng, 1, min(4096, most)) if rng.random() < 0.6 else 1, **c}
    if rng.random() < 0.6:                                        # decoding, one token or a few of each request
        R = _log(rng, 1, 96)
        most = max(2, 64 * 16384 * 1024 // (R * hkv * c["D"]))
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
    if case.get("mixed"):                                         # one in eight is over, one in eight waits, most others only decode
        adds = [-1 if i % 8 == 3 else 0 if i % 8 == 6 else 1 if i % 3 and i != full else a for i, a in enumerate(adds)]
    return have, adds


def _pages(tokens, page):
    return -(-tokens // page)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tables(have, width, page, spare, g):
    """Tables of scattered pages for what the requests have; the pages that are left over, and how many there are in all."""
    used = [_pages(h, page) for h in have]
    total = sum(used) + spare
    ids = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    tables = torch.full((len(have), width), -1, dtype=torch.int32, device=DEV)
    mask = torch.arange(width, device=DEV)[None, :] < _ints(used)[:, None]
    tables[mask] = ids[:sum(used)]
    return tables, ids[sum(used):].clone(), total


def _cache(pages, case, g):
    """Keys and values of earlier steps: e4m3 under scales that differ by page and head."""
    shape = (pages, case["hkv"], case["page"], case["D"])
    out = []
    for size in (2.0, 0.7):
        x = torch.empty(shape, dtype=E4M3, device=DEV)
        scale = torch.empty(pages, case["hkv"], dtype=torch.float32, device=DEV)
        for at in range(0, pages, 4096):
            part = torch.randn(x[at:at + 4096].shape, device=DEV, generator=g) * size * torch.exp(0.5 * torch.randn(x[at:at + 4096].shape[:2], device=DEV, generator=g))[:, :, None, None]
            s = _scale(part.abs().amax((2, 3)))
            x[at:at + 4096] = _e4m3(part / s[:, :, None, None])
            scale[at:at + 4096] = s
        out += [x, scale]
    return out[0], out[2], out[1], out[3]


def _e4m3(x):
    return x.clamp(-TOP, TOP).to(E4M3)


def _scale(amax):
    """The smallest power of two under which `amax` lies within e4m3."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, FLOOR).clamp(min=FLOOR))


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "sample":
        R, V = case["R"], case["V"]
        rank = torch.rand(R, V + case["pad"], device=DEV, generator=g).argsort(-1).float()
        x = 14.0 - 1.2 * torch.log(rank + 1) + 0.6 * torch.randn(R, V + case["pad"], device=DEV, generator=g)
        x[torch.rand(R, V + case["pad"], device=DEV, generator=g) < 0.01] = float("-inf")        # tokens that are not allowed
        i = torch.arange(R, device=DEV)

        def choose(*values):
            return torch.tensor(values, device=DEV)[(i + seed) % len(values)]

        state = {"kind": kind, "logits": x.to(DTYPES[case["dtype"]])[:, :V], "u": torch.rand(R, device=DEV, generator=g),
                 "temperature": None, "top_k": None, "top_p": None, "min_p": None}
        if case["mode"] == "nucleus":
            state.update(temperature=choose(0.8), top_p=choose(0.95))
        elif case["mode"] == "top_k":
            state.update(temperature=choose(0.7, 1.0), top_k=choose(50, 200, 20).to(torch.int32))
        elif case["mode"] == "mixed":
            state.update(temperature=choose(1.0, 0.6, 0.0, 1.3, 0.8), top_k=choose(0, 50, 20, 1000).to(torch.int32), top_p=choose(0.95, 1.0, 0.9),
                         min_p=choose(0.0, 0.05))
        return state
    have, adds = _lengths(case)
    page = case["page"]
    n = [max(a, 0) for a in adds]
    starts = [0]
    for a in n:
        starts.append(starts[-1] + a)
    spare = sum(_pages(h + a, page) - _pages(h, page) for h, a in zip(have, n)) + 7
    width = _pages(case["ctx"] + case["new"], page) + 1
    if kind == "plan":
        tables, free, total = _tables(have, width, page, spare, g)
        pool = torch.full((total,), -1, dtype=torch.int32, device=DEV)
        pool[:free.numel()] = free
        return {"kind": kind, "lengths": _ints(have), "new": _ints(adds), "tables": tables, "free": pool, "count": _ints([free.numel()]), "page": page,
                "tokens": starts[-1] + 5}
    seen = [h + a for h, a in zip(have, n)]
    tables, free, total = _tables(seen, width, page, 3, g)
    k, v, k_scale, v_scale = _cache(total, case, g)
    state = {"kind": kind, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "hq": case["hq"], "page": page, "tables": tables,
             "starts": _ints(starts), "seen": _ints(seen), "most": max(n), "longest": max(seen)}
    dt, T, D = DTYPES[case["dtype"]], starts[-1], case["D"]
    if kind == "attend":
        state["q"] = (1.5 * torch.randn(T, case["hq"], D, device=DEV, generator=g)).to(dt)
        return state
    row = torch.repeat_interleave(torch.arange(len(n), device=DEV), _ints(n).long())
    pos = torch.arange(T, device=DEV) - state["starts"][row] + _ints(have)[row]
    state["positions"] = pos.to(torch.int32)
    state["slots"] = (tables[row, pos // page] * page + pos % page).to(torch.int32)
    x = torch.randn(T, (case["hq"] + 2 * case["hkv"]) * D, device=DEV, generator=g)
    x *= torch.where(torch.rand(x.shape[1], device=DEV, generator=g) < 0.02, 8.0, 1.0)             # channels that stand out
    state["qkv"] = x.to(dt)
    angle = _angles(state["longest"], D)
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


def _angles(rows, D):
    inv = THETA ** -(torch.arange(0, D, 2, device=DEV).double() / D)
    return torch.arange(rows, device=DEV).double()[:, None] * inv


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _plan(s):
    lengths, new, tables, free, count, page, T = (s[x] for x in ("lengths", "new", "tables", "free", "count", "page", "tokens"))
    R, width = tables.shape
    lengths, new = lengths.long(), new.long()
    over, n = new < 0, new.clamp(min=0)
    ends = n.cumsum(0).clamp(max=T)
    starts = torch.cat([ends.new_zeros(1), ends])
    have = -(-lengths // page)
    fits = ~over & (n > 0) & (lengths + n <= width * page) & (n.cumsum(0) <= T)
    need = torch.where(fits, -(-(lengths + n) // page) - have, 0)
    back = tables[over[:, None] & (torch.arange(width, device=DEV) < have[:, None])]                # pages of the requests that are over
    supply = torch.cat([back, free[:int(count)].flip(0)])
    fits &= (need == 0) | (need.cumsum(0) <= supply.numel())
    need = torch.where(fits, need, 0)
    base, taken = need.cumsum(0) - need, int(need.sum())
    col = torch.arange(width, device=DEV) - have[:, None]
    grow = (col >= 0) & (col < need[:, None])
    tables[grow] = supply[(base[:, None] + col)[grow]]
    left = back[taken:]
    free[int(count):int(count) + left.numel()] = left
    lengths_out = torch.where(over, 0, torch.where(fits, lengths + n, lengths))
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(ends, t, right=True).clamp(max=R - 1)
    good = (t < ends[-1]) & fits[row]
    pos = torch.where(good, lengths[row] + t - starts[row], -1)
    slot = torch.where(good, tables[row, pos.clamp(min=0) // page] * page + pos % page, -1)
    seen = torch.where(fits, lengths + n, 0)
    whole = {"starts": starts, "positions": pos, "slots": slot, "seen": seen, "lengths": lengths_out, "count": count + (back.numel() - taken)}
    return {**{k: v.to(torch.int32) for k, v in whole.items()}, "tables": tables, "free": free}


def _rotated(x, cos, sin):
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _append(s):
    hq, page, slots = s["hq"], s["page"], s["slots"].long()
    hkv, D = s["k"].shape[1], s["k"].shape[3]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, D)
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]
    q = _rotated(x[:, :hq], cos, sin).to(s["qkv"].dtype)
    where, off = slots // page, slots % page
    first = torch.full((s["k"].shape[0],), page, dtype=torch.int64, device=DEV).scatter_reduce(0, where, off, "amin")
    for cache, scale, y in ((s["k"], s["k_scale"], _rotated(x[:, hq:hq + hkv], cos, sin)), (s["v"], s["v_scale"], x[:, hq + hkv:])):
        most = torch.zeros_like(scale).scatter_reduce(0, where[:, None].expand(-1, hkv), y.abs().amax(-1), "amax")
        touched = first < page
        old = torch.where((first == 0)[:, None], 0.0, scale)
        now = torch.where(touched[:, None], torch.maximum(old, _scale(most)), scale)
        ids = torch.nonzero(touched).squeeze(1)
        held = cache[ids].float()
        kept = torch.arange(page, device=DEV)[None, None, :, None] < first[ids][:, None, None, None]
        cache[ids] = torch.where(kept, _e4m3(held * (scale[ids] / now[ids])[:, :, None, None]).float(), held).to(E4M3)
        scale.copy_(now)
        cache.view(torch.uint8)[where, :, off] = _e4m3(y / scale[where][:, :, None]).view(torch.uint8)
    return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attend(s):
    q, starts, seen, page = s["q"].float(), s["starts"].long(), s["seen"].long(), s["page"]
    hq, D = q.shape[1:]
    hkv, R, L, N = s["k"].shape[1], seen.numel(), s["longest"], s["most"]
    ids = s["tables"][:, :-(-L // page)].long().clamp(min=0)

    def whole(cache, scale):                                      # [R, hkv, L, D], requests padded to the longest
        return (cache[ids].float() * scale[ids][..., None, None]).transpose(1, 2).reshape(R, hkv, -1, D)[:, :, :L]

    n = starts[1:] - starts[:-1]
    i = torch.arange(N, device=DEV)
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qq = q[rows].view(R, N, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(R, hkv, -1, D)
    pos = seen[:, None] - n[:, None] + i
    score = (qq @ whole(s["k"], s["k_scale"]).transpose(2, 3)).view(R, hkv, -1, N, L) * D ** -0.5
    hidden = torch.arange(L, device=DEV) > pos[:, :, None]
    score = score.masked_fill(hidden[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = (p.view(R, hkv, -1, L) @ whole(s["v"], s["v_scale"])).view(R, hkv, -1, N, D) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(R, N, hq, D)[i < n[:, None]].to(s["q"].dtype)


def _sample(s):
    x = s["logits"].double()
    R, V = x.shape
    t, k, p, least = s["temperature"], s["top_k"], s["top_p"], s["min_p"]
    t = torch.ones(R, device=DEV, dtype=torch.double) if t is None else t.double()
    greedy = t <= 0
    top, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((top - top[:, :1]) / torch.where(greedy, 1.0, t)[:, None])
    mass = w.cumsum(-1)
    keep = torch.full((R,), V, dtype=torch.int64, device=DEV)
    if k is not None:
        keep = torch.where(k > 0, k.long().clamp(max=V), keep)
    within = mass.gather(1, keep[:, None] - 1)
    if p is not None:
        keep = torch.where(p < 1, torch.minimum(keep, (mass < p.double()[:, None] * within).sum(-1) + 1), keep)
    if least is not None:
        keep = torch.where(least > 0, torch.minimum(keep, (w >= least.double()[:, None]).sum(-1)), keep)
    keep = torch.where(greedy, 1, keep.clamp(min=1))
    w = torch.where(torch.arange(V, device=DEV) < keep[:, None], w, 0.0)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    mass = by_index.cumsum(-1)
    token = (mass <= s["u"].double()[:, None] * mass[:, -1:]).sum(-1)
    return {"tokens": token, "logprobs": torch.log(by_index.gather(1, token[:, None]).squeeze(1) / mass[:, -1]).float()}


def run(state):
    kind = state["kind"]
    if not own:
        return {"plan": _plan, "append": _append, "attend": _attend, "sample": _sample}[kind](state)
    from htr_b200 import paged, sampling

    if kind == "plan":
        plan = paged.plan_step(state["lengths"], state["new"], state["tables"], state["free"], state["count"], state["page"], state["tokens"])
        return {"starts": plan.starts, "positions": plan.positions, "slots": plan.slots, "seen": plan.seen, "lengths": plan.lengths, "count": plan.count,
                "tables": state["tables"], "free": state["free"]}
    if kind == "append":
        cache = paged.LayerCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
        q = paged.rope_append(state["qkv"], state["positions"], state["slots"], state["cos"], state["sin"], cache, state["hq"])
        return {"q": q, "k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if kind == "attend":
        cache = paged.LayerCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
        return paged.attention(state["q"], state["starts"], state["seen"], state["tables"], cache, state["most"])
    tokens, logprobs = sampling.sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                                       min_p=state["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None                                               # whole numbers
    s = prepare(case, seed)
    if kind == "sample":
        return _exact_sample(s)
    if kind == "append":
        return _exact_append(case, s)
    out, rep = [], case["hq"] // case["hkv"]
    starts = s["starts"].tolist()
    for r, seen in enumerate(s["seen"].tolist()):                 # one request and head after the other
        q = s["q"][starts[r]:starts[r + 1]].double()
        pages = s["tables"][r, :_pages(seen, case["page"])].long()
        heads = []
        for h in range(case["hq"]):
            k, v = ((c[pages, h // rep].double() * f[pages, h // rep].double()[:, None, None]).reshape(-1, case["D"])[:seen]
                    for c, f in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
            a = q[:, h] @ k.T / math.sqrt(case["D"])
            a = a.masked_fill(torch.ones_like(a, dtype=torch.bool).triu(seen - q.shape[0] + 1), -math.inf)
            heads.append(a.softmax(-1) @ v)
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _exact_append(case, s):
    """Keys and values before they are rounded to 8 bits, in units of their page's scale."""
    hq, hkv, D, page = case["hq"], case["hkv"], case["D"], case["page"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    # the angles' sines and cosines are inputs
    z = torch.view_as_complex(x[:, :hq + hkv].reshape(x.shape[0], hq + hkv, D // 2, 2).contiguous())
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()]
    z = torch.view_as_real(z * turn[:, None]).flatten(-2)
    slots = s["slots"].tolist()
    pages = {}
    for t, slot in enumerate(slots):
        pages.setdefault(slot // page, []).append(t)
    found = {"q": z[:, :hq]}
    for name, y in (("k", z[:, hq:]), ("v", x[:, hq + hkv:])):
        held, scale = s[name].double(), s[name + "_scale"].double()
        for p, tokens in pages.items():
            new = y[tokens[0]:tokens[-1] + 1].transpose(0, 1)
            off = slots[tokens[0]] % page
            most = new.abs().amax((1, 2))
            fit = torch.exp2(torch.ceil(torch.log2(most / TOP)).clamp(min=FLOOR))
            fit = fit if off == 0 else torch.maximum(fit, scale[p])
            held[p, :, :off] *= (scale[p] / fit)[:, None, None]
            held[p, :, off:off + len(tokens)] = new / fit[:, None, None]
            scale[p] = fit
        found[name], found[name + "_scale"] = held, scale
    return found


def _exact_sample(s):
    """Row by row: the tokens in order, how many are kept, and the probability of the one that plays the random number's part."""
    found = []
    R, V = s["logits"].shape
    for r in range(R):
        x = s["logits"][r].double()
        t, k, p, least = (None if s[n] is None else float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t is not None and t <= 0:
            found.append(0.0)
            continue
        q = (x if t is None else x / t).softmax(-1)
        order = torch.argsort(x, descending=True, stable=True)
        n = V if not k else min(V, int(k))
        share = q[order[:n]] / q[order[:n]].sum()
        if p is not None and p < 1:
            n = min(n, int((share.cumsum(0) < p).sum()) + 1)
        if least:
            n = min(n, int((q[order] / q[order[0]] >= least).sum()))
        q[order[max(n, 1):]] = 0
        q /= q.sum()
        found.append(float(torch.log(q[min(V - 1, int(torch.searchsorted(q.cumsum(0), s["u"][r].double(), right=True)))])))
    return {"tokens": None, "logprobs": torch.tensor(found, dtype=torch.double)}


def work(case):
    kind = case["kind"]
    if kind == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["R"] * (case["V"] * size + 4 + 12), "flops": 3 * case["R"] * case["V"]}
    have, adds = _lengths(case)
    n = [max(a, 0) for a in adds]
    page, T = case["page"], sum(n)
    if kind == "plan":
        pages = sum(_pages(h + a, page) - _pages(h, page) for h, a in zip(have, n)) + sum(_pages(h, page) for h, a in zip(have, adds) if a < 0)
        return {"bytes": 4 * (5 * case["R"] + 2 * T + 2 * pages), "flops": 4 * T}
    hq, hkv, D = case["hq"], case["hkv"], case["D"]
    if kind == "append":
        return {"bytes": 2 * T * (2 * hq + 2 * hkv) * D + 2 * T * hkv * D + 8 * T + 4 * T * D, "flops": 3 * T * (hq + hkv) * D + 2 * T * hkv * D}
    seen = sum(h + a for h, a in zip(have, n))
    pairs = sum(a * h + a * (a + 1) // 2 for h, a in zip(have, n))
    return {"bytes": 2 * seen * hkv * D + 8 * hkv * seen // page + 4 * T * hq * D, "flops": 4 * hq * D * pairs}
