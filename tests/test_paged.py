"""Page plans, the paged 8-bit cache and attention over it, against plain evaluations in 64 bits and in lists."""
import pytest
import torch

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")
E4M3 = torch.float8_e4m3fn


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---- plan_step ------------------------------------------------------------------------------------------------------


def plan_by_hand(lengths, new, tables, free, count, page, T):
    """The same step in lists; `tables` (rows of page lists, -1 where none) and `free` are changed."""
    width, back, status = len(tables[0]), [], 0
    for r, (n, a) in enumerate(zip(lengths, new)):
        if a < 0 and 0 <= n <= width * page:
            back += tables[r][:-(-n // page)]
    supply = back + free[:count][::-1]
    starts, positions, slots, seen, after, at, taken = [0], [], [], [], [], 0, 0
    for r, (n, a) in enumerate(zip(lengths, new)):
        ok = a > 0
        if not 0 <= n <= width * page:
            status, ok = status | 4, False
        if at + max(a, 0) > T:
            status, ok = status | 8, False
        if ok and n + a > width * page:
            status, ok = status | 2, False
        need = -(-(n + a) // page) - -(-n // page) if ok else 0
        if need:
            if taken + need > len(supply):
                status, ok = status | 1, False
                taken = len(supply) + 1                      # later requests that need pages get none either
            else:
                tables[r][-(-n // page):-(-n // page) + need] = supply[taken:taken + need]
                taken += need
        for i in range(max(a, 0)):
            if at + i < T:
                p = n + i
                positions.append(p if ok else -1)
                slots.append(tables[r][p // page] * page + p % page if ok else -1)
        at += max(a, 0)
        starts.append(min(at, T))
        seen.append(n + a if ok else 0)
        after.append(0 if a < 0 else n + a if ok else n)
    if taken > len(supply):                                  # what was served before pages ran out
        taken = sum(-(-s // page) - -(-n // page) for s, n in zip(seen, lengths) if s)
    left = back[taken:]
    free[count:count + len(left)] = left
    positions += [-1] * (T - len(positions))
    slots += [-1] * (T - len(slots))
    return starts, positions, slots, seen, after, count + len(back) - taken, status


def check_plan(lengths, new, tables, free, count, page, T, pad=0):
    from htr_b200 import paged

    R, width = len(lengths), len(tables[0])
    dev_tables = torch.full((R, width + pad), -7, dtype=torch.int32, device=DEV)[:, :width]
    dev_tables.copy_(ints(tables))
    dev_free, status = ints(free), ints([0])
    plan = paged.plan_step(ints(lengths), ints(new), dev_tables, dev_free, ints([count]), page, T, status=status)
    want = plan_by_hand(lengths, new, tables, free, count, page, T)
    for name, w in zip(("starts", "positions", "slots", "seen", "lengths"), want):
        assert getattr(plan, name).tolist() == w, name
    assert plan.count.tolist() == [want[5]] and status.tolist() == [want[6]]
    assert dev_tables.tolist() == tables
    assert dev_free.tolist()[:want[5]] == free[:want[5]]
    return want


def a_state(g, R, width, page, spare, most):
    lengths = [int(torch.randint(0, most + 1, (1,), generator=g)) for _ in range(R)]
    used = [-(-n // page) for n in lengths]
    total = sum(used) + spare
    ids = torch.randperm(total, generator=g).tolist()
    tables, at = [], 0
    for u in used:
        tables.append(ids[at:at + u] + [-1] * (width - u))
        at += u
    return lengths, tables, ids[at:] + [-1] * at, spare


@gpu
@pytest.mark.parametrize("R,page,most,spare,T", ((1, 16, 0, 3, 40), (3, 16, 50, 20, 60), (33, 64, 500, 30, 2000), (513, 32, 200, 700, 9000), (2000, 128, 300, 100, 1500),
                                                 (8192, 16, 20, 4000, 30000)))
@pytest.mark.parametrize("kind", ("tokens", "mixed", "scarce"))
def test_plan_against_lists(R, page, most, spare, T, kind):
    g = torch.Generator().manual_seed(R + page)
    width = -(-(most + 130) // page)
    lengths, tables, free, count = a_state(g, R, width, page, spare, most)
    if kind == "tokens":
        new = [1] * R
    else:
        new = [int(torch.randint(-1, 2 if i % 3 else 120, (1,), generator=g)) for i in range(R)]
    if kind == "scarce":
        count = min(count, 2)
    check_plan(lengths, new, tables, free, count, page, T, pad=3)


@gpu
def test_plan_refuses_what_does_not_fit():
    page = 16
    free = [9, 8, 7, 6, -1, -1, -1, -1, -1, -1]
    tables = [[0, 1, -1], [2, -1, -1], [3, 4, 5], [-1, -1, -1]]
    assert check_plan([32, 5, 40, 0], [17, 12, 9, 3], [t[:] for t in tables], free[:], 4, page, 64)[-1] == 2           # two tables are full
    assert check_plan([32, 5, 40, 0], [16, 30, 8, 3], [t[:] for t in tables], free[:], 2, page, 64)[-1] == 1           # no pages left
    assert check_plan([32, 5, 40, 0], [16, 30, -1, 3], [t[:] for t in tables], free[:], 0, page, 64)[-1] == 1          # ... but for those that come back
    assert check_plan([-3, 5, 49, 0], [1, 2, -1, 3], [t[:] for t in tables], free[:], 4, page, 64)[-1] == 4            # impossible lengths
    assert check_plan([3, 5, 40, 0], [1, 2, 5, 3], [t[:] for t in tables], free[:], 4, page, 7)[-1] == 8               # more tokens than announced
    assert check_plan([3, 5, 40, 0], [0, 0, 0, 0], [t[:] for t in tables], free[:], 4, page, 0)[-1] == 0               # nothing to do


@gpu
@pytest.mark.parametrize("captured", (False, True))
def test_pages_are_conserved_over_many_steps(captured):
    """A server's life on the buffers of one cache, updated in place: no page is ever held twice or lost."""
    from htr_b200 import paged

    R, page, pages, most = 40, 16, 200, 300
    cache = paged.PagedCache(1, 1, 64, pages, page, R, most, DEV)
    g = torch.Generator().manual_seed(1)
    new = ints([0] * R)
    cache.plan(new, 700)
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.plan(new, 700)
    held = 0
    for step in range(60):
        a = torch.where(torch.rand(R, generator=g) < 0.08, -1, torch.where(torch.rand(R, generator=g) < 0.15, torch.randint(0, 60, (R,), generator=g), 1))
        new.copy_(a.to(torch.int32))
        before = cache.lengths.tolist()
        if captured:
            graph.replay()
        else:
            cache.plan(new, 700)
        lengths, tables, n = cache.lengths.tolist(), cache.tables.tolist(), int(cache.count)
        used = [p for r in range(R) for p in tables[r][:-(-lengths[r] // page)]]
        assert sorted(used + cache.free.tolist()[:n]) == list(range(pages))
        assert all(x == (0 if y < 0 else b + y) or x == b for x, y, b in zip(lengths, a.tolist(), before))
        held = max(held, len(used))
    assert held > pages // 2


# ---- rope_append ----------------------------------------------------------------------------------------------------


def angles(rows, D):
    a = torch.arange(rows, device=DEV).double()[:, None] * 1.0e4 ** -(torch.arange(0, D, 2, device=DEV).double() / D)
    return a.cos().float(), a.sin().float()


def rotated(x, cos, sin):
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def empty_cache(pages, hkv, page, D, fill=0x7F):
    """A cache of bytes that would show (0x7F is NaN) wherever something is read that was never written."""
    from htr_b200 import paged

    k = torch.full((pages, hkv, page, D), fill, dtype=torch.uint8, device=DEV).view(E4M3)
    s = torch.full((pages, hkv), 2.0 ** 20, device=DEV)
    return paged.LayerCache(k, k.clone(), s, s.clone())


def wanted_exponent(most):
    e = -100
    while most > 448.0 * 2.0 ** e:
        e += 1
    return e


def check_append(dtype, D, page, hq, hkv, steps, size=1.0, pages=40, slack=0):
    """Runs steps = [(tokens of request 0, of request 1, ...), ...] and checks the cache's contents after each of them."""
    from htr_b200 import paged

    R = len(steps[0])
    cache, g = empty_cache(pages, hkv, page, D), torch.Generator(device=DEV).manual_seed(D + page + hq)
    width = pages // R
    tables = torch.randperm(pages, generator=torch.Generator().manual_seed(3))[:R * width].view(R, width)
    cos, sin = angles(width * page, D)
    have = [0] * R
    truth = [[[] for _ in range(R)] for _ in range(2)]           # exact k and v of every request
    growths = {}
    for adds in steps:
        T = sum(adds)
        pos = [have[r] + i for r in range(R) for i in range(adds[r])]
        row = [r for r in range(R) for _ in range(adds[r])]
        slots = [int(tables[r, p // page]) * page + p % page for r, p in zip(row, pos)]
        wide = torch.randn(T, (hq + 2 * hkv) * D + slack, device=DEV, generator=g) * size * torch.exp(torch.randn(T, 1, device=DEV, generator=g))
        x = wide.to(dtype)[:, :(hq + 2 * hkv) * D]
        q = paged.rope_append(x, ints(pos), ints(slots), cos, sin, cache, hq)
        y = x.double().reshape(T, hq + 2 * hkv, D)
        c, s = (t.double()[torch.tensor(pos, device=DEV)][:, None] for t in (cos, sin))
        qw, kw = rotated(y[:, :hq], c, s), rotated(y[:, hq:hq + hkv], c, s)
        # float32 rotation: three roundings relative to the terms, then one to the output's type (half a step) or, near zero, its smallest steps
        terms = rotated(y[:, :hq].abs(), c.abs(), -s.abs()).abs() + rotated(y[:, :hq].abs(), c.abs(), s.abs()).abs()
        assert ((q.double() - qw).abs() <= torch.finfo(dtype).eps / 2 * qw.abs() + 3 * 2.0 ** -24 * terms + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()
        for r in range(R):
            at = [i for i in range(T) if row[i] == r]
            truth[0][r] += list(kw[at])
            truth[1][r] += list(y[at, hq + hkv:])
            have[r] += adds[r]
        for part, (data, scale) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
            for r in range(R):
                for j in range(-(-have[r] // page)):
                    exact = torch.stack(truth[part][r][j * page:(j + 1) * page])
                    id = int(tables[r, j])
                    got = data[id, :, :exact.shape[0]].double().transpose(0, 1) * scale[id].double()[None, :, None]
                    sc = scale[id].double()
                    for h in range(hkv):
                        e = wanted_exponent(float(exact[:, h].abs().max().float()))
                        assert float(sc[h]) == 2.0 ** e, (float(sc[h]), e)
                        if growths.get((part, id, h), e) != e:
                            growths[part, id, h, "n"] = growths.get((part, id, h, "n"), 0) + 1
                        growths[part, id, h] = e
                    # half a step of e4m3 (2^-4), or of its subnormals (2^-10 of the scale), once when written and once each time that the scale grew, the
                    # later ones in steps at most half as large as the last: below 2^-9 in all; the float32 rotation before it is 2^-20 of that
                    bound = torch.maximum(2.0 ** -4 * exact.abs(), 2.0 ** -9 * sc[None, :, None].expand_as(exact)) * (1 + 2.0 ** -12)
                    assert ((got - exact).abs() <= bound).all(), float(((got - exact).abs() / bound).max())
                    stale = data[id].view(torch.uint8)[:, exact.shape[0]:]
                    assert (stale == 0x7F).all()                 # places behind the last token are left as they were
    return sum(v for k, v in growths.items() if k[-1] == "n")


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,page,hq,hkv", ((128, 16, 4, 2), (64, 64, 3, 3), (128, 128, 5, 1), (64, 32, 16, 1)))
def test_cache_holds_what_was_appended(dtype, D, page, hq, hkv):
    check_append(dtype, D, page, hq, hkv, [(3, 1, 0, page + 5), (1, 0, 2 * page, 1), (0, 1, 1, 1), (2 * page, page - 2, 1, 1)])


@gpu
def test_cache_filled_token_by_token():
    grown = check_append(torch.bfloat16, 64, 16, 2, 2, [(1, 1)] * 40, slack=8)
    assert grown > 10                                            # scales grew under older tokens


@gpu
@pytest.mark.parametrize("size", (2.0 ** -30, 2.0 ** 30))
def test_scales_far_from_one(size):
    check_append(torch.bfloat16, 128, 32, 4, 1, [(40, 3), (1, 1), (1, 1)], size=size)


@gpu
def test_special_values_and_tokens_outside():
    from htr_b200 import paged

    D, page, hq, hkv = 64, 16, 2, 1
    cache, (cos, sin) = empty_cache(4, hkv, page, D, fill=0), angles(32, D)
    x = torch.ones(7, 4 * D, dtype=torch.bfloat16, device=DEV)
    x[1, 3 * D] = float("inf")
    x[2, 3 * D + 1] = float("nan")
    x[3, 3 * D + 2] = float("-inf")
    x[4:] = 5.0
    x[5] = 0.0
    status = ints([0])
    # tokens 0 to 3 on page 1; 4: not served; 5: zeros on page 2; 6: a slot behind the cache
    q = paged.rope_append(x, ints([0, 1, 2, 3, -1, 0, 0]), ints([16, 17, 18, 19, -1, 32, 64]), cos, sin, cache, hq, status=status)
    assert int(status) == 16
    assert (q[4] == 0).all() and (q[6] == 0).all() and (q[:4] != 0).any()
    s = cache.v_scale[1, 0].item()
    assert s == 2.0 ** -8                                        # the finite values alone: 1 <= 448 * 2^-8
    v = cache.v.float()[1, 0] * s
    assert v[1, 0] == 448 * s and v[2, 1].isnan() and v[3, 2] == -448 * s and (v[0] == 1).all() and v[2, 0] == 1
    assert cache.v_scale[2, 0].item() == 2.0 ** -100 and (cache.v.float()[2, 0, 0] == 0).all()
    assert (cache.k.view(torch.uint8)[0] == 0).all() and (cache.k.view(torch.uint8)[3] == 0).all()
    status.zero_()
    paged.rope_append(x[:2], ints([32, -5]), ints([0, 1]), cos, sin, cache, hq, status=status)        # positions without angles
    assert int(status) == 16 and (cache.k.view(torch.uint8)[0] == 0).all()


def runs_by_hand(slots, positions, page, total, rows):
    """[(page, [tokens that are written])] and the status: a page's tokens follow one another, others that are not written between them, in rising slots."""
    ok = [0 <= s < total and 0 <= p < rows for s, p in zip(slots, positions)]
    status = 16 if any(not o and s != -1 for o, s in zip(ok, slots)) else 0
    runs, closed, last = [], False, None
    for t, o in enumerate(ok):
        if not o:
            continue
        if last is None or t - last >= page or slots[last] // page != slots[t] // page:
            runs.append((slots[t] // page, []))
            closed = False
        elif slots[t] <= slots[last]:
            closed, status = True, 16
        if not closed:
            runs[-1][1].append(t)
        last = t
    return runs, ok, status


def check_runs(dtype, D, page, hkv, slots, positions, pages, rows, seed=0):
    from htr_b200 import paged

    hq, T = 2, len(slots)
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(T, (hq + 2 * hkv) * D, device=DEV, generator=g) * torch.exp(2 * torch.randn(T, 1, device=DEV, generator=g))).to(dtype)
    cos, sin = angles(rows, D)
    cache, status = empty_cache(pages, hkv, page, D, fill=0x38), ints([0])       # 1.0 everywhere
    for s in cache[2:]:
        s.fill_(2.0 ** -12)
    before = [t.clone() for t in cache]
    q = paged.rope_append(x, ints(positions), ints(slots), cos, sin, cache, hq, status=status)
    runs, ok, want = runs_by_hand(slots, positions, page, pages * page, rows)
    assert int(status) == want and len({p for p, _ in runs}) == len(runs)        # (no page twice: that is not for the operator to put right)
    assert (q[[not o for o in ok]] == 0).all() and all(bool((q[t] != 0).any()) for t in range(T) if ok[t])
    y = x.double().view(T, hq + 2 * hkv, D)
    at = torch.tensor([p if o else 0 for p, o in zip(positions, ok)], device=DEV)
    exact = [rotated(y[:, hq:hq + hkv], cos.double()[at][:, None], sin.double()[at][:, None]), y[:, hq + hkv:]]
    for data, scale, old, old_scale, new in ((cache.k, cache.k_scale, before[0], before[2], exact[0]), (cache.v, cache.v_scale, before[1], before[3], exact[1])):
        touched = torch.zeros(pages, dtype=torch.bool, device=DEV)
        for id, tokens in runs:
            touched[id] = True
            places = [slots[t] % page for t in tokens]
            for h in range(hkv):
                e = wanted_exponent(float(new[tokens, h].abs().max().float()))
                s = float(scale[id, h])
                assert s == 2.0 ** (max(e, -12) if places[0] else e)
                got = data[id, h].double() * s
                # half a step of e4m3 or of its subnormals, of the element as the float32 rotation gives it: off by d, three roundings of terms that are at
                # most sqrt(2) * 448 * s in sum, 3 * 2^-24 * 634 * s < 2^-13 * s; in all (1 + 2^-4) * d more than half a step of the exact one
                bound = torch.maximum(2.0 ** -4 * new[tokens, h].abs(), torch.tensor(2.0 ** -10 * s, device=DEV)) + 2.0 ** -12 * s
                assert ((got[places] - new[tokens, h]).abs() <= bound).all(), float(((got[places] - new[tokens, h]).abs() / bound).max())
                rest = [p for p in range(page) if p not in places]
                early, late = [p for p in rest if p < places[0]], [p for p in rest if p > places[0]]
                # the older ones keep their value, but for half a step of e4m3's subnormals; what lies behind the first place and is not written keeps its bytes
                assert ((got[early] - 2.0 ** -12).abs() <= 2.0 ** -10 * s).all() and (data[id, h].view(torch.uint8)[late] == 0x38).all()
        assert torch.equal(data[~touched].view(torch.uint8), old[~touched].view(torch.uint8)) and torch.equal(scale[~touched], old_scale[~touched])


@gpu
@pytest.mark.parametrize("dtype,D,page,hkv", ((torch.bfloat16, 128, 64, 2), (torch.float16, 64, 16, 3), (torch.bfloat16, 64, 128, 1), (torch.bfloat16, 128, 32, 8)))
@pytest.mark.parametrize("hole", ("positions", "slots", "order", "twice", "all"))
@pytest.mark.parametrize("pieces", (3, 40))
def test_pages_whose_tokens_are_not_all_written(dtype, D, page, hkv, hole, pieces):
    """Positions without angles, slots of -1 and slots that do not rise in the middle of a page: one thread block writes it all the same."""
    g = torch.Generator().manual_seed(page + pieces)
    rows, slots, positions = 4 * page, [], []
    for id in torch.randperm(pieces, generator=g).tolist():
        off = int(torch.randint(0, page - 3, (1,), generator=g)) if id % 3 else 0
        n = int(torch.randint(3, page - off + 1, (1,), generator=g))
        mine, at = [id * page + off + i for i in range(n)], list(range(n))
        for i in torch.randint(1, n, (max(1, n // 6),), generator=g).tolist():
            how = hole if hole != "all" else ("positions", "slots", "order", "twice")[i % 4]
            if how == "positions":
                at[i] = (-5, rows, 1 << 30)[i % 3]
            elif how == "slots":
                mine[i] = -1
            elif how == "order" and id % 2:
                mine[i - 1], mine[i] = mine[i], mine[i - 1]
            elif how == "twice" and id % 2:
                mine[i] = mine[i - 1]
        slots += mine
        positions += at
    check_runs(dtype, D, page, hkv, slots, positions, pieces + 1, rows, seed=page)


# ---- attention ------------------------------------------------------------------------------------------------------


def filled(dtype, D, page, hq, hkv, have, adds, seed=0, pages=None, spread=0):
    """Queries and a cache for requests with have[r] + adds[r] tokens; what is not a token's is NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed + D + page)
    R, seen = len(have), [h + a for h, a in zip(have, adds)]
    used = [-(-max(s, 0) // page) for s in seen]
    pages = pages or sum(used) + 2
    cache = empty_cache(pages, hkv, page, D)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    tables, at = torch.full((R, max(used) + 2), -1, dtype=torch.int32), 0
    for r in range(R):
        tables[r, :used[r]] = ids[at:at + used[r]]
        for j in range(used[r]):
            n, id = min(page, seen[r] - j * page), int(ids[at + j])
            for data, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                data[id, :, :n] = (torch.randn(hkv, n, D, device=DEV, generator=g) * 100).clamp(-448, 448).to(E4M3)
                scale[id] = 2.0 ** (torch.randint(-1 - spread, 2 + spread, (hkv,), device=DEV, generator=g) - 7).float()
        at += used[r]
    q = (torch.randn(sum(adds), hq, D, device=DEV, generator=g) * 2).to(dtype)
    starts = [0]
    for a in adds:
        starts.append(starts[-1] + a)
    return q, ints(starts), ints(seen), tables.to(DEV), cache


def attend_exactly(q, starts, seen, tables, cache, scale):
    """In 64 bits: the result, and the sum of p |v|, to which the roundings of the probabilities are relative."""
    hq, hkv, page, D = q.shape[1], cache.k.shape[1], cache.k.shape[2], cache.k.shape[3]
    out, spread = torch.zeros(q.shape, dtype=torch.double, device=DEV), torch.zeros(q.shape, dtype=torch.double, device=DEV)
    for r in range(seen.numel()):
        s, e, n = int(starts[r]), int(starts[r + 1]), int(seen[r])
        if e == s or n <= 0:
            continue
        ids = tables[r, :-(-n // page)].long()
        for h in range(hq):
            k, v = ((c[ids, h * hkv // hq].double() * f[ids, h * hkv // hq].double()[:, None, None]).reshape(-1, D)[:n]
                    for c, f in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            at = torch.arange(n - (e - s), n, device=DEV)
            hide = torch.arange(n, device=DEV)[None] > at[:, None]
            p = (q[s:e, h].double() @ k.T * scale).masked_fill(hide, float("-inf")).softmax(-1)
            p = torch.where(at[:, None] < 0, 0.0, p)
            v = torch.where(hide.all(0)[:, None], 0.0, v)
            out[s:e, h], spread[s:e, h] = p @ v, p @ v.abs()
    return out, spread


def widened(q, tables, cache):
    """The tables with so many more (unused) columns that many rows a request are taken to be much work: by their width, for lengths are not known on the host."""
    page, width = cache.k.shape[2], tables.shape[1]
    more = int(1.6e9 / (max(q.shape[0], 1) * q.shape[1] * q.shape[2] * page)) + 1 - width
    return tables if more <= 0 else torch.cat([tables, torch.full((tables.shape[0], more), -1, dtype=torch.int32, device=tables.device)], 1)


def check_attention(q, starts, seen, tables, cache, max_new, scale=None, **kw):
    """By both kernels where there are many rows a request."""
    if q.shape[1] // cache.k.shape[1] * min(max_new, q.shape[0]) * q.shape[2] > 6144:
        check_one_attention(q, starts, seen, widened(q, tables, cache), cache, max_new, scale, **kw)
    return check_one_attention(q, starts, seen, tables, cache, max_new, scale, **kw)


def check_one_attention(q, starts, seen, tables, cache, max_new, scale, **kw):
    from htr_b200 import paged

    got = paged.attention(q, starts, seen, tables, cache, max_new, scale=scale, **kw)
    want, spread = attend_exactly(q, starts, seen, tables, cache, q.shape[2] ** -0.5 if scale is None else scale)
    n = int(starts[-1])
    # half a step of the output; 2^-11 for each probability (fp16); 2^-11 for the float32 scores: D terms of |q k| * scale up to about 40 in
    # sum, 2^-24 each time the sum is rounded (128 * 40 * 2^-24 = 2^-11.7), and for the exponentials (2^-21)
    bound = torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -10 * spread + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    off = (got.double() - want).abs()[:n]
    assert (off <= bound[:n]).all(), float((off / bound[:n]).max())
    return got


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,page,hq,hkv", ((128, 64, 8, 2), (64, 16, 6, 2), (128, 16, 5, 5), (64, 128, 24, 1), (128, 32, 16, 1)))
@pytest.mark.parametrize("have,adds", (((0, 14, 15, 16, 130, 77), (1, 1, 1, 1, 1, 0)), ((0, 1, 60, 5, 200), (1, 3, 5, 0, 2)), ((0, 63, 100), (70, 1, 33)), ((517,), (1,)),
                                       ((300, 0, 45), (260, 129, 200))))
def test_attention(dtype, D, page, hq, hkv, have, adds):
    check_attention(*filled(dtype, D, page, hq, hkv, have, adds), max_new=max(adds))


@gpu
@pytest.mark.parametrize("adds", ((1, 1), (2, 30), (150, 3)))
def test_attention_scales_that_differ_and_its_own_scale(adds):
    q, starts, seen, tables, cache = filled(torch.bfloat16, 128, 16, 4, 2, (100, 333), adds, spread=5)
    check_attention(q, starts, seen, tables, cache, max(adds), scale=0.01)
    cache.v_scale.mul_(2.0 ** 40)
    check_attention(q, starts, seen, tables, cache, max(adds), scale=0.01)
    cache.v_scale.mul_(2.0 ** -90)
    check_attention(q, starts, seen, tables, cache, max(adds), scale=0.01)


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_attention_over_long_sequences(dtype):
    check_attention(*filled(dtype, 128, 64, 4, 1, (20011, 3, 9000), (1, 1, 1)), max_new=1)
    check_attention(*filled(dtype, 64, 128, 4, 2, (6000, 1), (40, 300)), max_new=300)


@gpu
def test_rows_that_see_nothing_and_rows_behind_the_last():
    q, starts, seen, tables, cache = filled(torch.bfloat16, 64, 16, 4, 2, (20, 3, 0, 30), (2, 5, 3, 140))
    seen[1], seen[2] = 2, 0                                      # three of the five tokens stand before the first position; not served
    big = torch.cat([q, torch.ones_like(q[:4])])
    out = torch.full_like(big, 7.0)
    got = check_attention(big, starts, seen, tables, cache, 140, out=out)
    assert got is out and (got[2:5] == 0).all() and (got[7:10] == 0).all() and (got[150:] == 7).all() and (got[5:7] != 0).any()
    one = torch.full_like(big, 7.0)
    check_attention(big, ints([0, 0, 0, 0, 0]), seen, tables, cache, 1, out=one)
    assert (one == 7).all()


@gpu
@pytest.mark.parametrize("adds,wide", (((3, 1), False), ((9, 2), False), ((100, 1), False), ((20, 1), True), ((100, 1), True)))
def test_a_nan_reaches_only_those_that_see_it(adds, wide):
    """Keys and values of a step's later tokens, and all behind the last, may be NaN: earlier tokens do not see them."""
    q, starts, seen, tables, cache = filled(torch.bfloat16, 128, 16, 8, 2, (40, 17), adds)
    from htr_b200 import paged

    if wide:
        tables = widened(q, tables, cache)
    want = paged.attention(q, starts, seen, tables, cache, max(adds))
    at, n = 40 + adds[0] - 2, adds[0]                            # the last token but one of request 0
    page = int(tables[0, at // 16])
    cache.v.view(torch.uint8)[page, 1, at % 16, 5] = 0xFF
    cache.k.view(torch.uint8)[page, 0, at % 16, 77] = 0x7F
    got = paged.attention(q, starts, seen, tables, cache, max(adds))
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[n - 2:n, :4] = True                                      # a NaN key takes the whole result of its heads
    hit[n - 2:n, 4:, 5] = True                                   # a NaN value its dimension
    assert torch.equal(got.isnan(), hit) and torch.equal(got[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("adds,wide", (((1, 1), False), ((60, 1), False), ((60, 1), True)))
def test_table_entries_that_are_no_page_hide_their_tokens(adds, wide):
    from htr_b200 import paged

    q, starts, seen, tables, cache = filled(torch.bfloat16, 64, 16, 2, 1, (100, 64), adds)
    if wide:
        tables = widened(q, tables, cache)
    status = ints([0])
    want = paged.attention(q, starts, seen, tables, cache, max(adds), status=status).clone()
    assert int(status) == 0
    tables[0, 2], tables[1, :] = 1 << 30, -1
    got = paged.attention(q, starts, seen, tables, cache, max(adds), status=status)
    assert int(status) == 32 and torch.isfinite(got).all() and (got[int(starts[1]):] == 0).all() and not torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,hq,hkv,adds", ((128, 1, 1, (127, 128, 129)), (64, 1, 1, (255, 256, 257)), (128, 3, 1, (42, 43, 85)), (64, 6, 2, (86, 85, 1)), (128, 7, 1, (73, 19)),
                                           (64, 256, 1, (1, 3)), (128, 200, 1, (2, 1)), (64, 300, 1, (2,)), (128, 34, 2, (4, 1))))
def test_attention_at_the_ends_of_tiles(dtype, D, hq, hkv, adds):
    check_attention(*filled(dtype, D, 32, hq, hkv, (70, 0, 300)[:len(adds)], adds), max_new=max(adds))


@gpu
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), float("-inf")))
@pytest.mark.parametrize("D,adds,wide", ((128, (2, 1), False), (64, (40, 1), False), (64, (40, 1), True), (128, (40, 1), True)))
def test_queries_that_are_not_finite(bad, D, adds, wide):
    """Their own rows become NaN, and no others change."""
    from htr_b200 import paged

    q, starts, seen, tables, cache = filled(torch.bfloat16, D, 16, 8, 2, (40, 17), adds)
    if wide:
        tables = widened(q, tables, cache)
    want = paged.attention(q, starts, seen, tables, cache, max(adds))
    q[1, 5, 3] = bad
    got = paged.attention(q, starts, seen, tables, cache, max(adds))
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, 5] = True
    assert torch.equal(got.isnan(), hit) and torch.equal(got[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,adds,R", ((128, 1, 64), (64, 3, 64), (128, 40, 20), (64, 70, 20), (128, 20, 20)))
@pytest.mark.parametrize("nats", (12, 15, 18))
@pytest.mark.parametrize("spread", (0.0, 1.0))
def test_a_token_that_takes_nearly_all_and_has_no_values(dtype, D, adds, R, nats, spread):
    """The first token's score lies `nats` above those of 16500 others, which are equal or differ by `spread`, and its values are zero: the result is made of
    the others' probabilities, which have all their bits.  So many requests and heads (of the same pages) that one thread block goes over most of them."""
    from htr_b200 import paged

    hkv, group = 8, 4
    q, starts, seen, tables, cache = filled(dtype, D, 64, hkv * group, hkv, (16500,), (adds,))
    q.zero_()
    q[..., 0] = 1
    g = torch.Generator(device=DEV).manual_seed(8)
    cache.k_scale.fill_(1)
    cache.v_scale.fill_(2.0 ** -7)
    cache.k[..., 0] = (torch.randn(cache.k.shape[:3], device=DEV, generator=g) * (16 * spread)).clamp(-448, 448).to(E4M3)       # the only dimension that counts
    cache.v.copy_((torch.randn(cache.v.shape, device=DEV, generator=g) * 60 + 100).clamp(-448, 448).to(E4M3))
    id = int(tables[0, 0])
    cache.k[id, :, 0, 0] = 16 * nats                             # (12, 15 and 18 times 16 are e4m3's)
    cache.v[id, :, 0] = 0
    want, spread = attend_exactly(q, starts, seen, tables, cache, 1 / 16)
    got = paged.attention(q.repeat(R, 1, 1), ints([adds * r for r in range(R + 1)]), seen.repeat(R), widened(q, tables, cache).repeat(R, 1), cache, adds, scale=1 / 16)
    # the bound of check_one_attention
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -10 * spread + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got.double().view(R, *q.shape) - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


@gpu
@pytest.mark.parametrize("D,adds", ((128, 2), (64, 40), (128, 60)))
@pytest.mark.parametrize("of_q,of_k", ((120, 0), (116, -20), (100, 0), (-90, 0), (-120, 110)))
def test_queries_at_the_ends_of_the_range(D, adds, of_q, of_k):
    """Finite queries of any magnitude under a scale that brings the scores back."""
    q, starts, seen, tables, cache = filled(torch.bfloat16, D, 16, 4, 2, (100, 33), (adds, 1))
    cache.k_scale.mul_(2.0 ** of_k)
    check_attention(q * 2.0 ** of_q, starts, seen, tables, cache, adds, scale=2.0 ** -(of_q + of_k) * D ** -0.5)


@gpu
@pytest.mark.parametrize("D,page,hq,hkv,most", ((128, 64, 8, 2, 1), (64, 16, 4, 4, 1), (128, 16, 4, 1, 9), (64, 32, 24, 2, 30)))
@pytest.mark.parametrize("seed", (1, 2, 3))
def test_lengths_of_all_kinds_in_one_step(D, page, hq, hkv, most, seed):
    """The cut of the work falls everywhere: inside long requests, between short ones, at ones that add nothing."""
    g = torch.Generator().manual_seed(seed)
    R = 60
    have = [int(2 ** float(x)) - 1 for x in torch.rand(R, generator=g) * 11.5]
    adds = [int(x) for x in torch.randint(0, most + 1, (R,), generator=g)]
    adds[seed] = most
    check_attention(*filled(torch.bfloat16, D, page, hq, hkv, have, adds, seed=seed), max_new=most)


@gpu
def test_attention_of_many_requests():
    adds = [1] * 1100
    adds[700], adds[3] = 90, 0
    check_attention(*filled(torch.bfloat16, 128, 16, 1, 1, [r % 5 for r in range(1100)], adds), max_new=90)


@gpu
def test_pages_beyond_four_gigabytes():
    from htr_b200 import paged

    hkv, page, D, pages = 8, 128, 128, 36000                     # 4.7 GB of keys
    g = torch.Generator(device=DEV).manual_seed(4)
    k = torch.empty(pages, hkv, page, D, dtype=torch.uint8, device=DEV).view(E4M3)
    cache = paged.LayerCache(k, torch.empty_like(k), torch.empty(pages, hkv, device=DEV), torch.empty(pages, hkv, device=DEV))
    ids = [35999, 0, 34000]
    for x in (0, 1):
        for id in ids:
            cache[x][id] = (torch.randn(hkv, page, D, device=DEV, generator=g) * 90).clamp(-448, 448).to(E4M3)     # (beyond 464 is NaN)
            cache[2 + x][id] = 2.0 ** -7
    q = torch.randn(1, 8, D, device=DEV, generator=g).bfloat16()
    check_attention(q, ints([0, 1]), ints([300]), ints([ids]), cache, 1)
    qkv = torch.randn(2, 33 * D, device=DEV, generator=g).bfloat16()[:, :32 * D]
    cos, sin = angles(400, D)
    paged.rope_append(qkv, ints([300, 301]), ints([34000 * page + 44, 34000 * page + 45]), cos, sin, cache, 16)
    got = cache.v[34000, :, 44:46].double() * cache.v_scale[34000].double()[:, None, None]
    want = qkv.double().reshape(2, 32, D)[:, 24:].transpose(0, 1)
    assert ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -9 * cache.v_scale[34000].double()[:, None, None])).all()


@gpu
@pytest.mark.parametrize("adds,wide", (((1, 1, 1), False), ((90, 1, 200), False), ((90, 1, 200), True)))
def test_two_graphs_and_another_stream(adds, wide):
    """Captured calls keep no buffers in common with one another or with eager ones: replayed at the same time they give what each gives alone."""
    from htr_b200 import paged

    sets = [filled(torch.bfloat16, 128, 16, 8, 2, have, adds, seed=s) for s, have in enumerate(((3000, 1, 50), (40, 2500, 700)))]
    if wide:
        sets = [(q, starts, seen, widened(q, tables, cache), cache) for q, starts, seen, tables, cache in sets]
    want = [paged.attention(*x, max(adds)).clone() for x in sets]
    graphs, outs = [], []
    for x in sets:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.attention(*x, max(adds)))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(30):
        for o in outs:
            o.fill_(9)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = paged.attention(*sets[0], max(adds))
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)) and torch.equal(eager, want[0])


@gpu
@pytest.mark.parametrize("D,adds", ((64, 1), (128, 3), (64, 130), (128, 60)))
@pytest.mark.parametrize("of_v", (-93, 125))
def test_values_at_the_ends_of_the_range_over_a_long_sequence(D, adds, of_v):
    """Scales of 2^-100 and 2^118, the ends of what `rope_append` gives (2^119 would be beyond bf16), over 150000 tokens of equal scores."""
    q, starts, seen, tables, cache = filled(torch.bfloat16, D, 128, 4, 1, (150000,), (adds,))
    q.zero_()
    cache.v_scale.fill_(2.0 ** (of_v - 7))
    check_attention(q, starts, seen, tables, cache, adds)


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,adds", ((128, 2), (64, 40), (128, 60)))
@pytest.mark.parametrize("size", (8, 256, 4096))
def test_queries_with_an_element_that_stands_out(dtype, D, adds, size):
    """One dimension of the queries is larger than the others, and of the keys as much smaller.  The tcgen05 kernel holds queries to 2^-17 of the largest of their row."""
    q, starts, seen, tables, cache = filled(dtype, D, 16, 4, 2, (300, 33), (adds, 1))
    q[..., 5] *= size
    cache.k[..., 5] = (cache.k[..., 5].float() / size).to(E4M3)
    from htr_b200 import paged

    for t in (tables, widened(q, tables, cache)):
        got = paged.attention(q, starts, seen, t, cache, adds).double()
        want, spread = attend_exactly(q, starts, seen, tables, cache, D ** -0.5)
        # as in check_one_attention, and a score that is off by 2^-17 of the row's largest for all dimensions: so are the probability and, at most, the sum
        keys = (cache.k.double().nan_to_num(0).abs().sum(-1) * cache.k_scale.double()[..., None]).max()
        most = q.double().abs().amax(-1, keepdim=True)
        bound = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -10 + 2 * 2.0 ** -17 * most * keys * D ** -0.5) * spread + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@gpu
@pytest.mark.parametrize("D,have,adds,wide,block", ((128, [3000] * 12, [1] * 12, False, 60), (64, [900] * 30, [3] * 30, False, 100), (128, [1500] * 6, [100] * 6, True, 60),
                                                    (64, [2500] * 9, [30] * 9, True, 75)))
def test_rows_of_an_expired_wait_are_nan(D, have, adds, wide, block):
    """The first keys of one thread block never arrive, so that bounded waits run out: the rows that it owes are NaN, the others as they are without, the
    status word is set, and the next call is served again.  Single tokens, a few, tiles of 256 rows and twins of 120."""
    from htr_b200 import _lib, paged

    q, starts, seen, tables, cache = filled(torch.bfloat16, D, 16, 8, 2, have, adds)
    if wide:
        tables = widened(q, tables, cache)
    status = ints([0])
    want = paged.attention(q, starts, seen, tables, cache, max(adds), status=status)
    assert int(status) == 0
    for word in (status, None):
        out = torch.full_like(q, 3.0)
        _lib.lib.htr_paged_attention_withhold(block)
        try:
            paged.attention(q, starts, seen, tables, cache, max(adds), out=out, status=word)
        finally:
            _lib.lib.htr_paged_attention_withhold(-1)
        lost = out.isnan().any(-1)
        assert 0 < int(lost.sum()) < lost.numel() // 4 and out[lost].isnan().all() and torch.equal(out[~lost], want[~lost])
    assert int(status) == 64
    assert torch.equal(paged.attention(q, starts, seen, tables, cache, max(adds), status=status.zero_()), want) and int(status) == 0


@gpu
def test_the_workspace_is_sized_for_the_device_of_the_tensors(monkeypatch):
    """It depends on the device's number of SMs: asked for, as the launch is, with that device as the current one."""
    from htr_b200 import _lib, paged

    inside, seen_by = [], []

    class Device(torch.cuda.device):
        def __enter__(self):
            inside.append(1)
            return super().__enter__()

        def __exit__(self, *a):
            inside.pop()
            return super().__exit__(*a)

    class Library:
        def __getattr__(self, name):
            if name.startswith("htr_paged_attention"):
                seen_by.append((name, bool(inside)))
            return getattr(real, name)

    real = _lib.lib
    q, starts, seen, tables, cache = filled(torch.bfloat16, 64, 16, 4, 2, (20, 3), (1, 1))
    want = paged.attention(q, starts, seen, tables, cache, 1)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "lib", Library())
    strided = torch.stack([q, q], 2)[:, :, 0]                    # not contiguous: not for the native front
    assert torch.equal(paged.attention(strided, starts, seen, tables, cache, 1), want)
    assert [n for n, _ in seen_by] == ["htr_paged_attention_workspace_bytes", "htr_paged_attention"] and all(i for _, i in seen_by)


# ---- refusals -------------------------------------------------------------------------------------------------------


def test_no_cpu_path():
    from htr_b200 import _lib, paged

    i = torch.zeros(1, dtype=torch.int32)
    k = torch.zeros(1, 1, 16, 64, dtype=torch.uint8).view(E4M3)
    cache = paged.LayerCache(k, k, torch.ones(1, 1), torch.ones(1, 1))
    for call in (lambda: paged.plan_step(i, i, i[None], i, i, 16, 1), lambda: paged.rope_append(torch.zeros(1, 192).bfloat16(), i, i, torch.ones(1, 32), torch.ones(1, 32), cache, 1),
                 lambda: paged.attention(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(2, dtype=torch.int32), i, i[None], cache, 1)):
        with pytest.raises(_lib.HTRError, match="no CPU path"):
            call()


def test_status_codes_without_a_gpu():
    import ctypes

    from htr_b200 import _lib

    L, f = _lib.lib, ctypes.c_float(1.0)
    p = 16                                                       # an address that the checks before a launch look at and nothing reads

    def plan(R=4, stride=3, width=3, pages=8, page=16, T=9, at=p):
        return L.htr_page_plan(at, p, R, p, stride, width, p, pages, p, page, T, p, p, p, p, p, p, None, None)

    assert [plan(R=0), plan(stride=2), plan(width=0), plan(pages=0), plan(page=24), plan(page=256), plan(T=-1)] == [-2] * 7
    assert [plan(R=8193), plan(pages=1 << 28), plan(stride=1 << 28, width=1 << 28), plan(T=(1 << 31) - 1)] == [-8] * 4
    assert plan(at=None) == -5

    def append(dt=0, stride=6 * 64, T=2, rows=9, hq=4, hkv=1, D=64, pages=8, page=16, at=p):
        return L.htr_paged_append(at, dt, stride, p, p, T, p, p, rows, hq, hkv, D, p, p, p, p, pages, page, p, None, None)

    assert append(dt=2) == -3
    assert [append(stride=6 * 64 - 8), append(stride=6 * 64 + 4), append(T=-1), append(rows=0), append(hq=0), append(hkv=0), append(D=96), append(pages=0), append(page=8)] == [-2] * 9
    assert append(pages=1 << 28) == -8 and append(T=0, at=None) == 0 and append(at=None) == -5 and append(at=24) == -6

    def attend(dt=0, T=3, R=2, stride=3, width=3, pages=8, page=16, hq=4, hkv=2, D=64, most=1, at=p, work=p, size=1 << 40):
        return L.htr_paged_attention(at, dt, T, p, p, R, p, stride, width, p, p, p, p, pages, page, hq, hkv, D, most, f, p, None, work, size, None)

    assert attend(dt=2) == -3
    assert [attend(T=-1), attend(R=0), attend(stride=2), attend(page=17), attend(hq=5), attend(hkv=0), attend(D=32), attend(most=0)] == [-2] * 8
    assert [attend(R=8193), attend(pages=1 << 28), attend(most=1 << 30)] == [-8] * 3
    assert attend(T=0, at=None) == 0 and attend(at=None) == -5 and attend(at=24) == -6
    assert [attend(work=None), attend(size=0), attend(work=None, T=900, most=900, stride=1 << 20, width=1 << 20),
            attend(size=1 << 16, T=900, most=900, stride=1 << 20, width=1 << 20)] == [-4] * 4
    need = L.htr_paged_attention_workspace_bytes
    assert need(3, 2, 4, 2, 64, 1, 3, 16) > 0 and [need(3, 2, 4, 2, 96, 1, 3, 16), need(3, 2, 4, 2, 64, 1, 0, 16), need(3, 2, 4, 2, 64, 1, 3, 24), need(0, 2, 4, 2, 64, 1, 3, 16)] == [0] * 4


@gpu
def test_refusals():
    from htr_b200 import _lib, paged

    q, starts, seen, tables, cache = filled(torch.bfloat16, 64, 16, 4, 2, (20, 3), (1, 1))
    cos, sin = angles(64, 64)
    good = dict(qkv=torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=DEV), positions=ints([20, 3]), slots=ints([0, 16]), cos=cos, sin=sin, cache=cache, q_heads=4)
    paged.rope_append(**good)
    bad_cache = [cache._replace(k=cache.k.float()), cache._replace(v=cache.v[:1]), cache._replace(k=cache.k.transpose(1, 2)), cache._replace(k_scale=cache.k_scale.half()),
                 cache._replace(v_scale=cache.v_scale[:1]), cache._replace(k=cache.k[:, :, :8], v=cache.v[:, :, :8]), cache._replace(k=cache.k.cpu())]
    for change in (dict(qkv=good["qkv"].float()), dict(qkv=good["qkv"][:, :-64]), dict(qkv=good["qkv"][0]), dict(positions=ints([1])), dict(slots=good["slots"].long()),
                   dict(cos=cos[:, :16]), dict(sin=sin.double()), dict(cos=cos[:3]), dict(q_heads=0), *[dict(cache=c) for c in bad_cache]):
        with pytest.raises(_lib.HTRError):
            paged.rope_append(**{**good, **change})
    good = dict(q=q, starts=starts, seen=seen, tables=tables, cache=cache, max_new=1)
    paged.attention(**good)
    for change in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(starts=starts[:2]), dict(seen=seen.long()), dict(tables=tables[:1]), dict(tables=tables.t().contiguous().t()),
                   dict(max_new=0), dict(out=torch.empty_like(q)[:1]), dict(out=torch.empty_like(q).half()), dict(status=torch.zeros(1, device=DEV)), *[dict(cache=c) for c in bad_cache]):
        with pytest.raises(_lib.HTRError):
            paged.attention(**{**good, **change})
    assert paged.attention(q[:0], ints([0, 0, 0]), seen, tables, cache, 1).shape == (0, 4, 64)
    good = dict(lengths=ints([3, 4]), new=ints([1, 1]), tables=tables, free=ints([5, 6]), count=ints([2]), page_size=16, max_tokens=4)
    paged.plan_step(**good)
    for change in (dict(lengths=ints([3])), dict(new=ints([1, 1]).long()), dict(tables=tables.long()), dict(tables=tables[0]), dict(count=ints([1, 2])), dict(page_size=20),
                   dict(max_tokens=-1), dict(lengths_out=ints([1])), dict(count_out=ints([1, 1])), dict(free=ints([])), dict(status=ints([0, 0]))):
        with pytest.raises(_lib.HTRError):
            paged.plan_step(**{**good, **change})
    for args in ((1, 1, 96, 4, 16, 1, 64), (1, 1, 64, 4, 20, 1, 64), (0, 1, 64, 4, 16, 1, 64), (1, 1, 64, 0, 16, 1, 64)):
        with pytest.raises(_lib.HTRError):
            paged.PagedCache(*args, DEV)
