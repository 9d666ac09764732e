"""The paged cache in 4 bits: what is appended, what is unpacked, and attention over it, against plain evaluations in 64 bits; angles of far positions."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
NAN = 0x7FC0
MANY = 32768                                                 # rows (tokens times heads) from which on an append goes through matrix products


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def values(codes, scale):
    """What codes and scales stand for, in 64 bits."""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.double, device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return table[code.long()] * scale.double()[..., None]


def sylvester(D):
    h = torch.ones(1, 1, dtype=torch.double, device=DEV)
    while h.shape[0] < D:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h


def angles(rows, r):
    a = torch.arange(rows, device=DEV).double()[:, None] * 1.0e4 ** -(torch.arange(0, r, 2, device=DEV).double() / r)
    return a.cos().float(), a.sin().float()


def rotated(x, cos, sin, layout):
    """x [tokens, heads, D] in 64 bits; cos, sin [tokens, r / 2]."""
    r, c, s = 2 * cos.shape[1], cos[:, None], sin[:, None]
    y = x.clone()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y


def empty_cache(pages, hkv, page, D):
    """A cache whose places would show wherever something is read that was never written: NaN."""
    from htr_b200 import paged

    k = torch.full((pages, hkv, page, D // 2), 0xFF, dtype=torch.uint8, device=DEV)
    s = torch.full((pages, hkv, page), NAN, dtype=torch.int16, device=DEV).view(torch.bfloat16)
    return paged.LayerCache4(k, k.clone(), s, s.clone())


# ---- rope_append ----------------------------------------------------------------------------------------------------


def check_rows(codes, scale, exact, slack):
    """Codes [n, hkv, D / 2] and scales [n, hkv] of rows whose exact elements are `exact`; `slack`: how far the elements that were rounded may be from them."""
    most = exact.abs().amax(-1)
    sc = scale.double()
    # bf16(most / 6): half a step of it (eight significant bits: 2^-8), and what `slack` moves it by; at least 2^-100
    assert ((sc - (most / 6).clamp(min=2.0 ** -100)).abs() <= 2.0 ** -8 * sc + slack / 6 * (1 + 2.0 ** -8)).all()
    y = exact / sc[..., None]
    got = values(codes, torch.ones_like(scale))
    off = (got - y).abs()
    levels = torch.tensor(LEVELS, dtype=torch.double, device=DEV)
    best = (y.abs()[..., None] - levels).abs().amin(-1)
    assert (off <= best + 2 * slack[..., None] / sc[..., None] + 2.0 ** -22 * y.abs()).all(), float((off - best).max())
    assert ((got == 0) | (got.sign() == y.sign()) | (y.abs() <= 2 * slack[..., None] / sc[..., None])).all()


def check_append(dtype, D, page, hq, hkv, layout, r, steps, size=1.0, pages=40, slack_columns=0):
    """Runs steps = [(tokens of request 0, of request 1, ...), ...] and checks queries and cache after each of them."""
    from htr_b200 import paged

    R, H = len(steps[0]), sylvester(D)
    cache, g = empty_cache(pages, hkv, page, D), torch.Generator(device=DEV).manual_seed(D + page + hq + r)
    width = pages // R
    tables = torch.randperm(pages, generator=torch.Generator().manual_seed(3))[:R * width].view(R, width)
    cos, sin = angles(width * page, r)
    have, status = [0] * R, ints([0])
    for adds in steps:
        T = sum(adds)
        pos = [have[x] + i for x in range(R) for i in range(adds[x])]
        row = [x for x in range(R) for _ in range(adds[x])]
        slots = [int(tables[x, p // page]) * page + p % page for x, p in zip(row, pos)]
        wide = torch.randn(T, (hq + 2 * hkv) * D + slack_columns, device=DEV, generator=g) * size * torch.exp(torch.randn(T, 1, device=DEV, generator=g))
        x = wide.to(dtype)[:, :(hq + 2 * hkv) * D]
        before = [t.clone() for t in cache]
        q = paged.rope_append(x, ints(pos), ints(slots), cos, sin, cache, hq, status=status, layout=layout)
        assert int(status) == 0 and q.shape == (T, hq, D) and q.dtype == dtype
        y = x.double().reshape(T, hq + 2 * hkv, D)
        c, s = (t.double()[torch.tensor(pos, device=DEV)] for t in (cos, sin))
        z = rotated(y[:, :hq + hkv], c, s, layout) @ H
        # float32: three roundings of a rotation, then log2 D of each sum, each relative to at most the sum of all magnitudes (of which a rotated pair has up to
        # sqrt 2 times as much); where there are many rows, their elements enter as two tf32, the second of which cuts what the first leaves (2^-10) at
        # 2^-10 of it, and the matrix unit adds up in four steps, each cut at 2^-22 of the largest or finer
        noise = ((3 + math.log2(D)) * 2.0 ** -24 + (2.0 ** -19 if T * (hq + 2 * hkv) >= MANY else 0)) * 2 ** 0.5 * y[:, :hq + hkv].abs().sum(-1)
        want = z[:, :hq] * 8 / D
        bound = torch.finfo(dtype).eps / 2 * want.abs() + noise[:, :hq, None] * 8 / D * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((q.double() - want).abs() <= bound).all(), float(((q.double() - want).abs() / bound).max())
        at, off = ints(slots).long() // page, ints(slots).long() % page
        check_rows(cache.k[at, :, off], cache.k_scale[at, :, off], z[:, hq:] / 8, noise[:, hq:] / 8)
        check_rows(cache.v[at, :, off], cache.v_scale[at, :, off], y[:, hq + hkv:], torch.zeros(T, hkv, dtype=torch.double, device=DEV))
        mine = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
        mine[at, off] = True
        for now, was in zip(cache, before):                      # all else is left as it was
            now, was = (t.view(torch.int16) if t.dtype == torch.bfloat16 else t for t in (now, was))
            assert torch.equal(now.transpose(1, 2)[~mine], was.transpose(1, 2)[~mine])
        have = [h + a for h, a in zip(have, adds)]


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("D,page,hq,hkv,r", ((128, 16, 4, 2, 128), (64, 64, 3, 3, 64), (128, 128, 5, 1, 48), (64, 32, 16, 1, 16), (128, 64, 32, 8, 96)))
def test_cache_holds_what_was_appended(dtype, layout, D, page, hq, hkv, r):
    check_append(dtype, D, page, hq, hkv, layout, r, [(3, 1, 0, page + 5), (1, 0, 2 * page, 1), (0, 1, 1, 1), (2 * page, page - 2, 1, 1)])


@gpu
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("dtype,D,T,r", ((torch.bfloat16, 128, 1, 128), (torch.bfloat16, 64, 1, 64), (torch.bfloat16, 128, 700, 128), (torch.bfloat16, 64, 1501, 64),
                                         (torch.bfloat16, 128, 2049, 128), (torch.float16, 64, 3001, 64), (torch.float16, 128, 2200, 48), (torch.bfloat16, 64, 2500, 32),
                                         (torch.bfloat16, 128, 2100, 16), (torch.float16, 128, 2051, 128)))
def test_append_of_one_token_and_of_many(dtype, layout, D, T, r):
    check_append(dtype, D, 64, 12, 2, layout, r, [(T,)], slack_columns=8, pages=60)


@gpu
@pytest.mark.parametrize("hq,hkv,T", ((1, 1, 11000), (3, 5, 2600), (33, 3, 900)))
def test_heads_that_do_not_fill_a_thread_block(hq, hkv, T):
    check_append(torch.bfloat16, 64, 128, hq, hkv, "half", 64, [(T // 2, T - T // 2)], pages=100)


@gpu
@pytest.mark.parametrize("size", (2.0 ** -60, 2.0 ** 60))
def test_scales_far_from_one(size):
    check_append(torch.bfloat16, 128, 32, 4, 1, "half", 64, [(40, 3), (1, 1)], size=size)


@gpu
def test_ties_go_to_the_even_code():
    from htr_b200 import paged

    D, page = 64, 16
    cache, (cos, sin) = empty_cache(1, 1, page, D), angles(4, D)
    x = torch.zeros(1, 3 * D, dtype=torch.bfloat16, device=DEV)
    ties = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -6.0]
    x[0, 2 * D:2 * D + 16] = torch.tensor(ties) * 3              # the scale is 3
    paged.rope_append(x, ints([0]), ints([5]), cos, sin, cache, 1)
    assert float(cache.v_scale[0, 0, 5]) == 3
    got = values(cache.v[0, 0, 5], torch.ones((), device=DEV))[:16]
    assert got.tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, -6]


@gpu
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("more", (0, MANY // 4))
def test_special_values_and_tokens_outside(layout, more):
    from htr_b200 import paged

    D, page, hq, hkv = 64, 16, 2, 1
    cache, (cos, sin) = empty_cache(4, hkv, page, D), angles(32, D)
    x = torch.ones(9, 4 * D, dtype=torch.bfloat16, device=DEV)
    x[1, 3 * D] = float("inf")
    x[2, 3 * D + 1] = float("nan")
    x[3, 2 * D + 3] = float("nan")                               # of a key
    x[4, 2 * D:] = 0
    x[5, 3 * D:] = 3e38                                          # beyond the largest scale
    x[6, 2 * D:3 * D] = 3e38                                     # a key whose transform leaves float32
    status = ints([0])
    x = torch.cat([x, x.nan_to_num(0, 0, 0)[:1].expand(more, -1)])             # tokens that are not written, so that there are many
    slots, rest = [0, 1, 2, 3, 4, 5, 6, -1, 99] + [-1] * more, [0] * more
    q = paged.rope_append(x, ints([0, 1, 2, 3, 4, 5, 0, 9, 9] + rest), ints(slots), cos, sin, cache, hq, status=status, layout=layout)
    assert int(status) == 16 and (q[7:] == 0).all() and (q[:7] != 0).any(-1).all()
    v = values(cache.v[0, 0], cache.v_scale[0, 0])
    assert float(v[1, 0]) == 6 * 2.0 ** 119 and (v[1, 1:] == 0).all()          # infinity: the largest value; what stands beside it is nothing then
    assert v[2].isnan().all() and torch.isfinite(v[:2]).all()
    assert values(cache.k[0, 0], cache.k_scale[0, 0])[3].isnan().all() and torch.isfinite(v[3]).all()
    assert (v[4] == 0).all() and float(cache.v_scale[0, 0, 4]) == 2.0 ** -100 and float(cache.k_scale[0, 0, 4]) == 2.0 ** -100
    assert (v[5] == 6 * 2.0 ** 119).all()
    k = values(cache.k[0, 0], cache.k_scale[0, 0])[6]
    assert float(k[0]) == 6 * 2.0 ** 119 and (k[1:] == 0).all()
    assert (cache.v[0, 0, 7:] == 0xFF).all() and (cache.v[1:] == 0xFF).all() and cache.v_scale[1:].isnan().all()
    status.zero_()
    q = paged.rope_append(x, ints([0, 1, 2, 32, -1, 5, 6, 7, 8] + rest), ints([0, 1, 2, 3, 4, -5, 64, 7, 8] + [-1] * more), cos, sin, cache, hq, status=status, layout=layout)
    assert int(status) == 16 and (q[3:7] == 0).all() and (q[7:9] != 0).any(-1).all() and (q[9:] == 0).all()


@gpu
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("more", (0, MANY // 4))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_an_infinity_among_what_is_transformed_takes_its_row(dtype, layout, more):
    from htr_b200 import paged

    D, page = 128, 16
    cache, (cos, sin) = empty_cache(1, 1, page, D), angles(32, D)
    x = torch.ones(5 + more, 4 * D, dtype=dtype, device=DEV)
    x[1, 5], x[2, D + 77], x[3, 2 * D], x[4, 3 * D - 1] = float("inf"), float("-inf"), float("-inf"), float("inf")
    q = paged.rope_append(x, ints([0, 1, 2, 3, 4] + [0] * more), ints([0, 1, 2, 3, 4] + [-1] * more), cos, sin, cache, 2, layout=layout)
    hit = torch.zeros(5 + more, 2, D, dtype=torch.bool, device=DEV)
    hit[1, 0] = hit[2, 1] = True
    assert torch.equal(q.isnan(), hit) and torch.isfinite(q[~hit]).all()
    assert cache.k_scale[0, 0, :5].isnan().tolist() == [False, False, False, True, True] and torch.isfinite(cache.v_scale[0, 0, :5]).all()


@gpu
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("more", (0, MANY // 3))
@pytest.mark.parametrize("D,r", ((64, 64), (128, 128), (128, 48)))
@pytest.mark.parametrize("size", (0.5 ** 0.5, 5.0))
def test_finite_pairs_whose_rotation_leaves_float32(layout, more, D, r, size):
    """Two elements of 3e38 that turn by 45 degrees make one of 4e38 (and more under angles with a magnitude): rows of keys stay finite, at most 6 * 2^119, and
    so do queries that come back within bf16."""
    from htr_b200 import paged

    cache = empty_cache(1, 1, 16, D)
    cos = torch.full((1, r // 2), size, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(D + r)
    x = torch.randn(6, 3 * D, device=DEV, generator=g)
    i, j = (4, 5) if layout == "interleaved" else (4, 4 + r // 2)
    x[0, i] = x[0, j] = 1e38                                     # of a query
    x[1, i], x[1, j] = -1e38, 1e38
    x[2, D + i] = x[2, D + j] = 3e38                             # of a key
    x[3, D:2 * D] = x[3, D:2 * D].sign() * 3e38
    x[4, D:2 * D] = 3e38
    x[5, D + i] = x[5, D + j] = 2e36
    x = torch.cat([x, x[:1].expand(more, -1)]).bfloat16()
    q = paged.rope_append(x, ints([0] * (6 + more)), ints([*range(6)] + [-1] * more), cos, cos.clone(), cache, 1, layout=layout)[:6]
    y = x[:6].double().view(6, 3, D)
    z = rotated(y[:, :2], cos.double().expand(6, -1), cos.double().expand(6, -1), layout) @ sylvester(D)
    # as in check_append, but that a pair grows by up to sqrt 2 times size
    noise = ((3 + math.log2(D)) * 2.0 ** -24 + (2.0 ** -19 if (6 + more) * 3 >= MANY else 0)) * 2 ** 0.5 * max(size, 1.0) * y[:, :2].abs().sum(-1)
    want = z[:, 0] * 8 / D
    assert ((q[:, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + noise[:, :1] * 8 / D * 1.01).all()
    check_rows(cache.k[0, :, :6].transpose(0, 1), cache.k_scale[0, :, :6].transpose(0, 1), (z[:, 1:] / 8).clamp(-6 * 2.0 ** 119, 6 * 2.0 ** 119), noise[:, 1:] / 8)


@gpu
@pytest.mark.parametrize("page", (16, 64, 128))
@pytest.mark.parametrize("D,hkv", ((128, 1), (64, 3), (64, 40), (128, 30)))
def test_every_place_has_one_writer(page, D, hkv):
    """Slots that stand twice or fall back, holes between them, and pages that begin anew far behind: a token whose slot does not lie above those of its page
    among the page - 1 tokens before it is not written."""
    from htr_b200 import paged

    g = torch.Generator().manual_seed(page + D)
    slots, pages = [], 12
    for id in torch.randperm(pages, generator=g).tolist():
        n = int(torch.randint(1, page + 1, (1,), generator=g))
        mine = [id * page + i for i in range(n)]
        for _ in range(1 + n // 8):
            i = int(torch.randint(0, n, (1,), generator=g))
            mine[i] = [-1, id * page, mine[max(i - 1, 0)], id * page + page - 1][int(torch.randint(0, 4, (1,), generator=g))]
        slots += mine
    slots += [slots[0], 10 ** 6, slots[-1]]
    T = len(slots)
    positions = list(range(T))
    positions[T // 2] = T + 5                                    # outside: not written, and in nobody's way
    cos, sin = angles(T, D)
    x = torch.randn(T, (1 + 2 * hkv) * D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()
    cache, status = empty_cache(pages, hkv, page, D), ints([0])
    q = paged.rope_append(x, ints(positions), ints(slots), cos, sin, cache, 1, status=status)
    fits = [0 <= s < pages * page and p < T for s, p in zip(slots, positions)]
    written, wrong = {}, False
    for t, s in enumerate(slots):
        ok = fits[t] and not any(fits[u] and slots[u] // page == s // page and slots[u] >= s for u in range(max(0, t - page + 1), t))
        wrong |= not ok and s != -1
        assert bool((q[t] != 0).any()) == ok, t
        if ok:
            written.setdefault(s, []).append(t)                  # (twice, where it stands a page's tokens apart)
    assert wrong and int(status) == 16
    # each written place has its own token's values and keys, but for those that two tokens wrote
    z = x.double().view(T, -1, D)
    cs, sn = (t.double()[torch.tensor(positions, device=DEV).clamp(max=T - 1)] for t in (cos, sin))
    exact = [rotated(z[:, 1:1 + hkv], cs, sn, "interleaved") @ sylvester(D) / 8, z[:, 1 + hkv:]]
    once = {s: by[0] for s, by in written.items() if len(by) == 1}
    at, of = torch.tensor(list(once), device=DEV), torch.tensor(list(once.values()), device=DEV)
    for codes, scale, want in ((cache.k, cache.k_scale, exact[0][of]), (cache.v, cache.v_scale, exact[1][of])):
        check_rows(codes[at // page, :, at % page], scale[at // page, :, at % page], want, 2.0 ** -15 * want.abs().sum(-1))
        never = torch.ones(pages * page, dtype=torch.bool, device=DEV)
        never[list(written)] = False
        assert (codes.transpose(1, 2)[never.view(pages, page)] == 0xFF).all() and scale.transpose(1, 2)[never.view(pages, page)].isnan().all()


@gpu
def test_products_of_queries_and_keys_stay():
    """What the transform is for: queries as they come back times keys as they are held are the products of the rotated ones, but for the keys' rounding, which
    moves no element by more than a scale."""
    from htr_b200 import paged

    for D in (64, 128):
        cache, (cos, sin) = empty_cache(2, 1, 64, D), angles(64, D)
        g = torch.Generator(device=DEV).manual_seed(D)
        x = torch.randn(40, 3 * D, device=DEV, generator=g)
        x[:, D + 3] *= 30                                        # a channel of the keys that stands out
        x = x.half()
        q = paged.rope_append(x, ints(range(40)), ints(range(40)), cos, sin, cache, 1).double()[:, 0]
        y = x.double().view(40, 3, D)
        z = rotated(y, cos.double()[:40], sin.double()[:40], "interleaved")
        held = values(cache.k[0, 0, :40], cache.k_scale[0, 0, :40])
        off = (q @ held.T - z[:, 0] @ z[:, 1].T).abs()
        moved = cache.k_scale[0, 0, :40].double()[None] * q.abs().sum(-1, keepdim=True)
        assert (off <= moved + 2.0 ** -9 * z[:, 0].norm(dim=-1)[:, None] * z[:, 1].norm(dim=-1)[None]).all()


# ---- unpack ---------------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("D,page,hkv", ((128, 16, 3), (64, 16, 1), (128, 128, 2), (64, 32, 5), (64, 128, 1)))
def test_unpacked_pages(dtype, D, page, hkv):
    from htr_b200 import paged

    g = torch.Generator(device=DEV).manual_seed(D + page)
    cache = empty_cache(7, hkv, page, D)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.copy_(torch.randint(0, 256, codes.shape, device=DEV, generator=g))
        scale.copy_(torch.exp(torch.randn(scale.shape, device=DEV, generator=g)))
    cache.v_scale[2, 0, 5] = float("nan")
    ids = ints([2, 0, 2, -1, 6, 7, 1 << 30])
    k, v = paged.unpack(cache, ids, dtype)
    assert k.shape == v.shape == (7, hkv, page, D) and k.dtype == dtype
    real = [2, 0, 2, 6]
    exact = values(cache.v[real], cache.v_scale[real])
    assert torch.equal(v[[0, 1, 2, 4]].nan_to_num(nan=99.0), exact.to(dtype).nan_to_num(nan=99.0)) and v[0, 0, 5].isnan().all() and int(v.isnan().sum()) == 2 * D
    exact = values(cache.k[real], cache.k_scale[real])
    want, terms = exact @ sylvester(D) * 8 / D, exact.abs().sum(-1, keepdim=True) * 8 / D
    # log2 D float32 sums, and the rounding at the end
    bound = math.log2(D) * 2.0 ** -24 * terms + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((k[[0, 1, 2, 4]].double() - want).abs() <= bound * 1.01).all()
    assert (k[[3, 5, 6]] == 0).all() and (v[[3, 5, 6]] == 0).all()
    assert [t.shape for t in paged.unpack(cache, ints([]), dtype)] == [(0, hkv, page, D)] * 2


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
        at += used[r]
    every = torch.tensor([[int(tables[r, p // page]) * page + p % page for p in range(s)] for r, s in enumerate(seen) if s > 0] if R == 1 else
                         [int(tables[r, p // page]) * page + p % page for r, s in enumerate(seen) for p in range(max(s, 0))], device=DEV).reshape(-1)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        n = every.numel()
        codes[every // page, :, every % page] = torch.randint(0, 256, (n, hkv, D // 2), device=DEV, generator=g).to(torch.uint8)
        size = 2.0 ** torch.randint(-2 - spread, 0 + spread, (n, hkv), device=DEV, generator=g).float() * (1 + torch.rand(n, hkv, device=DEV, generator=g))
        scale[every // page, :, every % page] = (size / 2).bfloat16()
    q = (torch.randn(sum(adds), hq, D, device=DEV, generator=g) * 2).to(dtype)
    starts = [0]
    for a in adds:
        starts.append(starts[-1] + a)
    return q, ints(starts), ints(seen), tables.to(DEV), cache


def attend_exactly(q, starts, seen, tables, cache, scale):
    """In 64 bits: the result, and the sum of p |v|, to which the roundings of the probabilities are relative.  In it also 2^-19 of the largest p times scale for
    each code that a row sees: the kernels round p times scale to fp16, whose step ends at 2^-24, with the row's largest at 2^4 or more, so that half a step
    is up to 2^-29 = 2^-10 * 2^-19 of that.  (Where there are many rows, the scale is the largest of 16 neighbours.)  (A zero code of a token that takes nearly all
    leaves a result to terms that small.)"""
    hq, hkv, page, D = q.shape[1], cache.k.shape[1], cache.k.shape[2], q.shape[2]
    out, spread = torch.zeros(q.shape, dtype=torch.double, device=DEV), torch.zeros(q.shape, dtype=torch.double, device=DEV)
    for r in range(seen.numel()):
        s, e, n = int(starts[r]), int(starts[r + 1]), int(seen[r])
        if e == s or n <= 0:
            continue
        ids = tables[r, :-(-n // page)].long()
        for h in range(hq):
            k, v = (values(c[ids, h * hkv // hq], f[ids, h * hkv // hq]).reshape(-1, D)[:n] for c, f in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            at = torch.arange(n - (e - s), n, device=DEV)
            hide = torch.arange(n, device=DEV)[None] > at[:, None]
            p = (q[s:e, h].double() @ k.T * scale).masked_fill(hide, float("-inf")).softmax(-1)
            p = torch.where(at[:, None] < 0, 0.0, p)
            v = torch.where(hide.all(0)[:, None], 0.0, v)
            vs = cache.v_scale[ids, h * hkv // hq].reshape(-1)[:n].double()
            code = (~hide).double() @ (v / vs[:, None]).abs().nan_to_num(0)
            near = torch.nn.functional.pad(vs.nan_to_num(0), (0, -n % 16)).view(-1, 16).amax(-1).repeat_interleave(16)[:n]
            out[s:e, h], spread[s:e, h] = p @ v, p @ v.abs() + 2.0 ** -19 * (p * torch.where(hide, 0.0, near)).amax(-1, keepdim=True) * code
    return out, spread


def many(q, tables, cache):
    """The same call as one of much work, which goes by what the host knows: rows of queries behind the last token and (unused) columns of the tables.  Returns
    q, tables and max_new."""
    page, group, D = cache.k.shape[2], q.shape[1] // cache.k.shape[1], q.shape[2]
    q = torch.cat([q, torch.ones_like(q[:1]).expand(max(24576 // (group * D) + 1 - q.shape[0], 0), -1, -1)])
    more = int(1.6e9 / (q.shape[0] * q.shape[1] * D * page)) + 1 - tables.shape[1]
    return q, tables if more <= 0 else torch.cat([tables, torch.full((tables.shape[0], more), -1, dtype=torch.int32, device=tables.device)], 1), q.shape[0]


def check_attention(q, starts, seen, tables, cache, max_new, scale=None, out=None):
    """By both kernels."""
    q2, tables2, most = many(q, tables, cache)
    check_one_attention(q2, starts, seen, tables2, cache, most, scale)
    return check_one_attention(q, starts, seen, tables, cache, max_new, scale, out=out)


def bound_of(dtype, want, spread):
    # half a step of the output; 2^-11 for each probability (fp16); 2^-11 for the float32 scores: D terms of |q k| * scale up to about 40 in
    # sum, 2^-24 each time the sum is rounded (128 * 40 * 2^-24 = 2^-11.7), and for the exponentials (2^-21)
    return torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -10 * spread + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def check_one_attention(q, starts, seen, tables, cache, max_new, scale, **kw):
    from htr_b200 import paged

    got = paged.attention(q, starts, seen, tables, cache, max_new, scale=scale, **kw)
    want, spread = attend_exactly(q, starts, seen, tables, cache, q.shape[2] ** -0.5 if scale is None else scale)
    n = int(starts[-1])
    bound = bound_of(q.dtype, want, spread)
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
@pytest.mark.parametrize("value", (False, True))
def test_a_nan_reaches_only_those_that_see_it(adds, wide, value):
    """The scale of a later token's key or value may be NaN, as all behind the last: earlier tokens and other heads do not see it."""
    q, starts, seen, tables, cache = filled(torch.bfloat16, 128, 16, 8, 2, (40, 17), adds)
    from htr_b200 import paged

    q, tables, most = many(q, tables, cache) if wide else (q, tables, max(adds))
    want = paged.attention(q, starts, seen, tables, cache, most, out=torch.zeros_like(q))
    at, n = 40 + adds[0] - 2, adds[0]                            # the last token but one of request 0
    (cache.v_scale if value else cache.k_scale)[int(tables[0, at // 16]), 1, at % 16] = float("nan")
    got = paged.attention(q, starts, seen, tables, cache, most, out=torch.zeros_like(q))
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[n - 2:n, 4:] = True
    assert torch.equal(got.isnan(), hit) and torch.equal(got[~hit], want[~hit])


def attend_by_scales(q, starts, seen, tables, cache, scale, wide):
    """As attend_exactly, with the bound of either kernel from what a row sees alone: half a step of fp16, 2^-25, for each code under a probability times the scale of
    its value, of which the row's largest lies at 2^4 or more: 2^-29 of that; where there are many rows (`wide`), the scale is one that lies less than 2^5 higher."""
    want, mass, floor = (torch.zeros(q.shape, dtype=torch.double, device=DEV) for _ in range(3))
    hq, hkv, D = q.shape[1], cache.k.shape[1], q.shape[2]
    for r in range(seen.numel()):
        s, e, n = int(starts[r]), int(starts[r + 1]), int(seen[r])
        ids = tables[r, :-(-n // cache.k.shape[2])].long()
        hide = torch.arange(n, device=DEV)[None] > torch.arange(n - (e - s), n, device=DEV)[:, None]
        for h in range(hq):
            g = h * hkv // hq
            k, v = (values(c[ids, g], f[ids, g]).reshape(-1, D)[:n] for c, f in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            vs = cache.v_scale[ids, g].reshape(-1)[:n].double()
            p = (q[s:e, h].double() @ k.T * scale).masked_fill(hide, float("-inf")).softmax(-1)
            want[s:e, h], mass[s:e, h] = p @ v, p @ v.abs()
            floor[s:e, h] = 2.0 ** (-24 if wide else -29) * (p * vs).amax(-1, keepdim=True) * ((~hide).double() @ (v / vs[:, None]).abs())
    return want, mass + 2.0 ** 10 * floor                    # (bound_of takes 2^-10 of it)


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,adds,wide", ((128, (3, 1), False), (64, (9, 2), False), (128, (100, 1), True), (64, (95, 33), True), (128, (30, 1), True)))
@pytest.mark.parametrize("above", (6, 12, 20, 30, 119))
@pytest.mark.parametrize("value", (False, True))
def test_tokens_that_a_row_does_not_see_do_not_reach_it(dtype, D, adds, wide, above, value):
    """The scale of a later token's key or value lies far above those of its neighbours: rows that do not see it stay within the bound of what they see."""
    from htr_b200 import paged

    q, starts, seen, tables, cache = filled(dtype, D, 16, 8, 2, (40, 17), adds)
    at, n = 40 + adds[0] - 2, adds[0] - 2                        # the last token but one of request 0; rows before it
    (cache.v_scale if value else cache.k_scale)[int(tables[0, at // 16]), :, at % 16] = 2.0 ** above
    want, spread = attend_by_scales(q, starts, seen, tables, cache, D ** -0.5, wide)
    q2, tables2, most = many(q, tables, cache) if wide else (q, tables, max(adds))
    got = paged.attention(q2, starts, seen, tables2, cache, most)
    for rows in (slice(0, n), slice(int(starts[1]), int(starts[2]))):
        off, bound = (got[rows].double() - want[rows]).abs(), bound_of(dtype, want, spread)[rows]
        assert (off <= bound).all(), float((off / bound).max())


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,hq,have,adds", ((128, 8, (3000, 100, 0, 700), (150, 3, 70, 40)), (64, 8, (2000, 33, 5, 900), (130, 300, 1, 64)), (64, 2, (5000, 17), (500, 3))))
def test_scales_of_all_sizes_over_long_sequences(dtype, D, hq, have, adds):
    """Scales of 19 binades, so that nearly all groups of 16 keep those of their tokens, by both kernels; parts of cut tiles and twins among them."""
    from htr_b200 import paged

    q, starts, seen, tables, cache = filled(dtype, D, 32, hq, 2, have, adds, spread=9)
    scale = 2.0 ** -9 * D ** -0.5                                # (scores as elsewhere: up to about 40 in sum)
    for wide in (False, True):
        want, spread = attend_by_scales(q, starts, seen, tables, cache, scale, wide)
        q2, tables2, most = many(q, tables, cache) if wide else (q, tables, 1 + 16 // (hq // 2))
        bound = bound_of(dtype, want, spread)
        for r, n in enumerate(adds if wide else [min(a, most) for a in adds]):
            rows = slice(int(starts[r]), int(starts[r]) + n)
            if wide or n == adds[r]:
                off = (paged.attention(q2, starts, seen, tables2, cache, most, scale=scale)[rows].double() - want[rows]).abs()
                assert (off <= bound[rows]).all(), (r, float((off / bound[rows]).max()))


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,adds,wide", ((128, (2, 1), False), (64, (60, 1), True), (128, (100, 7), True)))
@pytest.mark.parametrize("above", (8, 14, 18, 25, 60))
def test_keys_beside_much_larger_ones(dtype, D, adds, wide, above):
    """Each seventh key is many times its neighbours, in two dimensions in which the queries have nothing: what the neighbours' scores are does not change."""
    from htr_b200 import paged

    q, starts, seen, tables, cache = filled(dtype, D, 32, 8, 2, (300, 33), adds)
    q[..., 6:8] = 0
    cache.k[:, :, 3::7] = 0
    cache.k[:, :, 3::7, 3] = 0x77
    cache.k_scale[:, :, 3::7] = 2.0 ** above
    want, spread = attend_by_scales(q, starts, seen, tables, cache, D ** -0.5, wide)
    q2, tables2, most = many(q, tables, cache) if wide else (q, tables, max(adds))
    got, n = paged.attention(q2, starts, seen, tables2, cache, most), q.shape[0]
    off, bound = (got[:n].double() - want).abs(), bound_of(dtype, want, spread)
    assert (off <= bound).all(), float((off / bound).max())


@gpu
@pytest.mark.parametrize("adds,wide", (((1, 1), False), ((60, 1), False), ((60, 1), True)))
@pytest.mark.parametrize("page", (16, 64))
def test_table_entries_that_are_no_page_hide_their_tokens(adds, wide, page):
    from htr_b200 import paged

    q, starts, seen, tables, cache = filled(torch.bfloat16, 64, page, 2, 1, (200, 64), adds)
    q, tables, most = many(q, tables, cache) if wide else (q, tables, max(adds))
    status, total = ints([0]), int(starts[-1])
    full = paged.attention(q, starts, seen, tables, cache, most, status=status)[:total].clone()
    assert int(status) == 0
    tables[0, 2], tables[1, :] = 1 << 30, -1
    got = paged.attention(q, starts, seen, tables, cache, most, status=status)[:total]
    assert int(status) == 32 and torch.isfinite(got).all() and (got[int(starts[1]):] == 0).all() and not torch.equal(got, full)
    alone, gap = tables.clone(), ints([0])                       # -1 in the place of a page, too
    alone[0, 2], alone[1] = -1, alone[0]
    paged.attention(q, starts, seen, alone, cache, most, status=gap)
    assert int(gap) == 32
    # without the hidden tokens: request 0 alone, whose scores there are lower than anything that counts
    hidden = [t for t in range(int(seen[0])) if t // page == 2]
    n = int(starts[1])
    ids = tables[0, :-(-int(seen[0]) // page)].long().clamp(max=cache.k.shape[0] - 1)
    for h in range(2):
        k, v = (values(c[ids, 0], f[ids, 0]).reshape(-1, 64)[:int(seen[0])] for c, f in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        hide = torch.arange(k.shape[0], device=DEV)[None] > torch.arange(k.shape[0] - n, k.shape[0], device=DEV)[:, None]
        hide[:, hidden] = True
        p = (q[:n, h].double() @ k.nan_to_num(0).T / 8).masked_fill(hide, float("-inf")).softmax(-1)
        want, spread = p @ v.nan_to_num(0), p @ v.nan_to_num(0).abs() + 2.0 ** -19 * 6 * v.shape[0]      # (as in attend_exactly; scales are below 1)
        assert ((got[:n, h].double() - want).abs() <= bound_of(q.dtype, want, spread)).all()


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
    q, tables, most = many(q, tables, cache) if wide else (q, tables, max(adds))
    want = paged.attention(q, starts, seen, tables, cache, most, out=torch.zeros_like(q))
    q[1, 5, 3] = bad
    got = paged.attention(q, starts, seen, tables, cache, most, out=torch.zeros_like(q))
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
    the others' probabilities.  So many requests and heads (of the same pages) that one thread block goes over most of them."""
    from htr_b200 import paged

    hkv, group = 8, 4
    q, starts, seen, tables, cache = filled(dtype, D, 64, hkv * group, hkv, (16500,), (adds,))
    q.zero_()
    q[..., 0] = 1
    g = torch.Generator(device=DEV).manual_seed(8)
    cache.k_scale.copy_(torch.randn(cache.k.shape[:3], device=DEV, generator=g).abs().clamp(min=0.01) * (16 * spread) + 2.0 ** -100)      # the key's only dimension that counts is +-1 of it
    cache.k[..., 0] = (cache.k[..., 0] & 0xF0) | (torch.randint(0, 2, cache.k.shape[:3], device=DEV, generator=g) * 8 + 2).to(torch.uint8)
    cache.v_scale.fill_(2.0 ** -4)
    cache.v.bitwise_and_(0x77)                                   # not negative
    id = int(tables[0, 0])
    cache.k[id, :, 0, 0] = (cache.k[id, :, 0, 0] & 0xF0) | 7     # 6
    cache.k_scale[id, :, 0] = 16 * nats / 6 if nats != 15 else 40                     # (12, 15 and 18 times 16 / 6 are bf16's)
    cache.v[id, :, 0] = 0
    want, spread = attend_exactly(q, starts, seen, tables, cache, 1 / 16)
    got = paged.attention(q.repeat(R, 1, 1), ints([adds * r for r in range(R + 1)]), seen.repeat(R), many(q, tables, cache)[1].repeat(R, 1), cache, adds * R, scale=1 / 16)
    off, bound = (got.double().view(R, *q.shape) - want).abs(), bound_of(dtype, want, spread)
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


def source(name):
    import os

    return open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "htr_b200", "csrc", name)).read()


def test_sizes_that_the_tests_choose_kernels_by():
    """MANY and what `many` fills up to are the borders that the sources have."""
    import re

    assert int(re.search(r"kManyRows = (\d+);", source("paged4_kernels.cu"))[1]) == MANY
    rule = re.search(r"max_new \* head_dim > (\d+) &&\s*\(double\)tokens \* q_heads \* \(double\)width \* head_dim > ([\d.e]+);", source("paged4_attention_tc.cu"))
    assert int(rule[1]) == 24576 and float(rule[2]) <= 1.6e9


@gpu
@pytest.mark.parametrize("D,page,adds", ((128, 16, (3, 1)), (64, 64, (100, 1)), (128, 64, (517,)), (64, 16, (1, 1))))
def test_either_kernel_is_the_one_that_is_meant(D, page, adds):
    """Their workspaces differ: that of many rows has two parts of 256 rows for each multiprocessor."""
    from htr_b200 import _lib

    q, starts, seen, tables, cache = filled(torch.bfloat16, D, page, 8, 2, (40, 17)[:len(adds)], adds)
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    need = lambda q, tables, most: _lib.lib.htr_paged4_attention_workspace_bytes(q.shape[0], seen.numel(), 8, 2, D, most, tables.shape[1], page)
    assert need(*many(q, tables, cache)) == sms * (2 * 256 * (D + 2) * 4 + 16) != need(q, tables, max(adds))


@gpu
def test_attention_of_many_requests():
    adds = [1] * 1100
    adds[700], adds[3] = 90, 0
    check_attention(*filled(torch.bfloat16, 128, 16, 1, 1, [r % 5 for r in range(1100)], adds), max_new=90)


@gpu
def test_pages_beyond_four_gigabytes():
    from htr_b200 import paged

    hkv, page, D, pages = 8, 128, 128, 70000                     # 4.6 GB of keys
    g = torch.Generator(device=DEV).manual_seed(4)
    k = torch.empty(pages, hkv, page, D // 2, dtype=torch.uint8, device=DEV)
    s = torch.empty(pages, hkv, page, dtype=torch.bfloat16, device=DEV)
    cache = paged.LayerCache4(k, torch.empty_like(k), s, torch.empty_like(s))
    ids = [69999, 0, 68000]
    for x in (0, 1):
        for id in ids:
            cache[x][id] = torch.randint(0, 256, (hkv, page, D // 2), device=DEV, generator=g).to(torch.uint8)
            cache[2 + x][id] = 0.3
    q = torch.randn(1, 8, D, device=DEV, generator=g).bfloat16()
    check_attention(q, ints([0, 1]), ints([300]), ints([ids]), cache, 1)
    many = torch.randn(200, 8, D, device=DEV, generator=g).bfloat16()
    check_attention(many, ints([0, 200]), ints([300]), ints([ids]), cache, 200)
    qkv = torch.randn(2, 33 * D, device=DEV, generator=g).bfloat16()[:, :32 * D]
    cos, sin = angles(400, D)
    paged.rope_append(qkv, ints([300, 301]), ints([68000 * page + 44, 68000 * page + 45]), cos, sin, cache, 16)
    want = qkv.double().reshape(2, 32, D)[:, 24:].transpose(0, 1)
    got, sc = values(cache.v[68000, :, 44:46], cache.v_scale[68000, :, 44:46]), cache.v_scale[68000, :, 44:46].double()[..., None]
    assert ((got - want).abs() <= torch.maximum(want.abs() / 5, sc / 4) * (1 + 2.0 ** -7)).all()       # half a step: 0.25, then at most a fifth
    assert torch.equal(paged.unpack(cache, ints([68000]), torch.float32)[1][0, :, 44:46].double(), got)


@gpu
@pytest.mark.parametrize("adds,wide", (((1, 1, 1), False), ((90, 1, 200), False), ((90, 1, 200), True)))
def test_two_graphs_and_another_stream(adds, wide):
    """Captured calls keep no buffers in common with one another or with eager ones: replayed at the same time they give what each gives alone."""
    from htr_b200 import paged

    sets = [filled(torch.bfloat16, 128, 16, 8, 2, have, adds, seed=s) for s, have in enumerate(((3000, 1, 50), (40, 2500, 700)))]
    most = max(adds)
    if wide:
        sets = [(q2, starts, seen, tables2, cache) for q, starts, seen, tables, cache in sets for q2, tables2, most in (many(q, tables, cache),)]
        most = sets[0][0].shape[0]
    run = lambda x: paged.attention(*x, most, out=torch.zeros_like(x[0]))
    want = [run(x).clone() for x in sets]
    graphs, outs = [], []
    for x in sets:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(x))
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
        eager = run(sets[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)) and torch.equal(eager, want[0])


@gpu
@pytest.mark.parametrize("D,adds", ((64, 1), (128, 3), (64, 130), (128, 60)))
@pytest.mark.parametrize("of_v", (-99, 118))
def test_values_at_the_ends_of_the_range_over_a_long_sequence(D, adds, of_v):
    """Scales near the ends of what `rope_append` gives, over 150000 tokens of equal scores; at the upper end of values whose sum bf16 still has."""
    q, starts, seen, tables, cache = filled(torch.bfloat16, D, 128, 4, 1, (150000,), (adds,))
    q.zero_()
    cache.v_scale.copy_(2.0 ** of_v * (1 + torch.rand(cache.v_scale.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))))
    check_attention(q, starts, seen, tables, cache, adds)


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,adds", ((128, 2), (64, 40), (128, 60)))
@pytest.mark.parametrize("size", (8, 256, 4096))
def test_tokens_whose_keys_and_values_are_much_smaller(dtype, D, adds, size):
    """Tokens side by side whose scales differ by `size`, and queries one of whose elements stands out as much."""
    q, starts, seen, tables, cache = filled(dtype, D, 16, 4, 2, (300, 33), (adds, 1))
    q[..., 5] *= size
    cache.k_scale[:, :, ::3] /= size
    cache.v_scale[:, :, 1::3] /= size
    check_attention(q / size, starts, seen, tables, cache, adds)


@gpu
@pytest.mark.parametrize("D,have,adds,block", ((128, [1500] * 6, [100] * 6, 60), (64, [2500] * 9, [30] * 9, 75)))
def test_rows_of_an_expired_wait_are_nan(D, have, adds, block):
    """The first keys of one thread block never arrive, so that bounded waits run out: the rows that it owes are NaN, the others as they are without, the
    status word is set, and the next call is served again.  Tiles of 256 rows and twins of 120 (the kernel for few rows has no such waits)."""
    from htr_b200 import _lib, paged

    q, starts, seen, tables, cache = filled(torch.bfloat16, D, 16, 8, 2, have, adds)
    q, tables, most = many(q, tables, cache)
    status = ints([0])
    want = paged.attention(q, starts, seen, tables, cache, most, out=torch.full_like(q, 3.0), status=status)
    assert int(status) == 0
    for word in (status, None):
        for one in range(block, block + 4):                      # (a thread block whose share is what an item costs besides its tokens has none)
            out = torch.full_like(q, 3.0)
            _lib.lib.htr_paged_attention_withhold(one)
            try:
                paged.attention(q, starts, seen, tables, cache, most, out=out, status=word)
            finally:
                _lib.lib.htr_paged_attention_withhold(-1)
            lost = out.isnan().any(-1)
            if lost.any():
                break
        assert 0 < int(lost.sum()) < lost.numel() // 4 and out[lost].isnan().all() and torch.equal(out[~lost], want[~lost])
    assert int(status) == 64
    assert torch.equal(paged.attention(q, starts, seen, tables, cache, most, out=torch.full_like(q, 3.0), status=status.zero_()), want) and int(status) == 0


# ---- the operators in a row -----------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("captured", (False, True))
@pytest.mark.parametrize("layout,r", (("interleaved", 128), ("half", 64)))
def test_steps_of_a_server(captured, layout, r):
    """Plan, append, attend and unpack on one cache, step after step, on a stream of their own; captured, the same steps replayed."""
    from htr_b200 import paged, rotary

    R, hq, hkv, D, page, T = 5, 8, 2, 128, 16, 60
    cache = paged.PagedCache(1, hkv, D, 60, page, R, 160, DEV, bits=4)
    cos, sin = rotary.angles(160, r, 1.0e4, factor=2.0, original=64, device=DEV)
    new, qkv, layer = ints([0] * R), torch.zeros(T, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=DEV), cache.layer(0)

    def step():
        plan = cache.plan(new, T)
        q = paged.rope_append(qkv, plan.positions, plan.slots, cos, sin, layer, hq, status=cache.status, layout=layout)
        return plan, q, paged.attention(q, plan.starts, plan.seen, cache.tables, layer, T, status=cache.status), paged.unpack(layer, cache.tables[2], torch.float32)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()                                                   # of no tokens
        stream.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                results = step()
        g = torch.Generator(device=DEV).manual_seed(r)
        for adds in ((3, 0, 40, 1, 1), (1, 17, 1, 20, 1), (1, 1, 1, 1, 1), (-1, 1, 1, 30, 1), (50, 1, 1, 1, 1)):
            new.copy_(ints(adds))
            qkv.copy_(torch.randn(qkv.shape, device=DEV, generator=g))
            if captured:
                graph.replay()
            else:
                results = step()
            plan, q, out, (k, v) = results
            n = sum(max(a, 0) for a in adds)
            want, spread = attend_exactly(q, plan.starts, plan.seen, cache.tables, layer, D ** -0.5)
            assert ((out.double() - want).abs()[:n] <= bound_of(q.dtype, want, spread)[:n]).all() and (q[n:] == 0).all() and int(cache.status) == 0
            seen = int(plan.seen[2])
            first = max(seen - max(adds[2], 0), 0)
            at = range(int(plan.starts[2]), int(plan.starts[3]))
            put = qkv.double().view(T, -1, D)[list(at), hq + hkv:]
            sc = layer.v_scale[cache.tables[2].long()].double().transpose(1, 2).reshape(-1, hkv, 1)[first:seen]
            kept = v.double().transpose(1, 2).reshape(-1, hkv, D)[first:seen]
            assert ((kept - put).abs() <= torch.maximum(put.abs() / 5, sc / 4) * (1 + 2.0 ** -7)).all()
            turned = rotated(qkv.double().view(T, -1, D)[list(at), hq:hq + hkv], cos.double()[first:seen], sin.double()[first:seen], layout)
            sk = layer.k_scale[cache.tables[2].long()].double().transpose(1, 2).reshape(-1, hkv, 1)[first:seen]
            kept = k.double().transpose(1, 2).reshape(-1, hkv, D)[first:seen]
            # no code is off by more than its scale, and the transform back keeps the norm but for its factor
            assert ((kept - turned).norm(dim=-1) <= sk[..., 0] * D ** 0.5 * 8 / D ** 0.5 * 1.01).all()


# ---- rotary.angles --------------------------------------------------------------------------------------------------


def turns(rows, dim, theta, first=0, factor=1.0, original=None, low=1.0, high=32.0):
    p, found = torch.arange(first, first + rows, dtype=torch.double)[:, None], []
    for i in range(dim // 2):
        f = theta ** (-2.0 * i / dim) / (2 * math.pi)
        keep = 0.0 if original is None else min(max((original * f - low) / (high - low), 0.0), 1.0)
        found.append(f * (keep + (1 - keep) / factor))
    t = p * torch.tensor(found, dtype=torch.double)
    return (t - t.round()) * 2 * math.pi


@gpu
@pytest.mark.parametrize("rows,dim,theta,how", ((1, 2, 1e4, {}), (1000, 128, 1e6, {}), (777, 96, 1e4, dict(first=131072)), (300, 6, 500.0, dict(factor=3.0)), (513, 256, 1e6, dict(first=999999)),
                                                (4097, 64, 1e6, dict(factor=8.0, original=32768)), (100, 30, 1e4, dict(factor=4.0, original=2048, low=2.0, high=4.0, magnitude=1.3)),
                                                (64, 128, 1e6, dict(first=2 ** 30)),
                                                (20011, 128, 1e6, dict(first=77)), (10007, 30, 1e4, dict(factor=4.0, original=2048, magnitude=0.8)), (9999, 256, 1e6, {}), (12345, 2, 1e4, {})))
def test_angles(rows, dim, theta, how):
    from htr_b200 import rotary

    cos, sin = rotary.angles(rows, dim, theta, device=DEV, **how)
    size = how.get("magnitude", 1.0)
    a = turns(rows, dim, theta, **{k: v for k, v in how.items() if k != "magnitude"})
    assert cos.shape == sin.shape == (rows, dim // 2) and cos.dtype == torch.float32
    # sincospif is off by at most a step of float32 (2^-24), its correction and the factor are rounded once each (2^-25); where there are many rows the result is a product
    # of two such complex numbers: each error times at most sqrt 2 for both parts of the other, and two roundings more: 2 * 1.42 * 2 + 1 < 7 times 2^-24.  And the angle
    # in 64 bits, once for the frequency (pow: 2 steps) and once for the product: 2^-51 of it, here and in the expectation
    far = torch.arange(how.get("first", 0), how.get("first", 0) + rows, dtype=torch.double)[:, None]
    bound = size * (7 * 2.0 ** -24 + 2 * 2.0 ** -51 * far)
    for got, want in ((cos, a.cos()), (sin, a.sin())):
        off = (got.double().cpu() - size * want).abs()
        assert (off <= bound).all(), float((off / bound).max())


@gpu
def test_angles_are_those_of_the_decoder():
    from htr_b200 import rotary
    from htr_b200.decoder import DecoderConfig, PackedDecoder

    model = PackedDecoder.__new__(PackedDecoder)
    model.cfg, model.device = DecoderConfig(), DEV
    for got, want in zip(rotary.angles(70000, 128, model.cfg.rope_theta, device=DEV), model._far_angles(70000)):
        assert float((got - want).abs().max()) <= 8 * 2.0 ** -24   # (the bound of test_angles, and a rounding of the other)


# ---- refusals -------------------------------------------------------------------------------------------------------


def test_no_cpu_path():
    from htr_b200 import _lib, paged, rotary

    i = torch.zeros(1, dtype=torch.int32)
    k, s = torch.zeros(1, 1, 16, 32, dtype=torch.uint8), torch.ones(1, 1, 16, dtype=torch.bfloat16)
    cache = paged.LayerCache4(k, k, s, s)
    for call in (lambda: paged.rope_append(torch.zeros(1, 192).bfloat16(), i, i, torch.ones(1, 32), torch.ones(1, 32), cache, 1, layout="half"),
                 lambda: paged.attention(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(2, dtype=torch.int32), i, i[None], cache, 1),
                 lambda: paged.unpack(cache, i), lambda: rotary.angles(3, 64, device="cpu")):
        with pytest.raises(_lib.HTRError, match="no CPU path"):
            call()
    with pytest.raises(_lib.HTRError, match="8 or 4 bits"):
        paged.PagedCache(1, 1, 64, 4, 16, 1, 64, "cpu", bits=2)
    small = paged.PagedCache(2, 3, 64, 4, 16, 1, 64, "cpu", bits=4).layer(1)
    assert isinstance(small, paged.LayerCache4) and small.k.shape == (4, 3, 16, 32) and small.k_scale.shape == (4, 3, 16) and small.k_scale.dtype == torch.bfloat16


def test_status_codes_without_a_gpu():
    import ctypes

    from htr_b200 import _lib

    L, f = _lib.lib, ctypes.c_float(1.0)
    p = 16                                                       # an address that the checks before a launch look at and nothing reads

    def append(dt=0, stride=6 * 64, T=2, rows=9, r=64, hq=4, hkv=1, D=64, pages=8, page=16, at=p, scales=p):
        return L.htr_paged4_append(at, dt, stride, p, p, T, p, p, rows, r, 0, hq, hkv, D, p, p, scales, p, pages, page, p, None, None)

    assert append(dt=2) == -3
    assert [append(stride=6 * 64 - 8), append(stride=6 * 64 + 4), append(T=-1), append(rows=0), append(r=80), append(r=8), append(r=24), append(hq=0), append(hkv=0), append(D=96),
            append(pages=0), append(page=8)] == [-2] * 12
    assert append(pages=1 << 28) == -8 and append(T=0, at=None) == 0 and append(at=None) == -5 and append(at=24) == -6 and append(scales=18) == -6

    def unpack(pages=8, hkv=2, page=16, D=64, n=3, dt=0, at=p, out=p):
        return L.htr_paged4_unpack(at, p, p, p, pages, hkv, page, D, p, n, out, p, dt, None)

    assert unpack(dt=3) == -3 and [unpack(pages=0), unpack(hkv=0), unpack(page=48), unpack(D=32), unpack(n=-1)] == [-2] * 5
    assert [unpack(pages=1 << 28), unpack(n=1 << 30, hkv=4)] == [-8] * 2 and unpack(n=0, at=None) == 0 and unpack(at=None) == -5 and unpack(out=8) == -6

    def attend(dt=0, T=3, R=2, stride=3, width=3, pages=8, page=16, hq=4, hkv=2, D=64, most=1, at=p, work=p, size=1 << 40):
        return L.htr_paged4_attention(at, dt, T, p, p, R, p, stride, width, p, p, p, p, pages, page, hq, hkv, D, most, f, p, None, work, size, None)

    assert attend(dt=2) == -3
    assert [attend(T=-1), attend(R=0), attend(stride=2), attend(page=17), attend(hq=5), attend(hkv=0), attend(D=32), attend(most=0)] == [-2] * 8
    assert [attend(R=8193), attend(pages=1 << 28), attend(most=1 << 30)] == [-8] * 3
    assert attend(T=0, at=None) == 0 and attend(at=None) == -5 and attend(at=24) == -6
    assert [attend(work=None), attend(size=0), attend(work=None, T=900, most=900, stride=1 << 20, width=1 << 20),
            attend(size=1 << 16, T=900, most=900, stride=1 << 20, width=1 << 20)] == [-4] * 4
    need = L.htr_paged4_attention_workspace_bytes
    assert need(3, 2, 4, 2, 64, 1, 3, 16) > 0 and [need(3, 2, 4, 2, 96, 1, 3, 16), need(3, 2, 4, 2, 64, 1, 0, 16), need(3, 2, 4, 2, 64, 1, 3, 24), need(0, 2, 4, 2, 64, 1, 3, 16)] == [0] * 4

    def angles_of(first=0, rows=4, dim=64, theta=1e4, factor=1.0, original=0.0, low=1.0, high=32.0, at=p):
        return L.htr_rope_angles(first, rows, dim, theta, factor, original, low, high, 1.0, at, p, None)

    inf = float("inf")
    assert [angles_of(first=-1), angles_of(rows=-1), angles_of(dim=0), angles_of(dim=7), angles_of(theta=0.0), angles_of(theta=inf), angles_of(factor=0.0), angles_of(factor=float("nan")),
            angles_of(original=-1.0), angles_of(low=32.0), angles_of(high=inf)] == [-2] * 11
    assert [angles_of(dim=258), angles_of(first=2 ** 31 - 3)] == [-8] * 2 and angles_of(rows=0, at=None) == 0 and angles_of(at=None) == -5


@gpu
def test_refusals():
    from htr_b200 import _lib, paged, rotary

    q, starts, seen, tables, cache = filled(torch.bfloat16, 64, 16, 4, 2, (20, 3), (1, 1))
    cos, sin = angles(64, 64)
    good = dict(qkv=torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=DEV), positions=ints([20, 3]), slots=ints([0, 16]), cos=cos, sin=sin, cache=cache, q_heads=4, layout="half")
    paged.rope_append(**good)
    bad_cache = [cache._replace(k=cache.k.float()), cache._replace(v=cache.v[:1]), cache._replace(k=cache.k.transpose(1, 2)), cache._replace(k_scale=cache.k_scale.half()),
                 cache._replace(v_scale=cache.v_scale[:1]), cache._replace(v_scale=cache.v_scale[:, :, 0]), cache._replace(k=cache.k[:, :, :8], v=cache.v[:, :, :8]), cache._replace(k=cache.k.cpu())]
    eight = paged.PagedCache(1, 2, 64, 4, 16, 1, 64, DEV).layer(0)
    for change in (dict(qkv=good["qkv"].float()), dict(qkv=good["qkv"][:, :-64]), dict(qkv=good["qkv"][0]), dict(positions=ints([1])), dict(slots=good["slots"].long()),
                   dict(cos=cos[:, :16]), dict(cos=cos[:, :12].contiguous(), sin=sin[:, :12].contiguous()), dict(cos=torch.cat((cos, cos), 1), sin=torch.cat((sin, sin), 1)), dict(sin=sin.double()),
                   dict(cos=cos[:3]), dict(q_heads=0), dict(layout="halves"), dict(layout=None), dict(cache=eight), *[dict(cache=c) for c in bad_cache]):
        with pytest.raises(_lib.HTRError):
            paged.rope_append(**{**good, **change})
    good = dict(q=q, starts=starts, seen=seen, tables=tables, cache=cache, max_new=1)
    paged.attention(**good)
    for change in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(starts=starts[:2]), dict(seen=seen.long()), dict(tables=tables[:1]), dict(tables=tables.t().contiguous().t()),
                   dict(max_new=0), dict(out=torch.empty_like(q)[:1]), dict(out=torch.empty_like(q).half()), dict(status=torch.zeros(1, device=DEV)), *[dict(cache=c) for c in bad_cache]):
        with pytest.raises(_lib.HTRError):
            paged.attention(**{**good, **change})
    assert paged.attention(q[:0], ints([0, 0, 0]), seen, tables, cache, 1).shape == (0, 4, 64)
    paged.unpack(cache, ints([0]))
    for args in ((cache, ints([0]).long()), (cache, ints([[0, 1]])), (cache, ints([0]), torch.float64), (eight, ints([0])), *[(c, ints([0])) for c in bad_cache]):
        with pytest.raises(_lib.HTRError):
            paged.unpack(*args)
    for args, how in (((4, 63), {}), ((4, 258), {}), ((-1, 64), {}), ((4, 64, 0.0), {}), ((4, 64), dict(factor=0.0)), ((4, 64), dict(original=0)), ((4, 64), dict(low=4.0, high=4.0)),
                      ((4, 64), dict(first=-1)), ((4, 64), dict(first=2 ** 31 - 2))):
        with pytest.raises(_lib.HTRError):
            rotary.angles(*args, device=DEV, **how)
    assert [t.shape for t in rotary.angles(0, 64, device=DEV)] == [(0, 32)] * 2
