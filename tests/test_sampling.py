"""The sampler against its definition in 64 bits, row by row."""
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")


def by_definition(x, u, t, k, p, least):
    """(token, logprob, whether u or p lies so near a border that another 64-bit sum may decide otherwise)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, math.nan, False
    if not t > 0:
        return int(x.argmax()), 0.0, False
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    order = np.argsort(-x, kind="stable")
    n = k if 0 < k < x.size else x.size
    mass, near = np.cumsum(w[order]), False
    if p < 1:
        within = p * mass[n - 1]
        near |= bool((np.abs(mass[:n] - within) < 1e-9 * mass[n - 1]).any())
        n = min(n, int((mass[:n] < within).sum()) + 1)
    if least > 0:
        near |= bool((np.abs(w - least) < 1e-11).any() and least < 1)
        n = min(n, int((w >= min(least, 1.0)).sum()))
    keep = order[:max(n, 1)]
    share = np.zeros_like(w)
    share[keep] = w[keep]
    run = np.cumsum(share)
    target = min(max(float(np.float32(u)), 0.0), 0.99999994) * run[-1]
    near |= bool((np.abs(run - target)[share > 0] < 1e-9 * run[-1]).any() and u > 0)
    token = int((run <= target).sum())
    return token, float((0.0 if x[token] == x.max() else (x[token] - x.max()) / t) - np.log(run[-1])), near


def check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    from htr_b200 import sampling

    tokens, logprobs = sampling.sample(logits, u, temperature, top_k, top_p, min_p)
    rows = logits.float().cpu().numpy()
    of = [[d] * len(rows) if s is None else [float(np.float32(s))] * len(rows) if not torch.is_tensor(s) else s.tolist() for s, d in
          ((temperature, 1.0), (top_k, 0), (top_p, 1.0), (min_p, 0.0))]
    skipped = 0
    for r, row in enumerate(rows):
        token, lp, near = by_definition(row, float(u[r]), of[0][r], int(of[1][r]), of[2][r], of[3][r])
        if near:
            skipped += 1
            continue
        assert int(tokens[r]) == token, (r, int(tokens[r]), token, [o[r] for o in of])
        # weights are held to 2^-42 and a sum of them is at least one: 2^-42 a token for the sum, and float32 for the result
        assert math.isnan(lp) and math.isnan(float(logprobs[r])) or abs(float(logprobs[r]) - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -42 * row.size, r
    assert skipped <= len(rows) // 8, skipped
    return tokens


def rows_of(R, V, dtype, seed, size=3.0, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(R, V + pad, device=DEV, generator=g) * size).to(dtype)[:, :V]
    return x, torch.rand(R, device=DEV, generator=g), g


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("R,V,pad", ((1, 1, 0), (3, 2, 1), (16, 7, 0), (9, 1000, 3), (5, 1025, 0), (3, 32003, 125), (2, 151936, 0), (33, 4096, 0)))
@pytest.mark.parametrize("mode", ("all", "k", "p", "min", "every"))
def test_rows_against_the_definition(dtype, R, V, pad, mode):
    x, u, g = rows_of(R, V, dtype, R + V, pad=pad)
    i = torch.arange(R, device=DEV)
    kw = {}
    if mode in ("k", "every"):
        kw["top_k"] = torch.tensor([0, 1, 5, 50, V, V + 9], dtype=torch.int32, device=DEV)[i % 6]
    if mode in ("p", "every"):
        kw["top_p"] = torch.tensor([0.9, 0.5, 1.0, 0.0, 0.999], device=DEV)[i % 5]
    if mode in ("min", "every"):
        kw["min_p"] = torch.tensor([0.1, 0.0, 1.0, 0.003], device=DEV)[i % 4]
    if mode != "all":
        kw["temperature"] = torch.tensor([1.0, 0.7, 0.0, 2.5, 0.05, 30.0, -1.0], device=DEV)[i % 7]
    check(x, u, **kw)


@gpu
@pytest.mark.parametrize("k,p", ((4, 1.0), (0, 0.5), (300, 0.9), (1, 0.1)))
def test_ties_go_to_the_lowest_index(k, p):
    """Equal logits everywhere, and few distinct ones: the kept tokens are the first of those that tie."""
    from htr_b200 import sampling

    V = 777
    x = torch.zeros(64, V, dtype=torch.bfloat16, device=DEV)
    x[32:] = (torch.arange(V, device=DEV) * 7919 % 5).bfloat16()
    u = (torch.arange(64, device=DEV) + 0.37) / 64
    check(x, u, top_k=k, top_p=p)
    tokens, logprobs = sampling.sample(x[:1], torch.tensor([0.99999994], device=DEV), top_k=k, top_p=p)
    n = min(k or V, math.ceil(np.float32(p) * np.float64(k or V)))
    assert int(tokens[0]) == n - 1 and abs(float(logprobs[0]) + math.log(n)) < 1e-6
    assert int(sampling.sample(x[32:33], u[:1], temperature=0.0)[0]) == next(i for i in range(V) if i * 7919 % 5 == 4)


@gpu
def test_special_logits():
    from htr_b200 import sampling

    inf, nan = math.inf, math.nan
    x = torch.zeros(6, 300, device=DEV)
    x[0] = -inf
    x[1] = nan
    x[2], x[2, 17] = -inf, -3.0                                  # one token alone
    x[3, 5], x[3, 200] = inf, inf                                # two infinite ones share everything
    x[4, :150] = nan
    x[5, ::2], x[5, 1::2] = 3.0e38, -3.0e38                      # the ends of the range
    u = torch.tensor([0.5, 0.5, 0.5, 0.6, 0.0, 0.9], device=DEV)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.8), dict(min_p=0.5), dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=inf, top_k=200)):
        if kw.get("temperature") != inf:
            check(x, u, **kw)
        tokens, logprobs = sampling.sample(x, u, **kw)
        assert tokens[:3].tolist() == [-1, -1, 17] and logprobs[:2].isnan().all() and int(tokens[3]) in (5, 200) and int(tokens[4]) >= 150 and int(tokens[5]) % 2 == 0
    x[4, :] = 0
    assert sampling.sample(x[4:5], u[4:5])[0].tolist() == [0]
    assert sampling.sample(torch.tensor([[0.0, -0.0]], device=DEV), torch.tensor([0.0], device=DEV), temperature=0.0)[0].tolist() == [0]


@gpu
def test_random_numbers_at_their_ends():
    x = torch.randn(8, 5000, generator=torch.Generator().manual_seed(2)).to(DEV)
    check(x, torch.tensor([0.0, 0.99999994, 2.0 ** -24, 1e-30, 0.5, 1.0, -0.5, 2.0], device=DEV))


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("power", (25, 39, 40, 41, 43, 47, 52, 56))
def test_random_numbers_far_below_one(dtype, power):
    """u times the sum of the weights at a fourth of the first token's weight, and at four times that: the first token, and the second."""
    from htr_b200 import sampling

    V, u = 131073, 2.0 ** -power                                 # fp16: 4 * 2^17 * 2^-25 is a weight of 2^-6 and 2^-10, a logit of -4 and -7
    x = torch.zeros(2, V, device=DEV)
    # weights are kept to 2^-43 of the largest: 2^-41 at the least, an eighth of it; a logit of -28 rounded to bf16 is off by 2^-4, a sixteenth
    x[0, 0], x[1, 0] = math.log(4 * V * u), math.log(V * u / 4)
    tokens, _ = sampling.sample(x.to(dtype), torch.full((2,), u, device=DEV))
    assert tokens.tolist() == [0, 1]


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("V", (1 << 20, 151936))
@pytest.mark.parametrize("below", (20, 25, 28, 30, 40))
def test_a_wide_tail_far_below_the_largest(dtype, V, below):
    """One token, and all others `below` nats under it: weights are multiples of 2^-42, and borders within V * 2^-42 of their place."""
    from htr_b200 import sampling

    x = torch.zeros(6, V, device=DEV)
    x[:, 0] = below
    w, off = math.exp(-below), V * 2.0 ** -42
    total = 1 + (V - 1) * w
    u = np.float32([0.0, 0.5, 1 / total - 2 * off - 2.0 ** -23, (1 + 0.25 * V * w) / total, (1 + 0.75 * V * w) / total, 0.99999994])
    tokens, logprobs = sampling.sample(x.to(dtype), torch.from_numpy(u).to(DEV))
    for target, token, logprob in zip(u.astype(np.float64) * total, tokens.tolist(), logprobs.tolist()):
        # the running weight passes the target at the token, but for the bound on both sides of it and on the total
        assert (token == 0 or 1 + (token - 1) * w <= target + 2 * off) and 1 + token * w >= target - 2 * off
        want = (-below if token else 0.0) - math.log(total)
        assert abs(logprob - want) <= off + 2.0 ** -24 * abs(want) + 2.0 ** -50
        assert token == 0 or below < 30                          # (0.41 of 2^-42 is none)


@gpu
def test_frequencies_follow_the_weights():
    from htr_b200 import sampling

    n, p = 20000, torch.tensor([0.5, 0.25, 0.125, 0.125])
    x = p.log().to(DEV).expand(n, 4)                             # rows that share their memory are copied
    got = torch.bincount(sampling.sample(x, ((torch.arange(n, device=DEV) + 0.5) / n))[0], minlength=4).cpu().double() / n
    assert float((got - p).abs().max()) <= 1 / n


@gpu
def test_a_large_vocabulary_and_many_rows():
    x, u, _ = rows_of(2, 1 << 20, torch.bfloat16, 5, size=1.0)
    check(x, u, top_p=0.95)
    check(x.float(), u)
    x, u, _ = rows_of(300, 500, torch.bfloat16, 6)
    check(x, u, top_k=40, temperature=0.8)


@gpu
def test_results_do_not_depend_on_the_run_and_replay():
    from htr_b200 import sampling

    x, u, g = rows_of(12, 50000, torch.bfloat16, 9, size=1.0)
    kw = dict(temperature=torch.full((12,), 0.9, device=DEV), top_p=torch.full((12,), 0.98, device=DEV))
    first = sampling.sample(x, u, **kw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = sampling.sample(x, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = sampling.sample(x, u, **kw)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first[0], second[0]) and torch.equal(first[0], third[0]) and torch.equal(first[1], third[1])
    u.copy_(torch.rand(12, device=DEV, generator=g))
    graph.replay()
    assert torch.equal(third[0], sampling.sample(x, u, **kw)[0])


def test_refusals_without_a_gpu():
    from htr_b200 import _lib, sampling

    with pytest.raises(_lib.HTRError, match="no CPU path"):
        sampling.sample(torch.zeros(1, 4), torch.zeros(1))
    L, p = _lib.lib, 16

    def call(dt=0, stride=8, rows=2, vocab=8, at=p, u=p, out=p):
        return L.htr_sample(at, dt, stride, rows, vocab, u, None, None, None, None, out, None, None)

    assert call(dt=3) == -3 and [call(rows=-1), call(vocab=0), call(stride=7)] == [-2] * 3 and call(vocab=(1 << 20) + 1, stride=1 << 21) == -8
    assert [call(at=None), call(u=None), call(out=None)] == [-5] * 3 and call(rows=0, at=None) == 0


@gpu
def test_refusals():
    from htr_b200 import _lib, sampling

    x, u = torch.zeros(3, 9, device=DEV), torch.zeros(3, device=DEV)
    for args, kw in (((x[0], u), {}), ((x.double(), u), {}), ((x, u.double()), {}), ((x, u[:2]), {}), ((x, u.cpu()), {}), ((x[:, :0], u), {}), ((x, u), dict(top_k=u)),
                     ((x, u), dict(top_p=u.half())), ((x, u), dict(min_p=u[:1])), ((x, u), dict(temperature=u.cpu()))):
        with pytest.raises(_lib.HTRError):
            sampling.sample(*args, **kw)
    assert sampling.sample(x[:0], u[:0])[0].shape == (0,)
