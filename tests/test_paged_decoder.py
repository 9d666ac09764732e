"""The packed decoder over the paged 8-bit cache: plan, append, attend and sample as a run, against dense evaluation."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def a_model(dtype=torch.bfloat16, head_dim=128, fused=True, seed=3):
    from htr_b200.decoder import DecoderConfig, PackedDecoder

    cfg = DecoderConfig(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=head_dim, intermediate=512, vocab=1024, K=4, K_head=4, max_len=64)
    return PackedDecoder(cfg, DEV, seed=seed, dtype=dtype, fused=fused)


def some_prompts(lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (n,), generator=g) for n in lens]


def held(cache, layer, r, n):
    """Keys and values [n, kv_heads, head_dim] of a request, as the cache has them."""
    page = cache.page_size
    ids = cache.tables[r, :-(-n // page)].long()
    c = cache.layer(layer)
    return [(x[ids].float() * s[ids][..., None, None]).transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n] for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]


def dense_logits(model, cache, r, seq):
    """float32 evaluation of one sequence with dense weights; attention over the cache's keys and values, which are compared with its own."""
    from htr_b200 import wire
    from htr_b200.decoder import _rms_norm

    cfg, T = model.cfg, seq.numel()
    dense = lambda w: wire.dequant(*w, dtype=torch.float32)
    x = model.embed[seq].float()
    pos = torch.arange(T, device=DEV)
    causal = (pos[None, :] <= pos[:, None])[None, None]
    rep = cfg.q_heads // cfg.kv_heads
    cos, sin = cache.cos[:T, None], cache.sin[:T, None]

    def rope(t):
        a, b = t[..., ::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    for li, L in enumerate(model.layers):
        qkv = _rms_norm(x, L["ln1"].float(), cfg.eps) @ dense(L["qkv"]).T
        q, k, v = (t.view(T, -1, cfg.head_dim) for t in qkv.split([n * cfg.head_dim for n in (cfg.q_heads, cfg.kv_heads, cfg.kv_heads)], -1))
        ck, cv = held(cache, li, r, T)
        for mine, theirs in ((rope(k), ck), (v, cv)):           # e4m3: half a step is 2^-4, 2^-3 when a page was scaled anew; plus the bf16 chain's 2e-2
            assert float((mine - theirs).norm() / mine.norm()) <= 2.0 ** -3 + 2e-2
        q, k, v = (t.permute(1, 0, 2).repeat_interleave(n, 0)[None] for t, n in ((rope(q), 1), (ck, rep), (cv, rep)))
        att = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=causal)[0].permute(1, 0, 2).reshape(T, -1)
        x = x + att @ dense(L["o"]).T
        gu = _rms_norm(x, L["ln2"].float(), cfg.eps) @ dense(L["gate_up"]).T
        x = x + (torch.nn.functional.silu(gu[:, :cfg.intermediate]) * gu[:, cfg.intermediate:]) @ dense(L["down"]).T
    return _rms_norm(x, model.ln_f.float(), cfg.eps) @ dense(model.head).T


@pytest.mark.parametrize("dtype,head_dim,fused", ((torch.bfloat16, 128, True), (torch.bfloat16, 64, True), (torch.bfloat16, 128, False), (torch.float16, 128, True)))
@pytest.mark.parametrize("steps", (((5, 1, 40), (1, 1, 1), (30, 0, 1), (1, 1, 1)), ((1, 2, 3), (1, 1, 1)), ((100, 0, 0), (1, 33, 0), (1, 1, 17), (0, 0, 1))))
def test_steps_of_many_sequences_match_dense_evaluation(dtype, head_dim, fused, steps):
    """Prompts, parts of prompts and single tokens in one step, padded rows behind them; both folded and separate forms."""
    model = a_model(dtype, head_dim, fused)
    R = 3
    seqs = [p.to(DEV) for p in some_prompts([sum(s[r] for s in steps) for r in range(R)])]
    cache = model.paged_cache(R, 30, page_size=16, max_len=160)
    at = [0] * R
    for adds in steps:
        pad = 2
        plan = cache.plan(torch.tensor(adds, dtype=torch.int32, device=DEV), sum(adds) + pad)
        ids = torch.cat([s[d:d + n] for s, d, n in zip(seqs, at, adds)] + [torch.zeros(pad, dtype=torch.long, device=DEV)])
        logits = model.forward_paged(ids, plan, cache, max(adds)).float()
        at = [d + n for d, n in zip(at, adds)]
        assert logits.shape == (R, 1024) and int(cache.status) == 0 and cache.lengths.tolist() == at
        for r in range(R):
            if adds[r]:
                want = dense_logits(model, cache, r, seqs[r][:at[r]])[-1]
                assert float((logits[r] - want).norm() / want.norm()) <= 2e-2      # the bound of the dense decoder's test: roundings of the chain


@pytest.mark.parametrize("lens,chunk", (((9,), 4096), ((1, 30, 64, 65, 17), 50), (tuple(range(1, 20)), 7)))
def test_generation_in_a_graph_equals_its_steps(lens, chunk):
    model, prompts = a_model(), some_prompts(lens)
    cache = model.paged_cache(len(lens), sum(-(-(n + 12) // 16) for n in lens) + 3, page_size=16, max_len=96)
    tokens, logprobs = model.generate_batch(prompts, 12, chunk=chunk, cache=cache)
    assert int(cache.count) == cache.free.numel() and cache.lengths.max() == 0     # the pages are back
    eager, _ = model.generate_batch(prompts, 12, chunk=chunk, cache=cache, use_graph=False)
    assert torch.equal(tokens, eager) and tokens.shape == (len(lens), 12) and (logprobs == 0).all() and ((tokens >= 0) & (tokens < 1024)).all()
    own, _ = model.generate_batch(prompts, 12, chunk=chunk, page_size=16)
    assert torch.equal(tokens, own)
    first, _ = model.generate_batch(prompts, 12, chunk=chunk, temperature=0.7, top_k=1, cache=cache)
    assert torch.equal(tokens, first)                                               # one token kept: the largest again


def test_greedy_tokens_are_those_of_the_dense_evaluation():
    model, prompts = a_model(), some_prompts((9, 40, 3))
    tokens, _ = model.generate_batch(prompts, 10, page_size=16)
    cache = model.paged_cache(3, 12, page_size=16)
    seqs = [torch.cat([p.to(DEV), t[:-1]]) for p, t in zip(prompts, tokens)]
    adds = [s.numel() for s in seqs]
    model.forward_paged(torch.cat(seqs), cache.plan(torch.tensor(adds, dtype=torch.int32, device=DEV), sum(adds)), cache, max(adds))
    for r, p in enumerate(prompts):
        want = dense_logits(model, cache, r, seqs[r])[p.numel() - 1:]
        # a chosen token's logit is the largest but for what two chains, each off by at most 2e-2 of the logits' norm, may differ at one place
        short = want.max(-1).values - want.gather(1, tokens[r][:, None])[:, 0]
        assert (short <= 2 * 2e-2 * want.norm(dim=1)).all()
        assert (want.argmax(-1) == tokens[r]).float().mean() >= 0.7


def test_sampled_sequences_that_end():
    model, prompts = a_model(), some_prompts((5, 20, 33, 2))
    how = dict(temperature=torch.tensor([1.0, 0.5, 2.0, 0.0]), top_k=[0, 50, 0, 0], top_p=0.9, min_p=torch.tensor([0.0, 0.0, 0.01, 0.0]), page_size=16)
    tokens, logprobs = model.generate_batch(prompts, 20, seed=7, **how)
    again, _ = model.generate_batch(prompts, 20, seed=7, **how)
    other, _ = model.generate_batch(prompts, 20, seed=8, **how)
    assert torch.equal(tokens, again) and not torch.equal(tokens[:3], other[:3]) and torch.equal(tokens[3], other[3])
    assert (logprobs <= 0).all() and (logprobs[3] == 0).all() and (logprobs[0] < 0).any()
    eos = int(tokens[0, 4])
    cut, lp = model.generate_batch(prompts, 20, seed=7, eos=eos, **how)
    # (once a sequence has ended a step has other rows, and their sums may have another order: equal up to there)
    for row in cut:
        ends = (row == eos).nonzero()
        assert (row[int(ends[0]) + 1:] == -1).all() if ends.numel() else (row >= 0).all()
    assert torch.equal(cut[0, :5], tokens[0, :5]) and (cut[0, 5:] == -1).all() and (lp[0, 5:] == 0).all()


def test_generation_refuses():
    from htr_b200 import _lib

    model, prompts = a_model(), some_prompts((5, 20))
    for bad in (dict(prompts=[]), dict(prompts=[prompts[0], prompts[0][:0]]), dict(prompts=[torch.tensor([1024])]), dict(prompts=[torch.tensor([-1])]), dict(new_tokens=0),
                dict(chunk=0), dict(cache=model.paged_cache(3, 9)), dict(temperature=torch.ones(3))):
        with pytest.raises(_lib.HTRError):
            model.generate_batch(**{**dict(prompts=prompts, new_tokens=4), **bad})
    small = model.paged_cache(2, 2, page_size=16, max_len=64)
    with pytest.raises(_lib.HTRError, match="no pages left"):
        model.generate_batch(prompts, 4, cache=small)
    assert int(small.count) == 2 and int(small.status) == 0
    tokens, _ = model.generate_batch([p[:5] for p in prompts], 4, cache=small)     # and it serves again
    assert (tokens >= 0).all()
    used = model.paged_cache(2, 9, page_size=16)
    used.plan(torch.tensor([3, 0], dtype=torch.int32, device=DEV), 3)
    with pytest.raises(_lib.HTRError):
        model.generate_batch(prompts, 4, cache=used)
    plan = used.plan(torch.tensor([1, 1], dtype=torch.int32, device=DEV), 2)
    with pytest.raises(_lib.HTRError):
        model.forward_paged(torch.zeros(0, dtype=torch.long, device=DEV), plan, used, 1)
    used.cos = None
    with pytest.raises(_lib.HTRError):
        model.forward_paged(torch.zeros(2, dtype=torch.long, device=DEV), plan, used, 1)


def test_generation_does_not_answer_for_earlier_steps():
    """A status word that an earlier step has set is refused before anything is done, and is not taken for this call's."""
    from htr_b200 import _lib

    model, prompts = a_model(), some_prompts((5, 20))
    cache = model.paged_cache(2, 9, page_size=16)
    cache.status.fill_(16)
    with pytest.raises(_lib.HTRError, match="an earlier step"):
        model.generate_batch(prompts, 4, cache=cache)
    assert int(cache.status) == 16 and int(cache.count) == 9 and int(cache.lengths.max()) == 0
    cache.status.zero_()
    tokens, _ = model.generate_batch(prompts, 4, cache=cache)
    assert (tokens >= 0).all()
