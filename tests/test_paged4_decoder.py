"""The packed decoder over the paged cache in 4 bits: plan, append, attend and sample as a run, against dense evaluation."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
STRETCH = dict(factor=4.0, original=48, magnitude=1.1)


def a_model(dtype=torch.bfloat16, head_dim=128, fused=True, seed=3):
    from htr_b200.decoder import DecoderConfig, PackedDecoder

    cfg = DecoderConfig(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=head_dim, intermediate=512, vocab=1024, K=4, K_head=4, max_len=64)
    return PackedDecoder(cfg, DEV, seed=seed, dtype=dtype, fused=fused)


def some_prompts(lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (n,), generator=g) for n in lens]


def held(cache, layer, r, n):
    """Keys and values [n, kv_heads, head_dim] of a request, as the cache has them, and the scales of both [n, kv_heads, 1]."""
    from htr_b200 import paged

    c, ids = cache.layer(layer), cache.tables[r, :-(-n // cache.page_size)].contiguous()
    flat = lambda t: t.transpose(1, 2).reshape(-1, t.shape[1], t.shape[3])[:n]
    return [flat(t) for t in (*paged.unpack(c, ids, torch.float32), c.k_scale[ids.long()].float()[..., None], c.v_scale[ids.long()].float()[..., None])]


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
        ck, cv, sk, sv = held(cache, li, r, T)
        # a code is off by at most a fifth of its value or a quarter of its scale (half a step each); keys in the basis of the transform, whose norm is that of the
        # key times sqrt(head_dim) / 8; plus the bf16 chain's 2e-2
        for mine, theirs, s in ((rope(k), ck, sk * 8 / cfg.head_dim ** 0.5), (v, cv, sv)):
            most = 0.2 + float((0.25 * s).square().sum().sqrt()) * cfg.head_dim ** 0.5 / float(mine.norm())
            assert float((mine - theirs).norm() / mine.norm()) <= most + 2e-2
        q, k, v = (t.permute(1, 0, 2).repeat_interleave(n, 0)[None] for t, n in ((rope(q), 1), (ck, rep), (cv, rep)))
        att = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=causal)[0].permute(1, 0, 2).reshape(T, -1)
        x = x + att @ dense(L["o"]).T
        gu = _rms_norm(x, L["ln2"].float(), cfg.eps) @ dense(L["gate_up"]).T
        x = x + (torch.nn.functional.silu(gu[:, :cfg.intermediate]) * gu[:, cfg.intermediate:]) @ dense(L["down"]).T
    return _rms_norm(x, model.ln_f.float(), cfg.eps) @ dense(model.head).T


@pytest.mark.parametrize("dtype,head_dim,fused,stretch", ((torch.bfloat16, 128, True, {}), (torch.bfloat16, 64, True, STRETCH), (torch.bfloat16, 128, False, STRETCH), (torch.float16, 128, True, {})))
@pytest.mark.parametrize("steps", (((5, 1, 40), (1, 1, 1), (30, 0, 1), (1, 1, 1)), ((1, 2, 3), (1, 1, 1)), ((100, 0, 0), (1, 33, 0), (1, 1, 17), (0, 0, 1))))
def test_steps_of_many_sequences_match_dense_evaluation(dtype, head_dim, fused, stretch, steps):
    """Prompts, parts of prompts and single tokens in one step, padded rows behind them; both folded and separate forms; angles as learned and stretched."""
    model = a_model(dtype, head_dim, fused)
    R = 3
    seqs = [p.to(DEV) for p in some_prompts([sum(s[r] for s in steps) for r in range(R)])]
    cache = model.paged_cache(R, 30, page_size=16, max_len=160, bits=4, **stretch)
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
    cache = model.paged_cache(len(lens), sum(-(-(n + 12) // 16) for n in lens) + 3, page_size=16, max_len=96, bits=4)
    tokens, logprobs = model.generate_batch(prompts, 12, chunk=chunk, cache=cache)
    assert int(cache.count) == cache.free.numel() and cache.lengths.max() == 0     # the pages are back
    eager, _ = model.generate_batch(prompts, 12, chunk=chunk, cache=cache, use_graph=False)
    assert torch.equal(tokens, eager) and tokens.shape == (len(lens), 12) and (logprobs == 0).all() and ((tokens >= 0) & (tokens < 1024)).all()
    own, _ = model.generate_batch(prompts, 12, chunk=chunk, page_size=16, bits=4)
    assert torch.equal(tokens, own)


def test_an_8_bit_cache_with_stretched_angles():
    """The angles of `rotary.angles` serve both kinds of cache."""
    model, (prompt,) = a_model(), some_prompts((40,))
    cache = model.paged_cache(1, 8, page_size=16, **STRETCH)
    plain = model.paged_cache(1, 8, page_size=16)
    assert not torch.equal(cache.cos, plain.cos) and cache.layer(0).k.dtype == torch.float8_e4m3fn
    tokens, _ = model.generate_batch([prompt], 5, cache=cache)
    assert ((tokens >= 0) & (tokens < 1024)).all()
