"""Angles of far positions: the paged cache of the decoder is not bound by the rows of its dense caches."""
import math

import torch


def test_angles_of_far_positions():
    """Within a float32 rounding (2^-25 next to 1) of the 64-bit ones, at positions where a float32 angle is off by 2^-7 and more."""
    from htr_b200.decoder import DecoderConfig, PackedDecoder

    model = PackedDecoder.__new__(PackedDecoder)                 # no weights: what lays out a cache looks at sizes alone
    model.cfg, model.device = DecoderConfig(layers=1, hidden=128, q_heads=1, kv_heads=1, head_dim=64, intermediate=128, vocab=128, K=4, K_head=4, max_len=64), torch.device("cpu")
    cache = model.paged_cache(1, 4, page_size=128, max_len=300007)
    rows = cache.tables.shape[1] * 128
    assert tuple(cache.cos.shape) == tuple(cache.sin.shape) == (rows, 32) and rows >= 300007 and cache.cos.dtype == torch.float32 and cache.cos.is_contiguous()
    for pos in (0, 1, 63, 1024, 65535, 65536, 131071, 131072, 200003, rows - 1):
        for i in (0, 1, 7, 31):
            a = pos * model.cfg.rope_theta ** (-2 * i / 64)
            # half a step of float32 and the 64-bit angle's own rounding: pos * 2^-51
            assert abs(float(cache.cos[pos, i]) - math.cos(a)) <= 2.0 ** -25 + pos * 2.0 ** -51
            assert abs(float(cache.sin[pos, i]) - math.sin(a)) <= 2.0 ** -25 + pos * 2.0 ** -51
