"""The decode harness with its rotation, KV cache and attention on the GPU (PagedDecoder) against the same decode with
them on the host, matmuls through the plugin in both.  The host decoder here rounds what the GPU's cache and its chunk
queries hold in F16 the same way, so what differs are F32 roundings, values next to an F16 border (one step of one key
or value, 2^-10 of it) and the softmax weights of a chunk (2^-11 of each): under 2e-3 of an attention output, which a
cosine of 0.99999 (4.5e-3) bounds through two layers."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TINY = dict(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, inter=512, vocab=992, theta=1.0e6, eps=1.0e-6)


def f16(a):
    return a.astype(np.float16).astype(np.float32)


def rounding_decoder(D, prompt_len):
    class Rounding(D.Decoder):
        def rope(self, v, nheads, pos):
            out = super().rope(v, nheads, pos)
            return f16(out) if nheads == self.cfg["kv_heads"] or pos < prompt_len else out

    return Rounding


def test_paged_decode_matches_host_attention(cuda, G):
    import decode_harness as D

    prompt = D.prompt_ids(TINY, 9, 45)
    with G.Backend(0) as be:
        m = D.PluginModel(cuda, be, TINY, 9)

        def matmul(keys, x):  # values go into the host's cache as the GPU's cache holds them
            ys = m.matmul(keys, x)
            return [f16(y) if k[1] == "v" else y for k, y in zip(keys, ys)]

        want, logits_want = rounding_decoder(D, len(prompt))(TINY, 9, matmul).generate(prompt, 24)
        got, logits_got = D.PagedDecoder(TINY, 9, m, len(prompt) + 24).generate(prompt, 24)
        m.free()
    assert got == want
    for a, b in zip(logits_got, logits_want):
        cos = float(a.astype(np.float64) @ b / (np.linalg.norm(a) * np.linalg.norm(b)))
        assert cos >= 0.99999, cos


def test_paged_decode_refuses_more_than_its_cache(cuda, G):
    import decode_harness as D

    att = D.DeviceAttention(cuda, TINY, 32)
    att.begin(32)
    with pytest.raises(RuntimeError, match="32 tokens"):
        att.begin(1)
