"""Refusals of the paged KV cache operators at the ends of their ranges, without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest

from test_paged_cpu import attn, cache, refused, rope


@pytest.mark.parametrize("n_seqs", [2 ** 24 + 1, 2 ** 31 - 1])
def test_attention_refuses_more_requests_than_it_counts(G, n_seqs):
    """The threads' shares of the requests are counted in 32 bits: near 2^31 the last ones would pass them."""
    L, p, c = G.lib(), attn(G, n_seqs=n_seqs), cache(G)
    refused(G, L.b200_paged_attention(C.byref(p), C.byref(c), None), "n_seqs")
    assert L.b200_paged_attention_workspace(C.byref(p), C.byref(c)) == 0


@pytest.mark.parametrize("kw", [dict(scale=0.1, logit_softcap=1e-39), dict(scale=-2e38), dict(scale=3e38)], ids=str)
def test_attention_refuses_factors_past_f32(G, kw):
    """The factor that takes q.k to tanh's argument, or to an exponent of 2: an infinite one would turn scores of 0 into
    NaN."""
    refused(G, G.lib().b200_paged_attention(C.byref(attn(G, **kw)), C.byref(cache(G)), None), "scale")


@pytest.mark.parametrize("kw", [dict(out_type=1), dict(n_tokens=2, nb_q=4096), dict(n_tokens=2, nb_q_out=4096)], ids=str)
def test_rope_in_place_refuses_another_type_or_stride(G, kw):
    """Rows written over rows that are still to be read."""
    refused(G, G.lib().b200_qk_norm_rope(C.byref(rope(G, **kw)), C.byref(cache(G)), None), "q_out is q")
