"""The paged KV cache operators without a GPU: argument records laid out as the header has them, and every refusal made
before anything is launched."""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # a 16-byte aligned address that no refused call touches


def test_records_match_the_header(G, tmp_path):
    recs = {"b200_kv_cache": G.KvCache, "b200_kv_plan_args": G.KvPlan, "b200_qk_norm_rope_args": G.QkNormRope,
            "b200_paged_attention_args": G.PagedAttention}
    lines = []
    for name, rec in recs.items():
        lines += [f'printf("%zu\\n", offsetof(struct {name}, {f[0]}));' for f in rec._fields_]
        lines.append(f'printf("%zu\\n", sizeof(struct {name}));')
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ggml-b200.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0; }\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe],
                   check=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for rec in recs.values():
        want += [getattr(rec, f[0]).offset for f in rec._fields_] + [C.sizeof(rec)]
    assert got == want


def cache(G, **kw):
    return G.KvCache(**{**dict(type=G.F16, head_dim=128, kv_heads=2, block_size=16, num_blocks=10, k=P, v=P), **kw})


def plan(G, **kw):
    return G.KvPlan(**{**dict(n_seqs=2, block_size=16, cached_lens=P, new_lens=P, block_table=P, table_width=4,
                              free_blocks=P, n_free=8, cu_new=P, kv_lens=P, positions=P, slots=P, max_tokens=2,
                              status=P), **kw})


def rope(G, **kw):
    return G.QkNormRope(**{**dict(n_tokens=1, heads=4, in_type=G.F32, out_type=G.F32, n_rot=128, q=P, k=P, v=P, q_out=P,
                                  positions=P, slots=P, eps=1e-6, freq_base=1e4, freq_scale=1.0), **kw})


def attn(G, **kw):
    return G.PagedAttention(**{**dict(n_tokens=1, n_seqs=1, heads=4, q_type=G.F32, out_type=G.F32, q=P, out=P, cu_new=P,
                                      kv_lens=P, block_table=P, table_width=4, max_new=1, max_kv=64, scale=0.1,
                                      workspace=P, workspace_bytes=1 << 30), **kw})


def refused(G, rc, word):
    assert rc == -1 and word in G.last_error(), (rc, G.last_error())


BAD_CACHE = [(dict(type=0), "type"), (dict(type=8), "type"), (dict(head_dim=80), "head_dim"), (dict(head_dim=0), "head_dim"),
             (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=-1), "kv_heads"), (dict(block_size=0), "block_size"),
             (dict(block_size=24), "block_size"), (dict(block_size=512), "block_size"), (dict(num_blocks=0), "num_blocks"),
             (dict(num_blocks=2 ** 27), "num_blocks"), (dict(k=None), "aligned"), (dict(v=P + 8), "aligned"),
             (dict(nb_token=256), "stride"), (dict(nb_token=264, nb_head=8192, nb_block=16384), "stride"),
             (dict(nb_token=256, nb_head=4096, nb_block=2 ** 40), "stride")]


@pytest.mark.parametrize("kw,word", BAD_CACHE, ids=str)
def test_cache_refusals(G, kw, word):
    L, c = G.lib(), cache(G, **kw)
    refused(G, L.b200_qk_norm_rope(C.byref(rope(G, n_rot=0)), C.byref(c), None), word)
    refused(G, L.b200_paged_attention(C.byref(attn(G)), C.byref(c), None), word)
    assert L.b200_paged_attention_workspace(C.byref(attn(G)), C.byref(c)) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(n_seqs=-1), "n_seqs"), (dict(n_seqs=16385), "n_seqs"), (dict(block_size=10), "block_size"),
    (dict(table_width=-1), "table_width"), (dict(n_free=2 ** 31), "n_free"), (dict(max_tokens=-1), "max_tokens"),
    (dict(cached_lens=None), "null"), (dict(new_lens=None), "null"), (dict(block_table=None), "null"),
    (dict(free_blocks=None), "null"), (dict(cu_new=None), "null"), (dict(kv_lens=None), "null"),
    (dict(slots=None), "null"), (dict(status=None), "null")], ids=str)
def test_plan_refusals(G, kw, word):
    refused(G, G.lib().b200_kv_plan(C.byref(plan(G, **kw)), None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(n_tokens=-1), "n_tokens"), (dict(heads=0), "heads"), (dict(in_type=2), "types"), (dict(out_type=24), "types"),
    (dict(n_rot=4), "n_rot"), (dict(n_rot=136), "n_rot"), (dict(n_rot=-8), "n_rot"), (dict(freq_base=0.0), "freq_base"),
    (dict(freq_base=float("nan")), "freq_base"), (dict(freq_scale=float("inf")), "freq_scale"),
    (dict(q_norm=P, eps=-1.0), "eps"), (dict(k_norm=P + 4), "aligned"), (dict(q=None), "q must"), (dict(k=P + 4), "k must"),
    (dict(v=None), "v must"), (dict(q_out=P + 2), "q_out"), (dict(nb_q=2032), "stride"), (dict(nb_k=1032), "stride"),
    (dict(positions=None), "null"), (dict(slots=None), "null")], ids=str)
def test_rope_refusals(G, kw, word):
    refused(G, G.lib().b200_qk_norm_rope(C.byref(rope(G, **kw)), C.byref(cache(G)), None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(q_type=30), "type"), (dict(out_type=30), "type"), (dict(n_tokens=-1), "n_tokens"), (dict(n_seqs=-1), "n_seqs"),
    (dict(heads=5), "heads"), (dict(heads=0), "heads"), (dict(n_tokens=2 ** 30), "n_tokens"),
    (dict(table_width=-1), "table_width"), (dict(max_new=-1), "max_new"), (dict(max_kv=-1), "max_kv"),
    (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"), (dict(logit_softcap=-1.0), "logit_softcap"),
    (dict(max_bias=float("inf")), "max_bias"), (dict(cu_new=None), "null"), (dict(kv_lens=None), "null"),
    (dict(block_table=None), "null"), (dict(q=P + 8), "q must"), (dict(out=None), "out must"), (dict(nb_q=2040), "stride"),
    (dict(nb_out=16), "stride")], ids=str)
def test_attention_refusals(G, kw, word):
    refused(G, G.lib().b200_paged_attention(C.byref(attn(G, **kw)), C.byref(cache(G)), None), word)


def test_null_records_and_empty_calls(G):
    L = G.lib()
    refused(G, L.b200_kv_plan(None, None), "null")
    refused(G, L.b200_qk_norm_rope(None, C.byref(cache(G)), None), "null")
    refused(G, L.b200_qk_norm_rope(C.byref(rope(G)), None, None), "null")
    refused(G, L.b200_paged_attention(C.byref(attn(G)), None, None), "null")
    assert L.b200_paged_attention_workspace(None, None) == 0
    # no tokens: nothing to launch
    assert L.b200_qk_norm_rope(C.byref(rope(G, n_tokens=0, q=None, k=None, v=None)), C.byref(cache(G)), None) == 0
    assert L.b200_paged_attention(C.byref(attn(G, n_tokens=0, q=None)), C.byref(cache(G)), None) == 0
    assert L.b200_paged_attention(C.byref(attn(G, n_seqs=0)), C.byref(cache(G)), None) == 0
