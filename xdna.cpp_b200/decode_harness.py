#!/usr/bin/env python
"""Greedy decode of a random-init Qwen2.5-3B-shaped model with every M = 1
MUL_MAT offloaded to the B200 plugin.

This stands in for llama.cpp when only MUL_MAT is claimed by the plugin
(src/ggml-xdna.cpp:95-147 claims MUL_MAT alone): the token embedding, RMSNorm,
RoPE, grouped-query attention, SwiGLU and the residual adds run on the host in
float32, and each matmul goes through ggml_backend_xdna_compute_graph with
host activations, as ggml's scheduler would hand them over.  The matmul is a
parameter of the decoder, so the same host arithmetic can be driven by
another implementation of the matmuls (the tests drive it with the CPU
oracle) and the greedy tokens compared.

Model (Qwen2.5-3B shapes): hidden 2048, 36 layers, 16 query / 2 KV heads of
128, SwiGLU intermediate 11008, vocab 151936, RMSNorm eps 1e-6, RoPE theta
1e6.  Random init: every linear weight N(0, 0.02), drawn and quantised to
Q4_0 on the GPU (b200_fill_normal + b200_quantize) and uploaded into a B200
buffer; embedding rows N(0, 0.02) drawn on the host per token id from a
seeded generator; norm weights 1; no biases; lm_head untied.  253 MUL_MATs
(1,735,704,576 weight bytes) per token.

With --attention device the rotation, the KV cache and the attention run on the
GPU too, through the paged KV cache operators (b200_kv_plan, b200_qk_norm_rope,
b200_paged_attention): q, k, v and the attention's output stay in device memory
between the matmuls, and the prompt goes through as one chunk.

Usage: python xdna.cpp_b200/decode_harness.py [--layers 36] [--prompt 16] [--new 128] [--seed 3]
                                              [--attention host|device]
"""
from __future__ import annotations

import argparse
import ctypes as C
import json
import os
import sys
import time
import zlib

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)

import ggml_b200 as G  # noqa: E402

QWEN25_3B = dict(hidden=2048, layers=36, heads=16, kv_heads=2, head_dim=128, inter=11008, vocab=151936,
                 theta=1.0e6, eps=1.0e-6)
LAYER_MATS = ("q", "k", "v", "o", "gate", "up", "down")


def mat_shapes(cfg: dict) -> dict:
    """(N, K) of each linear weight name."""
    h, kv, d, f = cfg["hidden"], cfg["kv_heads"] * cfg["head_dim"], cfg["heads"] * cfg["head_dim"], cfg["inter"]
    return {"q": (d, h), "k": (kv, h), "v": (kv, h), "o": (h, d), "gate": (f, h), "up": (f, h), "down": (h, f),
            "lm_head": (cfg["vocab"], h)}


def weight_keys(cfg: dict) -> list[tuple[int, str]]:
    return [(layer, n) for layer in range(cfg["layers"]) for n in LAYER_MATS] + [(cfg["layers"], "lm_head")]


def embedding_row(cfg: dict, seed: int, token: int) -> np.ndarray:
    rng = np.random.default_rng([seed, 7, token])
    return rng.normal(0.0, 0.02, cfg["hidden"]).astype(np.float32)


def prompt_ids(cfg: dict, seed: int, n: int) -> list[int]:
    return [int(t) for t in np.random.default_rng([seed, 11]).integers(0, cfg["vocab"], n)]


class Decoder:
    """Host side of the decode.  matmul(keys, x) returns W_key @ x for each
    (layer, name) key of a group that shares x (q/k/v, gate/up, or one)."""

    def __init__(self, cfg: dict, seed: int, matmul):
        self.cfg, self.seed, self.matmul = cfg, seed, matmul
        hd = cfg["head_dim"]
        self.inv_freq = (cfg["theta"] ** (-np.arange(0, hd, 2, dtype=np.float64) / hd)).astype(np.float64)
        self.kcache = [[] for _ in range(cfg["layers"])]
        self.vcache = [[] for _ in range(cfg["layers"])]

    def rmsnorm(self, x: np.ndarray) -> np.ndarray:
        return (x / np.sqrt(np.mean(x.astype(np.float64) ** 2) + self.cfg["eps"])).astype(np.float32)

    def rope(self, v: np.ndarray, nheads: int, pos: int) -> np.ndarray:
        hd = self.cfg["head_dim"]
        a = pos * self.inv_freq
        cos, sin = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
        v = v.reshape(nheads, hd)
        x1, x2 = v[:, : hd // 2], v[:, hd // 2:]  # rotate-half pairing (i, i + hd/2)
        return np.concatenate([x1 * cos - x2 * sin, x2 * cos + x1 * sin], axis=1)

    def step(self, token: int, pos: int) -> np.ndarray:
        cfg = self.cfg
        H, KVH, hd = cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
        x = embedding_row(cfg, self.seed, token)
        for layer in range(cfg["layers"]):
            h = self.rmsnorm(x)
            q, k, v = self.matmul([(layer, "q"), (layer, "k"), (layer, "v")], h)
            q = self.rope(q, H, pos)
            self.kcache[layer].append(self.rope(k, KVH, pos))
            self.vcache[layer].append(v.reshape(KVH, hd))
            K = np.stack(self.kcache[layer])  # [T, KVH, hd]
            V = np.stack(self.vcache[layer])
            att = np.empty((H, hd), np.float32)
            for head in range(H):
                g = head // (H // KVH)
                s = (K[:, g, :] @ q[head]) / np.float32(np.sqrt(hd))
                p = np.exp(s - s.max())
                att[head] = (p / p.sum()) @ V[:, g, :]
            (o,) = self.matmul([(layer, "o")], att.reshape(-1))
            x = x + o
            h2 = self.rmsnorm(x)
            gate, up = self.matmul([(layer, "gate"), (layer, "up")], h2)
            a = (gate / (1.0 + np.exp(-gate)) * up).astype(np.float32)
            (d,) = self.matmul([(layer, "down")], a)
            x = x + d
        (logits,) = self.matmul([(cfg["layers"], "lm_head")], self.rmsnorm(x))
        return logits

    def generate(self, prompt: list[int], n_new: int):
        """Feeds the prompt one token at a time (M = 1), then decodes n_new
        tokens greedily.  Returns the generated tokens and each step's logits."""
        tokens, logits_all = [], []
        pos, tok = 0, None
        for t in prompt:
            logits = self.step(t, pos)
            pos += 1
        for _ in range(n_new):
            tok = int(np.argmax(logits))
            tokens.append(tok)
            logits_all.append(logits)
            logits = self.step(tok, pos)
            pos += 1
        return tokens, logits_all


class DeviceAttention:
    """Rotation, paged KV cache and attention of one request on the GPU: caches
    of `max_tokens` tokens for every layer in blocks of `block_size`, F16 (the
    type a ggml host keeps them in), one block table for all layers.

    begin(n) plans a step of n new tokens; attend(layer, q, k, v) rotates the
    step's rows (F32, [n, heads * head_dim] on the device), writes keys and
    values into the layer's cache and returns the attention's F32 output.  The
    queries of a single token stay F32; those of a chunk are rotated into F16,
    which the tensor-core kernel takes."""

    def __init__(self, torch, cfg: dict, max_tokens: int, block_size: int = 16):
        self.torch, self.cfg, self.bs = torch, cfg, block_size
        n = -(-max_tokens // block_size)
        shape = (n, cfg["kv_heads"], block_size, cfg["head_dim"])
        kinds = dict(type=G.F16, head_dim=cfg["head_dim"], kv_heads=cfg["kv_heads"], block_size=block_size, num_blocks=n)
        self.mem = [[torch.empty(shape, dtype=torch.float16, device="cuda") for _ in range(2)]
                    for _ in range(cfg["layers"])]
        self.caches = [G.KvCache(k=k.data_ptr(), v=v.data_ptr(), **kinds) for k, v in self.mem]
        ints = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((1, n), -1, **ints)
        self.free = torch.arange(n, **ints)
        self.head, self.cached, self.status = (torch.zeros(1, **ints) for _ in range(3))
        self.length, self.steps, self.step = 0, {}, None

    def begin(self, n: int) -> None:
        """Positions and cache slots of n new tokens; lengths and table move on, on the device."""
        if self.length + n > self.table.shape[1] * self.bs:
            raise RuntimeError(f"the KV cache holds {self.table.shape[1] * self.bs} tokens")
        if n not in self.steps:
            self.steps[n] = self._step(n)
        self.step = self.steps[n]
        G.check(G.lib().b200_kv_plan(C.byref(self.step["plan"]), self._stream()), "kv_plan")
        self.length += n

    def attend(self, layer: int, q, k, v):
        s, L, cache = self.step, G.lib(), C.byref(self.caches[layer])
        s["rope"].q, s["rope"].k, s["rope"].v = q.data_ptr(), k.data_ptr(), v.data_ptr()
        G.check(L.b200_qk_norm_rope(C.byref(s["rope"]), cache, self._stream()), "qk_norm_rope")
        G.check(L.b200_paged_attention(C.byref(s["attn"]), cache, self._stream()), "paged_attention")
        return s["out"]

    def _stream(self) -> int:
        return self.torch.cuda.current_stream().cuda_stream

    def _step(self, n: int) -> dict:
        """Buffers and argument records of a step of n tokens."""
        torch, cfg = self.torch, self.cfg
        H, D = cfg["heads"], cfg["head_dim"]
        dev = dict(device="cuda")
        single = n == 1
        b = dict(new=torch.full((1,), n, dtype=torch.int32, **dev), cu=torch.empty(2, dtype=torch.int32, **dev),
                 pos=torch.empty(n, dtype=torch.int32, **dev), slots=torch.empty(n, dtype=torch.int64, **dev),
                 q=torch.empty((n, H * D), dtype=torch.float32 if single else torch.float16, **dev),
                 out=torch.empty((n, H * D), dtype=torch.float32, **dev))
        width = self.table.shape[1]
        b["plan"] = G.KvPlan(n_seqs=1, block_size=self.bs, cached_lens=self.cached.data_ptr(),
                             new_lens=b["new"].data_ptr(), block_table=self.table.data_ptr(), table_width=width,
                             free_blocks=self.free.data_ptr(), n_free=width, free_head=self.head.data_ptr(),
                             free_head_out=self.head.data_ptr(), cu_new=b["cu"].data_ptr(),
                             kv_lens=self.cached.data_ptr(), positions=b["pos"].data_ptr(), slots=b["slots"].data_ptr(),
                             max_tokens=n, status=self.status.data_ptr())
        kind = G.F32 if single else G.F16
        b["rope"] = G.QkNormRope(n_tokens=n, heads=H, in_type=G.F32, out_type=kind, n_rot=D, q_out=b["q"].data_ptr(),
                                 positions=b["pos"].data_ptr(), slots=b["slots"].data_ptr(), freq_base=cfg["theta"],
                                 freq_scale=1.0, neox=1)
        b["attn"] = G.PagedAttention(n_tokens=n, n_seqs=1, heads=H, q_type=kind, out_type=G.F32, q=b["q"].data_ptr(),
                                     out=b["out"].data_ptr(), cu_new=b["cu"].data_ptr(), kv_lens=self.cached.data_ptr(),
                                     block_table=self.table.data_ptr(), table_width=width, max_new=n,
                                     max_kv=width * self.bs, scale=D ** -0.5)
        need = G.lib().b200_paged_attention_workspace(C.byref(b["attn"]), C.byref(self.caches[0]))
        b["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, **dev)
        b["attn"].workspace, b["attn"].workspace_bytes = b["workspace"].data_ptr(), b["workspace"].numel()
        return b


class PagedDecoder(Decoder):
    """The decoder with its attention on the GPU.  model is a PluginModel: its
    matmul serves host rows, its matmul_device rows in device memory."""

    def __init__(self, cfg: dict, seed: int, model, max_tokens: int, block_size: int = 16):
        super().__init__(cfg, seed, model.matmul)
        self.model = model
        self.attention = DeviceAttention(model.torch, cfg, max_tokens, block_size)

    def extend(self, tokens: list[int]) -> np.ndarray:
        """Feeds tokens behind those so far, as one chunk; the logits of the last one."""
        cfg, torch = self.cfg, self.model.torch
        x = np.stack([embedding_row(cfg, self.seed, t) for t in tokens])
        self.attention.begin(len(tokens))
        for layer in range(cfg["layers"]):
            h = torch.from_numpy(np.stack([self.rmsnorm(r) for r in x])).cuda()
            q, k, v = self.model.matmul_device([(layer, "q"), (layer, "k"), (layer, "v")], h)
            (o,) = self.model.matmul_device([(layer, "o")], self.attention.attend(layer, q, k, v))
            x = x + o.cpu().numpy()
            for i in range(len(tokens)):
                gate, up = self.matmul([(layer, "gate"), (layer, "up")], self.rmsnorm(x[i]))
                (d,) = self.matmul([(layer, "down")], (gate / (1.0 + np.exp(-gate)) * up).astype(np.float32))
                x[i] = x[i] + d
        (logits,) = self.matmul([(cfg["layers"], "lm_head")], self.rmsnorm(x[-1]))
        return logits

    def generate(self, prompt: list[int], n_new: int):
        """Feeds the prompt as one chunk, then decodes n_new tokens greedily."""
        tokens, logits_all = [], []
        logits = self.extend(prompt)
        for _ in range(n_new):
            tokens.append(int(np.argmax(logits)))
            logits_all.append(logits)
            logits = self.extend(tokens[-1:])
        return tokens, logits_all


class PluginModel:
    """The model's Q4_0 weights in one B200 buffer, and the matmul through
    ggml_backend_xdna_compute_graph (host activations)."""

    def __init__(self, torch, be, cfg: dict, seed: int):
        self.cfg, self.be, self.torch = cfg, be, torch
        shapes = mat_shapes(cfg)
        keys = weight_keys(cfg)
        total = sum(shapes[n][0] * G.row_bytes(G.Q4_0, shapes[n][1]) for _, n in keys)
        self.buf = G.Buffer(total + 4096 * (len(keys) + 2), dev=be.dev)
        self.w = {}
        L = G.lib()
        for layer, name in keys:
            N, K = shapes[name]
            t = self.buf.alloc(G.tensor(G.Q4_0, [K, N, 1, 1], name=f"{name}.{layer}"))
            w = torch.empty(N * K, dtype=torch.float32, device="cuda")
            G.check(L.b200_fill_normal(w.data_ptr(), w.numel(), zlib.crc32(f"{seed}:{layer}:{name}".encode()),
                                       0.02, 0), "fill_normal")
            q = torch.empty(N * G.row_bytes(G.Q4_0, K), dtype=torch.uint8, device="cuda")
            G.check(L.b200_quantize(G.Q4_0, w.data_ptr(), q.data_ptr(), N, K, 0), "quantize")
            torch.cuda.synchronize()
            self.buf.set_device(t, q.data_ptr(), 0, q.numel())
            self.w[(layer, name)] = (t, N, K)
        self._keep = []

    def raw(self, key) -> np.ndarray:
        """GGUF bytes of one weight (the unpacked view of the buffer)."""
        t, N, K = self.w[key]
        out = np.empty(N * G.row_bytes(G.Q4_0, K), np.uint8)
        self.buf.get(t, out.ctypes.data, 0, out.nbytes)
        return out

    def matmul(self, keys, x: np.ndarray):
        x = np.ascontiguousarray(x, dtype=np.float32)
        ys, nodes = [], []
        for key in keys:
            t, N, K = self.w[key]
            y = np.empty(N, np.float32)
            xt = G.tensor(G.F32, [K, 1, 1, 1], data=x.ctypes.data)
            nodes.append(G.mul_mat_node(t, xt, y.ctypes.data, N, name=f"{key[1]}.{key[0]}"))
            ys.append(y)
            self._keep.append(xt)
        if not self.be.compute(nodes):
            raise RuntimeError(f"compute_graph failed: {G.last_error()}")
        self._keep.clear()
        return ys

    def matmul_device(self, keys, x):
        """W_key @ x for the rows of an F32 device tensor, as device tensors."""
        rows, ys, nodes, keep = x.shape[0], [], [], []
        self.torch.cuda.current_stream().synchronize()  # compute_graph runs on the backend's stream
        for key in keys:
            t, N, K = self.w[key]
            y = self.torch.empty((rows, N), dtype=self.torch.float32, device="cuda")
            xt = G.tensor(G.F32, [K, rows, 1, 1], data=x.data_ptr())
            nodes.append(G.mul_mat_node(t, xt, y.data_ptr(), N, rows, name=f"{key[1]}.{key[0]}"))
            ys.append(y)
            keep.append(xt)
        if not self.be.compute(nodes):
            raise RuntimeError(f"compute_graph failed: {G.last_error()}")
        return ys

    def free(self) -> None:
        self.buf.free()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=QWEN25_3B["layers"])
    ap.add_argument("--prompt", type=int, default=16)
    ap.add_argument("--new", type=int, default=128)
    ap.add_argument("--seed", type=int, default=3)
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--attention", choices=("host", "device"), default="host")
    a = ap.parse_args()
    import torch

    if not torch.cuda.is_available():
        sys.exit("decode_harness needs a CUDA device")
    torch.cuda.set_device(a.device)
    cfg = dict(QWEN25_3B, layers=a.layers)
    with G.Backend(a.device) as be:
        m = PluginModel(torch, be, cfg, a.seed)
        dec = (PagedDecoder(cfg, a.seed, m, a.prompt + a.new + 1) if a.attention == "device"
               else Decoder(cfg, a.seed, m.matmul))
        t0 = time.perf_counter()
        toks, _ = dec.generate(prompt_ids(cfg, a.seed, a.prompt), a.new)
        el = time.perf_counter() - t0
        m.free()
    steps = a.prompt + a.new
    print(json.dumps({"model": "qwen2.5-3b-shaped Q4_0 (random init)", "layers": cfg["layers"], "prompt": a.prompt,
                      "new_tokens": a.new, "attention": a.attention, "tok_s": round(steps / el, 2), "tokens": toks[:32]}))


if __name__ == "__main__":
    main()
