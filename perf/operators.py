"""The paged KV cache operators of libggml-b200.so on the workloads they serve: the plan of a step (block tables and
slots from request lengths), query/key norm and rotation with the cache write, and attention of new tokens over the
paged cache.

With ``own`` false, run() computes them with elementary torch operations in 32 bits (angles in 64); with ``own`` true it
makes the library calls.  A case's request lengths follow from the case alone, the values from the seed.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # every request of a running batch gets one token: the per-step plan of a decode loop
        plan("plan decode 64", seqs=64, new=1, ctx=4096, bs=16),
        # a step that mixes prompt chunks and running requests
        plan("plan mixed step", seqs=256, new=96, ctx=8191, bs=32),
        # many prompts admitted at once
        plan("plan many prompts", seqs=1024, new=255, ctx=0, bs=16),
        # one token of the 3B decode (16 query heads, 2 KV heads, no norms): straight from the F32 GEMV outputs
        rope("rope one token", tokens=1, heads=16, kv_heads=2, dim=128, src="f32", out="f32", cache="f16", norm=False,
             n_rot=128, neox=True, base=1.0e6, factors=False, bs=16),
        # a decode batch of a 64-head model with normed heads and scaled frequencies, far positions
        rope("rope batch 64", tokens=64, heads=64, kv_heads=8, dim=128, src="f32", out="bf16", cache="bf16", norm=True,
             n_rot=128, neox=True, base=5.0e5, factors=True, bs=16),
        # small heads, interleaved pairs, half the dimensions rotated
        rope("rope small heads 1001", tokens=1001, heads=12, kv_heads=12, dim=64, src="f16", out="f16", cache="f16",
             norm=False, n_rot=32, neox=False, base=1.0e4, factors=False, bs=32),
        # a long prompt chunk
        rope("rope chunk 8191", tokens=8191, heads=32, kv_heads=8, dim=128, src="bf16", out="bf16", cache="bf16",
             norm=True, n_rot=128, neox=True, base=1.0e6, factors=False, bs=16),
        # single-token decode of the 3B model's heads: latency
        attn("attn one token", seqs=1, new=1, ctx=1000, heads=16, kv_heads=2, dim=128, q="f32", cache="f16", bs=16),
        # one request with a long context: few rows, a long axis
        attn("attn long context", seqs=1, new=1, ctx=130000, heads=64, kv_heads=8, dim=128, q="bf16", cache="bf16",
             bs=64),
        # a ragged decode batch, F32 in and out as the GEMVs have it
        attn("attn batch 64", seqs=64, new=1, ctx=8192, heads=64, kv_heads=8, dim=128, q="f32", cache="f16", bs=16),
        # a step of a prompt chunk among running requests, capped scores, a window, wide heads
        attn("attn mixed window", seqs=12, new=509, ctx=6000, heads=16, kv_heads=8, dim=256, q="f16", cache="f16",
             bs=32, softcap=50.0, window=4096, mixed=True),
        # a chunk of a long prompt
        attn("attn chunk 4096", seqs=1, new=4096, ctx=12288, heads=32, kv_heads=8, dim=128, q="bf16", cache="bf16",
             bs=16),
    ]


def plan(name, **kw):
    return dict(op="plan", name=name, mixed=False, **kw)


def rope(name, **kw):
    return dict(op="rope", name=name, **kw)


def attn(name, softcap=0.0, max_bias=0.0, window=0, mixed=False, **kw):
    return dict(op="attn", name=name, softcap=softcap, max_bias=max_bias, window=window, mixed=mixed, **kw)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "attn", "attn", "attn"])
    if op == "plan":
        seqs = _log(rng, 1, 1024)
        c = plan("", seqs=seqs, new=_log(rng, 1, max(1, min(4096, 131072 // seqs))), ctx=_log(rng, 1, 16384) - 1,
                 bs=rng.choice([16, 32, 64, 128, 256]))
    elif op == "rope":
        dim, kv_heads = rng.choice([64, 96, 128, 256]), rng.choice([1, 2, 4, 8, 12])
        heads, cache = kv_heads * rng.choice([1, 2, 4, 5, 8]), rng.choice(["f16", "bf16"])
        c = rope("", tokens=_log(rng, 1, max(1, min(8192, 8191 * 48 * 128 // ((heads + 2 * kv_heads) * dim)))),
                 heads=heads, kv_heads=kv_heads, dim=dim, src=rng.choice(["f32", cache]), out=rng.choice(["f32", cache]),
                 cache=cache, norm=rng.random() < 0.5, n_rot=rng.choice([dim, dim, dim // 2, 0]),
                 neox=rng.random() < 0.7, base=rng.choice([1.0e4, 5.0e5, 1.0e6]), factors=rng.random() < 0.3,
                 bs=rng.choice([16, 32, 64]))
    else:
        dim, kv_heads, cache = rng.choice([64, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice(["f16", "bf16"])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
        kind = rng.choice(["decode", "decode", "few", "chunk", "mixed"])
        seqs = 1 if kind == "chunk" and rng.random() < 0.5 else _log(rng, 1, 48 if kind == "decode" else 8)
        new = 1 if kind == "decode" else _log(rng, 2, 8) if kind == "few" else _log(rng, 16, 2048)
        most = min(32768, (1 << 28) // (seqs * heads * new), (1 << 28) // (seqs * kv_heads * dim))
        c = attn("", seqs=seqs, new=new, ctx=_log(rng, 1, max(2, most - new)) - 1, heads=heads, kv_heads=kv_heads,
                 dim=dim, q=rng.choice(["f32", cache, cache]), cache=cache, bs=rng.choice([16, 32, 64, 128]),
                 softcap=30.0 if rng.random() < 0.2 else 0.0, max_bias=8.0 if rng.random() < 0.15 else 0.0,
                 window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0, mixed=kind == "mixed")
    del c["name"]
    return c


def _lens(case):
    """[(cached, new)] of the case's requests: the first has the most of both, the others spread below it; the other
    requests of a mixed step are running ones with one new token."""
    rng = random.Random("%d %d %d %s" % (case["seqs"], case["new"], case["ctx"], case["mixed"]))
    got = [(case["ctx"], case["new"])]
    for _ in range(case["seqs"] - 1):
        cached = int(case["ctx"] * math.exp(rng.uniform(math.log(0.05), 0.0)))
        new = 1 if case["mixed"] else max(1, int(case["new"] * math.exp(rng.uniform(math.log(0.05), 0.0))))
        got.append((cached, new))
    return got


# -------------------------------------------------------------------------------------------------------------- inputs
def _normal(gen, shape, dtype=torch.float32, sigma=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * sigma).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn}[case["op"]](case, seed, gen)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _prepare_plan(case, seed, gen):
    lens, bs = _lens(case), case["bs"]
    random.Random(seed).shuffle(lens)
    owned = [-(-c // bs) for c, _ in lens]
    need = [-(-(c + n) // bs) - o for (c, n), o in zip(lens, owned)]
    width, total = max(o + n for o, n in zip(owned, need)), sum(n for _, n in lens)
    pages = torch.randperm(sum(owned) + sum(need) + 64, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < _ints(owned)[:, None]
    table[held] = pages[: sum(owned)]
    z = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
    return dict(case=case, bs=bs, total=total, cached=_ints([c for c, _ in lens]), new=_ints([n for _, n in lens]),
                table=table, free=pages[sum(owned):].contiguous(), head=_ints([3]), head_out=z(1), cu=z(len(lens) + 1),
                kv=z(len(lens)), pos=z(total), slots=z(total, torch.int64), status=z(1))


def _prepare_rope(case, seed, gen):
    T, H, KH, D, bs = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "bs"))
    src = DTYPES[case["src"]]
    blocks = -(-T // bs) + 2
    start = random.Random(seed).randrange(100000)  # a chunk somewhere in a long request
    perm = torch.randperm(blocks, generator=gen, device="cuda")
    at = torch.arange(T, device="cuda")
    cache = lambda: torch.zeros((blocks, KH, bs, D), dtype=DTYPES[case["cache"]], device="cuda")  # noqa: E731
    weight = lambda: 1.0 + _normal(gen, D, sigma=0.2) if case["norm"] else None  # noqa: E731
    factors = None
    if case["factors"] and case["n_rot"]:
        factors = 1.0 + 7.0 * torch.rand(case["n_rot"] // 2, generator=gen, device="cuda")
    return dict(case=case, q=_normal(gen, (T, H, D), src, 2.0), k=_normal(gen, (T, KH, D), src, 2.0),
                v=_normal(gen, (T, KH, D), src), qw=weight(), kw=weight(), factors=factors,
                pos=(start + at).to(torch.int32), slots=perm[at // bs] * bs + at % bs, kc=cache(), vc=cache(),
                out=torch.zeros((T, H, D), dtype=DTYPES[case["out"]], device="cuda"))


def _prepare_attn(case, seed, gen):
    H, KH, D, bs = (case[k] for k in ("heads", "kv_heads", "dim", "bs"))
    lens = _lens(case)
    kv, new = [c + n for c, n in lens], [n for _, n in lens]
    pages = [-(-n // bs) for n in kv]
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(max(pages), device="cuda")[None, :] < _ints(pages)[:, None]
    blocks = sum(pages) + 3
    table[held] = torch.randperm(blocks, generator=gen, device="cuda")[: sum(pages)].to(torch.int32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    # keys of unit variance, queries somewhat wider than that: peaked rows, as a model has them
    cache = lambda: _normal(gen, (blocks, KH, bs, D), DTYPES[case["cache"]])  # noqa: E731
    kc, vc = cache(), cache()
    q = _normal(gen, (cu[-1], H, D), DTYPES[case["q"]], 1.5)
    return dict(case=case, q=q, kc=kc, vc=vc, table=table, cu=_ints(cu), kv=_ints(kv), new=_ints(new), max_q=max(new),
                max_kv=max(kv), out=torch.zeros_like(q), scale=1.0 / math.sqrt(D))


# ----------------------------------------------------------------------------------------------------------- the passes
def run(s):
    if own:
        return _own(s)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn}[s["case"]["op"]](s)


def _plain_plan(s):
    bs, table = s["bs"], s["table"]
    cached, new = s["cached"].long(), s["new"].long()
    owned, kv = (cached + bs - 1) // bs, cached + new
    need = (kv + bs - 1) // bs - owned
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    first = s["head"].long() + torch.cumsum(need, 0) - need
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new, output_size=s["total"])
    pos = cached[seq] + torch.arange(s["total"], device="cuda") - cu[seq]
    page = pos // bs
    fresh = page >= owned[seq]
    taken = torch.where(fresh, first[seq] + page - owned[seq], 0)
    block = torch.where(fresh, s["free"][taken], table[seq, page])
    table[seq, page] = block
    slots = block.long() * bs + pos % bs
    head = s["head"] + need.sum().to(torch.int32)
    return [cu.to(torch.int32), kv.to(torch.int32), pos.to(torch.int32), slots, table, head, torch.zeros_like(s["status"])]


def _plain_turn(x, w, cos, sin, n, neox):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    if not n:
        return x
    a, b = (x[..., : n // 2], x[..., n // 2: n]) if neox else (x[..., 0:n:2], x[..., 1:n:2])
    y, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([y, z], -1) if neox else torch.stack([y, z], -1).flatten(-2)
    return torch.cat([turned, x[..., n:]], -1)


def _plain_rope(s):
    c = s["case"]
    n, bs = c["n_rot"], c["bs"]
    freq = c["base"] ** (-torch.arange(0, n, 2, dtype=torch.float64, device="cuda") / max(n, 1))
    if s["factors"] is not None:
        freq = freq / s["factors"]
    angle = s["pos"].double()[:, None, None] * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    s["out"].copy_(_plain_turn(s["q"], s["qw"], cos, sin, n, c["neox"]))
    block, off = s["slots"] // bs, s["slots"] % bs
    s["kc"][block, :, off] = _plain_turn(s["k"], s["kw"], cos, sin, n, c["neox"]).to(s["kc"].dtype)
    s["vc"][block, :, off] = s["v"].to(s["vc"].dtype)
    return [s["out"], s["kc"], s["vc"]]


def _slopes(heads, max_bias):
    near = 2 ** int(math.log2(heads))
    m0, m1 = 2.0 ** (-max_bias / near), 2.0 ** (-max_bias / 2.0 / near)
    return [m0 ** (h + 1) if h < near else m1 ** (2 * (h - near) + 1) for h in range(heads)]


def _plain_attn(s):
    c = s["case"]
    H, KH, D, bs = (c[k] for k in ("heads", "kv_heads", "dim", "bs"))
    B, mq, mkv, G = s["kv"].numel(), s["max_q"], s["max_kv"], H // KH
    ids = s["table"].clamp(min=0).long()
    k = s["kc"][ids].permute(0, 2, 1, 3, 4).reshape(B, KH, -1, D)[:, :, :mkv].float()  # [B, KH, keys, D]
    v = s["vc"][ids].permute(0, 2, 1, 3, 4).reshape(B, KH, -1, D)[:, :, :mkv].float()
    i, j = torch.arange(mq, device="cuda"), torch.arange(mkv, device="cuda")
    real = i[None, :] < s["new"][:, None]
    row = torch.where(real, s["cu"][:-1, None] + i[None, :], 0)
    q = s["q"][row].float().reshape(B, mq, KH, G, D).permute(0, 2, 3, 1, 4).reshape(B, KH, G * mq, D)
    x = ((q @ k.transpose(-1, -2)) * s["scale"]).reshape(B, H, mq, mkv)
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    away = j[None, None, :] - (s["kv"] - s["new"])[:, None, None] - i[None, :, None]  # [B, mq, keys]: key less query
    if c["max_bias"]:
        slope = torch.tensor(_slopes(H, c["max_bias"]), device="cuda")
        x = x + slope[None, :, None, None] * away[:, None].float()
    seen = away <= 0
    if c["window"]:
        seen &= away > -c["window"]
    x = x.masked_fill(~seen[:, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = x.reshape(B, KH, G * mq, mkv) @ v.masked_fill(~(j[None, :] < s["kv"][:, None])[:, None, :, None], 0.0)
    o = o.reshape(B, H, mq, D).permute(0, 2, 1, 3)  # [B, mq, H, D]
    s["out"].copy_(o[real])
    return s["out"]


# ------------------------------------------------------------------------------------------------------------- the calls
def _own(s):
    """The library's call on this state.  The argument records hold the state's addresses and sizes; a decode loop keeps
    them from one step to the next, so they are filled by a state's first pass."""
    call = s.get("call")
    if call is None:
        call = s["call"] = {"plan": _call_plan, "rope": _call_rope, "attn": _call_attn}[s["case"]["op"]](s)
    function, args, what, out = call
    G.check(function(*args, torch.cuda.current_stream().cuda_stream), what)
    return out


G = None


def _library():
    global G
    if G is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "xdna.cpp_b200"))
        import ggml_b200

        G = ggml_b200
    return G


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call_plan(s):
    g = _library()
    p = g.KvPlan(n_seqs=len(s["new"]), block_size=s["bs"], cached_lens=_ptr(s["cached"]), new_lens=_ptr(s["new"]),
                 block_table=_ptr(s["table"]), table_width=s["table"].shape[1], free_blocks=_ptr(s["free"]),
                 n_free=len(s["free"]), free_head=_ptr(s["head"]), free_head_out=_ptr(s["head_out"]), cu_new=_ptr(s["cu"]),
                 kv_lens=_ptr(s["kv"]), positions=_ptr(s["pos"]), slots=_ptr(s["slots"]), max_tokens=s["total"],
                 status=_ptr(s["status"]))
    out = [s["cu"], s["kv"], s["pos"], s["slots"], s["table"], s["head_out"], s["status"]]
    return g.lib().b200_kv_plan, (ctypes.byref(p),), "kv_plan", out


def _types(g):
    return {torch.float32: g.F32, torch.float16: g.F16, torch.bfloat16: g.BF16}


def _cache(g, s):
    blocks, kv_heads, bs, dim = s["kc"].shape
    return g.KvCache(type=_types(g)[s["kc"].dtype], head_dim=dim, kv_heads=kv_heads, block_size=bs, num_blocks=blocks,
                     k=_ptr(s["kc"]), v=_ptr(s["vc"]))


def _call_rope(s):
    g, c = _library(), s["case"]
    types = _types(g)
    p = g.QkNormRope(n_tokens=c["tokens"], heads=c["heads"], in_type=types[s["q"].dtype], out_type=types[s["out"].dtype],
                     q=_ptr(s["q"]), k=_ptr(s["k"]), v=_ptr(s["v"]), q_out=_ptr(s["out"]), q_norm=_ptr(s["qw"]),
                     k_norm=_ptr(s["kw"]), eps=1e-6, positions=_ptr(s["pos"]), slots=_ptr(s["slots"]), n_rot=c["n_rot"],
                     neox=int(c["neox"]), freq_base=c["base"], freq_scale=1.0, freq_factors=_ptr(s["factors"]))
    kv = _cache(g, s)
    return g.lib().b200_qk_norm_rope, (ctypes.byref(p), ctypes.byref(kv)), "qk_norm_rope", [s["out"], s["kc"], s["vc"]]


def _call_attn(s):
    g, c = _library(), s["case"]
    types, kv = _types(g), _cache(g, s)
    p = g.PagedAttention(n_tokens=s["q"].shape[0], n_seqs=len(s["kv"]), heads=c["heads"], q_type=types[s["q"].dtype],
                         out_type=types[s["out"].dtype], q=_ptr(s["q"]), out=_ptr(s["out"]), cu_new=_ptr(s["cu"]),
                         kv_lens=_ptr(s["kv"]), block_table=_ptr(s["table"]), table_width=s["table"].shape[1],
                         max_new=s["max_q"], max_kv=s["max_kv"], scale=s["scale"], logit_softcap=c["softcap"],
                         max_bias=c["max_bias"], window=c["window"])
    need = g.lib().b200_paged_attention_workspace(ctypes.byref(p), ctypes.byref(kv))
    s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = _ptr(s["workspace"]), s["workspace"].numel()
    return g.lib().b200_paged_attention, (ctypes.byref(p), ctypes.byref(kv)), "paged_attention", s["out"]


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "plan":
        lens, bs = _lens(case), case["bs"]
        tokens = sum(n for _, n in lens)
        pages = sum(-(-(c + n) // bs) - c // bs for c, n in lens)
        return {"bytes": 20 * len(lens) + 12 * tokens + 8 * pages, "flops": 0}
    if case["op"] == "rope":
        rows_kv, rows_q = case["tokens"] * 2 * case["kv_heads"], case["tokens"] * case["heads"]
        moved = (rows_q + rows_kv) * BYTES[case["src"]] + rows_q * BYTES[case["out"]] + rows_kv * BYTES[case["cache"]]
        return {"bytes": moved * case["dim"] + 12 * case["tokens"], "flops": (rows_q + rows_kv / 2) * case["dim"] * 7}
    D, H, KH, w = case["dim"], case["heads"], case["kv_heads"], case["window"]
    keys = pairs = tokens = 0
    for cached, new in _lens(case):
        tokens += new
        oldest = max(0, cached + 1 - w) if w else 0
        keys += cached + new - oldest
        if w:
            short = min(max(w - cached, 0), new)  # rows whose window reaches back to the first key
            pairs += short * cached + short * (short + 1) // 2 + (new - short) * w
        else:
            pairs += new * cached + new * (new + 1) // 2
    moved = 2 * keys * KH * D * BYTES[case["cache"]] + 2 * tokens * H * D * BYTES[case["q"]]
    return {"bytes": moved + 4 * (keys // case["bs"] + 2 * case["seqs"]), "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    return (_exact_rope if case["op"] == "rope" else _exact_attn)(case, s)


def _exact_rope(case, s):
    n, D, bs = case["n_rot"], case["dim"], case["bs"]

    def turned(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(torch.sum(y ** 2, dim=2, keepdim=True) / D + 1e-6) * w.double()
        z = y.clone()
        for i in range(n // 2):
            f = case["base"] ** (-2.0 * i / n)
            a = s["pos"].double() * (f / s["factors"][i].double() if s["factors"] is not None else f)
            u, v = (i, i + n // 2) if case["neox"] else (2 * i, 2 * i + 1)
            z[:, :, u] = y[:, :, u] * torch.cos(a)[:, None] - y[:, :, v] * torch.sin(a)[:, None]
            z[:, :, v] = y[:, :, u] * torch.sin(a)[:, None] + y[:, :, v] * torch.cos(a)[:, None]
        return z

    kc, vc = torch.zeros_like(s["kc"], dtype=torch.float64), torch.zeros_like(s["vc"], dtype=torch.float64)
    where = (torch.div(s["slots"], bs, rounding_mode="floor"), slice(None), torch.remainder(s["slots"], bs))
    kc[where] = turned(s["k"], s["kw"])
    vc[where] = s["v"].double()
    return [turned(s["q"], s["qw"]), kc, vc]


def _exact_attn(case, s):
    H, KH, D, bs, w = (case[k] for k in ("heads", "kv_heads", "dim", "bs", "window"))
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    slopes = _slopes(H, case["max_bias"]) if case["max_bias"] else None
    cu, kv = s["cu"].tolist(), s["kv"].tolist()
    for b, total in enumerate(kv):
        pages = s["table"][b, : -(-total // bs)].long()
        for h in range(H):
            g = h * KH // H
            K = s["kc"][pages, g].reshape(-1, D)[:total].double()
            V = s["vc"][pages, g].reshape(-1, D)[:total].double()
            for r0 in range(cu[b], cu[b + 1], 2048):
                r1 = min(r0 + 2048, cu[b + 1])
                p = torch.arange(r0, r1, device="cuda")[:, None] - cu[b + 1] + total  # position of each query row
                z = s["q"][r0:r1, h].double() @ K.T * s["scale"]
                if case["softcap"]:
                    z = torch.tanh(z / case["softcap"]) * case["softcap"]
                d = p - torch.arange(total, device="cuda")[None, :]
                if slopes:
                    z = z - slopes[h] * d.double()
                hidden = d < 0
                if w:
                    hidden |= d >= w
                z[hidden] = -math.inf
                out[r0:r1, h] = torch.softmax(z, dim=1) @ V
    return out
