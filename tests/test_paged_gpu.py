"""The paged KV cache operators on the GPU against their definitions in 64 bits (or whole numbers), at the sizes, masks,
strides and lengths where they can go wrong."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from paged_helpers import (HALF, U, Cache, attention_ref, ints, ptr, run_attention, spread_tables, stream, type_id)

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def no_wait_ran_out(cuda, G):
    yield
    status = C.c_int(-1)
    G.check(G.lib().b200_paged_attention_error(C.byref(status)), "paged_attention_error")
    assert status.value == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


# -------------------------------------------------------------------------------------------------------------- kv_plan
def plan_ref(cached, new, table, free, head, bs, max_tokens):
    table = [list(r) for r in table]
    cu, pos, slots = [0], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        for i in range(c, c + n):
            if i % bs == 0:
                table[b][i // bs] = free[head]
                head += 1
            pos.append(i)
            slots.append(table[b][i // bs] * bs + i % bs)
        cu.append(cu[-1] + n)
    pad = max_tokens - len(pos)
    return cu, [c + n for c, n in zip(cached, new)], pos + [0] * pad, slots + [-1] * pad, table, head


class Plan:
    def __init__(self, G, cached, new, bs, width, n_free, max_tokens, head=0, seed=0, in_place=False):
        B = len(cached)
        owned = [-(-c // bs) for c in cached]
        g = torch.Generator().manual_seed(seed)
        ids = torch.randperm(sum(owned) + n_free, generator=g).tolist()
        self.rows, at = [], 0
        for o in owned:
            self.rows.append(ids[at: at + o] + [-7] * (width - o))
            at += o
        self.free_list = ids[at:]
        self.table = ints(self.rows).reshape(B, width) if B else torch.empty((0, width), dtype=torch.int32, device="cuda")
        self.cached, self.new, self.free = ints(cached), ints(new), ints(self.free_list)
        self.head = ints([head])
        self.head_out = self.head if in_place else ints([-9])
        self.kv = self.cached if in_place else ints([-9] * B)
        self.cu, self.status = ints([-9] * (B + 1)), ints([-9])
        self.pos = ints([-9] * max_tokens)
        self.slots = ints([-9] * max_tokens, torch.int64)
        self.rec = G.KvPlan(n_seqs=B, block_size=bs, cached_lens=ptr(self.cached), new_lens=ptr(self.new),
                            block_table=ptr(self.table), table_width=width, free_blocks=ptr(self.free), n_free=n_free,
                            free_head=ptr(self.head), free_head_out=ptr(self.head_out), cu_new=ptr(self.cu),
                            kv_lens=ptr(self.kv), positions=ptr(self.pos), slots=ptr(self.slots), max_tokens=max_tokens,
                            status=ptr(self.status))

    def run(self, G):
        G.check(G.lib().b200_kv_plan(C.byref(self.rec), stream()), "kv_plan")
        torch.cuda.synchronize()

    def got(self):
        return (self.cu.tolist(), self.kv.tolist(), self.pos.tolist(), self.slots.tolist(), self.table.tolist(),
                self.head_out.item())


def lens_of(B, most_cached, most_new, seed):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, most_cached + 1, (B,), generator=g).tolist()
    new = torch.randint(0, most_new + 1, (B,), generator=g).tolist()
    return cached, new


@pytest.mark.parametrize("B,most_cached,most_new,bs,pad", [
    (1, 0, 1, 16, 0), (1, 31, 5, 16, 0), (3, 64, 1, 32, 2), (33, 100, 40, 16, 7), (1024, 300, 1, 64, 0),
    (1025, 50, 3, 256, 100), (7, 0, 1000, 128, 0), (300, 17, 33, 16, 2000),
    (20, 100, 3000, 32, 500), (900, 50, 60, 16, 3)])
def test_kv_plan(cuda, G, B, most_cached, most_new, bs, pad):
    cached, new = lens_of(B, most_cached, most_new, B + bs)
    if B == 1:
        cached, new = [most_cached], [most_new]
    width = max(-(-(c + n) // bs) for c, n in zip(cached, new)) + 2
    total = sum(new) + pad
    p = Plan(G, cached, new, bs, width, sum(new) + 5, total, head=3, seed=B)
    ref = plan_ref(cached, new, p.rows, p.free_list, 3, bs, total)
    p.run(G)
    assert p.status.item() == 0
    assert p.got() == ref


def test_kv_plan_most_requests_and_none(cuda, G):
    B = 16384
    cached, new = lens_of(B, 40, 9, 1)
    p = Plan(G, cached, new, 16, 4, sum(new), sum(new), seed=2)
    ref = plan_ref(cached, new, p.rows, p.free_list, 0, 16, sum(new))
    p.run(G)
    assert p.status.item() == 0 and p.got() == ref
    none = Plan(G, [], [], 16, 4, 1, 5)
    none.run(G)
    assert none.status.item() == 0 and none.cu.tolist() == [0]
    assert none.slots.tolist() == [-1] * 5 and none.pos.tolist() == [0] * 5


@pytest.mark.parametrize("B,pad", [(40, 0), (40, 4000)])
def test_kv_plan_in_place_graph_replay(cuda, G, B, pad):
    """Lengths and head updated in place, the step replayed as a graph: each replay appends to the last."""
    cached, new = lens_of(B, 50, 20, 5)
    bs, steps = 16, 4
    width = max(-(-(c + steps * n) // bs) for c, n in zip(cached, new))
    p = Plan(G, cached, new, bs, width, steps * sum(new), sum(new) + pad, head=0, in_place=True)
    rows, head = p.rows, 0
    start = p.cached.clone()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            G.check(G.lib().b200_kv_plan(C.byref(p.rec), side.cuda_stream), "kv_plan")
    assert torch.equal(p.cached, start)
    for _ in range(steps):
        ref = plan_ref(cached, new, rows, p.free_list, head, bs, sum(new) + pad)
        graph.replay()
        torch.cuda.synchronize()
        assert p.status.item() == 0 and p.got() == ref
        cached, rows, head = ref[1], ref[4], ref[5]


def test_kv_plan_status(cuda, G):
    """What the lengths can get wrong is reported and stays inside the arrays."""
    p = Plan(G, [5, 10], [30, 30], 16, 8, 2, 60)   # 2 + 2 blocks are needed, 2 are free
    p.run(G)
    assert p.status.item() == G.KV_NO_FREE_BLOCK and p.head_out.item() == 2
    slots, rows = p.slots.tolist(), p.table.tolist()
    assert rows[0][1:3] == p.free_list[:2] and rows[1][1:] == [-7] * 7
    assert slots[:30] == [rows[0][i // 16] * 16 + i % 16 for i in range(5, 35)]
    assert slots[30:36] == [rows[1][0] * 16 + i for i in range(10, 16)] and slots[36:] == [-1] * 24

    p = Plan(G, [5, 10], [30, 30], 16, 2, 10, 60)  # three blocks each, rows of two
    p.run(G)
    assert p.status.item() == G.KV_ROW_TOO_SHORT
    assert p.slots.tolist()[27:30] == [-1] * 3 and p.table.shape == (2, 2)

    p = Plan(G, [5, 10], [30, 30], 16, 8, 10, 50)
    p.run(G)
    assert p.status.item() == G.KV_TOO_MANY_TOKENS and p.cu.tolist() == [0, 30, 50] and -1 not in p.slots.tolist()

    p = Plan(G, [5, 10, 3], [2, 4, 1], 16, 8, 10, 7)
    p.new.copy_(ints([2, -4, 0x7FFFFFFF]))
    p.run(G)
    assert p.status.item() == G.KV_BAD_LENGTH and p.cu.tolist() == [0, 2, 2, 2] and p.slots.tolist()[2:] == [-1] * 5


# --------------------------------------------------------------------------------------------------------- qk_norm_rope
def rope_ref(x, w, pos, n, neox, base, scale, factors, eps):
    """The 64-bit value, and the sum of absolute values of its rotation pair (what its roundings are relative to)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + eps) * w.double()
    out, size = y.clone(), y.abs()
    if n:
        f = scale * base ** (-torch.arange(0, n, 2, dtype=torch.float64, device=x.device) / n)
        if factors is not None:
            f = f / factors.double()
        a = (pos.double()[:, None] * f)[:, None, :]
        u, v = (slice(0, n // 2), slice(n // 2, n)) if neox else (slice(0, n, 2), slice(1, n, 2))
        out[..., u] = y[..., u] * a.cos() - y[..., v] * a.sin()
        out[..., v] = y[..., u] * a.sin() + y[..., v] * a.cos()
        size[..., u] = size[..., v] = y[..., u].abs() + y[..., v].abs()
    return out, size


def near(got, ref, bound, what):
    """got within its own rounding, and `bound`, of ref."""
    far = (got.double() - ref).abs() - bound - HALF[got.dtype] * (ref.abs() + bound)
    worst = far.max().item() if far.numel() else 0.0
    # a subnormal F16 result is rounded to a multiple of 2^-24
    assert worst <= (2.0 ** -25 if got.dtype == F16 else 0.0), (what, worst)
    assert torch.isfinite(got).all(), what


# one norm: 8 + 5 roundings of the sum of squares count half, then root, division and two products: 12 U; one
# rotation: sine and cosine within 4 U (turns rounded once, times 2 pi; 2 U of the function), three roundings
ROPE_U = 20 * U


def check_rope(G, T, H, KH, D, src, out, cache, norm, n_rot, neox, factors, bs, layout="head", fused=False,
               base=1.0e6, scale=1.0, pos0=0, in_place=False, seed=0):
    g = gen(seed)
    if fused:  # q, k and v are columns of one projection's output
        qkv = (2 * normal(g, T, (H + 2 * KH) * D)).to(src)
        q, k, v = (s.unflatten(1, (-1, D)) for s in qkv.split([H * D, KH * D, KH * D], 1))
        nb = dict.fromkeys(("nb_q", "nb_k", "nb_v"), qkv.stride(0) * qkv.element_size())
    else:
        q, k, v = ((2 * normal(g, T, h, D)).to(src) for h in (H, KH, KH))
        nb = {}
    w = [1 + 0.3 * normal(g, D) if n else None for n in ((norm, norm) if isinstance(norm, bool) else norm)]
    ff = 1 + 7 * torch.rand(n_rot // 2, generator=g, device="cuda") if factors and n_rot else None
    blocks = -(-T // bs) + 2
    c = Cache(G, blocks, KH, bs, D, cache, layout)
    order = torch.randperm(blocks, generator=g, device="cuda")
    at = torch.arange(T, device="cuda")
    slots = order[at // bs] * bs + at % bs
    if T > 3:
        slots[1], slots[3] = -1, blocks * bs  # outside the cache: nothing is written
    pos = (pos0 + at).to(torch.int32)
    refs = [rope_ref(x, wi, pos, n_rot, neox, base, scale, ff, 1e-5) for x, wi in ((q, w[0]), (k, w[1]))]
    v0 = v.clone()
    dst = q if in_place else torch.full((T, H, D), math.nan, dtype=out, device="cuda")
    if in_place:
        nb["nb_q_out"] = nb.get("nb_q", 0)
    p = G.QkNormRope(n_tokens=T, heads=H, in_type=type_id(G, src), out_type=type_id(G, dst.dtype), n_rot=n_rot,
                     q=ptr(q), k=ptr(k), v=ptr(v), q_out=ptr(dst), q_norm=ptr(w[0]), k_norm=ptr(w[1]),
                     positions=ptr(pos), slots=ptr(slots), freq_factors=ptr(ff), eps=1e-5, freq_base=base,
                     freq_scale=scale, neox=int(neox), **nb)
    G.check(G.lib().b200_qk_norm_rope(C.byref(p), C.byref(c.rec), stream()), "qk_norm_rope")
    torch.cuda.synchronize()
    near(dst, refs[0][0], ROPE_U * refs[0][1], "q")
    ok = (slots >= 0) & (slots < blocks * bs)
    b, o = slots[ok] // bs, slots[ok] % bs
    near(c.k[b, :, o], refs[1][0][ok], ROPE_U * refs[1][1][ok], "k")
    assert torch.equal(c.v[b, :, o], v0[ok].to(cache))
    c.k[b, :, o] = math.nan
    c.v[b, :, o] = math.nan
    assert c.k.isnan().all() and c.v.isnan().all()  # no other slot was touched


@pytest.mark.parametrize("src,out,cache", [(F32, F32, F16), (F32, BF16, BF16), (F16, F16, F16), (BF16, BF16, BF16),
                                           (F32, F16, BF16), (BF16, F32, F16), (F16, BF16, BF16)])
@pytest.mark.parametrize("D,n_rot,neox", [(64, 64, True), (64, 24, False), (96, 96, True), (96, 48, False),
                                          (128, 128, True), (128, 128, False), (128, 0, True), (256, 64, True),
                                          (256, 256, False)])
def test_qk_norm_rope(cuda, G, src, out, cache, D, n_rot, neox):
    check_rope(G, 37, 6, 2, D, src, out, cache, True, n_rot, neox, D == 128, 16, seed=D + n_rot)
    check_rope(G, 1, 3, 3, D, src, out, cache, False, n_rot, neox, False, 32, seed=D)


@pytest.mark.parametrize("kw", [
    dict(norm=(True, False)), dict(norm=(False, True)), dict(layout="token"), dict(layout="both", fused=True),
    dict(fused=True, in_place=True), dict(pos0=1_000_000, base=10000.0), dict(pos0=200_000, scale=0.25, factors=True),
    dict(T=5000, H=1, KH=1), dict(T=3, H=64, KH=8), dict(T=130, H=24, KH=24)])
def test_qk_norm_rope_forms(cuda, G, kw):
    args = dict(T=70, H=8, KH=2, D=128, src=BF16, out=BF16, cache=BF16, norm=True, n_rot=128, neox=True,
                factors=False, bs=16, seed=3)
    check_rope(G, **{**args, **kw})


# ------------------------------------------------------------------------------------------------------ paged_attention
def check_attention(G, lens, H, KH, D, q_type, cache_type, bs, out_type=None, layout="head", pad_rows=2, seed=0,
                    fused=False, **opts):
    """lens: (key count, new tokens) of each request.  Keys, blocks and table entries that no request owns hold NaN or
    garbage; rows of no request keep what they held."""
    g = gen(seed)
    kv, new = [a for a, _ in lens], [b for _, b in lens]
    lists, table, blocks = spread_tables([max(a, 0) for a in kv], bs, seed=seed)
    c = Cache(G, blocks, KH, bs, D, cache_type, layout)
    for n, ids in zip(kv, lists):
        if n > 0:
            c.put(ids, normal(g, n, KH, D), normal(g, n, KH, D))
    T = sum(new) + pad_rows
    if fused:
        wide = normal(g, T, (H + 3) * D).to(q_type)
        q = wide[:, : H * D].unflatten(1, (H, D))
        opts["nb_q"] = wide.stride(0) * wide.element_size()
    else:
        q = normal(g, T, H, D).to(q_type)
    q.mul_(1.5)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    out_type = out_type or q_type
    out = torch.full((T, H, D), 7.0, dtype=out_type, device="cuda")
    scale = 1 / math.sqrt(D)
    run_attention(G, q, out, c, ints(cu), ints(kv), table, scale, **opts)
    torch.cuda.synchronize()
    half = 0.0 if q_type == F32 else HALF[cache_type]
    ref_opts = {k: v for k, v in opts.items() if k in ("cap", "max_bias", "window")}
    for b, (n, m) in enumerate(lens):
        k, v = c.get(lists[b], max(n, 0))
        for r0 in range(cu[b], cu[b + 1], 1024):  # the 64-bit scores of 1024 rows at a time
            r1 = min(r0 + 1024, cu[b + 1])
            ref, bound = attention_ref(q[r0:r1], k, v, n - m + r0 - cu[b], scale, weight_half=half, **ref_opts)
            near(out[r0:r1], ref, bound, f"request {b} of {lens}, rows {r0}..")
    assert (out[cu[-1]:] == 7.0).all()
    return out


LENS = [
    [(1, 1)], [(16, 1), (17, 1), (15, 1), (1, 1)], [(64, 1), (63, 1), (65, 1), (200, 1)],
    [(3, 3), (0, 0), (70, 2), (129, 129)], [(300, 65)], [(5, 9), (0, 4), (40, 17)],
]
TYPES = [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("q_type,cache_type", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_paged_attention(cuda, G, lens, D, q_type, cache_type):
    check_attention(G, lens, 6, 2, D, q_type, cache_type, 16, seed=D)
    check_attention(G, lens, 6, 2, D, q_type, cache_type, 16, seed=D, max_kv=100000)  # another work split


@pytest.mark.parametrize("q_type,cache_type", TYPES)
@pytest.mark.parametrize("H,KH", [(1, 1), (5, 5), (8, 1), (14, 2), (17, 1), (64, 8), (72, 2)])
def test_paged_attention_groups(cuda, G, H, KH, q_type, cache_type):
    check_attention(G, [(100, 1), (33, 3), (257, 20)], H, KH, 128, q_type, cache_type, 32, seed=H)
    check_attention(G, [(100, 1), (33, 2), (257, 1)], H, KH, 128, q_type, cache_type, 32, seed=H)
    check_attention(G, [(100, 1), (33, 2), (257, 1)], H, KH, 128, q_type, cache_type, 32, seed=H, max_kv=100000)


@pytest.mark.parametrize("q_type,cache_type", TYPES)
@pytest.mark.parametrize("lens", [[(700, 1), (64, 1), (2000, 2)], [(700, 300), (130, 130)]], ids=str)
@pytest.mark.parametrize("opts", [dict(cap=5.0), dict(max_bias=8.0), dict(window=1), dict(window=100),
                                  dict(window=2 ** 31 - 1), dict(cap=20.0, max_bias=4.0, window=333)], ids=str)
def test_paged_attention_masks(cuda, G, opts, lens, q_type, cache_type):
    check_attention(G, lens, 12, 4, 128, q_type, cache_type, 64, seed=11, **opts)
    check_attention(G, lens, 3, 1, 64, q_type, cache_type, 16, seed=12, **opts)
    check_attention(G, lens, 3, 1, 64, q_type, cache_type, 16, seed=12, max_kv=100000, **opts)


@pytest.mark.parametrize("lens", [[(3000, 1)], [(5000, 1), (1, 1), (1024, 1)], [(1500, 700), (900, 1), (257, 64)]], ids=str)
@pytest.mark.parametrize("bs", [16, 128, 256])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_long(cuda, G, lens, bs, q_type, cache_type):
    check_attention(G, lens, 16, 2, 128, q_type, cache_type, bs, seed=bs)
    check_attention(G, lens, 16, 2, 128, q_type, cache_type, bs, seed=bs, max_kv=100000)  # another work split


# few tall items with many parts: one item, two, and more than their bound from the token count
@pytest.mark.parametrize("lens", [[(5000, 20)], [(6000, 40)], [(2100, 40), (1900, 35), (2500, 45)]], ids=str)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_few_long_items(cuda, G, lens, D, q_type, cache_type):
    check_attention(G, lens, 8, 1, D, q_type, cache_type, 32)


@pytest.mark.parametrize("lens", [[(200, 1), (90, 1)], [(200, 100), (90, 1)]], ids=str)
@pytest.mark.parametrize("kw", [dict(layout="token"), dict(layout="both"), dict(fused=True), dict(out_type="other"),
                                dict(max_new=0, max_kv=0), dict(max_new=100000, max_kv=1000000)], ids=str)
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_forms(cuda, G, kw, lens, q_type, cache_type):
    if kw.get("out_type"):
        kw = dict(out_type=cache_type if q_type == F32 else F32)
    check_attention(G, lens, 8, 2, 128, q_type, cache_type, 16, seed=5, **kw)


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_far_blocks(cuda, G, new, q_type, cache_type):
    """Blocks whose offsets pass 2^31 elements and 2^32 bytes."""
    bs, KH, D, blocks = 256, 8, 128, 8400
    c = Cache(G, blocks, KH, bs, D, cache_type)
    assert c.k.numel() > 2 ** 31
    g = gen(1)
    ids = [blocks - 1, 3, blocks - 2]
    c.put(ids, normal(g, 600, KH, D), normal(g, 600, KH, D))
    q = normal(g, new, 8, D).to(q_type)
    out = torch.zeros_like(q)
    run_attention(G, q, out, c, ints([0, new]), ints([600]), ints([ids]), 0.1)
    torch.cuda.synchronize()
    k, v = c.get(ids, 600)
    half = 0.0 if q_type == F32 else HALF[cache_type]
    ref, bound = attention_ref(q, k, v, 600 - new, 0.1, weight_half=half)
    near(out, ref, bound, "far blocks")


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_bad_device_data(cuda, G, new, q_type, cache_type):
    """A block id outside the cache reads as zeros, keys behind the table's row are not there, and row counts that do
    not fit the arrays are cut: nothing is accessed outside them."""
    g = gen(2)
    bs, KH, D = 16, 2, 128
    c = Cache(G, 8, KH, bs, D, cache_type)
    c.put(list(range(8)), normal(g, 128, KH, D), normal(g, 128, KH, D))
    q = normal(g, new, 4, D).to(q_type)
    half = 0.0 if q_type == F32 else HALF[cache_type]
    for bad in (8, -1, 2 ** 31 - 1, -2 ** 31):
        out = torch.zeros_like(q)
        run_attention(G, q, out, c, ints([0, new]), ints([60]), ints([[2, bad, 5, 1]]), 0.1)
        torch.cuda.synchronize()
        k, v = c.get([2, 0, 5, 1], 60)
        k[16:32], v[16:32] = 0, 0
        ref, bound = attention_ref(q, k, v, 60 - new, 0.1, weight_half=half)
        near(out, ref, bound, f"block {bad}")
    out = torch.zeros_like(q)  # 100 keys, two blocks in the row: the rows still stand at positions up to 99
    run_attention(G, q, out, c, ints([0, new]), ints([100]), ints([[2, 7]]), 0.1)
    torch.cuda.synchronize()
    k, v = c.get([2, 7], 32)
    ref, bound = attention_ref(q, k, v, 100 - new, 0.1, weight_half=half)
    near(out, ref, bound, "short table row")
    out = torch.zeros_like(q)
    run_attention(G, q, out, c, ints([-5, new + 1000, 3]), ints([60, -3]), ints([[2, 6, 5, 1], [0, 0, 0, 0]]), 0.1,
                  max_new=new, max_kv=60)
    torch.cuda.synchronize()
    k, v = c.get([2, 6, 5, 1], 60)
    ref, bound = attention_ref(q, k, v, 60 - new, 0.1, weight_half=half)
    near(out, ref, bound, "row counts")


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_size_of_scores(cuda, G, new, q_type, cache_type):
    """Queries far from 1 (scores of +-10^4, of 10^-8, a row of zeros): the maximum is taken off before the
    exponential, and F32 queries keep their precision at any size."""
    g = gen(3)
    c = Cache(G, 10, 1, 16, 64, cache_type)
    ids = list(range(9))
    c.put(ids, normal(g, 130, 1, 64), normal(g, 130, 1, 64))
    for size in (3000.0, 1e-6, 0.0) + ((1e6, 1e-30) if q_type == F32 else ()):
        q = (normal(g, new, 4, 64) * size).to(q_type)
        out = torch.zeros_like(q)
        run_attention(G, q, out, c, ints([0, new]), ints([130]), ints([ids]), 0.125)
        torch.cuda.synchronize()
        k, v = c.get(ids, 130)
        ref, bound = attention_ref(q, k, v, 130 - new, 0.125, weight_half=0.0 if q_type == F32 else HALF[cache_type])
        bound = torch.where(bound > 1, math.inf, bound) if size > 1e5 else bound  # scores known to 10^-2 at best
        near(out, ref, torch.nan_to_num(bound, posinf=100.0), f"size {size}")


@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_scale_not_positive(cuda, G, new, scale, q_type, cache_type):
    g = gen(7)
    c = Cache(G, 10, 2, 16, 128, cache_type)
    ids = list(range(9))
    c.put(ids, normal(g, 140, 2, 128), normal(g, 140, 2, 128))
    q = normal(g, new, 4, 128).to(q_type)
    out = torch.zeros_like(q)
    run_attention(G, q, out, c, ints([0, new]), ints([140]), ints([ids]), scale)
    torch.cuda.synchronize()
    k, v = c.get(ids, 140)
    ref, bound = attention_ref(q, k, v, 140 - new, scale, weight_half=0.0 if q_type == F32 else HALF[cache_type])
    near(out, ref, bound, f"scale {scale}")


@pytest.mark.parametrize("max_kv", [200, 100000])
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_nan_stays_in_its_request(cuda, G, new, max_kv, q_type, cache_type):
    """A NaN key or query makes the rows that see it NaN, and no row of another request."""
    g = gen(8)
    lens = [150, 150, 150, 33]
    lists, table, blocks = spread_tables(lens, 16, seed=3)
    c = Cache(G, blocks, 2, 16, 64, cache_type)
    for n, ids in zip(lens, lists):
        c.put(ids, normal(g, n, 2, 64), normal(g, n, 2, 64))
    at = 150 - new // 2 - 1  # request 0: a key that half of the rows see
    c.k[lists[0][at // 16], 0, at % 16, 5] = math.nan
    c.k[lists[3][:1], :] = math.nan  # request 3: its first 16 keys
    n3 = min(new, 33)
    cu = ints([0, new, 2 * new, 3 * new, 3 * new + n3])
    q = normal(g, 3 * new + n3, 6, 64).to(q_type)
    q[2 * new] = math.nan  # request 2: its first row
    out = torch.zeros_like(q)
    run_attention(G, q, out, c, cu, ints(lens), table, 0.125, max_kv=max_kv)
    torch.cuda.synchronize()
    first = at - (150 - new)
    assert out[max(first, 0): new, :3].isnan().all() and not out[: max(first, 0), :3].isnan().any()
    assert not out[:new, 3:].isnan().any()
    assert out[2 * new].isnan().all() and not out[2 * new + 1: 3 * new].isnan().any()
    assert out[3 * new:].isnan().all()
    k, v = c.get(lists[1], 150)
    ref, bound = attention_ref(q[new: 2 * new], k, v, 150 - new, 0.125,
                               weight_half=0.0 if q_type == F32 else HALF[cache_type])
    near(out[new: 2 * new], ref, bound, "request 1")


@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_largest_hints(cuda, G, q_type, cache_type):
    """Hints at the ends of their range choose a work split, nothing else."""
    for hints in (dict(max_new=2 ** 31 - 1, max_kv=2 ** 31 - 1), dict(max_new=0, max_kv=2 ** 31 - 1),
                  dict(max_new=2 ** 31 - 1, max_kv=0)):
        check_attention(G, [(90, 1), (200, 20), (64, 64)], 8, 2, 64, q_type, cache_type, 32, seed=9, **hints)


def test_paged_attention_many_requests(cuda, G):
    """More requests than any kernel has threads."""
    lens = [(1 + (i * 37) % 70, 1) for i in range(700)]
    check_attention(G, lens, 4, 2, 64, F16, F16, 16, seed=13)
    check_attention(G, lens[:400] + [(300, 90)], 4, 2, 64, BF16, BF16, 16, seed=14)
    check_attention(G, lens[:400] + [(300, 90)], 4, 2, 64, F32, F16, 16, seed=15)


@pytest.mark.parametrize("new", [1, 3, 70])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_graph_replay(cuda, G, new, q_type, cache_type):
    """A captured call serves other lengths, tables and values on replay, beside another call on another stream."""
    g = gen(4)
    bs, KH, H, D, B = 16, 2, 16, 128, 3
    width = 40
    c = Cache(G, B * width, KH, bs, D, cache_type)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(0)).reshape(B, width)
    for b in range(B):
        c.put(table[b].tolist(), normal(g, bs * width, KH, D), normal(g, bs * width, KH, D))
    q = normal(g, B * new, H, D).to(q_type)
    out, other = torch.zeros_like(q), torch.zeros_like(q)
    cu, kv, dev_table = ints([i * new for i in range(B + 1)]), ints([new] * B), table.to(torch.int32).cuda()
    args = dict(max_new=new, max_kv=bs * width)
    keep = run_attention(G, q, out, c, cu, kv, dev_table, 0.09, call=False, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            G.check(G.lib().b200_paged_attention(C.byref(keep[0]), C.byref(c.rec), side.cuda_stream), "capture")
    half = 0.0 if q_type == F32 else HALF[cache_type]
    for lens in ([new, 77, 640], [500, new + 1, 16], [640, 640, 640]):
        kv.copy_(ints(lens))
        q.copy_(normal(g, B * new, H, D))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        run_attention(G, q, other, c, cu, kv, dev_table, 0.09, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, other)
        for b, n in enumerate(lens):
            k, v = c.get(table[b].tolist(), n)
            ref, bound = attention_ref(q[b * new: (b + 1) * new], k, v, n - new, 0.09, weight_half=half)
            near(out[b * new: (b + 1) * new], ref, bound, f"replay {lens}")


# -------------------------------------------------------------------------------------------------- a run of all three
@pytest.mark.parametrize("src,cache_type", [(F32, F16), (F32, BF16), (BF16, BF16)])
def test_decode_steps(cuda, G, src, cache_type):
    """Prompt chunks, then mixed and single-token steps of three requests: plan, rotation and cache write, attention,
    against 64-bit attention over each request's whole history."""
    g = gen(6)
    H, KH, D, bs, B, width = 8, 2, 64, 16, 3, 16
    c = Cache(G, B * width + 2, KH, bs, D, cache_type)
    state = dict(cached=ints([0] * B), table=torch.full((B, width), -1, dtype=torch.int32, device="cuda"),
                 free=torch.randperm(B * width + 2, generator=torch.Generator().manual_seed(9)).to(torch.int32).cuda(),
                 head=ints([0]))
    history = [[] for _ in range(B)]
    qw, kw = 1 + 0.3 * normal(g, D), 1 + 0.3 * normal(g, D)
    for new in ([37, 1, 90], [1, 16, 1], [1, 1, 1], [0, 1, 5], [1, 1, 1]):
        T = sum(new) + 3  # padded rows, as a captured step has them
        cu, pos, slots, status = ints([0] * (B + 1)), ints([0] * T), ints([0] * T, torch.int64), ints([-1])
        plan = G.KvPlan(n_seqs=B, block_size=bs, cached_lens=ptr(state["cached"]), new_lens=ptr(new_d := ints(new)),
                        block_table=ptr(state["table"]), table_width=width, free_blocks=ptr(state["free"]),
                        n_free=state["free"].numel(), free_head=ptr(state["head"]), free_head_out=ptr(state["head"]),
                        cu_new=ptr(cu), kv_lens=ptr(state["cached"]), positions=ptr(pos), slots=ptr(slots),
                        max_tokens=T, status=ptr(status))
        G.check(G.lib().b200_kv_plan(C.byref(plan), stream()), "kv_plan")
        qkv = (2 * normal(g, T, (H + 2 * KH) * D)).to(src)
        q, k, v = (s.unflatten(1, (-1, D)) for s in qkv.split([H * D, KH * D, KH * D], 1))
        row = qkv.stride(0) * qkv.element_size()
        turned = torch.empty((T, H, D), dtype=src, device="cuda")
        rope = G.QkNormRope(n_tokens=T, heads=H, in_type=type_id(G, src), out_type=type_id(G, src), n_rot=D, q=ptr(q),
                            k=ptr(k), v=ptr(v), nb_q=row, nb_k=row, nb_v=row, q_out=ptr(turned), q_norm=ptr(qw),
                            k_norm=ptr(kw), positions=ptr(pos), slots=ptr(slots), eps=1e-6, freq_base=1e4,
                            freq_scale=1.0, neox=1)
        G.check(G.lib().b200_qk_norm_rope(C.byref(rope), C.byref(c.rec), stream()), "qk_norm_rope")
        out = torch.full((T, H, D), 7.0, dtype=src, device="cuda")
        run_attention(G, turned, out, c, cu, state["cached"], state["table"], 0.125, max_new=max(new), max_kv=200)
        torch.cuda.synchronize()
        assert status.item() == 0
        at = 0
        for b, n in enumerate(new):
            rows = slice(at, at + n)
            history[b].append((k[rows].clone(), v[rows].clone()))
            ks, vs = (torch.cat([h[i] for h in history[b]]) for i in range(2))
            p0 = ks.shape[0] - n
            every = torch.arange(ks.shape[0], device="cuda")
            # keys as the cache holds them: a 16-bit value next to the 64-bit one counts as one more rounding of a score
            kr = rope_ref(ks, kw, every, D, True, 1e4, 1.0, None, 1e-6)[0].to(cache_type)
            qr = rope_ref(q[rows], qw, every[p0:], D, True, 1e4, 1.0, None, 1e-6)[0].to(src)
            half = HALF[cache_type] if src != F32 else 0.0
            ref, bound = attention_ref(qr, kr, vs.to(cache_type), p0, 0.125, weight_half=half)
            # a key that lies next to a border of its type may round the other way: a score off by one step of one
            # product, at most 2 HALF |q| |k| scale, on few keys; counted on all of them
            size = torch.einsum("nhd,khd->nhk", qr.double().abs(), kr.double().abs().repeat_interleave(H // KH, 1))
            slack = (2 * (HALF[cache_type] + HALF[src]) * 0.125 * size.amax()).item() if n else 0.0
            near(out[rows], ref, bound + slack * vs.double().abs().amax() * 0.02, f"step {new}, request {b}")
            at += n
        assert (out[at:] == 7.0).all()
