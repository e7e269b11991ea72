"""The paged KV cache operators at the ends of their ranges: softmax weights and queries far below a row's largest, the
largest caps, request counts next to a shared-memory limit, calls on several streams.  Bounds as in paged_helpers."""
from __future__ import annotations

import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

from paged_helpers import HALF, U, Cache, attention_ref, ints, run_attention
from test_paged_gpu import (BF16, F16, F32, TYPES, check_attention, gen, near, no_wait_ran_out,  # noqa: F401 (a fixture)
                            normal)

pytestmark = pytest.mark.gpu


def one_request(G, g, n, KH, D, bs, cache_type, keys=None, values=None):
    """A cache with one request of n keys: (cache, block table, keys, values)."""
    ids = torch.randperm(-(-n // bs), generator=torch.Generator().manual_seed(n)).tolist()
    c = Cache(G, len(ids), KH, bs, D, cache_type)
    c.put(ids, normal(g, n, KH, D) if keys is None else keys, normal(g, n, KH, D) if values is None else values)
    return c, ints([ids]), *c.get(ids, n)


def attend(G, q, c, table, n, scale, **opts):
    out = torch.full_like(q, 7.0)
    run_attention(G, q, out, c, ints([0, q.shape[0]]), ints([n]), table, scale, **opts)
    torch.cuda.synchronize()
    return out


# new tokens of one request, and the hint that chooses between its forms: joined in a cluster, joined from partials
# (of the stream kernel), and the kernels of many rows
FORMS = [(1, None), (1, 100000), (3, 100000), (90, None)]


@pytest.mark.parametrize("new,max_kv", FORMS)
@pytest.mark.parametrize("q_type,cache_type,nats", [(F32, F16, 17), (F32, F16, 22), (F32, BF16, 22), (F16, F16, 17),
                                                    (BF16, BF16, 22)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_paged_attention_tail_far_below_the_largest_key(cuda, G, D, q_type, cache_type, nats, new, max_kv):
    """One key in 32 (its value is 0) lies `nats` above all others, so that the output is made of weights of e^-nats.

    A weight is rounded relative to itself down to the smallest normal number of its pieces, and by an absolute amount
    below it, in units of the weight of the running maximum: F16 weights are held times 2^7 and end at 2^-24 (off by
    2^-25 / 2^7); of F32 queries the second piece is held times 2^11 more (off by 2^-25 / 2^18); BF16 pieces end where
    F32 does.  The row's sum is at least that of the weights relative to its largest."""
    g = gen(nats + D)
    n, scale = 2100, 0.125
    keys = normal(g, n, 2, D)
    keys[..., 0] = -8.0 * nats / 4.0
    keys[::32] = 0.0
    values = 1000.0 * (1.0 + 0.3 * normal(g, n, 2, D))
    values[::32] = 0.0
    c, table, k, v = one_request(G, g, n, 2, D, 16, cache_type, keys, values)
    q = 0.25 * math.sqrt(64 / D) * normal(g, new, 6, D)
    q[..., 0] = 4.0
    q = q.to(q_type)
    out = attend(G, q, c, table, n, scale, max_kv=max_kv)
    ref, bound = attention_ref(q, k, v, n - new, scale, weight_half=0.0 if q_type == F32 else HALF[cache_type])
    floor = {(F32, F16): 2.0 ** -43, (F16, F16): 2.0 ** -32}.get((q_type, cache_type), 0.0)
    top = n // 32 - new // 32  # keys whose weight is 1 that every row sees: a lower bound of its sum
    bound = bound + floor * v.double().abs().sum(0).repeat_interleave(3, 0)[None] / top
    assert (bound < 0.02 * ref.abs()).all()  # what is asked for can fail
    near(out, ref, bound, f"{nats} nats below")


@pytest.mark.parametrize("new,max_kv", FORMS)
@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -128, 1e-39, 1e-44])
def test_paged_attention_subnormal_queries(cuda, G, size, cache_type, new, max_kv):
    """F32 queries around and below the smallest normal number, zeros among them: scores of 0 but for a rounding, so
    the output is the mean of the values seen."""
    g = gen(21)
    n = 130
    c, table, k, v = one_request(G, g, n, 2, 64, 16, cache_type)
    q = torch.sign(normal(g, new, 6, 64)) * size
    q[..., ::3] = 0.0
    assert ((q != 0) & (q.abs() <= 2.0 ** -126)).any()
    out = attend(G, q, c, table, n, 0.125, max_kv=max_kv)
    ref, bound = attention_ref(q, k, v, n - new, 0.125)
    near(out, ref, bound, f"size {size}")


@pytest.mark.parametrize("new,max_kv", FORMS)
@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_paged_attention_small_queries_beside_a_large_one(cuda, G, D, cache_type, new, max_kv):
    """F32 queries of about 2^-15 of the row's largest value, where keys are about 10^4 and the largest value's key is
    0: the scores are made of the small ones, which carry their 22 bits all the same."""
    g = gen(22 + D)
    n = 300
    keys = 20000.0 * normal(g, n, 2, D).clamp(-3, 3)
    keys[..., 5] = 0.0
    c, table, k, v = one_request(G, g, n, 2, D, 32, cache_type, keys)
    q = 2.0 ** -15 * math.sqrt(64 / D) * normal(g, new, 6, D)
    q[..., 5] = 1.0
    out = attend(G, q, c, table, n, 0.5, max_kv=max_kv)
    ref, bound = attention_ref(q, k, v, n - new, 0.5)
    near(out, ref, bound, "small queries")


PLAN_IN_A_FRESH_PROCESS = """
import sys
import ggml_b200 as G
from test_paged_gpu import Plan, lens_of, plan_ref
B = int(sys.argv[1])
for most_new, most in ((1, 2000), (1, 1 << 30), (9, 1 << 30)):  # a CTA, 8 CTAs, 16 CTAs
    cached, new = lens_of(B, 40, most_new, B)
    while sum(new) > most:
        new = [x if i % 4 == 0 else 0 for i, x in enumerate(new)]
    p = Plan(G, cached, new, 16, 4, sum(new), sum(new), seed=2)
    ref = plan_ref(cached, new, p.rows, p.free_list, 0, 16, sum(new))
    p.run(G)
    assert p.status.item() == 0 and p.got() == ref, (B, most_new)
print("same plans")
"""


@pytest.mark.parametrize("B", [6079, 6144])
def test_kv_plan_first_call_next_to_the_shared_memory_limit(cuda, G, B):
    """Request counts whose sums fit 48 KB of shared memory alone, but not beside what a kernel declares, as the first
    call of a process."""
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join([here, os.path.join(here, os.pardir, "xdna.cpp_b200")])
    got = subprocess.run([sys.executable, "-c", PLAN_IN_A_FRESH_PROCESS, str(B)], capture_output=True, text=True,
                         env={**os.environ, "PYTHONPATH": path}, timeout=300)
    assert got.returncode == 0 and "same plans" in got.stdout, got.stderr[-2000:]


def test_paged_attention_error_waits_for_every_stream(cuda, G):
    """The status is that of all calls made before it, also of those still in work on a stream that the legacy stream
    does not wait for."""
    side, status = torch.cuda.Stream(), C.c_int(-1)
    g = gen(23)
    c, table, _, _ = one_request(G, g, 40, 2, 64, 16, F16)
    q = normal(g, 1, 4, 64)
    out, cu, kv = torch.empty_like(q), ints([0, 1]), ints([40])
    args, _workspace = run_attention(G, q, out, c, cu, kv, table, 0.125)
    G.check(G.lib().b200_paged_attention_error(C.byref(status)), "warm-up: what is loaded at its first use")
    ran = torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # about 0.2 s
        G.check(G.lib().b200_paged_attention(C.byref(args), C.byref(c.rec), side.cuda_stream), "paged_attention")
        ran.record()
    assert not ran.query()
    G.check(G.lib().b200_paged_attention_error(C.byref(status)), "paged_attention_error")
    assert ran.query() and status.value == 0


@pytest.mark.parametrize("new,max_kv", FORMS)
@pytest.mark.parametrize("q_type,cache_type", TYPES)
@pytest.mark.parametrize("cap", [50.0, 64.0, 65.0, 1e3, 1e4, 1e6])
def test_paged_attention_large_caps(cuda, G, cap, q_type, cache_type, new, max_kv):
    """A cap far above the scores changes them by less and less: no term of the error grows with the cap.

    tanh's argument and value, and their products, are off by a few roundings of the score itself (8 U counted); up to
    a cap of 64 the kernel of many rows takes tanh from an exponential instead, off by 2^-21 of the cap."""
    g = gen(24)
    n = 260
    c, table, k, v = one_request(G, g, n, 2, 64, 16, cache_type)
    q = (3 * normal(g, new, 6, 64)).to(q_type)
    out = attend(G, q, c, table, n, 0.125, max_kv=max_kv, cap=cap)
    half = 0.0 if q_type == F32 else HALF[cache_type]
    ref, _ = attention_ref(q, k, v, n - new, 0.125, cap=cap)
    _, bound = attention_ref(q, k, v, n - new, 0.125, weight_half=half)  # all but the cap's own error
    kk, vv = (x.double().repeat_interleave(3, 1) for x in (k, v))
    s = torch.einsum("nhd,khd->hnk", q.double(), kk) * 0.125
    seen = torch.arange(n, device="cuda")[None, :] <= torch.arange(n - new, n, device="cuda")[:, None]
    w = torch.softmax((cap * torch.tanh(s / cap)).masked_fill(~seen, -math.inf), -1)
    off = 8 * U * s.abs().amax() + (2.0 ** -21 * cap if cap <= 64 and new == 90 and q_type != F32 else 0.0)
    # a score off by d: a weight and the row's sum off by d each; the bound's own weights are those without the cap
    most = torch.einsum("hnk,khd->nhd", w, vv.abs())
    plain = torch.einsum("hnk,khd->nhd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), vv.abs())
    near(out, ref, bound * (most / plain).clamp(min=1) + 2 * off * most, f"cap {cap}")


def test_paged_decode_goes_on_after_a_refused_step(cuda, G):
    """A step that the cache has no room for leaves the length as it was: a shorter one still fits."""
    import decode_harness as D

    tiny = dict(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=64, inter=512, vocab=992, theta=1.0e6, eps=1.0e-6)
    att = D.DeviceAttention(cuda, tiny, 32)
    att.begin(20)
    with pytest.raises(RuntimeError, match="32 tokens"):
        att.begin(13)
    att.begin(12)
    torch.cuda.synchronize()
    assert att.status.item() == 0 and att.cached.item() == 32


@pytest.mark.parametrize("new,max_kv", FORMS)
@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("power", [20, 60, 100, -20, -60, -100])
def test_paged_attention_queries_of_any_power(cuda, G, power, cache_type, new, max_kv):
    """F32 queries times a power of two, with the scale divided by it, are the same scores: the normal bound holds, at
    10^30 and at 10^-30 too."""
    g = gen(25)
    n = 130
    c, table, k, v = one_request(G, g, n, 2, 64, 16, cache_type)
    q = 1.5 * normal(g, new, 6, 64)
    out = attend(G, q * 2.0 ** power, c, table, n, 0.125 * 2.0 ** -power, max_kv=max_kv)
    ref, bound = attention_ref(q, k, v, n - new, 0.125)
    near(out, ref, bound, f"2^{power}")


@pytest.mark.parametrize("lens", [[(4000, 1)], [(20000, 1), (300, 1)], [(3000, 400), (900, 1), (5000, 1)], [(2000, 700)]],
                         ids=str)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_repeats_itself(cuda, G, lens, D, q_type, cache_type):
    """The same call gives the same bits, whatever else the GPU does beside it."""
    g = gen(26)
    pages = [-(-n // 16) for n, _ in lens]
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32)
    cu, at = [0], 0
    for b, (_, m) in enumerate(lens):
        table[b, : pages[b]] = torch.arange(at, at + pages[b])
        at += pages[b]
        cu.append(cu[-1] + m)
    c = Cache(G, at, 4, 16, D, cache_type)
    c.k.copy_(normal(g, *c.k.shape))
    c.v.copy_(normal(g, *c.v.shape))
    q = (1.5 * normal(g, cu[-1], 16, D)).to(q_type)
    outs, table, cu, kv = [torch.empty_like(q) for _ in range(4)], table.cuda(), ints(cu), ints([n for n, _ in lens])
    hints, side, x = dict(max_new=max(m for _, m in lens), max_kv=max(n for n, _ in lens)), torch.cuda.Stream(), None
    for i, out in enumerate(outs):
        if i % 2:
            with torch.cuda.stream(side):
                x = torch.randn(2048, 2048, device="cuda") @ torch.randn(2048, 2048, device="cuda")
        run_attention(G, q, out, c, cu, kv, table, 0.09, **hints)
        torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:]) and x is not None


@pytest.mark.parametrize("q_type,cache_type", TYPES)
@pytest.mark.parametrize("new", [1, 12, 200])
def test_paged_attention_two_calls_at_once(cuda, G, new, q_type, cache_type):
    """Two calls on two streams, each with a workspace of its own, in work at the same time."""
    g = gen(27)
    n, sides = 3000, [torch.cuda.Stream(), torch.cuda.Stream()]
    c, table, k, v = one_request(G, g, n, 2, 128, 16, cache_type)
    calls = []
    for side in sides:
        q = normal(g, new, 16, 128).to(q_type)
        out, cu, kv = torch.zeros_like(q), ints([0, new]), ints([n])
        calls.append((q, out, cu, kv, run_attention(G, q, out, c, cu, kv, table, 0.09, max_kv=100000, call=False)))
    torch.cuda.synchronize()
    for _ in range(5):
        for side, (_, _, _, _, (args, _)) in zip(sides, calls):
            G.check(G.lib().b200_paged_attention(C.byref(args), C.byref(c.rec), side.cuda_stream), "paged_attention")
    torch.cuda.synchronize()
    for q, out, *_ in calls:
        ref, bound = attention_ref(q, k, v, n - new, 0.09, weight_half=0.0 if q_type == F32 else HALF[cache_type])
        near(out, ref, bound, "two streams")


@pytest.mark.parametrize("q_type,cache_type", TYPES)
@pytest.mark.parametrize("H,KH", [(300, 1), (40, 40)])
def test_paged_attention_many_heads(cuda, G, H, KH, q_type, cache_type):
    check_attention(G, [(100, 1), (33, 2), (257, 20)], H, KH, 64, q_type, cache_type, 32, seed=H)


@pytest.mark.parametrize("new,max_kv", FORMS)
@pytest.mark.parametrize("q_type,cache_type", TYPES)
def test_paged_attention_window_behind_the_table_row(cuda, G, q_type, cache_type, new, max_kv):
    """Keys behind a table row do not exist: rows whose window lies behind it all see none and are 0."""
    g = gen(28)
    c, _, _, _ = one_request(G, g, 32, 2, 64, 16, cache_type)
    q = normal(g, new, 6, 64).to(q_type)
    for table in (ints([[1, 0]]), torch.empty((1, 0), dtype=torch.int32, device="cuda")):
        out = torch.full_like(q, 7.0)
        run_attention(G, q, out, c, ints([0, new]), ints([400]), table, 0.125, window=10, max_kv=max_kv)
        torch.cuda.synchronize()
        assert (out == 0).all()
