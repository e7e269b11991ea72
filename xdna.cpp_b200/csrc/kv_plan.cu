// The plan of a step over a paged KV cache: block tables, cache slots and
// positions of every request's new tokens, from the request lengths.
//
// Mathematics: with owned_b = ceil(cached_b / bs) and need_b =
// ceil((cached_b + new_b) / bs) - owned_b, the exclusive prefix sums of new
// and need give each request its first token and its first free-list entry.
// Token t of request b has position pos = cached_b + t - cu_b and lies in the
// request's block pos / bs: a block the request owns (read from its table
// row), or free[head + first_b + pos / bs - owned_b].
//
// The work is a few bytes per token, so the call is bound by latency: one
// launch, in which every CTA forms the prefix sums of all requests for itself
// (8 bytes a request, from L2) and then takes its share of the tokens.  The
// CTAs form one cluster: its barrier stands between the last read of the
// lengths and the head and the first write to them, so both may be updated in
// place, and no counter in memory has to be kept.
#include <cuda_runtime.h>

#include "gemv.cuh"
#include "paged.cuh"

namespace xb {
namespace {

constexpr int kThreads = 1024;
constexpr int kCluster = 8, kWide = 16;  // CTAs (16: more than the portable size, which every B200 has)
constexpr int kOneCtaTokens = 2048;  // up to here one CTA takes the tokens in two rounds
// Up to here 8 CTAs whose lanes take one token at a time (two rounds), beyond 16
// whose lanes take four: 83000 tokens of 1024 requests took 20 us with 8 CTAs and
// one token, 13.3 us with four, 9.7 us with 16 CTAs and four.
constexpr int kShortTokens = 16384;

struct Sum {
    long long tokens, blocks;
};

__device__ __forceinline__ Sum warp_inclusive(Sum v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, v.tokens, d);
        const long long n = __shfl_up_sync(0xffffffffu, v.blocks, d);
        if (lane >= d) {
            v.tokens += t;
            v.blocks += n;
        }
    }
    return v;
}

struct Lens {
    int cached, fresh;
    bool bad;
};

__device__ __forceinline__ Lens read_lens(const struct b200_kv_plan_args& p, int b) {
    const int c = p.cached_lens[b], n = p.new_lens[b];
    Lens l{c, n, false};
    if (c < 0 || n < 0 || static_cast<long long>(c) + n > 0x7fffffffLL) l = Lens{c < 0 ? 0 : c, 0, true};
    return l;
}

// kEach: tokens a lane has in work at once.
template <int kCtas, int kEach>
__global__ void __launch_bounds__(kThreads) kv_plan_kernel(const __grid_constant__ struct b200_kv_plan_args p, int log_bs) {
    // Held to 32 bits: sums past max_tokens or 2^31 - 1 blocks are cut there, and
    // no token that is written lies behind a cut (the status says so).
    extern __shared__ int prefix[];  // [n_seqs] first token, then [n_seqs] first free-list entry
    int* first_token = prefix;
    int* first_block = prefix + p.n_seqs;
    __shared__ Sum warp_sum[32];
    __shared__ int flags;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = static_cast<int>(blockIdx.x);
    const int B = p.n_seqs, bs = 1 << log_bs;
    if (tid == 0) flags = 0;
    grid_wait();
    __syncthreads();

    // prefix sums: a thread owns `per` consecutive requests
    const int per = (B + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    const int head = p.free_head ? *p.free_head : 0;
    Sum mine{0, 0};
    int bad = 0;
    for (int b = b0; b < b1; ++b) {
        const Lens l = read_lens(p, b);
        const long long owned = (static_cast<long long>(l.cached) + bs - 1) >> log_bs;
        const long long held = (static_cast<long long>(l.cached) + l.fresh + bs - 1) >> log_bs;
        if (l.bad) bad |= B200_KV_BAD_LENGTH;
        if (held > p.table_width) bad |= B200_KV_ROW_TOO_SHORT;
        mine.tokens += l.fresh;
        mine.blocks += held - owned;
    }
    const Sum inc = warp_inclusive(mine);
    if (lane == 31) warp_sum[warp] = inc;
    if (bad) atomicOr(&flags, bad);
    __syncthreads();
    if (warp == 0) warp_sum[lane] = warp_inclusive(warp_sum[lane]);
    __syncthreads();
    const Sum before = warp ? warp_sum[warp - 1] : Sum{0, 0};
    const Sum all = warp_sum[31];
    Sum run{before.tokens + inc.tokens - mine.tokens, before.blocks + inc.blocks - mine.blocks};
    for (int b = b0; b < b1; ++b) {
        const Lens l = read_lens(p, b);
        first_token[b] = static_cast<int>(run.tokens < p.max_tokens ? run.tokens : p.max_tokens);
        first_block[b] = static_cast<int>(run.blocks < 0x7fffffffLL ? run.blocks : 0x7fffffffLL);
        run.tokens += l.fresh;
        run.blocks += ((static_cast<long long>(l.cached) + l.fresh + bs - 1) >> log_bs) -
                      ((static_cast<long long>(l.cached) + bs - 1) >> log_bs);
    }
    if (tid == 0) {
        int f = flags;
        if (head < 0 || head + all.blocks > p.n_free) f |= B200_KV_NO_FREE_BLOCK;
        if (all.tokens > p.max_tokens) f |= B200_KV_TOO_MANY_TOKENS;
        if (rank == 0) *p.status = f;
    }
    __syncthreads();

    // the tokens of this CTA (cached_lens is read here for the last time): a warp
    // takes 32 kEach consecutive ones, a lane every 32nd of them, in step.  The
    // requests of the first and the last are searched for by two lanes at once, the
    // others between them.
    const int most = static_cast<int>(p.max_tokens), total = static_cast<int>(all.tokens < most ? all.tokens : most);
    const int width = static_cast<int>(p.table_width), free_left = static_cast<int>(p.n_free) - max(head, 0);
    constexpr int kSpan = 32 * kEach;
    for (long long s0 = (static_cast<long long>(warp) * kCtas + rank) * kSpan; s0 < most;
         s0 += static_cast<long long>(kCtas) * (kThreads / 32) * kSpan) {
        int lo[kEach], hi[kEach], cached[kEach], block[kEach];
        const int t0 = static_cast<int>(s0) + lane, there = min(most - static_cast<int>(s0), kSpan);
        if (kEach == 1) {
            lo[0] = 0, hi[0] = B;
            if (lane < there && t0 < total)
                while (hi[0] - lo[0] > 1) {  // the last request whose first token is at or before the token
                    const int mid = (lo[0] + hi[0]) >> 1;
                    if (first_token[mid] <= t0) lo[0] = mid; else hi[0] = mid;
                }
        } else {
            int from = 0, to = B;
            if (s0 < total) {
                const int t = lane ? min(static_cast<int>(s0) + there, total) - 1 : static_cast<int>(s0);
                while (to - from > 1) {
                    const int mid = (from + to) >> 1;
                    if (first_token[mid] <= t) from = mid; else to = mid;
                }
            }
            const int lowest = __shfl_sync(0xffffffffu, from, 0), highest = __shfl_sync(0xffffffffu, from, 1) + 1;
#pragma unroll
            for (int i = 0; i < kEach; ++i) lo[i] = lowest, hi[i] = highest;
            for (int n = highest - lowest; n > 1; n = (n + 1) >> 1)
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int mid = (lo[i] + hi[i]) >> 1;
                    if (mid > lo[i]) {
                        if (first_token[mid] <= t0 + i * 32) lo[i] = mid; else hi[i] = mid;
                    }
                }
        }
        // token i of the lane exists: i * 32 + lane < there; it is a request's: t < total
        auto real = [&](int i) { return i * 32 + lane < there && t0 + i * 32 < total; };
#pragma unroll
        for (int i = 0; i < kEach; ++i) cached[i] = real(i) ? max(p.cached_lens[lo[i]], 0) : 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            block[i] = -1;
            if (!real(i)) continue;
            const int pos = cached[i] + (t0 + i * 32 - first_token[lo[i]]), page = pos >> log_bs;
            const int owned = static_cast<int>((static_cast<unsigned>(cached[i]) + bs - 1) >> log_bs);
            if (page >= width) continue;
            if (page < owned) {
                block[i] = p.block_table[static_cast<long long>(lo[i]) * width + page];
            } else if (head >= 0) {
                const unsigned x = static_cast<unsigned>(first_block[lo[i]]) + static_cast<unsigned>(page - owned);
                if (free_left > 0 && x < static_cast<unsigned>(free_left)) block[i] = p.free_blocks[head + x];
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i * 32 + lane >= there) continue;
            const int t = t0 + i * 32, pos = real(i) ? cached[i] + (t - first_token[lo[i]]) : 0;
            // a new block's first token is new, and its thread alone writes the entry
            if (block[i] >= 0 && (pos & (bs - 1)) == 0)
                p.block_table[static_cast<long long>(lo[i]) * width + (pos >> log_bs)] = block[i];
            if (p.positions) p.positions[t] = pos;
            p.slots[t] = block[i] < 0 ? -1 : static_cast<int64_t>(block[i]) * bs + (pos & (bs - 1));
        }
    }

    // every CTA has read the lengths and the head: now they may be overwritten
    if (kCtas > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    if (rank == 0) {
        for (int b = tid; b <= B; b += kThreads) {
            p.cu_new[b] = b < B ? first_token[b] : static_cast<int32_t>(total);
            if (b < B) {
                const Lens l = read_lens(p, b);
                p.kv_lens[b] = l.cached + l.fresh;
            }
        }
        if (tid == 0 && p.free_head_out) {
            const long long h = head + all.blocks;
            *p.free_head_out = static_cast<int32_t>(head < 0 ? head : h < p.n_free ? h : p.n_free);
        }
    }
}

template <int kCtas, int kEach>
cudaError_t launch_ctas(const struct b200_kv_plan_args& p, cudaStream_t stream) {
    constexpr auto kernel = kv_plan_kernel<kCtas, kEach>;
    int log_bs = 4;
    while ((1 << log_bs) < p.block_size) ++log_bs;
    if (kCtas == kWide) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    // Without the attribute a kernel has 48 KB, of which its static shared memory is
    // part.  It is set to the most any call needs: calls at once need one limit.
    constexpr int kEachSeq = 2 * sizeof(int), kAlways = 32 * 1024;
    const size_t smem = static_cast<size_t>(p.n_seqs) * kEachSeq;
    if (smem > kAlways) {
        const cudaError_t e = allow_smem<kernel>(kMaxSeqs * kEachSeq);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kernel, dim3(kCtas), dim3(kThreads), smem, stream, kCtas, p, log_bs);
}

}  // namespace

cudaError_t kv_plan_launch(const struct b200_kv_plan_args& p, cudaStream_t stream) {
    if (p.max_tokens <= kOneCtaTokens) return launch_ctas<1, 1>(p, stream);
    if (p.max_tokens <= kShortTokens) return launch_ctas<kCluster, 1>(p, stream);
    return launch_ctas<kWide, 4>(p, stream);
}

}  // namespace xb
