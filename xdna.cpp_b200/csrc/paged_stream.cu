// Causal attention over a paged KV cache for requests with few rows (decode):
// every warp streams keys and values of its own.
//
// Mathematics as in paged_attention.cu.  With few rows the pass is bound by
// reading K and V once from HBM, so it is cut along the keys: a request's rows
// of one KV head (new tokens x group, R = 8 NT at a time) are an item, 32 keys
// of an item (16 at head_dim 256) a unit, and the units of all items, in order,
// are dealt out as one equal contiguous run to each of 4 streams per SM, whatever
// the lengths.  A stream is a warp that works and a warp that loads for it: TMA
// boxes, page by page, into a ring of 48 KB (with warps that issue their own loads
// one token over 1001 keys took 0.9 us more).  No stream waits for another one.  An
// item that ends in another stream than it began in leaves a partial (m, l, o) in the workspace for each
// stream; combine_kernel joins them in stream order, so results do not depend on
// timing.  Where there are few items with few keys, a cluster takes each instead
// and joins its sums in shared memory (kJoin).
//
// The products run transposed, S^T = K q^T and O^T = V^T P^T, with keys (then
// dimensions of V) as the 16 rows of mma.m16n8k16 and the item's rows as its 8
// columns: with up to 8 query heads a KV head nothing is multiplied in vain.  The
// rate of the fifth-generation tensor cores would not help: a unit's products take
// about a fifth of the time its bytes take.
// With 16-bit queries the weights are rounded to the cache's type, as the chunk
// kernel has to: BF16 outputs are off by 2.3e-3 of their size against 1.7e-3 for a
// 32-bit form rounded once (F16 2.9e-4 against 2.1e-4).  A second piece of every
// weight costs 1 to 1.5 % with 8 rows an item and 5 to 10 % with 32.
// The running maximum is moved only when a score passes it by 8 (a weight then
// is at most 2^8; what F16 makes of small ones: Half16), which a vote finds out;
// moving it takes the shuffles.
//
// Measured on a B200: one request of 130001 BF16 keys, 64 query and 8 KV heads of
// 128: 93 us, 5.7 TB/s of K and V; 64 requests of up to 8193 F16 keys with F32
// queries: 111 us, 5.5 TB/s; one token over 1001 keys: 7 us (joining form; 11 us
// with partials and a second launch).
#include <algorithm>

#include "paged_split.cuh"
#include "paged_tma.cuh"

namespace xb {
namespace {

constexpr float kSlack = 8.f;    // log2 of the largest weight (before kWeightLog2)
constexpr int kCluster = 8;      // CTAs that share an item of the joining form
// Keys up to which the joining form is taken: it uses 8 SMs an item.  2, 8 KV
// heads: 6.9, 6.9 us at 1024 keys, 12.5, 12.8 us at 8192, against 10.7, 11.9 us and
// 20, 19 us with partials; at 32768 about 33 us against 24 and 36 us.
constexpr int kJoinKeys = 16384;

// A unit is kKeys keys of an item: K and V in kHalves blocks of 64 values a row,
// each row 128 swizzled bytes.
template <int D>
struct Ring {
    static constexpr int kKeys = D > 128 ? 16 : 32;
    static constexpr int kWarps = 4;  // streams; as many warps more load for them
    static constexpr int kThreads = kWarps * 64;
    static constexpr int kStages = D == 64 ? 6 : 3;
    static constexpr int kHalves = (D + 63) / 64;
    static constexpr int kBlock = kKeys * 128;         // bytes of 64 values of every key
    static constexpr int kStage = 2 * kHalves * kBlock;  // K, then V
    static constexpr int kWarpBytes = kStages * kStage;
    static constexpr int kBytes = kWarps * kWarpBytes + 1024;  // 1024: alignment
};

struct StreamArgs {
    SplitArgs g;
    CUtensorMap k, v;
    int box_tokens;  // tokens per TMA box: a block, or a unit of one
};

// Walks the units of a stream.
struct Cursor {
    int b, kvh, tile, unit;
    Request rq;
    Work w;

    template <int R, int kKeys>
    __device__ __forceinline__ void enter(const AttnArgs& a) {
        rq = read_request(a, b);
        w = request_work<kKeys>(a, rq, R);
    }
    // The next unit (there is one).
    template <int R, int kKeys>
    __device__ __forceinline__ void next(const AttnArgs& a) {
        if (++unit < w.units) return;
        unit = 0;
        if (++tile < w.tiles) return;
        tile = 0;
        if (++kvh < a.kv.kv_heads) return;
        kvh = 0;
        do {
            ++b;
            enter<R, kKeys>(a);
        } while (!w.rows);
    }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Joins the partials that the warps of a cluster hold in shared memory, one at
// the start of each warp's ring, and writes the item's rows: first the warps of
// each CTA, then the CTAs' sums over distributed shared memory (rank r writes the
// rows r, r + kCluster, ...).
template <int D, int R, int kThreads, int kWarps, int kRingBytes>
__device__ __forceinline__ void cluster_join(const AttnArgs& a, const Request& rq, int kvh, int tile, int rows,
                                             uint8_t* smem) {
    constexpr int kEach = R * D / kThreads;
    const int tid = threadIdx.x, rank = static_cast<int>(blockIdx.x) % kCluster;
    auto part = [&](int w) { return reinterpret_cast<float*>(smem + static_cast<size_t>(w) * kRingBytes); };
    __syncthreads();
    float o[kEach], top[kEach], sum[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int x = i * kThreads + tid, r = x / D;
        top[i] = -INFINITY, sum[i] = 0.f, o[i] = 0.f;
        if (r >= rows) continue;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top[i] = fmaxf(top[i], part(w)[R * D + r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float m = part(w)[R * D + r];
            if (part(w)[R * D + R + r] == 0.f) continue;  // no key seen; a warp without units wrote no sums
            const float c = top[i] == -INFINITY ? 1.f : exp2f(m - top[i]);
            sum[i] = fmaf(c, part(w)[R * D + R + r], sum[i]);
            o[i] = fmaf(c, part(w)[x], o[i]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int x = i * kThreads + tid, r = x / D;
        part(0)[x] = o[i];
        if (x % D == 0) part(0)[R * D + r] = top[i], part(0)[R * D + R + r] = sum[i];
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    uint32_t from[kCluster];
#pragma unroll
    for (int c = 0; c < kCluster; ++c)
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from[c]) : "r"(smem_addr(part(0))), "r"(c));
    auto get = [&](int c, int x) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(from[c] + 4 * x) : "memory");
        return v;
    };
    for (int x = tid; x < (R + kCluster - 1) / kCluster * D; x += kThreads) {
        const int r = rank + x / D * kCluster, col = x % D;
        if (r >= rows) continue;
        float m[kCluster], v[kCluster], l[kCluster], t = -INFINITY, all = 0.f, y = 0.f;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) m[c] = get(c, R * D + r), l[c] = get(c, R * D + R + r), v[c] = get(c, r * D + col);
#pragma unroll
        for (int c = 0; c < kCluster; ++c) t = fmaxf(t, m[c]);
        t = t == -INFINITY ? 0.f : t;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            const float f = exp2f(m[c] - t);
            all = fmaf(f, l[c], all);
            y = fmaf(f, v[c], y);
        }
        const int rr = tile * R + r, i = rr / a.group;
        store_one(a, rq.first + i, kvh * a.group + rr - i * a.group, col, all == 0.f ? 0.f : y / all);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // before the next item's copies
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // until here the sums stay
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// kJoin: a cluster of kCluster CTAs takes one item (and those g.tiles row tiles
// further on), its warps equal runs of the item's units, and joins them in shared
// memory: one launch and no workspace, for few items with few keys.
template <typename T, int D, int NP, int NT, bool kJoin>
__global__ void __launch_bounds__(Ring<D>::kThreads, 1) attn_stream_kernel(const __grid_constant__ StreamArgs c) {
    using L = Ring<D>;
    constexpr int R = 8 * NT, kThreads = L::kThreads, kSteps = D / 16, kKeys = L::kKeys;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[L::kWarps][L::kStages], empty[L::kWarps][L::kStages];
    __shared__ int dead_word;
    volatile int* dead = &dead_word;
    const SplitArgs& g = c.g;
    uint8_t* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    __shared__ long long before[kThreads + 1];  // units of the requests before each thread's
    __shared__ long long warp_units[kThreads / 32];
    const AttnArgs& a = g.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.p.n_seqs;
    const int own = warp % L::kWarps;  // the stream of this CTA that the warp loads for or works on
    const bool loads = warp >= L::kWarps;
    if (tid == 0) {
        dead_word = 0;
        for (int i = 0; i < L::kWarps * L::kStages; ++i) bar_init(&full[0][0] + i, 1), bar_init(&empty[0][0] + i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    grid_wait();
    __syncthreads();
    if (!kJoin) grid_release();  // combine_kernel may take its place on the SMs; it waits for this grid's end

    Cursor at;
    int left = 0;         // units to fetch
    long long item0 = 0;  // units before the item `at` is in
    long long me = 0, all = 0, streams = 0;
    if constexpr (kJoin) {
        const int item = static_cast<int>(blockIdx.x) / kCluster;
        at.kvh = item % a.kv.kv_heads;
        at.tile = item / a.kv.kv_heads % g.tiles;
        at.b = item / a.kv.kv_heads / g.tiles;
        at.enter<R, kKeys>(a);
    } else {
        // units of all requests, summed up over the threads
        const int per = (B + kThreads - 1) / kThreads;
        {
            long long mine = 0;
            for (int b = min(tid * per, B); b < min(tid * per + per, B); ++b) {
                const Work w = request_work<kKeys>(a, read_request(a, b), R);
                mine += static_cast<long long>(w.units) * w.tiles * a.kv.kv_heads;
            }
            long long inc = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const long long o = __shfl_up_sync(0xffffffffu, inc, d);
                if (lane >= d) inc += o;
            }
            if (lane == 31) warp_units[warp] = inc;
            __syncthreads();
            for (int w = 0; w < warp; ++w) inc += warp_units[w];
            before[tid + 1] = inc;
            if (tid == 0) before[0] = 0;
            __syncthreads();
        }
        all = before[kThreads];
        streams = min(static_cast<long long>(g.streams), max(1LL, all));
        // neighbouring streams lie on different SMs: a short run of units uses all of them
        me = static_cast<long long>(own) * gridDim.x + blockIdx.x;
        if (lane == 0 && !loads && me < g.streams) g.heads[me].parts = 0;
        if (me >= streams || all == 0) return;
        const long long u0 = all * me / streams, u1 = all * (me + 1) / streams;
        left = static_cast<int>(u1 - u0);

        // the first unit
        {
            int lo = 0, hi = kThreads;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (before[mid] <= u0) lo = mid; else hi = mid;
            }
            long long u = before[lo];
            at.b = lo * per;
            at.enter<R, kKeys>(a);
            for (;;) {
                const long long n = static_cast<long long>(at.w.units) * at.w.tiles * a.kv.kv_heads;
                if (u0 < u + n) break;
                u += n;
                ++at.b;
                at.enter<R, kKeys>(a);
            }
            const long long item = (u0 - u) / at.w.units;
            at.unit = static_cast<int>(u0 - u - item * at.w.units);
            at.kvh = static_cast<int>(item / at.w.tiles);
            at.tile = static_cast<int>(item - static_cast<long long>(at.kvh) * at.w.tiles);
            item0 = u0 - at.unit;
        }
    }
    const uint32_t ring = smem_addr(smem) + own * L::kWarpBytes;
    uint32_t done = 0;  // units loaded, or worked off, by this warp
    for (; !kJoin || at.tile < at.w.tiles; at.tile += g.tiles) {
        if constexpr (kJoin) {
            const int n = at.w.units, i = own * kCluster + static_cast<int>(blockIdx.x) % kCluster;
            constexpr int kAll = kCluster * L::kWarps;
            at.unit = static_cast<int>(static_cast<long long>(n) * i / kAll);
            left = static_cast<int>(static_cast<long long>(n) * (i + 1) / kAll) - at.unit;
        }
        bool fresh = true;  // no unit of the item worked off yet

        // ------------------------------------------------------------------- loads
        if (loads) {
            const int boxes = kKeys / c.box_tokens;  // lane i < boxes loads box i of a unit
            // the table entry of a box's block, not looked at before the unit is loaded
            auto block_of = [&](const Cursor& f) {
                const int j = f.w.lo + f.unit * kKeys + lane * c.box_tokens, page = j >> a.log_bs;
                return lane < boxes && j < f.w.hi ? __ldg(a.p.block_table + static_cast<int64_t>(f.b) * a.p.table_width + page)
                                                  : 0;
            };
            Cursor fetch = at;
            int id = block_of(fetch);
            bool ok = true;
            for (int todo = left; todo > 0; ++done) {
                const int j = fetch.w.lo + fetch.unit * kKeys + lane * c.box_tokens, kvh = fetch.kvh;
                const bool on = lane < boxes && j < fetch.w.hi;
                // a block outside the cache: behind the last one, zeros
                const int block = id >= 0 && id < a.kv.num_blocks ? id : static_cast<int>(a.kv.num_blocks);
                if (--todo > 0) {
                    fetch.next<R, kKeys>(a);
                    id = block_of(fetch);
                }
                const uint32_t stage = done % L::kStages;
                if (done >= L::kStages) ok = bar_wait(&empty[own][stage], ((done / L::kStages) & 1) ^ 1, dead);
                if (!ok) break;
                uint64_t* bar = &full[own][stage];
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, on)) * c.box_tokens * 128 * 2 * L::kHalves;
                if (lane == 0) bar_expect(bar, bytes);
                __syncwarp();
                if (on) {
                    const uint32_t to = ring + stage * L::kStage + lane * c.box_tokens * 128;
#pragma unroll
                    for (int h = 0; h < L::kHalves; ++h)
                        tma_box(to + h * L::kBlock, &c.k, bar, h * 64, j & (a.kv.block_size - 1), kvh, block);
#pragma unroll
                    for (int h = 0; h < L::kHalves; ++h)
                        tma_box(to + (L::kHalves + h) * L::kBlock, &c.v, bar, h * 64, j & (a.kv.block_size - 1), kvh, block);
                }
                __syncwarp();
            }
            // Copies in flight land before the CTA ends, also where the warp that they are
            // for has given up.
            for (uint32_t i = done < L::kStages ? 0 : done - L::kStages; i < done; ++i)
                bar_wait(&full[own][i % L::kStages], (i / L::kStages) & 1, nullptr);
            if constexpr (!kJoin) return;
        }

        // Addresses of this lane's matrix rows: 16-byte column x of row r lies at
        // column x ^ (r & 7) of it.
        uint32_t k_at[4], v_at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k_at[i] = (lane & 15) * 128 + (((2 * i + (lane >> 4)) ^ (lane & 7)) << 4);
            v_at[i] = ((lane & 7) + ((lane >> 4) & 1) * 8) * 128 + (((2 * i + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
        }
        uint32_t qf[NP][NT][kSteps][2];
        float o[NT][kSteps][4], m[NT][2], l[NT][2], mul[NT][2], slope[NT][2];
        int pos[NT][2];
        int rows = 0, all_lo = 0, all_hi = 0;  // keys [all_lo, all_hi) are seen by every row

        bool begun_here = at.unit == 0, ok = true;
        int todo = loads ? 0 : left;  // units to work off
        while (todo > 0) {
            if (fresh) {  // a new item: its queries, and nothing seen yet
                fresh = false;
                const int G = a.group, r0 = at.tile * R;
                rows = min(R, at.w.rows - r0);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int r = nt * 8 + (lane >> 2);
                    const bool on = r < rows;
                    const int i = (r0 + r) / G, h = at.kvh * G + (r0 + r) - i * G;
                    const char* src = static_cast<const char*>(a.p.q) + (at.rq.first + (on ? i : 0)) * a.p.nb_q;
                    float up = 1.f;
                    if constexpr (NP == 1) {
                        const uint32_t* s = reinterpret_cast<const uint32_t*>(src) + static_cast<int64_t>(h) * (D / 2) + (lane & 3);
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            qf[0][nt][k][0] = on ? __ldg(s + k * 8) : 0u;
                            qf[0][nt][k][1] = on ? __ldg(s + k * 8 + 4) : 0u;
                        }
                    } else {
                        const float2* s = reinterpret_cast<const float2*>(src) + static_cast<int64_t>(h) * (D / 2) + (lane & 3);
                        float2 x[kSteps][2];
                        float big = 0.f;
#pragma unroll
                        for (int k = 0; k < kSteps; ++k)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                x[k][e] = on ? __ldg(s + k * 8 + e * 4) : make_float2(0.f, 0.f);
                                big = fmaxf(big, fmaxf(fabsf(x[k][e].x), fabsf(x[k][e].y)));
                            }
                        if (NP == 2) {  // 4 lanes hold a row
                            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                            up = row_power(big);
                        }
                        const float down = 1.f / up;
#pragma unroll
                        for (int k = 0; k < kSteps; ++k)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                uint32_t piece[NP];
                                split_pair<T, NP>(x[k][e].x * down, x[k][e].y * down, piece);
#pragma unroll
                                for (int c = 0; c < NP; ++c) qf[c][nt][k][e] = piece[c];
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {  // this lane's columns of S^T
                        const int col = 2 * (lane & 3) + e, rr = r0 + nt * 8 + col, it = rr / G;
                        mul[nt][e] = a.pre * __shfl_sync(0xffffffffu, up, col * 4);
                        slope[nt][e] = head_slope(a, at.kvh * G + rr - it * G);
                        pos[nt][e] = at.rq.pos0() + it;
                        m[nt][e] = -INFINITY;
                        l[nt][e] = 0.f;
                    }
#pragma unroll
                    for (int n = 0; n < kSteps; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[nt][n][e] = 0.f;
                }
                const int p0 = at.rq.pos0() + r0 / G, p1 = at.rq.pos0() + (r0 + rows - 1) / G;
                all_hi = min(p0 + 1, at.w.hi);
                all_lo = a.p.window > 0 && p1 >= a.p.window ? p1 - a.p.window + 1 : 0;
            }
            const uint32_t stage = done % L::kStages, kt = ring + stage * L::kStage, vt = kt + L::kHalves * L::kBlock;
            ok = bar_wait(&full[own][stage], (done / L::kStages) & 1, dead);
            if (!ok) break;
            ++done;
            const int j0 = at.w.lo + at.unit * kKeys, exist = at.w.hi - j0;
            if (exist < kKeys) {  // values of keys that do not exist: a weight of 0 would not hide a NaN
                for (int x = lane; x < (kKeys - max(exist, 0)) * 8 * L::kHalves; x += 32) {
                    const int r = max(exist, 0) + x / (8 * L::kHalves), col = x % (8 * L::kHalves);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + (col >> 3) * L::kBlock + r * 128 +
                                                                                 (col & 7) * 16),
                                 "r"(0)
                                 : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into the stage
                __syncwarp();
            }

            // scores: two chains of matrix instructions per 16 keys, joined by an addition
            float s[kKeys / 16][NT][4];
#pragma unroll
            for (int kb = 0; kb < kKeys / 16; ++kb) {
                float t[NT][2][4] = {};
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t kf[4];
                    ldsm4(kf, kt + (k >> 2) * L::kBlock + kb * 2048 + k_at[k & 3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = NP - 1; i >= 0; --i) mma16816<T>(t[nt][k & 1], kf, qf[i][nt][k][0], qf[i][nt][k][1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kb][nt][e] = t[nt][0][e] + t[nt][1][e];
            }
            const bool whole = j0 >= all_lo && j0 + kKeys <= all_hi;
            bool higher = false;
#pragma unroll
            for (int kb = 0; kb < kKeys / 16; ++kb)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int q = e & 1, j = j0 + kb * 16 + (lane >> 2) + 8 * (e >> 1);
                        float x = s[kb][nt][e] * mul[nt][q];
                        if (a.post != 0.f) x = a.post * tanhf(x);
                        if (a.bias_near) x = fmaf(slope[nt][q], static_cast<float>(j - pos[nt][q]), x);
                        if (!whole && (j > min(pos[nt][q], at.w.hi - 1) || (a.p.window > 0 && pos[nt][q] - j >= a.p.window)))
                            x = -INFINITY;
                        s[kb][nt][e] = x;
                        higher |= x > m[nt][q] + kSlack;
                    }
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float top = m[nt][q];
#pragma unroll
                        for (int kb = 0; kb < kKeys / 16; ++kb) top = fmaxf(top, fmaxf(s[kb][nt][q], s[kb][nt][2 + q]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float f = top == -INFINITY ? 1.f : exp2f(m[nt][q] - top);
                        m[nt][q] = top;
                        l[nt][q] *= f;
#pragma unroll
                        for (int n = 0; n < kSteps; ++n) o[nt][n][q] *= f, o[nt][n][2 + q] *= f;
                    }
            }
            uint32_t pf[kKeys / 16][NP][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // 16-bit queries: the weights' factor goes into the exponent, whose rounding
                // is far below that of the weights; F32 queries: an exact product
                constexpr float kUp = NP > 1 ? 1 << Half16<T>::kWeightLog2 : 1, kOff = NP > 1 ? 0 : Half16<T>::kWeightLog2;
                const float base[2] = {m[nt][0] == -INFINITY ? 0.f : m[nt][0] - kOff,
                                       m[nt][1] == -INFINITY ? 0.f : m[nt][1] - kOff};
#pragma unroll
                for (int kb = 0; kb < kKeys / 16; ++kb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[kb][nt][e] = exp2f(s[kb][nt][e] - base[e & 1]) * kUp;
                        l[nt][e & 1] += s[kb][nt][e];
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {  // keys 0-7, then 8-15
                        uint32_t piece[NP];
                        split_pair<T, NP>(s[kb][nt][2 * e], s[kb][nt][2 * e + 1], piece, Half16<T>::kLow);
#pragma unroll
                        for (int i = 0; i < NP; ++i) pf[kb][i][nt][e] = transpose8x8(piece[i]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < kSteps; ++n) {
                // the matrix unit cuts its sums off: with F32 queries every unit's sum starts
                // at 0 and is added by a rounded addition, or a long axis would show it
                constexpr int kSums = weight_sums(NP);
                float t[kSums][NT][4] = {};
#pragma unroll
                for (int kb = 0; kb < kKeys / 16; ++kb) {
                    uint32_t vf[4];
                    ldsm4_t(vf, vt + (n >> 2) * L::kBlock + kb * 2048 + v_at[n & 3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = NP - 1; i >= 0; --i)
                            mma16816<T>(NP > 1 ? t[i % kSums][nt] : o[nt][n], vf, pf[kb][i][nt][0], pf[kb][i][nt][1]);
                }
                if (NP > 1)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[nt][n][e] += kSums == 2 ? fmaf(t[kSums - 1][nt][e], 1.f / Half16<T>::kLow, t[0][nt][e]) : t[0][nt][e];
            }
            __syncwarp();  // every lane has read the stage
            if (lane == 0) bar_arrive(&empty[own][stage]);
            --todo;
            const bool ends = at.unit + 1 == at.w.units;
            if constexpr (kJoin) {
                if (todo > 0) ++at.unit;
                continue;
            }
            if (!ends && todo > 0) {
                ++at.unit;
                continue;
            }

            // the item ends here, or goes on in the next stream
            const bool whole_item = ends && begun_here;
            const int part = begun_here ? 1 : 0;
            float* to = g.parts + (static_cast<size_t>(me) * 2 + part) * part_floats(R, D);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float sum = l[nt][q];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    const int r = nt * 8 + 2 * (lane & 3) + q;
                    if (r >= rows) continue;
                    if (whole_item) {
                        const int rr = at.tile * R + r, i = rr / a.group, h = at.kvh * a.group + rr - i * a.group;
                        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                        for (int n = 0; n < kSteps; ++n) {
                            store_one(a, at.rq.first + i, h, n * 16 + (lane >> 2), sum == 0.f ? 0.f : o[nt][n][q] * inv);
                            store_one(a, at.rq.first + i, h, n * 16 + 8 + (lane >> 2),
                                      sum == 0.f ? 0.f : o[nt][n][2 + q] * inv);
                        }
                    } else {
#pragma unroll
                        for (int n = 0; n < kSteps; ++n) {
                            to[r * D + n * 16 + (lane >> 2)] = o[nt][n][q];
                            to[r * D + n * 16 + 8 + (lane >> 2)] = o[nt][n][2 + q];
                        }
                        if ((lane >> 2) == 0) {
                            to[R * D + r] = m[nt][q];
                            to[R * D + R + r] = sum;
                        }
                    }
                }
            if (begun_here && !ends && lane == 0) {
                const long long w1 = stream_of(item0 + at.w.units - 1, all, streams);
                g.heads[me] = SplitHead{at.b, at.kvh, at.tile, static_cast<int>(w1 - me + 1)};
            }
            if (todo > 0) {
                item0 += at.w.units;
                at.next<R, kKeys>(a);
                fresh = begun_here = true;
            }
        }
        if constexpr (!kJoin) {
            break;
        } else {
            // this warp's sums to the start of its ring (all of it has been read)
            __syncwarp();
            float* to = reinterpret_cast<float*>(smem + own * L::kWarpBytes);
            const bool any = at.w.units > 0 && !fresh;
            const int r0 = at.tile * R;
            rows = min(R, at.w.rows - r0);
            if (!loads)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int r = nt * 8 + 2 * (lane & 3) + q;
                    float sum = any ? l[nt][q] : 0.f;
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    if (any)
#pragma unroll
                        for (int n = 0; n < kSteps; ++n) {
                            to[r * D + n * 16 + (lane >> 2)] = o[nt][n][q];
                            to[r * D + n * 16 + 8 + (lane >> 2)] = o[nt][n][2 + q];
                        }
                    if ((lane >> 2) == 0) {
                        to[R * D + r] = any ? m[nt][q] : -INFINITY;
                        to[R * D + R + r] = sum;
                    }
                }
            cluster_join<D, R, kThreads, L::kWarps, L::kWarpBytes>(a, at.rq, at.kvh, at.tile, rows, smem);
        }
    }
}

template <int D>
size_t workspace_of(int R) {
    return split_bytes(static_cast<size_t>(sm_count()) * Ring<D>::kWarps, R, D);
}

// The joining form is taken where its clusters fit on the SMs at once and no
// warp gets a long run.
struct Items {
    int tiles;      // row tiles of a request (as the hints have it)
    int64_t count;  // items of the call, 2^40 at most
    bool join;
};
Items count_items(const AttnArgs& a, int R) {
    Items i;
    const int64_t rows = std::min<int64_t>(a.p.max_new, a.p.n_tokens) * a.group;  // < 2^31
    i.tiles = static_cast<int>(std::max<int64_t>(1, (rows + R - 1) / R));
    i.count = static_cast<int64_t>(
        std::min(static_cast<double>(i.tiles) * a.p.n_seqs * a.kv.kv_heads, static_cast<double>(int64_t(1) << 40)));
    i.join = i.count * kCluster <= sm_count() && a.p.max_kv <= kJoinKeys;
    return i;
}

template <typename T, int D, int NP, int NT, bool kJoin>
cudaError_t launch_form(const StreamArgs& c, int ctas, cudaStream_t stream) {
    using L = Ring<D>;
    constexpr auto kernel = attn_stream_kernel<T, D, NP, NT, kJoin>;
    const cudaError_t e = allow_smem<kernel>(L::kBytes);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3(ctas), dim3(L::kThreads), L::kBytes, stream, kJoin ? kCluster : 1, c);
}

template <typename T, int D, int NP, int NT>
cudaError_t launch_rows(const AttnArgs& a, cudaStream_t stream) {
    using L = Ring<D>;
    const Items items = count_items(a, 8 * NT);
    const int sms = sm_count();
    StreamArgs c;
    SplitArgs& g = c.g;
    g = split_args(a, static_cast<size_t>(sms) * L::kWarps);
    c.box_tokens = std::min(a.kv.block_size, L::kKeys);
    if (!cache_map(&c.k, a.kv, a.kv.k, c.box_tokens) || !cache_map(&c.v, a.kv, a.kv.v, c.box_tokens))
        return cudaErrorInvalidValue;
    g.tiles = items.tiles;
    if (items.join) return launch_form<T, D, NP, NT, true>(c, static_cast<int>(items.count) * kCluster, stream);
    // no more streams than the hints give work for
    const int64_t units = std::min<int64_t>(items.count, 1 << 30) * std::max<int64_t>(1, (int64_t(a.p.max_kv) + L::kKeys - 1) / L::kKeys);
    g.streams = static_cast<int>(std::min<int64_t>(sms * L::kWarps, std::max<int64_t>(1, units)));
    const cudaError_t e = launch_form<T, D, NP, NT, false>(c, std::min(sms, g.streams), stream);
    if (e != cudaSuccess) return e;
    return combine_launch<D, 8 * NT>(g, items.count, stream);
}

// Rows of an item: as few 8-column blocks as the hints ask for, as many as the
// registers hold beside q's NP pieces and o (255 a thread: four blocks of heads of 96
// spill 124 bytes, two with F32 queries up to 32, the others none).
constexpr int most_blocks(int D, bool f32) { return D > 128 ? 1 : f32 || D > 96 ? 2 : 4; }
int row_blocks(const AttnArgs& a) {
    const int64_t rows = static_cast<int64_t>(a.p.max_new) * a.group;
    const int want = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    return std::min(want, most_blocks(a.kv.head_dim, a.p.q_type == GGML_TYPE_F32));
}

template <typename T, int D, int NP, int kMost>
cudaError_t launch_blocks(const AttnArgs& a, cudaStream_t stream) {
    const int n = row_blocks(a);
    if constexpr (kMost >= 4)
        if (n == 4) return launch_rows<T, D, NP, 4>(a, stream);
    if constexpr (kMost >= 2)
        if (n == 2) return launch_rows<T, D, NP, 2>(a, stream);
    return launch_rows<T, D, NP, 1>(a, stream);
}
template <typename T, int D>
cudaError_t launch_pieces(const AttnArgs& a, cudaStream_t stream) {
    if (a.p.q_type == GGML_TYPE_F32)
        return launch_blocks<T, D, Half16<T>::kPieces, most_blocks(D, true)>(a, stream);
    return launch_blocks<T, D, 1, most_blocks(D, false)>(a, stream);
}
template <typename T>
cudaError_t launch_type(const AttnArgs& a, cudaStream_t stream) {
    switch (a.kv.head_dim) {
        case 64: return launch_pieces<T, 64>(a, stream);
        case 96: return launch_pieces<T, 96>(a, stream);
        case 128: return launch_pieces<T, 128>(a, stream);
        default: return launch_pieces<T, 256>(a, stream);
    }
}

}  // namespace

size_t stream_workspace(const AttnArgs& a) {
    const int R = 8 * row_blocks(a);
    if (count_items(a, R).join) return 0;
    switch (a.kv.head_dim) {
        case 64: return workspace_of<64>(R);
        case 96: return workspace_of<96>(R);
        case 128: return workspace_of<128>(R);
        default: return workspace_of<256>(R);
    }
}

cudaError_t stream_error(int* out) { return take_wait_error(out); }

cudaError_t stream_launch(const AttnArgs& a, cudaStream_t stream) {
    return a.kv.type == GGML_TYPE_F16 ? launch_type<__half>(a, stream) : launch_type<__nv_bfloat16>(a, stream);
}

}  // namespace xb
