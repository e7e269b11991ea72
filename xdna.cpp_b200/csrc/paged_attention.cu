// Causal attention of new tokens over a paged KV cache: the tile kernel.
//
// Mathematics: a row (token i, head h) at position p sees the keys j <= p (and
// j > p - window).  One pass over the keys keeps the row's running maximum m,
// its sum l = sum 2^(s_j - m) and o = sum 2^(s_j - m) v_j, where s_j is the
// score times log2(e); a larger maximum scales l and o by 2^(m - m').  The
// row's output is o / l.
//
// The query heads that share a KV head are rows of the same tile (row r is
// token r / group, head r % group), so a K/V tile is read once for all of
// them.  A warp takes 16 rows, a CTA 128 (64 at head_dim 256, whose pieces of q
// fill shared memory); K and V tiles of kKeys keys come through a two-stage
// cp.async ring, in rows padded by 16 bytes (an odd number of 16-byte columns:
// ldmatrix reads 8 rows without a bank conflict).  The F32 queries run as NP
// 16-bit pieces of q and of the softmax weights, whose products with the exact
// 16-bit K and V add up in F32.  The work of all items is dealt out in equal
// runs to the CTAs (paged_walk.cuh) and cut items are joined.
//
// Bound by issue: 2048 rows of 32 heads of 128 over 4096 keys take 798 us with an
// F16 cache (two pieces), 975 us with BF16 (three), a third of it matrix
// instructions; the chunk kernel takes 140 us with 16-bit queries.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "paged_walk.cuh"

namespace xb {
namespace {

constexpr int kMinTiles = 2;   // key tiles per CTA below which fewer CTAs run
constexpr float kSlack = 8.f;  // log2 of the largest weight (before kWeightLog2)

template <int D, int NP>
struct Tile {
    static constexpr int kWarps = D > 128 ? 4 : 8;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRows = kWarps * 16;
    static constexpr int kCtas = D == 64 ? 2 : 1;  // on an SM
    static constexpr int kKeys = D > 128 ? 32 : 64;
    static constexpr int kStride = D + 8;  // elements per row
    static constexpr int kQ = kRows * kStride;
    static constexpr int kK = kKeys * kStride;
    static constexpr size_t kBytes = (NP * kQ + 4 * kK) * sizeof(uint16_t) + kRows * sizeof(float);
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    const int bytes = on ? 16 : 0;  // 0: fills with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <typename T, int D, int NP>
__global__ void __launch_bounds__(Tile<D, NP>::kThreads, Tile<D, NP>::kCtas)
    attn_tile_kernel(const __grid_constant__ SplitArgs g) {
    using L = Tile<D, NP>;
    constexpr int kKeys = L::kKeys, kS = L::kStride, kThreads = L::kThreads, kRows = L::kRows;
    constexpr int kSums = weight_sums(NP);
    constexpr float kUp = 1 << Half16<T>::kWeightLog2;
    extern __shared__ __align__(16) uint16_t smem[];
    __shared__ RunUnits<kThreads> units;
    const AttnArgs& a = g.a;
    uint16_t* qs = smem;
    uint16_t* ks = qs + NP * L::kQ;
    uint16_t* vs = ks + 2 * L::kK;
    float* row_scale = reinterpret_cast<float*>(vs + 2 * L::kK);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_wait();

    Run run;
    start_run<kRows, kKeys, kThreads>(a, gridDim.x, kMinTiles, units, run);
    const long long me = blockIdx.x;
    if (tid == 0) g.heads[me].parts = 0;
    if (!run.units) return;
    Walk w = run.first;
    bool first_item = true;
    do {
        const Request rq = w.rq;
        const int kvh = w.kvh, G = a.group, r0 = w.tile * kRows, rows = min(kRows, w.rows - r0);
        const int lo = w.s0 * kKeys, hi = min(w.hi, w.s1 * kKeys);  // this run's keys of the item

        auto load = [&](int j0, int stage) {
            constexpr int kChunks = D / 8;
#pragma unroll
            for (int x = 0; x < kKeys * kChunks / kThreads; ++x) {
                const int i = x * kThreads + tid, r = i / kChunks, c = i - r * kChunks, j = j0 + r;
                const int id = j < hi ? key_block(a, w.b, j >> a.log_bs) : -1;
                const int64_t at = id < 0 ? 0
                                          : id * a.kv.nb_block + kvh * a.kv.nb_head +
                                                (j & (a.kv.block_size - 1)) * a.kv.nb_token + c * 16;
                const int d = stage * L::kK + r * kS + c * 8;
                cp_async16(smem_addr(ks + d), static_cast<const char*>(a.kv.k) + at, id >= 0);
                cp_async16(smem_addr(vs + d), static_cast<const char*>(a.kv.v) + at, id >= 0);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if (lo < hi) load(lo, 0);

        // the tile's queries, as NP pieces
        for (int r = warp; r < kRows; r += L::kWarps) {
            const bool on = r < rows;
            const int i = (r0 + r) / G, h = kvh * G + (r0 + r) - i * G;
            const char* src = static_cast<const char*>(a.p.q) + (rq.first + (on ? i : 0)) * a.p.nb_q;
            const float2* s = reinterpret_cast<const float2*>(src) + static_cast<int64_t>(h) * (D / 2);
            float big = 0.f, up = 1.f;
            if (NP == 2) {
                for (int c = lane; on && c < D / 2; c += 32) big = fmaxf(big, fmaxf(fabsf(s[c].x), fabsf(s[c].y)));
#pragma unroll
                for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                up = row_power(big);
            }
            if (lane == 0) row_scale[r] = up;
            const float down = 1.f / up;
            for (int c = lane; c < D / 2; c += 32) {
                const float2 x = on ? s[c] : make_float2(0.f, 0.f);
                uint32_t piece[NP];
                split_pair<T, NP>(x.x * down, x.y * down, piece);
#pragma unroll
                for (int k = 0; k < NP; ++k) *reinterpret_cast<uint32_t*>(qs + k * L::kQ + r * kS + 2 * c) = piece[k];
            }
        }
        __syncthreads();

        // this thread's two rows
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, slope[2], mul[2];
        int p[2], last[2], row[2];  // position, last key it sees, row of the tile
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            row[e] = warp * 16 + (lane >> 2) + 8 * e;
            const int i = (r0 + row[e]) / G;
            p[e] = rq.pos0() + i;
            last[e] = min(p[e], w.hi - 1);
            slope[e] = head_slope(a, kvh * G + (r0 + row[e]) - i * G);
            mul[e] = a.pre * row_scale[row[e]];
        }
        // keys [all_lo, all_hi) are seen by every row of the tile
        const int p0 = rq.pos0() + r0 / G, p1 = rq.pos0() + (r0 + rows - 1) / G;
        const int all_hi = min(p0 + 1, w.hi), all_lo = a.p.window > 0 && p1 >= a.p.window ? p1 - a.p.window + 1 : 0;
        float o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

        int stage = 0;
        for (int j0 = lo; j0 < hi; j0 += kKeys, stage ^= 1) {
            if (j0 + kKeys < hi) {
                load(j0 + kKeys, stage ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncthreads();
            const uint16_t* kt = ks + stage * L::kK;
            const uint16_t* vt = vs + stage * L::kK;

            float s[kKeys / 8][4];
#pragma unroll
            for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t qf[NP][4];
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    ldsm4(qf[i], smem_addr(qs + i * L::kQ + (warp * 16 + (lane & 15)) * kS + k * 16 + (lane >> 4) * 8));
#pragma unroll
                for (int n = 0; n < kKeys / 16; ++n) {
                    uint32_t kf[4];
                    ldsm4(kf, smem_addr(kt + (n * 16 + (lane & 7) + (lane >> 4) * 8) * kS + k * 16 + ((lane >> 3) & 1) * 8));
#pragma unroll
                    for (int i = NP - 1; i >= 0; --i) {
                        mma16816<T>(s[2 * n], qf[i], kf[0], kf[1]);
                        mma16816<T>(s[2 * n + 1], qf[i], kf[2], kf[3]);
                    }
                }
            }

            // scores in units of log 2, hidden keys at -inf
#pragma unroll
            for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] *= mul[e >> 1];
            if (a.post != 0.f)
#pragma unroll
                for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = a.post * tanhf(s[n][e]);
            if (a.bias_near)
#pragma unroll
                for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + n * 8 + 2 * (lane & 3) + (e & 1);
                        s[n][e] = fmaf(slope[e >> 1], static_cast<float>(j - p[e >> 1]), s[n][e]);
                    }
            if (j0 < all_lo || j0 + kKeys > all_hi)
#pragma unroll
                for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int q = e >> 1, j = j0 + n * 8 + 2 * (lane & 3) + (e & 1);
                        if (j > last[q] || (a.p.window > 0 && p[q] - j >= a.p.window)) s[n][e] = -INFINITY;
                    }
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
            // the maximum moves only when a score passes it by kSlack (a weight is 2^kSlack at most)
            if (__any_sync(0xffffffffu, top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 1));
                    top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 2));
                    top[q] = fmaxf(top[q], m[q]);
                    const float c = top[q] == -INFINITY ? 1.f : exp2f(m[q] - top[q]);
                    m[q] = top[q];
                    l[q] *= c;
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[n][2 * q] *= c;
                        o[n][2 * q + 1] *= c;
                    }
                }
            }
            const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};  // no key yet: 0
            uint32_t pf[kKeys / 16][NP][4];
#pragma unroll
            for (int k = 0; k < kKeys / 16; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float* x = &s[2 * k + (e >> 1)][2 * (e & 1)];
                    x[0] = exp2_fast(x[0] - base[e & 1]) * kUp;
                    x[1] = exp2_fast(x[1] - base[e & 1]) * kUp;
                    l[e & 1] += x[0] + x[1];
                    uint32_t piece[NP];
                    split_pair<T, NP>(x[0], x[1], piece, Half16<T>::kLow);
#pragma unroll
                    for (int i = 0; i < NP; ++i) pf[k][i][e] = piece[i];
                }
            // The matrix unit cuts its sums off instead of rounding them, which adds up
            // over a long axis: every tile's sum starts at 0 and is added by a rounded
            // addition.
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                float t[kSums][2][4] = {};
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k) {
                    uint32_t vf[4];
                    ldsm4_t(vf, smem_addr(vt + (k * 16 + (lane & 15)) * kS + n * 16 + (lane >> 4) * 8));
#pragma unroll
                    for (int i = NP - 1; i >= 0; --i) {
                        mma16816<T>(t[i % kSums][0], pf[k][i], vf[0], vf[1]);
                        mma16816<T>(t[i % kSums][1], pf[k][i], vf[2], vf[3]);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[2 * n + h][e] +=
                            kSums == 2 ? fmaf(t[kSums - 1][h][e], 1.f / Half16<T>::kLow, t[0][h][e]) : t[0][h][e];
            }
            __syncthreads();
        }

        // the rows' output, or the item's partial
        const bool whole = w.s0 == w.t0 && w.s1 == w.t1;
        float* part = g.parts + (static_cast<size_t>(me) * 2 + (w.s0 == w.t0)) * part_floats(kRows, D);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            l[q] += __shfl_xor_sync(0xffffffffu, l[q], 1);
            l[q] += __shfl_xor_sync(0xffffffffu, l[q], 2);
            if (row[q] >= rows) continue;
            const bool none = l[q] == 0.f;  // no key, or only scores of -inf
            const float inv = whole ? 1.f / l[q] : 1.f;
            const int i = (r0 + row[q]) / G, h = kvh * G + (r0 + row[q]) - i * G;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                const int col = n * 8 + 2 * (lane & 3);
                const float2 x = none ? make_float2(0.f, 0.f) : make_float2(o[n][2 * q] * inv, o[n][2 * q + 1] * inv);
                if (whole)
                    store_out(a, rq.first + i, h, col, x.x, x.y);
                else
                    *reinterpret_cast<float2*>(part + static_cast<size_t>(row[q]) * D + col) = x;
            }
            if (!whole && (lane & 3) == 0) {
                part[kRows * D + row[q]] = m[q];
                part[kRows * D + kRows + row[q]] = l[q];
            }
        }
        if (tid == 0 && w.s0 == w.t0 && w.s1 < w.t1) g.heads[me] = run.head(w, first_item, me);
        first_item = false;
        __syncthreads();  // before the next item's queries
    } while (w.next<kRows, kKeys>(a));
}

template <int D, int NP>
int tile_streams() {
    return sm_count() * Tile<D, NP>::kCtas;
}

template <typename T, int D>
cudaError_t launch_tile(const AttnArgs& a, cudaStream_t stream) {
    constexpr int NP = Half16<T>::kPieces;
    using L = Tile<D, NP>;
    constexpr auto kernel = attn_tile_kernel<T, D, NP>;
    const cudaError_t e = allow_smem<kernel>(static_cast<int>(L::kBytes));
    if (e != cudaSuccess) return e;
    const int streams = tile_streams<D, NP>();
    const SplitArgs g = split_args(a, streams);
    const cudaError_t f = launch_pdl(kernel, dim3(streams), dim3(L::kThreads), L::kBytes, stream, 1, g);
    if (f != cudaSuccess) return f;
    const int64_t items = (a.p.n_tokens * a.group / L::kRows + 1) * a.kv.kv_heads;
    return combine_launch<D, L::kRows>(g, items, stream);
}
template <typename T>
cudaError_t launch_type(const AttnArgs& a, cudaStream_t stream) {
    switch (a.kv.head_dim) {
        case 64: return launch_tile<T, 64>(a, stream);
        case 96: return launch_tile<T, 96>(a, stream);
        case 128: return launch_tile<T, 128>(a, stream);
        default: return launch_tile<T, 256>(a, stream);
    }
}

template <typename T>
size_t tile_workspace(const AttnArgs& a) {
    constexpr int NP = Half16<T>::kPieces;
    switch (a.kv.head_dim) {
        case 64: return split_bytes(tile_streams<64, NP>(), Tile<64, NP>::kRows, 64);
        case 96: return split_bytes(tile_streams<96, NP>(), Tile<96, NP>::kRows, 96);
        case 128: return split_bytes(tile_streams<128, NP>(), Tile<128, NP>::kRows, 128);
        default: return split_bytes(tile_streams<256, NP>(), Tile<256, NP>::kRows, 256);
    }
}

AttnArgs make_args(const struct b200_paged_attention_args& p, const struct b200_kv_cache& kv) {
    AttnArgs a = {};
    a.p = p;
    a.kv = kv;
    a.group = p.heads / kv.kv_heads;
    while ((1 << a.log_bs) < kv.block_size) ++a.log_bs;
    a.pre = p.logit_softcap != 0.f ? p.scale / p.logit_softcap : p.scale * kLog2e;
    a.post = p.logit_softcap * kLog2e;
    if (p.max_bias != 0.f) {
        a.bias_near = 1;
        while (2 * a.bias_near <= p.heads) a.bias_near *= 2;
        a.log2_m0 = -p.max_bias / a.bias_near;
        a.log2_m1 = -p.max_bias / 2.f / a.bias_near;
    }
    a.min_rows = 0;
    a.max_rows = 0x7fffffff;
    return a;
}

}  // namespace

int sm_count() {
    static std::atomic<int> count[kMaxDevices];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 0;
    if ((n = count[dev].load(std::memory_order_relaxed)) == 0 &&
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
        count[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Requests of up to kStreamRows rows go to the stream kernel, the others to the
// chunk kernel (16-bit queries) or the tile kernel (F32); where the hints (or a
// single request) leave no doubt, one kernel takes everything.  The kernels run
// one after the other and share the workspace.
namespace {
struct Split {
    bool stream, chunk, tile;
};
Split split(const AttnArgs& a) {
    const bool few = static_cast<int64_t>(a.p.max_new) * a.group <= kStreamRows;
    const bool f32 = a.p.q_type == GGML_TYPE_F32;
    return Split{few || a.p.n_seqs > 1, !few && !f32, !few && f32};
}
}  // namespace

size_t paged_attention_workspace(const struct b200_paged_attention_args& p, const struct b200_kv_cache& kv) {
    const AttnArgs a = make_args(p, kv);
    const Split s = split(a);
    const size_t tile = kv.type == GGML_TYPE_F16 ? tile_workspace<__half>(a) : tile_workspace<__nv_bfloat16>(a);
    return std::max(s.stream ? stream_workspace(a) : 0, s.chunk ? chunk_workspace(a) : s.tile ? tile : 0);
}

cudaError_t paged_attention_launch(const struct b200_paged_attention_args& p, const struct b200_kv_cache& kv,
                                   cudaStream_t stream) {
    AttnArgs a = make_args(p, kv);
    const Split s = split(a);
    if (s.stream) {
        if (s.chunk || s.tile) a.max_rows = kStreamRows;
        const cudaError_t e = stream_launch(a, stream);
        if (e != cudaSuccess || !(s.chunk || s.tile)) return e;
        a.min_rows = kStreamRows;
        a.max_rows = 0x7fffffff;
    }
    if (s.chunk) return chunk_launch(a, stream);
    return kv.type == GGML_TYPE_F16 ? launch_type<__half>(a, stream) : launch_type<__nv_bfloat16>(a, stream);
}

cudaError_t paged_error_status(int* out) {
    // all streams: the copy that reads a word waits for the legacy stream alone
    cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return e;
    int stream = 0, chunk = 0;
    e = stream_error(&stream);
    const cudaError_t f = chunk_error(&chunk);
    *out = stream || chunk;
    return e != cudaSuccess ? e : f;
}

}  // namespace xb
