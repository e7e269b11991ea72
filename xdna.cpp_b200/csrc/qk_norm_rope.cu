// RMS norm of every query and key head, rotation by position, and the write of
// keys and values into the paged cache, in one pass over the q/k/v rows.
//
// Mathematics (per head row x of D values): y = x rsqrt(mean(x^2) + eps) w,
// then the pairs (u, v) of y turn by a_i = pos f_i with f_i = freq_scale
// freq_base^(-2i/n) / factor_i.  At positions of 10^5 an F32 angle is off by
// 10^-2, so the angle is formed as turns, pos * (f_i / 2 pi), in 64 bits; its
// distance to the nearest whole turn is exact there and then fits F32.
//
// The pass is bound by HBM: tokens x (heads + 2 kv_heads) x D values are read
// and written once.  A lane holds 8 values of a row as two 4-value chunks that
// contain its rotation pairs whole ((4l.., n/2 + 4l..) for split halves,
// 8 consecutive values for interleaved pairs), so no value crosses lanes
// except in the sum of squares.  D / 8 lanes make a row, 32 / (D / 8) rows a
// step, kDeep steps of one kind (queries, keys or values) of one token a chunk, a
// warp's item: its loads are in flight together, at constant distances from one
// address, and the norm weights, sines and cosines are fetched once for all of
// them (with kind and address worked out for every step, instructions bound the
// pass: 8191 tokens of 48 bf16 rows of 128 took 54 us at 69 % of the issue slots;
// now they take 43 us, 4.7 TB/s.  More warps with fewer registers, deeper loads and
// sines formed once per CTA were no faster.)
// One or more warps share a token's chunks; each forms the token's sines and
// cosines in shared memory while its first chunk is on its way, and has the next
// chunk in flight while it works on one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "gemv.cuh"
#include "paged.cuh"

namespace xb {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = 24;  // resident on an SM
constexpr int kRounds = 5;
constexpr int kMaxPairs = 128;

struct Turns {
    double f[kMaxPairs];  // turns per position of each pair, before the factors
};

template <typename T>
struct Chunk;  // 4 values as one load and store
template <>
struct Chunk<float> {
    using Raw = float4;
    static __device__ __forceinline__ void get(const Raw& x, float (&v)[4]) {
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    }
    static __device__ __forceinline__ void store(void* p, const float (&v)[4]) {
        *static_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
template <>
struct Chunk<__half> {
    using Raw = uint2;
    static __device__ __forceinline__ void get(const Raw& x, float (&v)[4]) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
    static __device__ __forceinline__ void store(void* p, const float (&v)[4]) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *static_cast<uint2*>(p) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
template <>
struct Chunk<__nv_bfloat16> {
    using Raw = uint2;
    static __device__ __forceinline__ void get(const Raw& x, float (&v)[4]) {
        v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u);
        v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void store(void* p, const float (&v)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        *static_cast<uint2*>(p) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};

// The pairs that turn together, of a lane's two chunks, and back.
template <bool kNeox>
__device__ __forceinline__ void pairs(const float (&x)[4], const float (&y)[4], float (&u)[4], float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        u[e] = kNeox ? x[e] : e < 2 ? x[2 * e] : y[2 * e - 4];
        v[e] = kNeox ? y[e] : e < 2 ? x[2 * e + 1] : y[2 * e - 3];
    }
}
template <bool kNeox>
__device__ __forceinline__ void unpair(const float (&u)[4], const float (&v)[4], float (&x)[4], float (&y)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = kNeox ? u[e] : e & 1 ? v[e / 2] : u[e / 2];
        y[e] = kNeox ? v[e] : e & 1 ? v[2 + e / 2] : u[2 + e / 2];
    }
}

struct RopeArgs {
    struct b200_qk_norm_rope_args p;
    struct b200_kv_cache kv;
    int log_bs;
    int parts;               // warps that share a token
    int q_chunks, k_chunks;  // chunks of the query heads, and of the KV heads
};

template <typename In, int D>
struct Rows {
    static constexpr int kLanes = D / 8;  // lanes that hold a row
    static constexpr int kGroup = kLanes <= 8 ? 8 : kLanes <= 16 ? 16 : 32;
    static constexpr int kPerStep = 32 / kGroup;  // rows
    static constexpr int kDeep = 8 / sizeof(In);  // steps of a chunk
    static constexpr int kPerChunk = kPerStep * kDeep;
};

// kNeox: the pairs are (i, i + n / 2), else (2 i, 2 i + 1).
template <typename In, typename Out, typename Cache, int D, bool kNeox>
__global__ void __launch_bounds__(kThreads, 768 / kThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a,
                                                                             const __grid_constant__ Turns turns) {
    using L = Rows<In, D>;
    using Raw = typename Chunk<In>::Raw;
    __shared__ __align__(16) float cosine[kThreads / 32][D / 2], sine[kThreads / 32][D / 2];
    const auto& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int l = lane & (L::kGroup - 1), sub = lane / L::kGroup, n = p.n_rot, half = n / 2;
    const bool on = l < L::kLanes;

    // the lane's two chunks of a row, and whether they turn
    const bool turn = on && 8 * l < n;
    int c0 = 8 * l, c1 = 8 * l + 4;
    if (kNeox && turn) c0 = 4 * l, c1 = half + 4 * l;
    if (!on) c0 = c1 = 0;

    const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp;
    const int64_t t = item / a.parts;
    const int chunks = a.q_chunks + 2 * a.k_chunks;
    grid_wait();
    if (t >= p.n_tokens) return;

    // chunk x: 0 queries, 1 keys, 2 values, this lane's first head, and its loads
    auto kind_of = [&](int x) { return x < a.q_chunks ? 0 : x < a.q_chunks + a.k_chunks ? 1 : 2; };
    auto head_of = [&](int x, int kind) {
        return (x - (kind == 0 ? 0 : kind == 1 ? a.q_chunks : a.q_chunks + a.k_chunks)) * L::kPerChunk + sub;
    };
    auto fetch = [&](int x, Raw (&raw_x)[L::kDeep], Raw (&raw_y)[L::kDeep]) {
        const int kind = kind_of(x), h0 = head_of(x, kind), heads = on ? (kind == 0 ? p.heads : a.kv.kv_heads) : 0;
        const char* src = (kind == 0   ? static_cast<const char*>(p.q) + t * p.nb_q
                           : kind == 1 ? static_cast<const char*>(p.k) + t * p.nb_k
                                       : static_cast<const char*>(p.v) + t * p.nb_v) +
                          h0 * D * static_cast<int>(sizeof(In));
        const Raw* from_x = reinterpret_cast<const Raw*>(src + c0 * sizeof(In));
        const Raw* from_y = reinterpret_cast<const Raw*>(src + c1 * sizeof(In));
#pragma unroll
        for (int u = 0; u < L::kDeep; ++u) {
            raw_x[u] = raw_y[u] = Raw{};
            if (h0 + u * L::kPerStep < heads) {
                raw_x[u] = from_x[u * L::kPerStep * D / 4];
                raw_y[u] = from_y[u * L::kPerStep * D / 4];
            }
        }
    };
    int x_chunk = static_cast<int>(item - t * a.parts);
    if (x_chunk >= chunks) return;
    Raw raw_x[L::kDeep], raw_y[L::kDeep];
    fetch(x_chunk, raw_x, raw_y);
    const int64_t slot = p.slots[t];
    if (n) {
        const double position = static_cast<double>(p.positions[t]);
        for (int j = lane; j < half; j += 32) {
            double f = turns.f[j];
            if (p.freq_factors) f /= static_cast<double>(p.freq_factors[j]);
            const double r = position * f;
            sincospif(2.0f * static_cast<float>(r - rint(r)), &sine[warp][j], &cosine[warp][j]);
        }
        __syncwarp();
    }
    for (; x_chunk < chunks; x_chunk += a.parts) {
        const int kind = kind_of(x_chunk), h0 = head_of(x_chunk, kind);
        const int heads = on ? (kind == 0 ? p.heads : a.kv.kv_heads) : 0;
        Raw next_x[L::kDeep], next_y[L::kDeep];
        const bool more = x_chunk + a.parts < chunks;
        if (more) fetch(x_chunk + a.parts, next_x, next_y);

        // where the rows go: the distance of heads in q_out, or in the cache
        char* dst = static_cast<char*>(p.q_out) + t * p.nb_q_out + h0 * D * static_cast<int>(sizeof(Out));
        int64_t step = L::kPerStep * D * static_cast<int>(sizeof(Out));
        bool stored = true;
        if (kind != 0) {
            const int64_t block = slot >> a.log_bs;
            stored = slot >= 0 && block < a.kv.num_blocks;
            dst = static_cast<char*>(kind == 1 ? a.kv.k : a.kv.v) + block * a.kv.nb_block +
                  (slot & (a.kv.block_size - 1)) * a.kv.nb_token + h0 * a.kv.nb_head;
            step = L::kPerStep * a.kv.nb_head;
        }
        if (kind == 2) {
#pragma unroll
            for (int u = 0; u < L::kDeep; ++u) {
                float x[4], y[4];
                Chunk<In>::get(raw_x[u], x);
                Chunk<In>::get(raw_y[u], y);
                if (stored && h0 + u * L::kPerStep < heads) {
                    Chunk<Cache>::store(dst + u * step + c0 * sizeof(Cache), x);
                    Chunk<Cache>::store(dst + u * step + c1 * sizeof(Cache), y);
                }
            }
        } else {
            // The pairs (u, v) of a lane, with the norm's weights in the rotation's
            // coefficients: u' = inv (u uc - v vs), v' = inv (u us + v vc).
            const float* w = kind == 0 ? p.q_norm : p.k_norm;
            float uc[4], vc[4], us[4] = {}, vs[4] = {};
#pragma unroll
            for (int e = 0; e < 4; ++e) uc[e] = vc[e] = 1.f;
            if (w) {
                const float4 wx = *reinterpret_cast<const float4*>(w + c0), wy = *reinterpret_cast<const float4*>(w + c1);
                const float x[4] = {wx.x, wx.y, wx.z, wx.w}, y[4] = {wy.x, wy.y, wy.z, wy.w};
                pairs<kNeox>(x, y, uc, vc);
            }
            if (turn) {
                const float4 cv = *reinterpret_cast<const float4*>(&cosine[warp][4 * l]);
                const float4 sv = *reinterpret_cast<const float4*>(&sine[warp][4 * l]);
                const float c[4] = {cv.x, cv.y, cv.z, cv.w}, s[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) us[e] = uc[e] * s[e], vs[e] = vc[e] * s[e], uc[e] *= c[e], vc[e] *= c[e];
            }
#pragma unroll
            for (int r = 0; r < L::kDeep; ++r) {
                float x[4], y[4], u[4], v[4];
                Chunk<In>::get(raw_x[r], x);
                Chunk<In>::get(raw_y[r], y);
                pairs<kNeox>(x, y, u, v);
                float inv = 1.f;
                if (w) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) ss = fmaf(u[e], u[e], fmaf(v[e], v[e], ss));
#pragma unroll
                    for (int d = L::kGroup / 2; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                    inv = rsqrtf(fmaf(ss, 1.0f / D, p.eps));  // 2 units in the last place
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float p0 = u[e] * uc[e], p1 = v[e] * vc[e];
                    if (turn) p0 = fmaf(-v[e], vs[e], p0), p1 = fmaf(u[e], us[e], p1);
                    u[e] = p0 * inv, v[e] = p1 * inv;
                }
                unpair<kNeox>(u, v, x, y);
                if (stored && h0 + r * L::kPerStep < heads) {
                    char* to = dst + r * step;
                    if (kind == 0) {
                        Chunk<Out>::store(to + c0 * sizeof(Out), x);
                        Chunk<Out>::store(to + c1 * sizeof(Out), y);
                    } else {
                        Chunk<Cache>::store(to + c0 * sizeof(Cache), x);
                        Chunk<Cache>::store(to + c1 * sizeof(Cache), y);
                    }
                }
            }
        }
        if (more)
#pragma unroll
            for (int u = 0; u < L::kDeep; ++u) raw_x[u] = next_x[u], raw_y[u] = next_y[u];
    }
}

template <typename In, typename Out, typename Cache, int D>
cudaError_t launch_pairs(const RopeArgs& a, const Turns& t, dim3 grid, cudaStream_t stream) {
    return launch_pdl(a.p.neox ? qk_norm_rope_kernel<In, Out, Cache, D, true> : qk_norm_rope_kernel<In, Out, Cache, D, false>,
                      grid, dim3(kThreads), 0, stream, 1, a, t);
}
template <typename In, typename Out, typename Cache>
cudaError_t launch_dim(const RopeArgs& a, const Turns& t, dim3 grid, cudaStream_t stream) {
    switch (a.kv.head_dim) {
        case 64: return launch_pairs<In, Out, Cache, 64>(a, t, grid, stream);
        case 96: return launch_pairs<In, Out, Cache, 96>(a, t, grid, stream);
        case 128: return launch_pairs<In, Out, Cache, 128>(a, t, grid, stream);
        default: return launch_pairs<In, Out, Cache, 256>(a, t, grid, stream);
    }
}
template <typename In, typename Out>
cudaError_t launch_cache(const RopeArgs& a, const Turns& t, dim3 grid, cudaStream_t stream) {
    return a.kv.type == GGML_TYPE_F16 ? launch_dim<In, Out, __half>(a, t, grid, stream)
                                      : launch_dim<In, Out, __nv_bfloat16>(a, t, grid, stream);
}
template <typename In>
cudaError_t launch_out(const RopeArgs& a, const Turns& t, dim3 grid, cudaStream_t stream) {
    switch (a.p.out_type) {
        case GGML_TYPE_F32: return launch_cache<In, float>(a, t, grid, stream);
        case GGML_TYPE_F16: return launch_cache<In, __half>(a, t, grid, stream);
        default: return launch_cache<In, __nv_bfloat16>(a, t, grid, stream);
    }
}

}  // namespace

cudaError_t qk_norm_rope_launch(const struct b200_qk_norm_rope_args& p, const struct b200_kv_cache& kv,
                                cudaStream_t stream) {
    RopeArgs a{p, kv, 0, 1, 0, 0};
    while ((1 << a.log_bs) < kv.block_size) ++a.log_bs;
    Turns turns;
    if (p.n_rot) {
        // powers by products: 64 roundings of 64-bit numbers, 10^-14 of an angle
        const double ratio = std::pow(static_cast<double>(p.freq_base), -2.0 / p.n_rot);
        double f = static_cast<double>(p.freq_scale) / 6.283185307179586476925286766559;
        for (int i = 0; i < p.n_rot / 2; ++i, f *= ratio) turns.f[i] = f;
    }
    const int per = (kv.head_dim <= 64 ? 4 : kv.head_dim <= 128 ? 2 : 1) *  // Rows::kPerChunk
                    (p.in_type == GGML_TYPE_F32 ? 2 : 4);
    a.q_chunks = (p.heads + per - 1) / per;
    a.k_chunks = (kv.kv_heads + per - 1) / per;
    const int chunks = a.q_chunks + 2 * a.k_chunks;
    // A token's chunks are shared by as many warps as it takes for kRounds rounds of
    // warps on all SMs (few tokens: one chunk a warp).
    const int64_t want = static_cast<int64_t>(sm_count()) * kWarps * kRounds;
    a.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(chunks, want / p.n_tokens)));
    const int64_t grid = (p.n_tokens * a.parts + kThreads / 32 - 1) / (kThreads / 32);
    switch (p.in_type) {
        case GGML_TYPE_F32: return launch_out<float>(a, turns, dim3(static_cast<unsigned>(grid)), stream);
        case GGML_TYPE_F16: return launch_out<__half>(a, turns, dim3(static_cast<unsigned>(grid)), stream);
        default: return launch_out<__nv_bfloat16>(a, turns, dim3(static_cast<unsigned>(grid)), stream);
    }
}

}  // namespace xb
