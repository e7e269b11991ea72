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
// except in the sum of squares.  D / 8 lanes make a row, and a lane keeps the
// 4 sines and cosines of its token for all the rows of that token it handles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "gemv.cuh"
#include "paged.cuh"

namespace xb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;

struct Turns {
    double f[kMaxPairs];  // turns per position of each pair, before the factors
};

template <typename T>
struct Chunk;  // 4 values as one load
template <>
struct Chunk<float> {
    static __device__ __forceinline__ void load(const void* p, float (&v)[4]) {
        const float4 x = *static_cast<const float4*>(p);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    }
    static __device__ __forceinline__ void store(void* p, const float (&v)[4]) {
        *static_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
template <>
struct Chunk<__half> {
    static __device__ __forceinline__ void load(const void* p, float (&v)[4]) {
        const uint2 x = *static_cast<const uint2*>(p);
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
    static __device__ __forceinline__ void load(const void* p, float (&v)[4]) {
        const uint2 x = *static_cast<const uint2*>(p);
        v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u);
        v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void store(void* p, const float (&v)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        *static_cast<uint2*>(p) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};

struct RopeArgs {
    struct b200_qk_norm_rope_args p;
    struct b200_kv_cache kv;
    int splits;   // warps that share one token's rows
    int log_bs;
};

template <typename In, typename Out, typename Cache, int D>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a,
                                                                const __grid_constant__ Turns turns) {
    constexpr int kLanes = D / 8;                                  // lanes that hold a row
    constexpr int kGroup = kLanes <= 8 ? 8 : kLanes <= 16 ? 16 : 32;
    constexpr int kRows = 32 / kGroup;                             // rows per warp
    const auto& p = a.p;
    const int lane = threadIdx.x & 31, l = lane & (kGroup - 1), sub = lane / kGroup;
    const bool on = l < kLanes;
    const int n = p.n_rot, half = n / 2;

    // the lane's chunks, and whether they turn
    const bool turn = on && 8 * l < n;
    int c0 = 8 * l, c1 = 8 * l + 4;
    if (p.neox && turn) c0 = 4 * l, c1 = half + 4 * l;
    if (!on) c0 = c1 = 0;

    double f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = turn ? turns.f[4 * l + i] : 0.0;
    grid_wait();
    if (turn && p.freq_factors) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] /= static_cast<double>(p.freq_factors[4 * l + i]);
    }

    const int rows = p.heads + 2 * a.kv.kv_heads;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
    const int64_t items = p.n_tokens * a.splits;
    for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); it < items; it += warps) {
        const int64_t t = it / a.splits;
        const int part = static_cast<int>(it - t * a.splits);
        const double pos = static_cast<double>(p.positions[t]);
        const int64_t slot = p.slots[t];
        float c[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double x = pos * f[i];
            sincospif(2.0f * static_cast<float>(x - rint(x)), &s[i], &c[i]);
        }
        const int64_t block = slot >> a.log_bs;
        const bool stored = slot >= 0 && block < a.kv.num_blocks;
        const int64_t at = stored ? block * a.kv.nb_block + (slot & (a.kv.block_size - 1)) * a.kv.nb_token : 0;

        for (int r0 = part * kRows; r0 < rows; r0 += a.splits * kRows) {
            const int r = r0 + sub;
            const bool row_on = on && r < rows;
            const bool is_q = r < p.heads, is_v = r >= p.heads + a.kv.kv_heads;
            const int h = is_q ? r : is_v ? r - p.heads - a.kv.kv_heads : r - p.heads;
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            if (row_on) {
                const char* src = static_cast<const char*>(is_q ? p.q : is_v ? p.v : p.k) +
                                  t * (is_q ? p.nb_q : is_v ? p.nb_v : p.nb_k) + static_cast<int64_t>(h) * D * sizeof(In);
                Chunk<In>::load(src + c0 * sizeof(In), x);
                Chunk<In>::load(src + c1 * sizeof(In), y);
            }
            const float* w = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
            if (p.q_norm || p.k_norm) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
                for (int d = kGroup / 2; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                if (w && row_on) {
                    const float inv = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
                    float wx[4], wy[4];
                    Chunk<float>::load(w + c0, wx);
                    Chunk<float>::load(w + c1, wy);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] *= inv * wx[i], y[i] *= inv * wy[i];
                }
            }
            if (turn && !is_v) {
                if (p.neox) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float u = x[i], v = y[i];
                        x[i] = u * c[i] - v * s[i];
                        y[i] = u * s[i] + v * c[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float u = x[2 * i], v = x[2 * i + 1];
                        x[2 * i] = u * c[i] - v * s[i];
                        x[2 * i + 1] = u * s[i] + v * c[i];
                        u = y[2 * i], v = y[2 * i + 1];
                        y[2 * i] = u * c[i + 2] - v * s[i + 2];
                        y[2 * i + 1] = u * s[i + 2] + v * c[i + 2];
                    }
                }
            }
            if (!row_on) continue;
            if (is_q) {
                char* dst = static_cast<char*>(p.q_out) + t * p.nb_q_out + static_cast<int64_t>(h) * D * sizeof(Out);
                Chunk<Out>::store(dst + c0 * sizeof(Out), x);
                Chunk<Out>::store(dst + c1 * sizeof(Out), y);
            } else if (stored) {
                char* dst = static_cast<char*>(is_v ? a.kv.v : a.kv.k) + at + h * a.kv.nb_head;
                Chunk<Cache>::store(dst + c0 * sizeof(Cache), x);
                Chunk<Cache>::store(dst + c1 * sizeof(Cache), y);
            }
        }
    }
}

template <typename In, typename Out, typename Cache>
cudaError_t launch_dim(const RopeArgs& a, const Turns& t, unsigned grid, cudaStream_t stream) {
    switch (a.kv.head_dim) {
        case 64: return launch_pdl(qk_norm_rope_kernel<In, Out, Cache, 64>, grid, kThreads, 0, stream, 1, a, t);
        case 96: return launch_pdl(qk_norm_rope_kernel<In, Out, Cache, 96>, grid, kThreads, 0, stream, 1, a, t);
        case 128: return launch_pdl(qk_norm_rope_kernel<In, Out, Cache, 128>, grid, kThreads, 0, stream, 1, a, t);
        default: return launch_pdl(qk_norm_rope_kernel<In, Out, Cache, 256>, grid, kThreads, 0, stream, 1, a, t);
    }
}
template <typename In, typename Out>
cudaError_t launch_cache(const RopeArgs& a, const Turns& t, unsigned grid, cudaStream_t stream) {
    return a.kv.type == GGML_TYPE_F16 ? launch_dim<In, Out, __half>(a, t, grid, stream)
                                      : launch_dim<In, Out, __nv_bfloat16>(a, t, grid, stream);
}
template <typename In>
cudaError_t launch_out(const RopeArgs& a, const Turns& t, unsigned grid, cudaStream_t stream) {
    switch (a.p.out_type) {
        case GGML_TYPE_F32: return launch_cache<In, float>(a, t, grid, stream);
        case GGML_TYPE_F16: return launch_cache<In, __half>(a, t, grid, stream);
        default: return launch_cache<In, __nv_bfloat16>(a, t, grid, stream);
    }
}

}  // namespace

cudaError_t qk_norm_rope_launch(const struct b200_qk_norm_rope_args& p, const struct b200_kv_cache& kv,
                                cudaStream_t stream) {
    RopeArgs a{p, kv, 1, 0};
    while ((1 << a.log_bs) < kv.block_size) ++a.log_bs;
    Turns turns;
    const double turn = 6.283185307179586476925286766559;
    for (int i = 0; i < p.n_rot / 2; ++i)
        turns.f[i] = static_cast<double>(p.freq_scale) *
                     std::pow(static_cast<double>(p.freq_base), -2.0 * i / p.n_rot) / turn;
    const int rows_per_warp = kv.head_dim <= 64 ? 4 : kv.head_dim <= 128 ? 2 : 1;
    const int rounds = (p.heads + 2 * kv.kv_heads + rows_per_warp - 1) / rows_per_warp;
    // Enough warps for every SM: a token's rows are shared by up to one warp per
    // round while tokens alone leave SMs idle.
    const int64_t want = 148 * 32;
    a.splits = static_cast<int>(p.n_tokens >= want ? 1 : std::min<int64_t>(rounds, (want + p.n_tokens - 1) / p.n_tokens));
    const int64_t warps = p.n_tokens * a.splits;
    const int64_t ctas = std::min<int64_t>((warps + kThreads / 32 - 1) / (kThreads / 32), 148 * 8);
    switch (p.in_type) {
        case GGML_TYPE_F32: return launch_out<float>(a, turns, static_cast<unsigned>(ctas), stream);
        case GGML_TYPE_F16: return launch_out<__half>(a, turns, static_cast<unsigned>(ctas), stream);
        default: return launch_out<__nv_bfloat16>(a, turns, static_cast<unsigned>(ctas), stream);
    }
}

}  // namespace xb
