// Partials of items that are cut along the keys, and the kernel that joins them.
//
// The attention kernels deal out the work of all requests as equal contiguous
// runs, one to each stream (a warp, or a CTA).  A stream leaves at most two
// partials: slot 0 for an item that began in an earlier stream, slot 1 for one
// that begins in it and goes on.  combine_kernel looks at every stream that
// began such an item and adds its parts up in stream order.
#pragma once
#include "paged_attn.cuh"

namespace xb {

// What a stream that begins an item, but does not end it, leaves for combine_kernel.
struct alignas(16) SplitHead {
    int b, kvh, tile;
    int parts;  // streams the item lies in; 0: none
};

// Floats of a partial of R rows: [R][D] sums of weighted values, [R] maxima, [R] sums of weights.
__host__ __device__ __forceinline__ size_t part_floats(int R, int D) { return static_cast<size_t>(R) * (D + 2); }

struct SplitArgs {
    AttnArgs a;
    SplitHead* heads;  // [streams]
    float* parts;      // [streams][2] partials
};

inline size_t split_bytes(size_t streams, int R, int D) {
    return streams * (sizeof(SplitHead) + 2 * part_floats(R, D) * sizeof(float));
}
inline SplitArgs split_args(const AttnArgs& a, size_t streams) {
    SplitArgs g{a, static_cast<SplitHead*>(a.p.workspace), nullptr};
    g.parts = reinterpret_cast<float*>(g.heads + streams);
    return g;
}

#ifdef __CUDACC__
// The last of `streams` streams that share `all` units equally (stream w has the
// units from all w / streams on) to begin at or before unit u.
__device__ __forceinline__ long long stream_of(long long u, long long all, long long streams) {
    return ((u + 1) * streams - 1) / all;
}

// Stream blockIdx.x's item: a warp per row, the rows dealt out over blockIdx.y.
template <int D, int R>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ SplitArgs g) {
    grid_wait();
    const AttnArgs& a = g.a;
    const SplitHead head = g.heads[blockIdx.x];
    if (!head.parts) return;
    const Request rq = read_request(a, head.b);
    const int rows = min(R, rq.count * a.group - head.tile * R), lane = threadIdx.x & 31;
    const size_t slot = part_floats(R, D);
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += 8 * gridDim.y) {
        // lane p holds part p, p + 32, ...: the row's largest maximum, then its parts' weights
        auto part = [&](int p) { return g.parts + (2 * (static_cast<size_t>(blockIdx.x) + p) + (p == 0)) * slot; };
        float top = -INFINITY;
        for (int p = lane; p < head.parts; p += 32) top = fmaxf(top, part(p)[R * D + r]);
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, o[D / 32] = {};
        for (int p0 = 0; p0 < head.parts; p0 += 32) {
            float w = 0.f;
            if (p0 + lane < head.parts) {
                const float* x = part(p0 + lane);
                w = exp2f(x[R * D + r] - base);
                sum += w * x[R * D + R + r];
            }
            const int n = min(32, head.parts - p0);
#pragma unroll 4
            for (int p = 0; p < n; ++p) {
                const float c = __shfl_sync(0xffffffffu, w, p);
                const float* x = part(p0 + p) + r * D + lane * 2;
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    const float2 v = *reinterpret_cast<const float2*>(x + i * 64);
                    o[2 * i] = fmaf(c, v.x, o[2 * i]);
                    o[2 * i + 1] = fmaf(c, v.y, o[2 * i + 1]);
                }
                if (D % 64) o[D / 32 - 1] = fmaf(c, part(p0 + p)[r * D + D / 64 * 64 + lane], o[D / 32 - 1]);
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int rr = head.tile * R + r, i = rr / a.group, h = head.kvh * a.group + rr - i * a.group;
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
            store_out(a, rq.first + i, h, k * 64 + lane * 2, sum == 0.f ? 0.f : o[2 * k] * inv,
                      sum == 0.f ? 0.f : o[2 * k + 1] * inv);
        if (D % 64)
            store_one(a, rq.first + i, h, D / 64 * 64 + lane, sum == 0.f ? 0.f : o[D / 32 - 1] * inv);
    }
}
#endif

}  // namespace xb
