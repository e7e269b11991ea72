// Partials of items that are cut along the keys, and the kernel that joins them.
//
// The attention kernels deal out the work of all requests as equal contiguous
// runs, one to each stream (a warp, or a CTA).  A stream leaves at most two
// partials: slot 0 for an item that began in an earlier stream, slot 1 for one
// that begins in it and goes on.  combine_kernel looks at every stream that
// began such an item and adds its parts up in stream order.
#pragma once
#include <algorithm>

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
    int streams;       // that may have work
    int tiles;         // joining form of the stream kernel: row tiles its grid has for each request
};

inline size_t split_bytes(size_t streams, int R, int D) {
    return streams * (sizeof(SplitHead) + 2 * part_floats(R, D) * sizeof(float));
}
inline SplitArgs split_args(const AttnArgs& a, size_t streams) {
    SplitArgs g{a, static_cast<SplitHead*>(a.p.workspace), nullptr, static_cast<int>(streams), 1};
    g.parts = reinterpret_cast<float*>(g.heads + streams);
    return g;
}

#ifdef __CUDACC__
// The last of `streams` streams that share `all` units equally (stream w has the
// units from all w / streams on) to begin at or before unit u.
__device__ __forceinline__ long long stream_of(long long u, long long all, long long streams) {
    return ((u + 1) * streams - 1) / all;
}

constexpr int kCombineWarps = 8;

// Joins the item that stream `me` began.  Block y takes the rows y, y +
// gridDim.y, ...; kSpread: all warps share the parts of one row at a time (few
// items, many parts), else every warp takes rows of its own.
template <int D, int R, bool kSpread>
__device__ __forceinline__ void combine_item(const SplitArgs& g, int me, const SplitHead& head,
                                             float (&shared_o)[kSpread ? kCombineWarps : 1][D],
                                             float (&shared_l)[kCombineWarps]) {
    const AttnArgs& a = g.a;
    const Request rq = read_request(a, head.b);
    const int rows = min(R, rq.count * a.group - head.tile * R), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t slot = part_floats(R, D);
    const float* mine = g.parts + 2 * static_cast<size_t>(me) * slot;
    auto part = [&](int p) { return mine + (2 * static_cast<size_t>(p) + (p == 0)) * slot; };
    const int step = kSpread ? gridDim.y : gridDim.y * kCombineWarps;
    for (int r = kSpread ? blockIdx.y : blockIdx.y + gridDim.y * warp; r < rows; r += step) {
        // the row's largest maximum
        float top = -INFINITY;
        for (int p = lane; p < head.parts; p += 32) top = fmaxf(top, part(p)[R * D + r]);
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float base = top == -INFINITY ? 0.f : top;
        // this warp's parts: lane i holds the weight of the i-th of 32 of them
        const int first = kSpread ? warp : 0, stride = kSpread ? kCombineWarps : 1;
        float sum = 0.f, o[D / 32] = {};
        for (int p0 = first; p0 < head.parts; p0 += 32 * stride) {
            float w = 0.f;
            if (p0 + lane * stride < head.parts) {
                const float* x = part(p0 + lane * stride);
                w = exp2f(x[R * D + r] - base);
                sum += w * x[R * D + R + r];
            }
            const int n = min(32, (head.parts - p0 + stride - 1) / stride);
#pragma unroll 8
            for (int i = 0; i < n; ++i) {
                const float c = __shfl_sync(0xffffffffu, w, i);
                const float* x = part(p0 + i * stride) + r * D;
#pragma unroll
                for (int k = 0; k < D / 64; ++k) {
                    const float2 v = *reinterpret_cast<const float2*>(x + k * 64 + lane * 2);
                    o[2 * k] = fmaf(c, v.x, o[2 * k]);
                    o[2 * k + 1] = fmaf(c, v.y, o[2 * k + 1]);
                }
                if (D % 64) o[D / 32 - 1] = fmaf(c, x[D / 64 * 64 + lane], o[D / 32 - 1]);
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int rr = head.tile * R + r, i = rr / a.group, h = head.kvh * a.group + rr - i * a.group;
        if constexpr (kSpread) {
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
                *reinterpret_cast<float2*>(&shared_o[warp][k * 64 + lane * 2]) = make_float2(o[2 * k], o[2 * k + 1]);
            if (D % 64) shared_o[warp][D / 64 * 64 + lane] = o[D / 32 - 1];
            if (lane == 0) shared_l[warp] = sum;
            __syncthreads();
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < kCombineWarps; ++w) l += shared_l[w];
            const float inv = l == 0.f ? 0.f : 1.f / l;
            for (int c = threadIdx.x; c < D; c += 32 * kCombineWarps) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < kCombineWarps; ++w) x += shared_o[w][c];
                store_one(a, rq.first + i, h, c, l == 0.f ? 0.f : x * inv);
            }
            __syncthreads();
        } else {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
                store_out(a, rq.first + i, h, k * 64 + lane * 2, sum == 0.f ? 0.f : o[2 * k] * inv,
                          sum == 0.f ? 0.f : o[2 * k + 1] * inv);
            if (D % 64) store_one(a, rq.first + i, h, D / 64 * 64 + lane, sum == 0.f ? 0.f : o[D / 32 - 1] * inv);
        }
    }
}

// Joins the items of stream blockIdx.x; kScan: of the blockIdx.x-th stream that has
// one to join, and of every gridDim.x-th after it.
template <int D, int R, bool kSpread, bool kScan>
__global__ void __launch_bounds__(32 * kCombineWarps) combine_kernel(const __grid_constant__ SplitArgs g) {
    __shared__ float shared_o[kSpread ? kCombineWarps : 1][D];
    __shared__ float shared_l[kCombineWarps];
    grid_wait();
    if (!kScan) {
        const SplitHead head = g.heads[blockIdx.x];
        if (head.parts) combine_item<D, R, kSpread>(g, blockIdx.x, head, shared_o, shared_l);
        return;
    }
    const int lane = threadIdx.x & 31;
    unsigned seen = 0;
    for (int from = 0; from < g.streams; from += 32) {  // alike in all warps
        const bool any = from + lane < g.streams && g.heads[from + lane].parts;
        for (unsigned left = __ballot_sync(0xffffffffu, any); left; left &= left - 1)
            if (seen++ % gridDim.x == blockIdx.x) {
                const int me = from + __ffs(left) - 1;
                combine_item<D, R, kSpread>(g, me, g.heads[me], shared_o, shared_l);
            }
    }
}

// Launches combine_kernel after a kernel whose items are about `items` (as the
// hints have it).  Few items have many parts each and leave most streams nothing to
// do: then a row is a CTA's (up to 32 rows an item) or a warp's, else a warp takes 4.
// Very few tall items: a row is a CTA's, and the CTAs look for the items, since a
// grid over all streams would be empty blocks for the most part (33 tokens of 8 heads
// over 19.9 K keys, 2 items: 40.8 -> 27.2 us with the attention kernel; 8 items, of
// 19 parts: 40.0 with a row a warp against 43.1).
template <int D, int R>
cudaError_t combine_launch(const SplitArgs& g, int64_t items, cudaStream_t stream) {
    const dim3 threads(32 * kCombineWarps);
    const bool few = g.streams >= 4 * items;
    if (few && R <= 32)
        return launch_pdl(combine_kernel<D, R, true, false>, dim3(g.streams, R), threads, 0, stream, 1, g);
    if (R > 32 && g.streams >= 32 * items)
        return launch_pdl(combine_kernel<D, R, true, true>, dim3(static_cast<unsigned>(std::max<int64_t>(items, 1)), R),
                          threads, 0, stream, 1, g);
    const int rows = few ? kCombineWarps : 4 * kCombineWarps;  // of a block
    return launch_pdl(combine_kernel<D, R, false, false>, dim3(g.streams, (R + rows - 1) / rows), threads, 0, stream, 1,
                      g);
}
#endif

}  // namespace xb
