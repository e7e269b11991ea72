// Device pieces the paged attention kernels share: the arguments, the score
// function and the search for a tile's request.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "gemv.cuh"
#include "paged.cuh"

namespace xb {

struct AttnArgs {
    struct b200_paged_attention_args p;
    struct b200_kv_cache kv;
    int group;        // query heads per KV head
    int log_bs;
    float pre, post;  // score in units of log 2: post * tanh(pre s) with a cap, pre s without
    int bias_near;    // ALiBi: heads below it have slopes m0^(h+1), the others m1^(2(h - near)+1); 0: no bias
    float log2_m0, log2_m1;
    int min_rows;     // this kernel takes the requests with more than min_rows rows (new tokens x group) ...
    int max_rows;     // ... and at most max_rows
};

constexpr float kLog2e = 1.4426950408889634f;

// The stream kernel (paged_stream.cu): rows (new tokens x group) up to which a
// request is its work, its workspace, and its launch.  It reads K and V once for
// every 8 to 32 rows, mostly from L2, but wastes no rows: 96 rows over 8012 keys
// take 16 us (F32 queries 22) against 31 (41) in the chunk (tile) kernel, 192 rows
// of 4 KV heads 36 (59) against 43 (69), 2400 rows of 2 KV heads 136 (273) against
// 60 (174).
constexpr int kStreamRows = 128;
size_t stream_workspace(const AttnArgs& a);
cudaError_t stream_launch(const AttnArgs& a, cudaStream_t stream);
cudaError_t stream_error(int* out);  // reads and clears the error word of its bounded waits

// The chunk kernel (paged_chunk.cu), for 16-bit queries: its workspace and launch.
size_t chunk_workspace(const AttnArgs& a);
cudaError_t chunk_launch(const AttnArgs& a, cudaStream_t stream);
cudaError_t chunk_error(int* out);

#ifdef __CUDACC__
// Slope of a query head, times log2(e).
__device__ __forceinline__ float head_slope(const AttnArgs& a, int h) {
    if (!a.bias_near) return 0.f;
    const float e = h < a.bias_near ? a.log2_m0 * (h + 1) : a.log2_m1 * (2 * (h - a.bias_near) + 1);
    return exp2f(e) * kLog2e;
}

// A request's rows of q and its key count, held inside the arrays whatever the device data says.
struct Request {
    int first, count, kv;
    __device__ __forceinline__ int pos0() const { return kv - count; }  // position of its first row
};
__device__ __forceinline__ Request read_request(const AttnArgs& a, int b) {
    const int n = static_cast<int>(a.p.n_tokens);
    const int s = min(max(a.p.cu_new[b], 0), n);
    const int e = min(max(a.p.cu_new[b + 1], s), n);
    return Request{s, e - s, max(a.p.kv_lens[b], 0)};
}
// The rows of a request this kernel takes (0: another kernel's).
__device__ __forceinline__ int my_rows(const AttnArgs& a, const Request& r) {
    const long long rows = static_cast<long long>(r.count) * a.group;
    return rows > a.min_rows && rows <= a.max_rows ? static_cast<int>(rows) : 0;
}
// Keys a table row has room for; there are none behind it.
__device__ __forceinline__ int table_keys(const AttnArgs& a) {
    const int64_t n = a.p.table_width << a.log_bs;
    return n < 0x7fffff00 ? static_cast<int>(n) : 0x7fffff00;  // the caches hold fewer than 2^31
}
// Keys that some row of tokens [i0, i1] of the request sees: [lo, hi).
__device__ __forceinline__ void key_range(const AttnArgs& a, const Request& r, int i0, int i1, int& lo, int& hi) {
    const int p0 = r.pos0() + i0;
    hi = min(max(0, r.pos0() + i1 + 1), table_keys(a));
    lo = a.p.window > 0 && p0 >= a.p.window ? p0 - a.p.window + 1 : 0;
}
// Work of one request in units of kKeys keys: `tiles` row tiles of R rows for
// each KV head, `units` units for each of those from key lo on (one even where
// no key is seen, so that the rows are written).
struct Work {
    int rows, tiles, lo, hi, units;
};
template <int kKeys>
__device__ __forceinline__ Work request_work(const AttnArgs& a, const Request& r, int R) {
    Work w;
    w.rows = my_rows(a, r);
    w.tiles = (w.rows + R - 1) / R;
    w.lo = w.hi = w.units = 0;
    if (w.rows) {
        key_range(a, r, 0, r.count - 1, w.lo, w.hi);
        w.lo = w.lo / kKeys * kKeys;
        w.units = max(1, (w.hi - w.lo + kKeys - 1) / kKeys);
    }
    return w;
}
// Cache block of a key, or -1 where the table has none (its keys read as zeros).
__device__ __forceinline__ int key_block(const AttnArgs& a, int b, int page) {
    if (page >= a.p.table_width) return -1;
    const int id = __ldg(a.p.block_table + static_cast<int64_t>(b) * a.p.table_width + page);
    return id >= 0 && id < a.kv.num_blocks ? id : -1;
}
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t row, int head, int col, float x, float y) {
    char* base = static_cast<char*>(a.p.out) + row * a.p.nb_out;
    const int64_t at = static_cast<int64_t>(head) * a.kv.head_dim + col;
    if (a.p.out_type == GGML_TYPE_F32)
        *reinterpret_cast<float2*>(base + at * 4) = make_float2(x, y);
    else if (a.p.out_type == GGML_TYPE_F16)
        *reinterpret_cast<__half2*>(base + at * 2) = __floats2half2_rn(x, y);
    else
        *reinterpret_cast<__nv_bfloat162*>(base + at * 2) = __floats2bfloat162_rn(x, y);
}
__device__ __forceinline__ void store_one(const AttnArgs& a, int64_t row, int head, int col, float x) {
    char* base = static_cast<char*>(a.p.out) + row * a.p.nb_out;
    const int64_t at = static_cast<int64_t>(head) * a.kv.head_dim + col;
    if (a.p.out_type == GGML_TYPE_F32)
        *reinterpret_cast<float*>(base + at * 4) = x;
    else if (a.p.out_type == GGML_TYPE_F16)
        *reinterpret_cast<__half*>(base + at * 2) = __float2half_rn(x);
    else
        *reinterpret_cast<__nv_bfloat16*>(base + at * 2) = __float2bfloat16_rn(x);
}

// 16-bit types: packing, and the pieces whose sum is an F32 value.
//
// A softmax weight is 2^8 at most (the running maximum moves when a score passes
// it by 8), and most of a long row's are small.  F16 ends at 2^-24, below which a
// weight would be lost for V while the sum of weights still counts it (31 keys in
// 32 at 17 nats below the 32nd: all of their share of the output); so weights are
// formed times 2^kWeightLog2, up to 2^15, and o and l carry the same factor until
// they are divided.
template <typename T>
struct Half16;
template <>
struct Half16<__half> {
    static constexpr int kPieces = 2;  // of an F32 value: 11 + 11 bits
    static constexpr int kWeightLog2 = 7;
    static constexpr float kLow = 2048.f;  // what the second piece of a weight is held times
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        return __half22float2(*reinterpret_cast<const __half2*>(&u));
    }
};
template <>
struct Half16<__nv_bfloat16> {
    static constexpr int kPieces = 3;  // 8 + 8 + 8 bits
    static constexpr int kWeightLog2 = 0;  // F32's range
    static constexpr float kLow = 1.f;
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
};
// Splits the pair (x, y) into NP 16-bit pairs, highest first, those behind the
// first held times `low` each.  The sum of the pieces is off by at most 2^-24
// (BF16), or 2^-22 of x or 2^-25 / low (F16; the smallest step is 2^-24).
template <typename T, int NP>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[NP], float low = 1.f) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        out[i] = Half16<T>::pack(x, y);
        if (i + 1 < NP) {
            const float2 h = Half16<T>::unpack(out[i]);
            x = (x - h.x) * low;
            y = (y - h.y) * low;
        }
    }
}
// Two pieces of a weight have a sum of products each: second[...] / kLow joins the
// first's (with one or three pieces there is one sum).
constexpr int weight_sums(int pieces) { return pieces == 2 ? 2 : 1; }
// F16 pieces reach down to 2^-24 only, so a row of F32 queries whose largest value
// is `big` is divided by a power of two that leaves it in [2^14, 2^15): values down
// to 2^-17 of it keep their 22 bits, and smaller ones are off by 2^-39 of it, which
// keys of 65504 do not show.  (In [1, 2) that was 2^-25, and a query of 2^-15 of the
// largest beside keys of 10^4 had scores off by 10^-3.)  BF16 pieces have F32's
// range.  The power and its reciprocal are normal numbers: a row of subnormal
// queries ends below 2^14.
__device__ __forceinline__ float row_power(float big) {
    return big > 0.f && big <= FLT_MAX ? ldexpf(1.f, max(ilogbf(big) - 14, -126)) : 1.f;
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2 units in the last place
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
#endif

}  // namespace xb
