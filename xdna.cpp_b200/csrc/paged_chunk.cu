// Causal attention of many new tokens over a paged KV cache on the
// fifth-generation tensor cores.
//
// Mathematics as in paged_attention.cu: per row a running maximum m, l = sum
// 2^(s - m) and o = sum 2^(s - m) v, in one pass over tiles of 128 keys.
//
// A CTA works on an item of up to 2 x 128 rows (query tile q: rows 128 q ..) of
// one request and KV head.  Per tile of keys: S = Q K^T into TMEM, weights
// P = 2^(s - m) back into TMEM over S in 16 bits, O += P V in TMEM.  Roles:
//   8 warps per query tile   half a row per thread: softmax, rescaling and output
//   one warp per query tile  issues its matrix instructions (one warp for both was
//                            the bound: its waits and issues in a row took longer
//                            than the matrix unit)
//   one warp each            TMA loads of K and of V, page by page, into rings
// While one query tile is in its softmax the matrix unit works on the other
// one: their warps take turns in the exponentials.  O is rescaled only when a row's
// maximum grows by more than 8 (weights stay below 2^8), which a vote of the warp
// finds out.  The weights are rounded
// to 16 bits (the cache's type; F16 times 2^7, see Half16) because the matrix unit
// takes both factors in one type; scores, sums and O are F32.
//
// The work of all items, counted in key tiles, is dealt out in equal contiguous
// runs to one CTA per SM; items that end up cut are joined by combine_kernel.
//
// K is held as the K-major, V as the MN-major operand in 128-byte swizzled rows:
// the layout a TMA box of 64 values by 16..128 tokens has in shared memory.  D is
// cut into halves of 64 values; a box past head_dim (96) or in a block outside
// the cache reads as zeros.  Rows of V behind the last key are zeroed before
// they are used, since a weight of 0 would not hide a NaN there.
//
// Every wait is bounded (2 s of %globaltimer): one that runs out sets the error
// word, all roles give up, copies and matrix instructions in flight are waited
// for (bounded again), and TMEM is freed.
//
// Measured on a B200: 4096 rows of 32 heads of 128, BF16, over 16384 keys: 850 us in
// short bursts (1.13 PFLOP/s), 960 to 1000 us under the power cap; matrix pipe 53 %,
// exponential unit 54 %, issue 49 %.  A key tile of a query tile is one chain: S, the
// maximum, its exchange between the halves of a row, the exponentials, O and the
// next S (about 4000 clocks, of which the matrix unit has 1024 for each query tile),
// and two query tiles fill TMEM.  Heads of 256 have one query tile; its S has two
// buffers instead, so that S of the next tile is formed during the softmax (509 new
// tokens of 16 heads beside 11 requests of one token, all launches: 143 -> 135 us; 131 us now).
// Tried and slower: 64-key tiles with two buffers of S for heads of 128 (923 us in
// bursts), a whole row per thread (1044 against 1013 us), a share of the exponentials
// by a polynomial (every share), turns by an mbarrier (1115 us).
#include <algorithm>

#include "paged_split.cuh"
#include "paged_tma.cuh"
#include "paged_walk.cuh"

namespace xb {
namespace {

constexpr int kKeys = 128;
constexpr int kMinTiles = 2;   // key tiles per CTA below which fewer CTAs run
constexpr float kSlack = 8.f;  // log2 of the largest weight (before kWeightLog2)
constexpr int kTurnClocks = 4000;  // longest wait for a turn (a courtesy: nothing depends on it)

template <int D>
struct Shape {
    static constexpr int kQ = D > 128 ? 1 : 2;  // query tiles
    static constexpr int kRows = 128 * kQ;
    static constexpr int kHalves = (D + 63) / 64;
    static constexpr int kChunks = kHalves * 4;  // 16 bytes of half a row of queries
    static constexpr int kStages = D == 64 ? 4 : D <= 128 ? 2 : 1;
    static constexpr int kTile = kHalves * 128 * 128;  // bytes of 128 rows
    // 8 softmax warps and a matrix warp per query tile, a loading warp; made up to
    // whole groups of 4 warps, so that with two query tiles the softmax warps can
    // take registers from the others.  The compiler works to the launch's 96 all the
    // same: 148 bytes of a thread are spilled at heads of 64 to 128 (288 with a cap or
    // bias), none to speak of at 256 (168 registers).
    static constexpr int kThreads = kQ * 256 + 128;
    static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 104, kOtherRegs = 64;
    static_assert(kQ == 1 || 512 * kSoftmaxRegs + 128 * kOtherRegs <= 640 * kLaunchRegs, "registers of the launch");
    static constexpr int kSmem = (kQ + 2 * kStages) * kTile + 1024;  // 1024: alignment
    static constexpr int kS = 0, kO = 256, kPitch = 128;             // TMEM columns of q's S and O: + 128 q
    // One query tile leaves room for two buffers of S (columns 0 and 128), used in turn.
    static constexpr bool kTwo = kQ == 1;
    static __device__ __forceinline__ uint32_t buffer(uint32_t n) { return kTwo ? n & 1 : 0; }
    static __device__ __forceinline__ uint32_t phase(uint32_t n) { return kTwo ? n >> 1 & 1 : n & 1; }
};

struct ChunkArgs {
    SplitArgs g;
    CUtensorMap k, v;
    int box_tokens;  // tokens per TMA box: a block, or a tile of one
};

// ------------------------------------------------------------------- barriers
struct Bars {
    uint64_t kfull[4], kempty[4], vfull[4], vempty[4];
    // of each query tile; of each buffer of S; pfull: keys 0-31 and 64-95, then the others
    uint64_t qfull[2], sfull[2][2], pfull[2][2][2], ofull[2][2], drain[2];
};

// ------------------------------------------------------------ matrix unit, TMEM
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b))
                 : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
// Shared-memory operand in rows of 128 swizzled bytes, groups of 8 rows 1024
// bytes apart.  K-major (Q, K): `lead` unused.  MN-major (V): `lead` bytes
// between 64-value groups.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fff) | static_cast<uint64_t>((lead >> 4) & 0x3fff) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// kind::f16 instruction descriptor: F32 sums, 128 x n, both factors of `T`.
template <typename T>
__device__ __forceinline__ constexpr uint32_t instruction(int n, bool b_mn_major) {
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | (b_mn_major ? 1u << 16 : 0u) | static_cast<uint32_t>(n / 8) << 17 |
           (128u / 16) << 24;
}

// Waits for this thread's TMEM loads; the values go through it, so that nothing
// that uses them is moved in front.
__device__ __forceinline__ void tm_wait16(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}
// Two F32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
        "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void tm_st8(uint32_t addr, const uint32_t* u) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(u[0]), "r"(u[1]),
                 "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// What the scores go through beside the scale: nothing; a bias, a scale that is not
// positive or a cap up to kFastCap; a larger cap.
enum class Form { kPlain, kGeneral, kLargeCap };
constexpr float kFastCap = 64.f;

// post tanh(pre s).  Up to kFastCap with tanh x = 1 - 2 / (e^2x + 1), off by at most
// 2^-21 of post (2 units in the last place of the exponential and one of the
// reciprocal, of a term up to 2): 3e-5 of a weight at most, whose F16 rounding is up
// to 4.9e-4.  That does not shrink with the score, so larger caps take tanhf, whose
// error does (2048 rows of 32 heads of 128 over 4096 keys: 299 us against 230; the
// mixed step with heads of 256: 160 against 133).
template <Form kForm>
__device__ __forceinline__ float capped(float s, float pre, float post) {
    if (kForm == Form::kLargeCap) return post * tanhf(pre * s);
    const float e = exp2_fast(s * (pre * (2.f * kLog2e)));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.f));
    return fmaf(-2.f * post, r, post);
}
// True on one lane of a converged warp.  Branches on it, with addresses that are
// the same on every lane, keep what a matrix instruction takes in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ const char* shfl_ptr(const char* p, int lane) {
    return reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), lane));
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_ld16(uint32_t addr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
        : "memory");
}
// ----------------------------------------------------------------- query tiles
// The key tiles of query tile q that fall into [s0, s1): [lo, hi), empty when lo == hi.
__device__ __forceinline__ void query_tiles(const AttnArgs& a, const Walk& w, int r0, int& lo, int& hi) {
    lo = hi = 0;
    if (r0 >= w.rows) return;
    int k0, k1;
    key_range(a, w.rq, r0 / a.group, (min(r0 + 128, w.rows) - 1) / a.group, k0, k1);
    lo = max(w.s0, k0 / kKeys);
    hi = max(lo, min(w.s1, (k1 + kKeys - 1) / kKeys));
}

// Form::kPlain: the scale is folded into the exponential.
template <typename T, int D, Form kForm>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1) attn_chunk_kernel(const __grid_constant__ ChunkArgs c) {
    using L = Shape<D>;
    constexpr bool kGeneral = kForm != Form::kPlain;
    constexpr int R = L::kRows;
    extern __shared__ uint8_t raw[];
    __shared__ Bars bars;
    __shared__ RunUnits<L::kThreads> units;
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_word;
    __shared__ volatile int turns[8 * L::kQ];  // key tiles whose weights a softmax warp has formed
    __shared__ float swap[L::kQ][2][2][128];   // what the two halves of a row tell each other, twice
    volatile int* dead = &dead_word;
    const AttnArgs& a = c.g.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kLoadWarp = L::kQ * 8, kMmaWarp = kLoadWarp + 2;  // two of each (one query tile: one kMmaWarp)
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    const uint32_t qs = base, ks = qs + L::kQ * L::kTile, vs = ks + L::kStages * L::kTile;

    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            bar_init(&bars.kfull[i], 1);
            bar_init(&bars.kempty[i], L::kQ);
            bar_init(&bars.vfull[i], 1);
            bar_init(&bars.vempty[i], L::kQ);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&bars.qfull[i], 256);
            for (int j = 0; j < 2; ++j) {
                bar_init(&bars.sfull[i][j], 1);
                bar_init(&bars.pfull[i][j][0], 8);
                bar_init(&bars.pfull[i][j][1], 8);
                bar_init(&bars.ofull[i][j], 1);
            }
            bar_init(&bars.drain[i], 1);
        }
        dead_word = 0;
        for (int i = 0; i < 8 * L::kQ; ++i) turns[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    grid_wait();

    tc_before();
    Run run;
    start_run<R, kKeys, L::kThreads>(a, gridDim.x, kMinTiles, units, run);
    tc_after();
    const uint32_t tmem = tmem_slot;
    const long long me = blockIdx.x;
    if (tid == 0) c.g.heads[me].parts = 0;

    if (run.units) {
        Walk w = run.first;
        if (warp >= kLoadWarp) {
            if constexpr (L::kQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));
            if (warp < kMmaWarp) {
                // ---------------------------------------------------------------- loads
                const bool values = uniform(warp) == kLoadWarp + 1;  // one warp for K, one for V
                const CUtensorMap* map = values ? &c.v : &c.k;
                uint64_t *full = values ? bars.vfull : bars.kfull, *empty = values ? bars.vempty : bars.kempty;
                const uint32_t ring = values ? vs : ks;
                const int boxes = kKeys / c.box_tokens;  // per half; lane i looks up the block of box i
                uint32_t n = 0;                          // tiles so far
                bool ok = true;
                do {
                    const int s0 = uniform(w.s0), s1 = uniform(w.s1), kvh = uniform(w.kvh);
                    for (int t = s0; t < s1 && ok; ++t, ++n) {
                        const int j = t * kKeys + lane * c.box_tokens;
                        const bool on = lane < boxes && j < w.hi;
                        const int id = on ? key_block(a, w.b, j >> a.log_bs) : 0;
                        const int block = id < 0 ? static_cast<int>(a.kv.num_blocks) : id;  // behind the last: zeros
                        const int count = __popc(__ballot_sync(0xffffffffu, on));
                        const uint32_t stage = n % L::kStages;
                        if (n >= L::kStages) ok = bar_wait(&empty[stage], ((n / L::kStages) & 1) ^ 1, dead);
                        if (!ok) break;
                        if (elect_one()) bar_expect(&full[stage], count * L::kHalves * c.box_tokens * 128);
                        __syncwarp();
                        for (int x = 0; x < count; ++x) {
                            const int from = __shfl_sync(0xffffffffu, block, x), token = (t * kKeys + x * c.box_tokens) & (a.kv.block_size - 1);
                            if (elect_one())
#pragma unroll
                                for (int h = 0; h < L::kHalves; ++h)
                                    tma_box(ring + stage * L::kTile + h * 128 * 128 + x * c.box_tokens * 128, map, &full[stage], h * 64,
                                            token, kvh, from);
                            __syncwarp();
                        }
                    }
                } while (ok && w.next<R, kKeys>(a));
                // Copies in flight land before the CTA ends, also where the warps that they
                // are for have given up.
                for (uint32_t i = n < L::kStages ? 0 : n - L::kStages; i < n; ++i)
                    bar_wait(&full[i % L::kStages], (i / L::kStages) & 1, nullptr);
            } else if (warp < kMmaWarp + L::kQ) {
                // ----------------------------------------------------- matrix instructions
                constexpr uint32_t kIdescS = instruction<T>(kKeys, false), kIdescO = instruction<T>(D, true);
                const int q = uniform(warp) - kMmaWarp;
                const uint32_t s_at = uniform(tmem) + L::kS + q * L::kPitch, o_at = uniform(tmem) + L::kO + q * L::kPitch;
                const uint64_t q_op = operand(qs + q * L::kTile, 16), k_op = operand(ks, 16), v_op = operand(vs, 128 * 128);
                uint32_t i = 0, nq = 0, ns = 0, np = 0;  // key tiles; phases of qfull; tiles of S, and of P, so far
                bool ok = true;
                do {
                    int lo, hi;
                    query_tiles(a, w, w.tile * R + q * 128, lo, hi);
                    lo = uniform(lo), hi = uniform(hi);
                    const int s0 = uniform(w.s0), s1 = uniform(w.s1);
                    // step t: with one buffer of S, O of tile t - 1, then S of tile t; what S
                    // needs is waited for before the weights, so that it follows at once.
                    // With two, S of tile t first (the weights in its buffer, of tile t - 2,
                    // have been taken by the instructions before it).
                    for (int t = s0; t <= s1 && ok; ++t, ++i) {
                        const uint32_t k_stage = i % L::kStages, v_stage = (i + L::kStages - 1) % L::kStages;
                        const bool value = t > lo && t <= hi && t > s0, score = t >= lo && t < hi && t < s1;
                        const uint64_t v = v_op + (v_stage * L::kTile >> 4), k_at = k_op + (k_stage * L::kTile >> 4);
                        auto scores = [&] {
                            if (score) {
#pragma unroll
                                for (int k = 0; k < D / 16; ++k) {
                                    const uint32_t off = ((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4;
                                    mma_ss(s_at + L::buffer(ns) * 128, q_op + off, k_at + off, kIdescS, k > 0);
                                }
                                tc_commit(&bars.sfull[q][L::buffer(ns)]);
                            } else if (t < s1) {
                                bar_arrive(&bars.kempty[k_stage]);
                            }
                        };
                        // 16 keys k: their weights lie in half k / 4 of S's columns
                        auto weighted = [&](int k, bool add) {
                            mma_ts(o_at, s_at + L::buffer(np) * 128 + (k >> 2) * 64 + (k & 3) * 8, v + (k * 2048 >> 4),
                                   kIdescO, add);
                        };
                        if (!L::kTwo && t > s0) ok = bar_wait(&bars.vfull[v_stage], ((i - 1) / L::kStages) & 1, dead);
                        if (ok && t < s1) ok = bar_wait(&bars.kfull[k_stage], (i / L::kStages) & 1, dead);
                        if (ok && score && t == lo) ok = bar_wait(&bars.qfull[q], nq++ & 1, dead);
                        if (L::kTwo) {
                            tc_after();
                            if (ok && elect_one()) scores();
                            __syncwarp();
                            if (ok && t > s0) ok = bar_wait(&bars.vfull[v_stage], ((i - 1) / L::kStages) & 1, dead);
                        }
                        if (ok && value) ok = bar_wait(&bars.pfull[q][L::buffer(np)][0], L::phase(np), dead);
                        tc_after();
                        if (ok && value && elect_one()) {
                            weighted(0, t - 1 > lo);
                            weighted(1, true);
                            weighted(4, true);
                            weighted(5, true);
                        }
                        __syncwarp();
                        if (ok && value) ok = bar_wait(&bars.pfull[q][L::buffer(np)][1], L::phase(np), dead);
                        tc_after();
                        if (ok && elect_one()) {
                            if (value) {
                                weighted(2, true);
                                weighted(3, true);
                                weighted(6, true);
                                weighted(7, true);
                                if (L::kTwo) tc_commit(&bars.vempty[v_stage]);
                                if (L::kTwo || t == hi) tc_commit(&bars.ofull[q][L::buffer(np)]);
                            } else if (t > s0) {
                                bar_arrive(&bars.vempty[v_stage]);
                            }
                            if (!L::kTwo) scores();
                        }
                        __syncwarp();
                        ns += score, np += value;
                    }
                    --i;  // the last step has no tile of its own
                } while (ok && w.next<R, kKeys>(a));
                // matrix instructions in flight end before TMEM is freed, whoever has given up
                if (elect_one()) tc_commit(&bars.drain[q]);
                __syncwarp();
                bar_wait(&bars.drain[q], 0, nullptr);
            }
        } else {
            // ------------------------------------------------------------------ softmax
            if constexpr (L::kQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegs));
            // Warps 8 q + 4 h + i: rows 32 i .. of query tile q, half h of the columns
            const int q = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
            const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
            const uint32_t s_base = tmem + lanes + L::kS + q * L::kPitch + half * 64;
            const uint32_t o_at = tmem + lanes + L::kO + q * L::kPitch + half * (D / 2);
            // 16 bytes x of the warp's row r in the query tile; x of its half, [kChunks half,
            // kChunks (half + 1)), are touched by this warp alone
            const uint32_t q_at = qs + q * L::kTile + (warp & 3) * 32 * 128;
            auto chunk_at = [&](int r, int x) {
                return q_at + r * 128 + (x >> 3) * 128 * 128 + (((x & 7) ^ (r & 7)) << 4);
            };
            uint32_t ns = 0, no = 0, nx = 0;  // key tiles of this query tile, items, exchanges so far
            uint32_t n = 0;                   // key tiles before the item's
            int mine = 0, theirs = 0;         // key tiles of this and of the other query tile before the item's
            bool first_item = true;
            // The value of the thread that holds the row's other half.  Both warps of a
            // pair pass here equally often, whatever their waits return: a warp whose wait
            // has run out goes through the rest of its tiles all the same.
            auto other_half = [&](float x) {
                swap[q][nx & 1][half][row] = x;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + q * 4 + (warp & 3)) : "memory");
                return swap[q][nx++ & 1][half ^ 1][row];
            };
            do {
                const int r0 = w.tile * R + q * 128, rr = r0 + row;
                if (r0 < w.rows) {
                    int lo, hi, other_lo = 0, other_hi = 0;
                    query_tiles(a, w, r0, lo, hi);
                    if (L::kQ == 2) query_tiles(a, w, w.tile * R + (q ^ 1) * 128, other_lo, other_hi);
                    const bool on = rr < w.rows;
                    const int token = (on ? rr : r0) / a.group, head = w.kvh * a.group + (on ? rr - token * a.group : 0);
                    const int pos = w.rq.pos0() + token;
                    const int last = min(pos, w.hi - 1), first = a.p.window > 0 && pos >= a.p.window ? pos - a.p.window + 1 : 0;
                    const float slope = kGeneral ? head_slope(a, head) : 0.f;
                    float m = -INFINITY, l = 0.f;
                    if (lo < hi) {
                        // Half of the rows' queries into the swizzled rows the matrix unit reads: lanes
                        // side by side take what is side by side of a row.
                        const char* src = static_cast<const char*>(a.p.q) + (w.rq.first + token) * a.p.nb_q +
                                          static_cast<int64_t>(head) * D * 2;
#pragma unroll
                        for (int i = 0; i < L::kChunks; ++i) {
                            const int r = i * (32 / L::kChunks) + lane / L::kChunks, x = half * L::kChunks + lane % L::kChunks;
                            const uint4* from = reinterpret_cast<const uint4*>(shfl_ptr(on ? src : nullptr, r));
                            uint4 v = make_uint4(0, 0, 0, 0);
                            if (from && x < D / 8) v = __ldg(from + x);
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(r, x)),
                                         "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                                         : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        tc_before();  // O of the last item has been read
                        bar_arrive(&bars.qfull[q]);
                        // keys that every row of this query tile sees
                        const int p0 = w.rq.pos0() + r0 / a.group;
                        const int p1 = w.rq.pos0() + (min(r0 + 128, w.rows) - 1) / a.group;
                        const int all_hi = min(p0 + 1, w.hi);
                        const int all_lo = a.p.window > 0 && p1 >= a.p.window ? p1 - a.p.window + 1 : 0;
                        for (int t = lo; t < hi; ++t, ++ns) {
                            bar_wait(&bars.sfull[q][L::buffer(ns)], L::phase(ns), dead);
                            // O of the tile two before was ordered ahead of S; its phase is passed on every
                            // tile, so that the one waited for below is never mistaken for it
                            if (L::kTwo && ns >= 2) bar_wait(&bars.ofull[q][L::buffer(ns)], L::phase(ns - 2), dead);
                            tc_after();
                            const uint32_t s_at = s_base + L::buffer(ns) * 128;
                            // S is there: K is free.  With one buffer of S, so are O of the tile
                            // before and that tile's V.
                            if (row == 0 && half == 0) {
                                const uint32_t x = n + t - w.s0;
                                bar_arrive(&bars.kempty[x % L::kStages]);
                                if (!L::kTwo && t > lo) bar_arrive(&bars.vempty[(x - 1) % L::kStages]);
                            }
                            const int j0 = t * kKeys + half * 64;
                            const bool cut = t * kKeys < all_lo || (t + 1) * kKeys > all_hi;
                            const float pre = kGeneral ? 1.f : a.pre;
                            const int k0 = first - j0, k1 = last - j0;
                            // Columns of S, 16 worked on and 16 on their way (16 softmax warps leave no
                            // registers for more).  First pass: the maximum of half the row, in eight
                            // chains.  Scores that the cap, the bias or a hidden key change go back
                            // for the second pass.
                            float s0[16], s1[16], tops[8];
                            auto look = [&](float (&s)[16], int col) {
                                if (kGeneral || cut) {
                                    if (kGeneral) {
                                        if (a.post != 0.f)
#pragma unroll
                                            for (int i = 0; i < 16; ++i) s[i] = capped<kForm>(s[i], a.pre, a.post);
                                        else
#pragma unroll
                                            for (int i = 0; i < 16; ++i) s[i] *= a.pre;
                                        if (a.bias_near)
#pragma unroll
                                            for (int i = 0; i < 16; ++i)
                                                s[i] = fmaf(slope, static_cast<float>(j0 + col + i - pos), s[i]);
                                    }
                                    if (cut)
#pragma unroll
                                    for (int i = 0; i < 16; ++i)
                                        if (i < k0 - col || i > k1 - col) s[i] = -INFINITY;
                                    tm_st16(s_at + col, reinterpret_cast<const uint32_t*>(s));
                                }
#pragma unroll
                                for (int i = 0; i < 8; ++i) tops[i] = col ? max3(tops[i], s[i], s[i + 8]) : fmaxf(s[i], s[i + 8]);
                            };
                            tm_ld16(s_at, s0);
                            tm_wait16(s0);
                            tm_ld16(s_at + 16, s1);
                            look(s0, 0);
                            tm_wait16(s1);
                            tm_ld16(s_at + 32, s0);
                            look(s1, 16);
                            tm_wait16(s0);
                            tm_ld16(s_at + 48, s1);
                            look(s0, 32);
                            tm_wait16(s1);
                            look(s1, 48);
                            if (kGeneral || cut) tm_wait_st();
                            tm_ld16(s_at, s0);
                            float top = max3(max3(tops[0], tops[1], tops[2]), max3(tops[3], tops[4], tops[5]),
                                             fmaxf(tops[6], tops[7]));
                            top *= pre;
                            top = fmaxf(top, other_half(top));
                            if (__any_sync(0xffffffffu, top > m + kSlack)) {  // both halves alike
                                const float was = m;
                                m = fmaxf(m, top);
                                const float f = m == -INFINITY ? 1.f : exp2_fast(was - m);
                                l *= f;
                                if (t > lo) {
                                    if (L::kTwo) {  // once O has the tile before
                                        bar_wait(&bars.ofull[q][L::buffer(ns - 1)], L::phase(ns - 1), dead);
                                        tc_after();
                                    }
#pragma unroll 1
                                    for (int i = 0; i < D / 32; ++i) {
                                        float o[16];
                                        tm_ld16(o_at + i * 16, o);
                                        tm_wait16(o);
#pragma unroll
                                        for (int e = 0; e < 16; ++e) o[e] *= f;
                                        tm_st16(o_at + i * 16, reinterpret_cast<const uint32_t*>(o));
                                    }
                                }
                            }
                            if ((t + 1) * kKeys > w.hi) {  // values of keys that do not exist: a weight of 0 would not hide a NaN
                                const uint32_t x = n + t - w.s0, stage = x % L::kStages;
                                bar_wait(&bars.vfull[stage], (x / L::kStages) & 1, dead);
                                const int gone = max(w.hi - t * kKeys, 0);
                                for (int y = half * 128 + row; y < (kKeys - gone) * 8 * L::kHalves; y += 256)
                                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                                                     vs + stage * L::kTile + (y % (8 * L::kHalves) >> 3) * 128 * 128 +
                                                     (gone + y / (8 * L::kHalves)) * 128 + (y & 7) * 16),
                                                 "r"(0)
                                                 : "memory");
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            }
                            const float off = m == -INFINITY ? 0.f : Half16<T>::kWeightLog2 - m;
                            // The two query tiles' warps on a scheduler take turns in the exponentials,
                            // so that the matrix unit has the other one's work meanwhile (left alone
                            // they run in step, and the matrix unit waits for both).
                            if (L::kQ == 2) {
                                const int due = theirs + min(max(t + q - other_lo, 0), other_hi - other_lo);
                                const long long since = clock64();
                                while (turns[warp ^ 8] < due && clock64() - since < kTurnClocks) {}
                                __syncwarp();
                            }
                            const float2 pre2 = make_float2(pre, pre), off2 = make_float2(off, off);
                            // Second pass: the weights.
                            float2 sum[2] = {};
                            auto weigh = [&](const float (&s)[16], int col) {
                                uint32_t p[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    float2 x = fma2(make_float2(s[2 * i], s[2 * i + 1]), pre2, off2);
                                    x = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                                    sum[i & 1] = add2(sum[i & 1], x);
                                    p[i] = Half16<T>::pack(x.x, x.y);
                                }
                                tm_st8(s_at + col / 2, p);
                            };
                            tm_wait16(s0);
                            tm_ld16(s_at + 16, s1);
                            weigh(s0, 0);
                            tm_wait16(s1);
                            tm_ld16(s_at + 32, s0);
                            weigh(s1, 16);
                            auto hand_over = [&](int part) {  // weights the matrix unit may take
                                tm_wait_st();
                                tc_before();
                                __syncwarp();
                                if (lane == 0) bar_arrive(&bars.pfull[q][L::buffer(ns)][part]);
                            };
                            hand_over(0);
                            tm_wait16(s0);
                            tm_ld16(s_at + 48, s1);
                            weigh(s0, 32);
                            tm_wait16(s1);
                            weigh(s1, 48);
                            hand_over(1);
                            if (L::kQ == 2 && lane == 0) turns[warp] = mine + t + 1 - lo;
                            const float2 both = add2(sum[0], sum[1]);
                            l += both.x + both.y;
                        }
                        l += other_half(l);
                        if (L::kTwo)
                            bar_wait(&bars.ofull[q][L::buffer(ns - 1)], L::phase(ns - 1), dead);
                        else
                            bar_wait(&bars.ofull[q][0], no++ & 1, dead);
                        tc_after();
                        if (!L::kTwo && row == 0 && half == 0)
                            bar_arrive(&bars.vempty[(n + hi - 1 - w.s0) % L::kStages]);
                    }
                    // half of O to the output, or to the item's partial
                    const bool whole = w.s0 == w.t0 && w.s1 == w.t1;
                    const float inv = l == 0.f ? 0.f : whole ? 1.f / l : 1.f;
                    float* part = c.g.parts + (static_cast<size_t>(me) * 2 + (w.s0 == w.t0)) * part_floats(R, D);
                    // A thread holds a row, and 32 rows at once would cost a store 32 transactions:
                    // 64 bytes of each go through the queries' place, which has been read, and out
                    // with four lanes a row.  With the loads of the queries that go the same way:
                    // 300 tokens of 32 heads over 4300 keys, 62.5 -> 54.3 us.
                    const bool wide = !whole || a.p.out_type == GGML_TYPE_F32;
                    const char* to = whole ? static_cast<const char*>(a.p.out) + (w.rq.first + token) * a.p.nb_out +
                                                 (static_cast<int64_t>(head) * D + half * (D / 2)) * (wide ? 4 : 2)
                                           : reinterpret_cast<const char*>(part + static_cast<size_t>(q * 128 + row) * D +
                                                                           half * (D / 2));
                    if (!on) to = nullptr;
                    auto put = [&](int x, uint4 v) {
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(lane, half * L::kChunks + x)),
                                     "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                                     : "memory");
                    };
                    auto flush = [&](int chunks, int offset) {  // of 16 bytes, to `offset` bytes on in each row
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < chunks; ++k) {
                            const int r = (k * 32 + lane) / chunks, x = (k * 32 + lane) % chunks;
                            uint4 v;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                         : "r"(chunk_at(r, half * L::kChunks + x)));
                            const char* p = shfl_ptr(to, r);
                            if (p) *reinterpret_cast<uint4*>(const_cast<char*>(p) + offset + x * 16) = v;
                        }
                        __syncwarp();
                    };
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        float o[16];
                        if (lo < hi) {
                            tm_ld16(o_at + i * 16, o);
                            tm_wait16(o);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = l == 0.f ? 0.f : o[e] * inv;
                        if (wide) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                put(e, make_uint4(__float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]),
                                                  __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3])));
                            flush(4, i * 64);
                        } else {
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                put((i & 1) * 2 + e, make_uint4(Half16<T>::pack(o[8 * e], o[8 * e + 1]),
                                                                Half16<T>::pack(o[8 * e + 2], o[8 * e + 3]),
                                                                Half16<T>::pack(o[8 * e + 4], o[8 * e + 5]),
                                                                Half16<T>::pack(o[8 * e + 6], o[8 * e + 7])));
                            if (i & 1)
                                flush(4, (i - 1) * 32);
                            else if (i == D / 32 - 1)
                                flush(2, i * 32);
                        }
                    }
                    if (!whole && on && half == 0) {
                        part[R * D + q * 128 + row] = m;
                        part[R * D + R + q * 128 + row] = l;
                    }
                }
                if (tid == 0 && w.s0 == w.t0 && w.s1 < w.t1) {
                    c.g.heads[me] = run.head(w, first_item, me);
                }
                first_item = false;
                int lo, hi;
                query_tiles(a, w, r0, lo, hi);
                mine += hi - lo;
                if (L::kQ == 2) query_tiles(a, w, w.tile * R + (q ^ 1) * 128, lo, hi);
                theirs += hi - lo;
                n += w.s1 - w.s0;
            } while (w.next<R, kKeys>(a));
        }
    }

    tc_before();
    __syncthreads();
    tc_after();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// ------------------------------------------------------------------------ host
template <typename T, int D, Form kForm>
cudaError_t launch_form(const ChunkArgs& c, cudaStream_t stream) {
    using L = Shape<D>;
    constexpr auto kernel = attn_chunk_kernel<T, D, kForm>;
    const cudaError_t e = allow_smem<kernel>(L::kSmem);
    if (e != cudaSuccess) return e;
    const unsigned sms = static_cast<unsigned>(sm_count());
    const cudaError_t f = launch_pdl(kernel, dim3(sms), dim3(L::kThreads), L::kSmem, stream, 1, c);
    if (f != cudaSuccess) return f;
    const AttnArgs& a = c.g.a;
    const int64_t items = (a.p.n_tokens * a.group / L::kRows + 1) * a.kv.kv_heads;
    return combine_launch<D, L::kRows>(c.g, items, stream);
}
template <typename T, int D>
cudaError_t launch_dim(const ChunkArgs& c, cudaStream_t stream) {
    const AttnArgs& a = c.g.a;
    if (a.p.logit_softcap > kFastCap) return launch_form<T, D, Form::kLargeCap>(c, stream);
    return a.post != 0.f || a.bias_near || !(a.pre > 0.f) ? launch_form<T, D, Form::kGeneral>(c, stream)
                                                          : launch_form<T, D, Form::kPlain>(c, stream);
}
template <typename T>
cudaError_t launch_type(const ChunkArgs& c, cudaStream_t stream) {
    switch (c.g.a.kv.head_dim) {
        case 64: return launch_dim<T, 64>(c, stream);
        case 96: return launch_dim<T, 96>(c, stream);
        case 128: return launch_dim<T, 128>(c, stream);
        default: return launch_dim<T, 256>(c, stream);
    }
}

}  // namespace

size_t chunk_workspace(const AttnArgs& a) {
    return split_bytes(static_cast<size_t>(sm_count()), a.kv.head_dim > 128 ? 128 : 256, a.kv.head_dim);
}

cudaError_t chunk_launch(const AttnArgs& a, cudaStream_t stream) {
    ChunkArgs c;
    c.g = split_args(a, static_cast<size_t>(sm_count()));
    c.box_tokens = std::min(a.kv.block_size, kKeys);
    if (!cache_map(&c.k, a.kv, a.kv.k, c.box_tokens) || !cache_map(&c.v, a.kv, a.kv.v, c.box_tokens))
        return cudaErrorInvalidValue;
    return a.kv.type == GGML_TYPE_F16 ? launch_type<__half>(c, stream) : launch_type<__nv_bfloat16>(c, stream);
}

cudaError_t chunk_error(int* out) { return take_wait_error(out); }

}  // namespace xb
