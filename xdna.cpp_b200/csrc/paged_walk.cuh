// The work list of the attention kernels whose streams are CTAs: row tiles of R
// rows for each KV head of a request are items, tiles of kKeys keys their units
// (as many as the item's rows see), and the units of all items, in order, are
// dealt out as one equal contiguous run to every CTA.
#pragma once
#include "paged_split.cuh"

namespace xb {

// Key tiles [t0, t1) of row tile `tile`, and of one of its query tiles.
template <int R, int kKeys>
__device__ __forceinline__ void item_tiles(const AttnArgs& a, const Request& rq, int rows, int tile, int& t0, int& t1,
                                           int& hi) {
    int lo;
    key_range(a, rq, tile * R / a.group, (min(tile * R + R, rows) - 1) / a.group, lo, hi);
    t0 = lo / kKeys;
    t1 = max(t0 + 1, (hi + kKeys - 1) / kKeys);
}
template <int R, int kKeys>
__device__ __forceinline__ int item_units(const AttnArgs& a, const Request& rq, int rows, int tile) {
    int t0, t1, hi;
    item_tiles<R, kKeys>(a, rq, rows, tile, t0, t1, hi);
    return t1 - t0;
}
__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Units of all row tiles of one request (the same one on every lane), for one KV head.
template <int R, int kKeys>
__device__ __forceinline__ long long request_units(const AttnArgs& a, const Request& rq, int rows) {
    const int lane = threadIdx.x & 31, tiles = (rows + R - 1) / R;
    long long n = 0;
    for (int t = lane; t < tiles; t += 32) n += item_units<R, kKeys>(a, rq, rows, t);
    return warp_sum(n);
}

// Walks the items of a CTA's run; all lanes of a warp hold the same values.
struct Walk {
    int b, kvh, tile;
    Request rq;
    int rows, tiles;
    int t0, t1, hi;   // the item's key tiles, and the end of its keys
    int s0, s1;       // those of this run
    long long left;   // units of the run from s0 on

    template <int R, int kKeys>
    __device__ __forceinline__ void enter_request(const AttnArgs& a) {
        rq = read_request(a, b);
        rows = my_rows(a, rq);
        tiles = (rows + R - 1) / R;
    }
    template <int R, int kKeys>
    __device__ __forceinline__ void enter_item(const AttnArgs& a, int skip) {
        item_tiles<R, kKeys>(a, rq, rows, tile, t0, t1, hi);
        s0 = t0 + skip;
        s1 = static_cast<int>(min(static_cast<long long>(t1), s0 + left));
    }
    // The next item of the run; false at its end.
    template <int R, int kKeys>
    __device__ __forceinline__ bool next(const AttnArgs& a) {
        left -= s1 - s0;
        if (left <= 0) return false;
        if (++tile == tiles) {
            tile = 0;
            if (++kvh == a.kv.kv_heads) {
                kvh = 0;
                do {
                    ++b;
                    enter_request<R, kKeys>(a);
                } while (!rows);
            }
        }
        enter_item<R, kKeys>(a, 0);
        return true;
    }
};


// What start_run needs of shared memory.
template <int kThreads>
struct RunUnits {
    long long before[kThreads + 1];  // units of the requests before each thread's
    long long warps[kThreads / 32];
};

// A CTA's run: `units` units (0: none) from `first` on.
struct Run {
    Walk first;
    long long units, end;            // of the run; the unit behind it
    long long item0, all, streams;   // units before the first item, of all items; streams with work

    // What the stream leaves of an item that it began, but does not end: its last one.
    __device__ __forceinline__ SplitHead head(const Walk& w, bool first_item, long long me) const {
        const long long behind = first_item ? item0 + (w.t1 - w.t0) : end + (w.t1 - w.s1);
        return SplitHead{w.b, w.kvh, w.tile, static_cast<int>(stream_of(behind - 1, all, streams) - me + 1)};
    }
};

// The run of CTA blockIdx.x of `most`; called by all threads.  Fewer CTAs work
// when there are less than min_units units for each.
template <int R, int kKeys, int kThreads>
__device__ __forceinline__ void start_run(const AttnArgs& a, long long most, int min_units, RunUnits<kThreads>& u_of,
                                          Run& run) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.p.n_seqs;
    const int per = (B + kThreads - 1) / kThreads;
    {
        long long mine = 0;
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            Request rq{0, 0, 0};
            int rows = 0;
            if (b < B) {
                rq = read_request(a, b);
                rows = my_rows(a, rq);
            }
            const int tiles = (rows + R - 1) / R;
            long long n = 0;
            if (tiles <= 4)
                for (int t = 0; t < tiles; ++t) n += item_units<R, kKeys>(a, rq, rows, t);
            for (unsigned big = __ballot_sync(0xffffffffu, tiles > 4); big; big &= big - 1) {
                const int from = __ffs(big) - 1;  // a long request: its row tiles over all lanes
                Request r{__shfl_sync(0xffffffffu, rq.first, from), __shfl_sync(0xffffffffu, rq.count, from),
                          __shfl_sync(0xffffffffu, rq.kv, from)};
                const long long s = request_units<R, kKeys>(a, r, __shfl_sync(0xffffffffu, rows, from));
                if (lane == from) n = s;
            }
            mine += n * a.kv.kv_heads;
        }
        long long inc = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 31) u_of.warps[warp] = inc;
        __syncthreads();
        for (int w = 0; w < warp; ++w) inc += u_of.warps[w];
        u_of.before[tid + 1] = inc;
        if (tid == 0) u_of.before[0] = 0;
        __syncthreads();
    }
    const long long me = blockIdx.x;
    run.all = u_of.before[kThreads];
    run.streams = min(most, max(1LL, run.all / min_units));
    run.units = 0;
    if (me >= run.streams || run.all == 0) return;
    const long long u0 = run.all * me / run.streams;
    run.end = run.all * (me + 1) / run.streams;
    run.units = run.end - u0;
    Walk& w = run.first;
    int lo = 0, hi = kThreads;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (u_of.before[mid] <= u0) lo = mid; else hi = mid;
    }
    long long u = u_of.before[lo], one = 0;
    for (w.b = lo * per;; ++w.b) {
        w.enter_request<R, kKeys>(a);
        one = request_units<R, kKeys>(a, w.rq, w.rows);
        if (u0 < u + one * a.kv.kv_heads) break;
        u += one * a.kv.kv_heads;
    }
    w.kvh = static_cast<int>((u0 - u) / one);
    u += one * w.kvh;
    for (w.tile = 0;; w.tile += 32) {  // 32 row tiles at a time
        const int t = w.tile + lane;
        const long long n = t < w.tiles ? item_units<R, kKeys>(a, w.rq, w.rows, t) : 0;
        long long inc = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, u0 < u + inc);
        if (hit) {
            const int at = __ffs(hit) - 1;
            u += __shfl_sync(0xffffffffu, inc - n, at);
            w.tile += at;
            break;
        }
        u += __shfl_sync(0xffffffffu, inc, 31);
    }
    run.item0 = u;
    w.left = run.units;
    w.enter_item<R, kKeys>(a, static_cast<int>(u0 - u));
}

}  // namespace xb
