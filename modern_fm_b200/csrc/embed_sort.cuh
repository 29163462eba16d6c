// embed_sort.cuh — stable radix sort of one batch's ids with their positions,
// into a workspace of the caller: no allocation, no host round trip, no block
// waits for another, so a call can be captured and its launches replayed.
//
// Ids outside the table get the key n_rows and sort behind every real id. Least
// significant digit first, 8 bits a pass, in the tiles of segsort.cuh's
// scatter: a tile is ranked by match_any per warp, reordered in shared memory
// and written in runs. Two things differ from the training plan's sort, because
// one batch of some 10^5 ids is bound by its launches, not by its bytes:
//  * a pass's scatter counts the next pass's digits while it writes (integer
//    adds, grouped per warp), so only the first pass has a counting launch;
//  * up to kFuseTiles tiles, each tile sums the counts before it by itself
//    (at most 192 KB of L2 reads), which saves the prefix launch; more
//    tiles take one prefix launch a pass.
// Up to kSmallSort ids one block does every pass in shared memory.
#pragma once

#include "scan.cuh"
#include "vecio.cuh"

namespace mfm {

constexpr int kETileNT = 256;
constexpr int kETileItems = 8;
constexpr int kETile = kETileNT * kETileItems;
constexpr int kFuseTiles = 192;
constexpr int kSmallNT = 1024;
constexpr int kSmallItems = 8;
constexpr int64_t kSmallSort = (int64_t)kSmallNT * kSmallItems;

// The key of entry q: its id, or n_rows for padding (an id outside the table, or
// an entry of no row).
template <class I>
__device__ __forceinline__ uint32_t id_key(const I* ids, const int32_t* row_of, int64_t q,
                                           int64_t n_rows) {
    const I id = ids[q];
    const bool live = id >= 0 && (int64_t)id < n_rows && (!row_of || row_of[q] >= 0);
    return live ? (uint32_t)id : (uint32_t)n_rows;
}

// Digit counts of the first pass by tile, and zeros for the passes after it.
template <class I>
__global__ void __launch_bounds__(kETileNT)
    id_count_kernel(const I* __restrict__ ids, const int32_t* __restrict__ row_of, int64_t n,
                    int64_t n_rows, int passes,
                    int64_t n_tiles, uint32_t* __restrict__ counts) {
    __shared__ uint32_t h[256];
    const int t = threadIdx.x;
    const int64_t tile = blockIdx.x, lo = tile * kETile;
    h[t] = 0;
    for (int p = 1; p < passes; ++p) counts[(p * n_tiles + tile) * 256 + t] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kETileItems; ++i) {
        const int64_t q = lo + t + i * kETileNT;
        if (q < n) atomicAdd(&h[id_key(ids, row_of, q, n_rows) & 255u], 1u);
    }
    __syncthreads();
    counts[tile * 256 + t] = h[t];
}

// For batches of more than kFuseTiles tiles: block d turns digit d's counts into
// their prefix over the tiles, in place, and writes the digit's total.
__global__ void __launch_bounds__(256)
    id_prefix_kernel(uint32_t* __restrict__ counts, int64_t n_tiles,
                     uint32_t* __restrict__ totals) {
    __shared__ uint32_t sm[8];
    const int d = blockIdx.x;
    uint32_t run = 0;
    for (int64_t b = 0; b < n_tiles; b += 256) {
        const int64_t t = b + threadIdx.x;
        const uint32_t c = t < n_tiles ? counts[t * 256 + d] : 0u;
        uint32_t all;
        const uint32_t ex = block_exclusive_scan<uint32_t, 256>(c, sm, all);
        if (t < n_tiles) counts[t * 256 + d] = run + ex;
        run += all;
    }
    if (threadIdx.x == 0) totals[d] = run;
}

// One pass of one tile. FIRST: keys come from the ids, values are positions.
// FUSED: `counts` holds digit counts and the tile adds up those before it;
// otherwise it holds their prefix over the tiles, and `totals` the digits' sums.
// next != NULL: the next pass's counts.
template <class I, bool FIRST, bool FUSED>
__global__ void __launch_bounds__(kETileNT)
    id_scatter_kernel(const I* __restrict__ ids, const int32_t* __restrict__ row_of,
                      const uint32_t* __restrict__ kin,
                      const uint32_t* __restrict__ vin, uint32_t* __restrict__ kout,
                      uint32_t* __restrict__ vout, int64_t n, int64_t n_rows, int64_t n_tiles,
                      int shift, const uint32_t* __restrict__ counts,
                      const uint32_t* __restrict__ totals, uint32_t* __restrict__ next) {
    constexpr int NW = kETileNT / 32;
    __shared__ uint32_t cnt[NW][256];
    __shared__ uint32_t base[256];
    __shared__ uint32_t scan_sm[NW];
    __shared__ uint2 skv[kETile];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t tile = blockIdx.x, lo = tile * kETile;
    const int m = (int)(n - lo < kETile ? n - lo : kETile);
    const int q0 = warp * (32 * kETileItems) + lane;  // striped: a warp's items are in position order
    for (int i = t; i < NW * 256; i += kETileNT) (&cnt[0][0])[i] = 0;
    uint32_t key[kETileItems], val[kETileItems], rank[kETileItems];
#pragma unroll
    for (int i = 0; i < kETileItems; ++i) {
        const int q = q0 + i * 32;
        key[i] = 0;
        val[i] = 0;
        if (q < m) {
            key[i] = FIRST ? id_key(ids, row_of, lo + q, n_rows) : kin[lo + q];
            val[i] = FIRST ? (uint32_t)(lo + q) : vin[lo + q];
        }
    }
    uint32_t dtotal = 0, before = 0, all;
    if (FUSED) {
#pragma unroll 8
        for (int64_t b = 0; b < n_tiles; ++b) {
            const uint32_t c = counts[b * 256 + t];
            dtotal += c;
            before += b < tile ? c : 0u;
        }
    } else {
        dtotal = totals[t];
        before = counts[tile * 256 + t];
    }
    const uint32_t goff = block_exclusive_scan<uint32_t, kETileNT>(dtotal, scan_sm, all) + before;
    const unsigned lt = (1u << lane) - 1u;
#pragma unroll
    for (int i = 0; i < kETileItems; ++i) {
        const bool valid = q0 + i * 32 < m;
        const uint32_t d = valid ? (key[i] >> shift) & 255u : 256u + (uint32_t)lane;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const int leader = __ffs(peers) - 1;
        uint32_t b = 0;
        if (valid && lane == leader) {
            b = cnt[warp][d];
            cnt[warp][d] = b + (uint32_t)__popc(peers);
        }
        b = __shfl_sync(0xffffffffu, b, leader);
        rank[i] = b + (uint32_t)__popc(peers & lt);
        __syncwarp();
    }
    __syncthreads();
    uint32_t tot = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const uint32_t c = cnt[w][t];
        cnt[w][t] = tot;
        tot += c;
    }
    const uint32_t dstart = block_exclusive_scan<uint32_t, kETileNT>(tot, scan_sm, all);
#pragma unroll
    for (int w = 0; w < NW; ++w) cnt[w][t] += dstart;
    base[t] = goff - dstart;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kETileItems; ++i)
        if (q0 + i * 32 < m) {
            const uint32_t d = (key[i] >> shift) & 255u;
            skv[cnt[warp][d] + rank[i]] = make_uint2(key[i], val[i]);
        }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kETileItems; ++u) {
        const int j = t + u * kETileNT;
        const bool valid = j < m;
        uint32_t bin = 0xffffffffu;
        if (valid) {
            const uint2 e = skv[j];
            const uint32_t dst = base[(e.x >> shift) & 255u] + (uint32_t)j;
            kout[dst] = e.x;
            vout[dst] = e.y;
            // n < 2^31 entries: at most 2^20 tiles, so tile and digit fit 28 bits
            bin = (dst / kETile) * 256u + ((e.x >> (shift + 8)) & 255u);
        }
        if (next) {  // uniform over the block
            const unsigned peers = __match_any_sync(0xffffffffu, bin);
            if (valid && lane == __ffs(peers) - 1) atomicAdd(next + bin, (uint32_t)__popc(peers));
        }
    }
}

// All passes of up to NT * ITEMS ids in one block.
template <class I, int NT, int ITEMS>
__global__ void __launch_bounds__(NT)
    id_sort_small_kernel(const I* __restrict__ ids, const int32_t* __restrict__ row_of, int n, int64_t n_rows, int key_bits,
                         uint32_t* __restrict__ kout, uint32_t* __restrict__ vout) {
    constexpr int NW = NT / 32;
    extern __shared__ uint32_t dyn[];
    uint32_t(*cnt)[256] = reinterpret_cast<uint32_t(*)[256]>(dyn);  // NW x 256
    uint2* skv = reinterpret_cast<uint2*>(dyn + NW * 256);          // NT * ITEMS
    __shared__ uint32_t scan_sm[NW];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int q0 = warp * (32 * ITEMS) + lane;
    uint32_t key[ITEMS], val[ITEMS], rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int q = q0 + i * 32;
        key[i] = q < n ? id_key(ids, row_of, q, n_rows) : 0u;
        val[i] = (uint32_t)q;
    }
    const unsigned lt = (1u << lane) - 1u;
    for (int shift = 0; shift < key_bits; shift += 8) {
        for (int i = t; i < NW * 256; i += NT) (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool valid = q0 + i * 32 < n;
            const uint32_t d = valid ? (key[i] >> shift) & 255u : 256u + (uint32_t)lane;
            const unsigned peers = __match_any_sync(0xffffffffu, d);
            const int leader = __ffs(peers) - 1;
            uint32_t b = 0;
            if (valid && lane == leader) {
                b = cnt[warp][d];
                cnt[warp][d] = b + (uint32_t)__popc(peers);
            }
            b = __shfl_sync(0xffffffffu, b, leader);
            rank[i] = b + (uint32_t)__popc(peers & lt);
            __syncwarp();
        }
        __syncthreads();
        uint32_t tot = 0;
        if (t < 256)
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const uint32_t c = cnt[w][t];
                cnt[w][t] = tot;
                tot += c;
            }
        uint32_t all;
        const uint32_t dstart = block_exclusive_scan<uint32_t, NT>(tot, scan_sm, all);
        if (t < 256)
#pragma unroll
            for (int w = 0; w < NW; ++w) cnt[w][t] += dstart;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (q0 + i * 32 < n) {
                const uint32_t d = (key[i] >> shift) & 255u;
                skv[cnt[warp][d] + rank[i]] = make_uint2(key[i], val[i]);
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int q = q0 + i * 32;
            if (q < n) {
                const uint2 e = skv[q];
                key[i] = e.x;
                val[i] = e.y;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int q = q0 + i * 32;
        if (q < n) {
            kout[q] = key[i];
            vout[q] = val[i];
        }
    }
}

inline int id_key_bits(int64_t n_rows) {  // keys 0 .. n_rows
    int b = 1;
    while (b < 32 && ((int64_t)1 << b) <= n_rows) ++b;
    return b;
}

// Workspace of a sort of n ids, in 32-bit words: two key / value pairs and the
// passes' counts.
struct IdSortPlan {
    int64_t n = 0, n_tiles = 0;
    int key_bits = 1, passes = 1;
    int64_t words = 0;
    IdSortPlan(int64_t n_, int64_t n_rows) : n(n_) {
        key_bits = id_key_bits(n_rows);
        passes = (key_bits + 7) / 8;
        n_tiles = ceil_div(n, kETile);
        words = 4 * n + (n > kSmallSort ? ((int64_t)passes * n_tiles + 1) * 256 : 0);
    }
};

struct IdSorted {
    const uint32_t* keys;
    const uint32_t* pos;
};

template <class I>
IdSorted sort_ids(const IdSortPlan& P, const I* ids, const int32_t* row_of, int64_t n_rows,
                  uint32_t* ws, cudaStream_t s) {
    const int64_t n = P.n;
    uint32_t *k0 = ws, *v0 = ws + n, *k1 = ws + 2 * n, *v1 = ws + 3 * n, *counts = ws + 4 * n;
    if (n <= kSmallSort) {
        if (n <= 1024) {
            constexpr int NT = 256, IT = 4, SM = (NT / 32) * 1024 + NT * IT * 8;
            id_sort_small_kernel<I, NT, IT><<<1, NT, SM, s>>>(ids, row_of, (int)n, n_rows, P.key_bits, k0, v0);
        } else {
            constexpr int SM = (kSmallNT / 32) * 1024 + (int)kSmallSort * 8;
            auto k = id_sort_small_kernel<I, kSmallNT, kSmallItems>;
            MFM_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SM), "id sort shared memory");
            k<<<1, kSmallNT, SM, s>>>(ids, row_of, (int)n, n_rows, P.key_bits, k0, v0);
        }
        MFM_CHECK_LAUNCH("id sort launch");
        return {k0, v0};
    }
    const unsigned g = (unsigned)P.n_tiles;
    const bool fused = P.n_tiles <= kFuseTiles;
    uint32_t* totals = counts + (int64_t)P.passes * P.n_tiles * 256;
    id_count_kernel<I><<<g, kETileNT, 0, s>>>(ids, row_of, n, n_rows, P.passes, P.n_tiles, counts);
    uint32_t *ki = k1, *vi = v1, *ko = k0, *vo = v0;
    for (int p = 0; p < P.passes; ++p) {
        uint32_t* c = counts + (int64_t)p * P.n_tiles * 256;
        uint32_t* next = p + 1 < P.passes ? c + P.n_tiles * 256 : nullptr;
        if (!fused) id_prefix_kernel<<<256, 256, 0, s>>>(c, P.n_tiles, totals);
        if (p == 0 && fused)
            id_scatter_kernel<I, true, true><<<g, kETileNT, 0, s>>>(ids, row_of, ki, vi, ko, vo, n, n_rows, P.n_tiles, 8 * p, c, totals, next);
        else if (p == 0)
            id_scatter_kernel<I, true, false><<<g, kETileNT, 0, s>>>(ids, row_of, ki, vi, ko, vo, n, n_rows, P.n_tiles, 8 * p, c, totals, next);
        else if (fused)
            id_scatter_kernel<I, false, true><<<g, kETileNT, 0, s>>>(ids, row_of, ki, vi, ko, vo, n, n_rows, P.n_tiles, 8 * p, c, totals, next);
        else
            id_scatter_kernel<I, false, false><<<g, kETileNT, 0, s>>>(ids, row_of, ki, vi, ko, vo, n, n_rows, P.n_tiles, 8 * p, c, totals, next);
        std::swap(ki, ko);
        std::swap(vi, vo);
    }
    MFM_CHECK_LAUNCH("id sort launch");
    return {ki, vi};
}

}  // namespace mfm
