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

#include <type_traits>

#include "scan.cuh"
#include "vecio.cuh"

namespace mfm {

constexpr int kETileNT = 256;
constexpr int kETileItems = 8;
constexpr int kETile = kETileNT * kETileItems;
constexpr int kFuseTiles = 192;
constexpr int64_t kSmallSort = 2048;

// The entries of a batch: their ids and, where they are summed by rows, the rows'
// bounds (indptr, n_out + 1; NULL: every entry is a row of its own).
template <class I>
struct Entries {
    const I* ids;
    int64_t n;
    const int64_t* indptr;
    int64_t n_out, n_rows;
    // The rows that M x 32 consecutive entries belong to, one warp, lane l's i-th
    // being q0 + 32 i + l; -1 for none: the first row whose end is behind the entry,
    // if it begins at or before it. The warp finds the first entry's row (32 probes
    // a round), takes the ends of the 32 rows from there, one a lane, and looks
    // its entries up among them; entries behind all of those bisect the rest. Any
    // bounds give an answer in [-1, n_out), decreasing ones too.
    template <int M>
    __device__ __forceinline__ void rows(int64_t q0, int32_t (&r)[M]) const {
        if (!indptr) {
#pragma unroll
            for (int i = 0; i < M; ++i) r[i] = 0;
            return;
        }
        const int lane = threadIdx.x & 31;
        int32_t base = 0, len = (int32_t)n_out;  // the first row is in [base, base + len]
        while (len > 0) {
            const int32_t step = (len + 31) / 32;
            const int64_t p = (int64_t)(lane + 1) * step;
            const bool ends = p <= len && indptr[base + p] <= q0;
            const int n = __popc(__ballot_sync(0xffffffffu, ends));
            base += n * step;
            const int32_t rest = len - n * step;
            len = rest < step - 1 ? (rest > 0 ? rest : 0) : step - 1;
        }
        const int64_t end = base + lane < n_out ? indptr[base + lane + 1] : INT64_MAX;
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int64_t q = q0 + 32 * i + lane;
            int32_t k = 0;  // how many of the 32 rows end at or before q
#pragma unroll
            for (int w = 16; w > 0; w >>= 1)
                if (__shfl_sync(0xffffffffu, end, k + w - 1) <= q) k += w;
            if (__shfl_sync(0xffffffffu, end, k) <= q) ++k;
            int64_t lo = (int64_t)base + k;
            if (k == 32) {
                int64_t hi = n_out;
                while (lo < hi) {
                    const int64_t mid = (lo + hi) >> 1;
                    if (indptr[mid + 1] > q)
                        hi = mid;
                    else
                        lo = mid + 1;
                }
            }
            r[i] = lo < n_out && indptr[lo] <= q ? (int32_t)lo : -1;
        }
    }
    // The sort key of entry q: its id, or n_rows for padding (an id outside the
    // table, or an entry of no row).
    __device__ __forceinline__ uint32_t key(int64_t q, int32_t row) const {
        const I id = ids[q];
        return id >= 0 && (int64_t)id < n_rows && row >= 0 ? (uint32_t)id : (uint32_t)n_rows;
    }
};

// Keys and rows of all entries, digit counts of the first pass by tile, and zeros
// for the passes after it and for the block count of the kernels behind the sort.
template <class I>
__global__ void __launch_bounds__(kETileNT)
    id_count_kernel(Entries<I> in, int passes, int64_t n_tiles, uint32_t* __restrict__ keys,
                    int32_t* __restrict__ row_of, uint32_t* __restrict__ counts,
                    unsigned* __restrict__ done) {
    __shared__ uint32_t h[256];
    const int t = threadIdx.x;
    const int64_t tile = blockIdx.x, lo = tile * kETile;
    h[t] = 0;
    if (tile == 0 && t == 0) *done = 0;
    for (int p = 1; p < passes; ++p) counts[(p * n_tiles + tile) * 256 + t] = 0;
    __syncthreads();
    const int64_t q0 = lo + (t / 32) * (32 * kETileItems);
    int32_t r[kETileItems];
    in.rows(q0, r);
#pragma unroll
    for (int i = 0; i < kETileItems; ++i) {
        const int64_t q = q0 + 32 * i + (t & 31);
        if (q < in.n) {
            if (in.indptr) row_of[q] = r[i];
            const uint32_t k = in.key(q, r[i]);
            keys[q] = k;
            atomicAdd(&h[k & 255u], 1u);
        }
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

// One pass of one tile. FIRST: the values are the positions.
// FUSED: `counts` holds digit counts and the tile adds up those before it;
// otherwise it holds their prefix over the tiles, and `totals` the digits' sums.
// next != NULL: the next pass's counts.
template <bool FIRST, bool FUSED>
__global__ void __launch_bounds__(kETileNT)
    id_scatter_kernel(const uint32_t* __restrict__ kin, const uint32_t* __restrict__ vin,
                      uint32_t* __restrict__ kout, uint32_t* __restrict__ vout, int64_t n,
                      int64_t n_tiles, int shift, const uint32_t* __restrict__ counts,
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
            key[i] = kin[lo + q];
            val[i] = FIRST ? (uint32_t)(lo + q) : vin[lo + q];
        }
    }
    uint32_t dtotal = 0, before = 0, all;
    if (FUSED) {
        constexpr int F = 32;  // tiles' counts in flight
        for (int b0 = 0; b0 < (int)n_tiles; b0 += F) {
            uint32_t c[F];
#pragma unroll
            for (int f = 0; f < F; ++f) c[f] = b0 + f < (int)n_tiles ? counts[(b0 + f) * 256 + t] : 0u;
#pragma unroll
            for (int f = 0; f < F; ++f) {
                dtotal += c[f];
                before += b0 + f < tile ? c[f] : 0u;
            }
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
    id_sort_small_kernel(Entries<I> in, int key_bits, uint32_t* __restrict__ kout,
                         uint32_t* __restrict__ vout, int32_t* __restrict__ row_of,
                         unsigned* __restrict__ done) {
    const int n = (int)in.n;
    constexpr int NW = NT / 32;
    extern __shared__ uint32_t dyn[];
    uint32_t(*cnt)[256] = reinterpret_cast<uint32_t(*)[256]>(dyn);  // NW x 256
    uint2* skv = reinterpret_cast<uint2*>(dyn + NW * 256);          // NT * ITEMS
    __shared__ uint32_t scan_sm[NW];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int q0 = warp * (32 * ITEMS) + lane;
    uint32_t key[ITEMS], val[ITEMS], rank[ITEMS];
    int32_t r[ITEMS];
    in.rows(q0 - lane, r);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int q = q0 + i * 32;
        key[i] = 0u;
        val[i] = (uint32_t)q;
        if (q < n) {
            if (in.indptr) row_of[q] = r[i];
            key[i] = in.key(q, r[i]);
        }
    }
    if (t == 0) *done = 0;
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

// Sorts the batch's keys; writes row_of (with indptr) and clears *done.
template <class I>
IdSorted sort_ids(const IdSortPlan& P, const Entries<I>& in, int32_t* row_of, unsigned* done,
                  uint32_t* ws, cudaStream_t s) {
    const int64_t n = P.n;
    uint32_t *k0 = ws, *v0 = ws + n, *k1 = ws + 2 * n, *v1 = ws + 3 * n, *counts = ws + 4 * n;
    if (n <= kSmallSort) {
        auto small = [&](auto nt, auto items) {
            constexpr int NT = decltype(nt)::value, IT = decltype(items)::value;
            constexpr int SM = (NT / 32) * 1024 + NT * IT * 8;
            auto k = id_sort_small_kernel<I, NT, IT>;
            static_assert(SM <= 48 * 1024, "id sort shared memory");
            k<<<1, NT, SM, s>>>(in, P.key_bits, k0, v0, row_of, done);
        };
        using std::integral_constant;
        if (n <= 256)
            small(integral_constant<int, 256>{}, integral_constant<int, 1>{});
        else if (n <= 512)
            small(integral_constant<int, 512>{}, integral_constant<int, 1>{});
        else
            small(integral_constant<int, 512>{}, integral_constant<int, 4>{});
        MFM_CHECK_LAUNCH("id sort launch");
        return {k0, v0};
    }
    const unsigned g = (unsigned)P.n_tiles;
    const bool fused = P.n_tiles <= kFuseTiles;
    uint32_t* totals = counts + (int64_t)P.passes * P.n_tiles * 256;
    id_count_kernel<I><<<g, kETileNT, 0, s>>>(in, P.passes, P.n_tiles, k1, row_of, counts, done);
    uint32_t *ki = k1, *vi = v1, *ko = k0, *vo = v0;
    for (int p = 0; p < P.passes; ++p) {
        uint32_t* c = counts + (int64_t)p * P.n_tiles * 256;
        uint32_t* next = p + 1 < P.passes ? c + P.n_tiles * 256 : nullptr;
        if (!fused) id_prefix_kernel<<<256, 256, 0, s>>>(c, P.n_tiles, totals);
        auto pass = [&](auto first, auto whole) {
            id_scatter_kernel<decltype(first)::value, decltype(whole)::value>
                <<<g, kETileNT, 0, s>>>(ki, vi, ko, vo, n, P.n_tiles, 8 * p, c, totals, next);
        };
        if (p == 0 && fused)
            pass(std::true_type{}, std::true_type{});
        else if (p == 0)
            pass(std::true_type{}, std::false_type{});
        else if (fused)
            pass(std::false_type{}, std::true_type{});
        else
            pass(std::false_type{}, std::false_type{});
        std::swap(ki, ko);
        std::swap(vi, vo);
    }
    MFM_CHECK_LAUNCH("id sort launch");
    return {ki, vi};
}

}  // namespace mfm
