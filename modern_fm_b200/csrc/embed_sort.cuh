// embed_sort.cuh — stable radix sort of one batch's ids with what the gradient
// reads by them, into a workspace of the caller: no allocation, no host round
// trip, no block waits for another, so a call can be captured and replayed.
//
// Ids outside the table get the key n_rows and sort behind every real id. Least
// significant digit first, in tiles of 2048 entries that are ranked by
// match_any per warp, reordered in shared memory and written in runs. One
// batch of 10^4 to 10^6 ids is bound by its launches and their latencies, not by
// its bytes, which decides the rest:
//  * digits of up to 12 bits where that saves a pass (17 to 24 bits: two passes
//    instead of three, 302k click ids of 23 bits: 52 -> 38 us), of 8 bits otherwise;
//  * a pass's scatter counts the next pass's digits while it writes (integer
//    adds, grouped per warp), so only the first pass has a counting launch;
//  * 8-bit digits of up to kFuseTiles tiles: each tile sums the counts before it
//    by itself (at most 192 KB of L2 reads); else one prefix launch a pass (a call for
//    the touched rows of 60000 x 4 by the first and the second: 4000 ids 37 and 39 us,
//    60000 41 and 43, 130000 43 and 45, 260000 51 and 49, 390000 65 and 61, 800000 112
//    and 80);
//  * the last pass leaves, beside the sorted keys, each entry's gradient row and
//    scale instead of its position, so the sums read them in order;
//  * up to kSmallSort ids one block does every pass in shared memory (touched rows of
//    60000 x 16: 600 ids 22 us, 31 us by tiles; 2048 ids 27 us and 37 us); up to
//    kFewIds, every block of the gradient's only launch sorts them for itself.
#pragma once

#include <type_traits>

#include "scan.cuh"
#include "vecio.cuh"

namespace mfm {

constexpr int kETileNT = 256;
constexpr int kETileItems = 8;
constexpr int kETile = kETileNT * kETileItems;
constexpr int kFuseTiles = 192;
constexpr int kWideBits = 12;
constexpr int64_t kSmallSort = 2048;
constexpr int kFewIds = 256;
constexpr int kSortPad = 16;  // places behind the last entry: key n_rows, row 0, scale 0

// The entries of a batch: their ids and, where they are summed by rows, the rows'
// bounds (indptr, n_out + 1; NULL: every entry is a row of its own).
struct Ids {  // int32 or int64
    const void* p;
    int is64;
    __device__ __forceinline__ int64_t operator[](int64_t q) const {
        return is64 ? static_cast<const int64_t*>(p)[q] : (int64_t)static_cast<const int32_t*>(p)[q];
    }
};

struct Entries {
    Ids ids;
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
            const int32_t step = len / 32 + (len % 32 != 0);  // len + 31 may pass 2^31
            const int64_t p = (int64_t)(lane + 1) * step;
            const bool ends = p <= len && indptr[base + p] <= q0;
            const int n = __popc(__ballot_sync(0xffffffffu, ends));
            base += n * step;
            const int32_t rest = len - n * step;
            len = rest < step - 1 ? (rest > 0 ? rest : 0) : step - 1;
        }
        const int64_t at = (int64_t)base + lane;
        const int64_t end = at < n_out ? indptr[at + 1] : INT64_MAX;
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
        const int64_t id = ids[q];
        return id >= 0 && id < n_rows && row >= 0 ? (uint32_t)id : (uint32_t)n_rows;
    }
};

// Zeros for the rows [lo, hi) of a table of `bytes` a row whose bits in `touched`
// are clear: the rows of a gradient that no id touches. A warp takes `per` rows
// (which divides 32) at a time. It only needs the first pass's bits, so its
// blocks ride along in the launches behind that, which are bound by latency.
struct Fill {
    char* base;
    int64_t bytes, lo, hi;
    const uint32_t* touched;
    int per;
    unsigned blocks;
};

__device__ __forceinline__ void clear_row(char* p, int64_t bytes, bool vec) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        for (int64_t i = lane; i < bytes / 16; i += 32) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
    } else {  // whole elements of at least two bytes
        for (int64_t i = lane; i < bytes / 2; i += 32) reinterpret_cast<uint16_t*>(p)[i] = 0;
    }
}

__device__ __forceinline__ void clear_rows(char* at, int64_t bytes, int rows, unsigned touched, bool vec) {
    const int lane = threadIdx.x & 31;
    if (vec && bytes <= 1024) {  // the rows' vectors as one stretch
        const unsigned vr = (unsigned)(bytes / 16), total = (unsigned)rows * vr;
        for (unsigned i = lane; i < total; i += 32)
            if (!(touched >> (i / vr) & 1u)) reinterpret_cast<uint4*>(at)[i] = make_uint4(0, 0, 0, 0);
    } else {
        for (unsigned m = ~touched & (rows == 32 ? 0xffffffffu : (1u << rows) - 1u); m; m &= m - 1)
            clear_row(at + (__ffs(m) - 1) * bytes, bytes, vec);
    }
}

__device__ __forceinline__ void fill_untouched(const Fill& f, unsigned block) {
    const bool vec = f.bytes % 16 == 0 && (uintptr_t)f.base % 16 == 0;
    const int64_t warps = (int64_t)f.blocks * (blockDim.x / 32);
    for (int64_t r = f.lo + ((int64_t)block * (blockDim.x / 32) + threadIdx.x / 32) * f.per; r < f.hi; r += warps * f.per) {
        const int rows = (int)(r + f.per < f.hi ? f.per : f.hi - r);
        clear_rows(f.base + r * f.bytes, f.bytes, rows, f.touched[r / 32] >> (r & 31), vec);
    }
}

// What the last pass writes beside a key: the row and scale of the entry at
// position p (row_of NULL: the position itself; scale NULL: none).
template <class A>
struct SortedOut {
    uint32_t* keys;
    uint32_t* rows;
    A* scales;
    const int32_t* row_of;
    const A* scale;
    uint32_t pad_key;
    __device__ __forceinline__ void load(uint32_t p, uint32_t& row, A& s) const {
        row = row_of ? (uint32_t)row_of[p] : p;
        s = scale ? scale[p] : A(1);
    }
    __device__ __forceinline__ void store(int64_t at, uint32_t k, uint32_t row, A s) const {
        keys[at] = k;
        rows[at] = row;
        if (scale) scales[at] = s;
    }
};

// Keys and rows of all entries, digit counts of the first pass by tile, and zeros
// for the passes after it, for the block count of the kernels behind the sort
// and for the touched rows' bits.
template <int BITS>
__global__ void __launch_bounds__(kETileNT)
    id_count_kernel(Entries in, int passes, uint32_t mask, int64_t n_tiles,
                    uint32_t* __restrict__ keys, int32_t* __restrict__ row_of,
                    uint32_t* __restrict__ counts, unsigned* __restrict__ done,
                    uint32_t* __restrict__ touched) {
    constexpr int D = 1 << BITS;
    __shared__ uint32_t h[D];
    const int t = threadIdx.x;
    const int64_t tile = blockIdx.x, lo = tile * kETile;
    for (int d = t; d < D; d += kETileNT) {
        h[d] = 0;
        for (int p = 1; p < passes; ++p) counts[(p * n_tiles + tile) * D + d] = 0;
    }
    if (tile == 0 && t == 0) *done = 0;
    if (touched)
        for (int64_t i = tile * kETileNT + t; i * 32 < in.n_rows; i += n_tiles * kETileNT) touched[i] = 0;
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
            atomicAdd(&h[k & mask], 1u);
        }
    }
    __syncthreads();
    for (int d = t; d < D; d += kETileNT) counts[tile * D + d] = h[d];
}

// Turns each digit's counts into their prefix over the tiles, in place, and writes
// its total: a block takes 32 digits, 8 threads each a stretch of the tiles.
__global__ void __launch_bounds__(256)
    id_prefix_kernel(uint32_t* counts, int64_t n_tiles, int digits, uint32_t* totals) {
    after_previous();
    constexpr int F = 20;  // counts in flight
    __shared__ uint32_t part[8][33];
    const int lane = threadIdx.x & 31, g = threadIdx.x / 32, d = blockIdx.x * 32 + lane;
    const int64_t per = ceil_div(n_tiles, (int64_t)8), t0 = g * per;
    const int64_t t1 = t0 + per < n_tiles ? t0 + per : n_tiles;
    uint32_t sum = 0, c[F];
    for (int64_t b = t0; b < t1; b += F) {
#pragma unroll
        for (int f = 0; f < F; ++f) c[f] = b + f < t1 ? counts[(b + f) * digits + d] : 0u;
#pragma unroll
        for (int f = 0; f < F; ++f) sum += c[f];
    }
    part[g][lane] = sum;
    __syncthreads();
    uint32_t run = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i < g) run += part[i][lane];
        all += part[i][lane];
    }
    if (g == 0) totals[d] = all;
    for (int64_t b = t0; b < t1; b += F) {
        if (per > F) {  // one stretch of F is still in registers
#pragma unroll
            for (int f = 0; f < F; ++f) c[f] = b + f < t1 ? counts[(b + f) * digits + d] : 0u;
        }
#pragma unroll
        for (int f = 0; f < F; ++f)
            if (b + f < t1) {
                counts[(b + f) * digits + d] = run;
                run += c[f];
            }
    }
}

// A thread's ranks of its items among the equal digits of its warp, in order;
// cnt: the warp's running counts (zero before).
template <int ITEMS, class C>
__device__ __forceinline__ void warp_ranks(const uint32_t (&digit)[ITEMS], C* cnt,
                                           uint32_t (&rank)[ITEMS]) {
    const int lane = threadIdx.x & 31;
    const unsigned lt = (1u << lane) - 1u;
    unsigned peers[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) peers[i] = __match_any_sync(0xffffffffu, digit[i]);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int leader = __ffs(peers[i]) - 1;
        uint32_t b = 0;
        if (lane == leader && !(digit[i] & 0x80000000u)) {
            b = cnt[digit[i]];
            cnt[digit[i]] = (C)(b + (uint32_t)__popc(peers[i]));
        }
        b = __shfl_sync(0xffffffffu, b, leader);
        rank[i] = b + (uint32_t)__popc(peers[i] & lt);
        __syncwarp();
    }
}

// N neighbouring words, four at a time where there are that many.
template <int N>
__device__ __forceinline__ void load_many(const uint32_t* p, uint32_t (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const uint4 x = reinterpret_cast<const uint4*>(p)[k];
            v[4 * k] = x.x;
            v[4 * k + 1] = x.y;
            v[4 * k + 2] = x.z;
            v[4 * k + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = p[k];
    }
}
template <int N>
__device__ __forceinline__ void store_many(uint32_t* p, const uint32_t (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k)
            reinterpret_cast<uint4*>(p)[k] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) p[k] = v[k];
    }
}

template <int BITS>
constexpr int scatter_smem() {  // counts per warp (16 bits), offsets, the tile
    return (kETileNT / 32) * (1 << BITS) * 2 + (1 << BITS) * 4 + kETile * 8;
}

// One pass of one tile. FIRST: the values are the positions. FUSED: `counts` holds
// digit counts and the tile adds up those before it; otherwise it holds their
// prefix over the tiles, and `totals` the digits' sums. next != NULL: the next
// pass's counts; NULL: the last pass, which writes through `out`.
template <class A, int BITS, bool FIRST, bool FUSED>
__global__ void __launch_bounds__(kETileNT)
    id_scatter_kernel(const uint32_t* kin, const uint32_t* vin, uint32_t* kout, uint32_t* vout,
                      int64_t n, int64_t n_tiles, int shift, int bits, const uint32_t* counts,
                      const uint32_t* totals, uint32_t* next, SortedOut<A> out, uint32_t* touched,
                      Fill fill) {
    after_previous();
    if (!FIRST && blockIdx.x >= n_tiles) {
        fill_untouched(fill, blockIdx.x - (unsigned)n_tiles);
        return;
    }
    constexpr int NW = kETileNT / 32, D = 1 << BITS, PT = D / kETileNT;  // digits per thread
    extern __shared__ uint4 scatter_mem[];
    uint16_t(*cnt)[D] = reinterpret_cast<uint16_t(*)[D]>(scatter_mem);
    uint32_t* base = reinterpret_cast<uint32_t*>(cnt + NW);
    uint2* skv = reinterpret_cast<uint2*>(base + D);
    __shared__ uint32_t scan_sm[NW];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t tile = blockIdx.x, lo = tile * kETile;
    const int m = (int)(n - lo < kETile ? n - lo : kETile);
    const uint32_t mask = (1u << bits) - 1u;
    const int q0 = warp * (32 * kETileItems) + lane;  // striped: a warp's items are in position order
    for (int i = t; i < NW * D / 8; i += kETileNT) scatter_mem[i] = make_uint4(0, 0, 0, 0);
    uint32_t key[kETileItems], val[kETileItems], digit[kETileItems], rank[kETileItems];
#pragma unroll
    for (int i = 0; i < kETileItems; ++i) {
        const int q = q0 + i * 32;
        key[i] = q < m ? kin[lo + q] : 0u;
        val[i] = FIRST ? (uint32_t)(lo + q) : (q < m ? vin[lo + q] : 0u);
    }
    // this thread's digits are PT t .. PT t + PT - 1: their places in the output
    uint32_t total[PT], before[PT];
    if (FUSED) {
        constexpr int F = 32;  // tiles' counts in flight
        static_assert(!FUSED || PT == 1, "summed by the tile: one digit a thread");
        total[0] = before[0] = 0;
        for (int b0 = 0; b0 < (int)n_tiles; b0 += F) {
            uint32_t c[F];
#pragma unroll
            for (int f = 0; f < F; ++f) c[f] = b0 + f < (int)n_tiles ? counts[(b0 + f) * D + t] : 0u;
#pragma unroll
            for (int f = 0; f < F; ++f) {
                total[0] += c[f];
                before[0] += b0 + f < tile ? c[f] : 0u;
            }
        }
    } else {
        load_many<PT>(totals + t * PT, total);
        load_many<PT>(counts + tile * D + t * PT, before);
    }
    uint32_t sum = 0, all;
#pragma unroll
    for (int k = 0; k < PT; ++k) sum += total[k];
    uint32_t at = block_exclusive_scan<uint32_t, kETileNT>(sum, scan_sm, all);  // its barriers end the zeroing
#pragma unroll
    for (int k = 0; k < PT; ++k) {
        before[k] += at;
        at += total[k];
    }
#pragma unroll
    for (int i = 0; i < kETileItems; ++i)
        digit[i] = q0 + i * 32 < m ? (key[i] >> shift) & mask : 0x80000000u + (uint32_t)lane;
    warp_ranks<kETileItems>(digit, cnt[warp], rank);
    __syncthreads();
    // the warps' counts -> their prefix over the warps, and the digits' counts in
    // the tile into base; two 16-bit counts a word (at most 2048 each: no carry),
    // words 256 apart, so that no two lanes meet in a bank
    uint32_t mine[PT];
    if (PT > 1) {
        constexpr int WT = PT > 1 ? PT / 2 : 1;  // words per thread
#pragma unroll
        for (int k = 0; k < WT; ++k) {
            const int word = t + k * kETileNT;
            uint32_t run = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                uint32_t* c = reinterpret_cast<uint32_t*>(cnt[w]) + word;
                const uint32_t v = *c;
                *c = run;
                run += v;
            }
            reinterpret_cast<uint2*>(base)[word] = make_uint2(run & 0xffffu, run >> 16);
        }
        __syncthreads();
        load_many<PT>(base + t * PT, mine);
    } else {
        uint32_t run = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const uint32_t c = cnt[w][t];
            cnt[w][t] = (uint16_t)run;
            run += c;
        }
        mine[0] = run;
    }
    sum = 0;
#pragma unroll
    for (int k = 0; k < PT; ++k) sum += mine[k];
    uint32_t start = block_exclusive_scan<uint32_t, kETileNT>(sum, scan_sm, all);
    uint32_t first[PT];
#pragma unroll
    for (int k = 0; k < PT; ++k) {
        first[k] = start;
        start += mine[k];
    }
    store_many<PT>(base + t * PT, first);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kETileItems; ++i)
        if (q0 + i * 32 < m) skv[base[digit[i]] + cnt[warp][digit[i]] + rank[i]] = make_uint2(key[i], val[i]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PT; ++k) before[k] -= first[k];  // output place less tile place
    store_many<PT>(base + t * PT, before);
    __syncthreads();
    uint32_t dst[kETileItems];
    uint2 e[kETileItems];
#pragma unroll
    for (int u = 0; u < kETileItems; ++u) {
        const int j = t + u * kETileNT;
        e[u] = j < m ? skv[j] : make_uint2(0, 0);
        dst[u] = base[(e[u].x >> shift) & mask] + (uint32_t)j;
    }
    if (FIRST && touched) {
        // popular ids share their words: the bit is looked at first, so that few
        // of their entries get as far as the atomic
        uint32_t seen[kETileItems];
#pragma unroll
        for (int u = 0; u < kETileItems; ++u) {
            const int j = t + u * kETileNT;
            const bool want = j < m && e[u].x != out.pad_key && (j == 0 || skv[j - 1].x != e[u].x);
            seen[u] = want ? __ldcg(touched + e[u].x / 32) : 0xffffffffu;
        }
#pragma unroll
        for (int u = 0; u < kETileItems; ++u)
            if (!(seen[u] >> (e[u].x & 31) & 1u)) atomicOr(touched + e[u].x / 32, 1u << (e[u].x & 31));
    }
    if (next) {
#pragma unroll
        for (int u = 0; u < kETileItems; ++u) {
            const bool valid = t + u * kETileNT < m;
            // fewer than 2^20 tiles of 2^12 digits, or 2^20 of 2^8
            const uint32_t bin = valid ? (dst[u] / kETile) * D + ((e[u].x >> (shift + bits)) & mask) : 0xffffffffu;
            if (valid) {
                kout[dst[u]] = e[u].x;
                vout[dst[u]] = e[u].y;
            }
            const unsigned peers = __match_any_sync(0xffffffffu, bin);
            if (valid && lane == __ffs(peers) - 1) atomicAdd(next + bin, (uint32_t)__popc(peers));
        }
    } else {
        uint32_t row[kETileItems];
        A s[kETileItems];
#pragma unroll
        for (int u = 0; u < kETileItems; ++u)
            if (t + u * kETileNT < m) out.load(e[u].y, row[u], s[u]);
#pragma unroll
        for (int u = 0; u < kETileItems; ++u)
            if (t + u * kETileNT < m) {
                out.store(dst[u], e[u].x, row[u], s[u]);
            }
        if (tile == 0 && t < kSortPad) out.store(n + t, out.pad_key, 0u, A(0));
    }
}

// All passes of up to NT * ITEMS ids in one block: on return skv holds (key,
// position) of the sorted entries. rows: where entry q's row goes, or NULL.
template <int NT, int ITEMS>
struct BlockSort {
    static constexpr int NW = NT / 32;
    uint32_t cnt[NW][256];
    uint2 skv[NT * ITEMS];
    uint32_t scan_sm[NW];

    __device__ __forceinline__ void run(const Entries& in, int key_bits, int32_t* rows) {
        const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n = (int)in.n;
        const int q0 = warp * (32 * ITEMS) + lane;
        uint32_t key[ITEMS], val[ITEMS], digit[ITEMS], rank[ITEMS];
        int32_t r[ITEMS];
        in.rows(q0 - lane, r);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int q = q0 + i * 32;
            key[i] = 0u;
            val[i] = (uint32_t)q;
            if (q < n) {
                if (rows) rows[q] = r[i];
                key[i] = in.key(q, r[i]);
            }
        }
        for (int shift = 0; shift < key_bits; shift += 8) {
            for (int i = t; i < NW * 256; i += NT) (&cnt[0][0])[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                digit[i] = q0 + i * 32 < n ? (key[i] >> shift) & 255u : 0x80000000u + (uint32_t)lane;
            warp_ranks<ITEMS>(digit, cnt[warp], rank);
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
                if (q0 + i * 32 < n) skv[cnt[warp][digit[i]] + rank[i]] = make_uint2(key[i], val[i]);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int q = q0 + i * 32;
                if (q < n) {
                    key[i] = skv[q].x;
                    val[i] = skv[q].y;
                }
            }
            __syncthreads();
        }
    }
};

template <class A, int NT, int ITEMS>
__global__ void __launch_bounds__(NT)
    id_sort_small_kernel(Entries in, int key_bits, int32_t* row_of, unsigned* __restrict__ done,
                         SortedOut<A> out) {
    __shared__ BlockSort<NT, ITEMS> sort;
    const int t = threadIdx.x, n = (int)in.n;
    if (t == 0) *done = 0;
    sort.run(in, key_bits, in.indptr ? row_of : nullptr);
    uint32_t row[ITEMS];
    A s[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)  // row_of was written by this block, before a barrier
        if (t + i * NT < n) out.load(sort.skv[t + i * NT].y, row[i], s[i]);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (t + i * NT < n) out.store(t + i * NT, sort.skv[t + i * NT].x, row[i], s[i]);
    if (t < kSortPad) out.store(n + t, out.pad_key, 0u, A(0));
}

inline int id_key_bits(int64_t n_rows) {  // keys 0 .. n_rows
    int b = 1;
    while (b < 32 && ((int64_t)1 << b) <= n_rows) ++b;
    return b;
}

// How n ids are sorted, and the workspace in 32-bit words: two key / value pairs,
// the passes' counts and the digits' totals.
struct IdSortPlan {
    int64_t n = 0, n_tiles = 0, pitch = 0;  // pitch: of the four arrays, with the padding
    int key_bits = 1, passes = 1, bits = 8;
    bool wide = false;
    int64_t words = 0;
    IdSortPlan(int64_t n_, int64_t n_rows) : n(n_) {
        key_bits = id_key_bits(n_rows);
        const int narrow = (key_bits + 7) / 8, few = (key_bits + kWideBits - 1) / kWideBits;
        // with 2^20 tiles of 2^12 digits the last count's index would be the mark of no entry
        wide = few < narrow && ceil_div(n, kETile) < 1 << 20;
        passes = wide ? few : narrow;
        bits = wide ? (key_bits + passes - 1) / passes : 8;
        n_tiles = ceil_div(n, kETile);
        pitch = ceil_div(n + kSortPad, (int64_t)64) * 64;
        const int64_t digits = wide ? 1 << kWideBits : 256;
        words = 4 * pitch + (n > kSmallSort ? ((int64_t)passes * n_tiles + 1) * digits : 0);
    }
};

// Sorts the batch's keys into out.keys with the entries' rows and scales (out's
// keys and rows are set here, in the workspace); writes row_of (with indptr),
// clears *done and sets the touched rows' bits. The launch of pass p >= 1 fills
// fills[p - 1].
template <class A>
void sort_ids(int device, const IdSortPlan& P, const Entries& in, int32_t* row_of, unsigned* done,
              uint32_t* ws, SortedOut<A>& out, uint32_t* touched, const Fill* fills, cudaStream_t s) {
    const int64_t n = P.n;
    uint32_t* counts = ws + 4 * P.pitch;
    out.keys = ws;
    out.rows = ws + P.pitch;
    out.row_of = in.indptr ? row_of : nullptr;
    out.pad_key = (uint32_t)in.n_rows;
    using std::integral_constant;
    if (n <= kSmallSort) {
        auto small = [&](auto nt, auto items) {
            constexpr int NT = decltype(nt)::value, IT = decltype(items)::value;
            id_sort_small_kernel<A, NT, IT><<<1, NT, 0, s>>>(in, P.key_bits, row_of, done, out);
        };
        if (n <= 512)
            small(integral_constant<int, 512>{}, integral_constant<int, 1>{});
        else
            small(integral_constant<int, 512>{}, integral_constant<int, 4>{});
        MFM_CHECK_LAUNCH("id sort launch");
        return;
    }
    // keys and values go back and forth between the two pairs and end in `out`
    uint32_t *k0 = out.keys, *v0 = out.rows, *k1 = ws + 2 * P.pitch, *v1 = ws + 3 * P.pitch;
    const unsigned g = (unsigned)P.n_tiles;
    auto run = [&](auto width) {
        constexpr int BITS = decltype(width)::value, D = 1 << BITS, SM = scatter_smem<BITS>();
        uint32_t* totals = counts + (int64_t)P.passes * P.n_tiles * D;
        const bool fused = BITS == 8 && P.n_tiles <= kFuseTiles;
        uint32_t *ki = P.passes % 2 ? k1 : k0, *vi = P.passes % 2 ? v1 : v0;
        uint32_t *ko = P.passes % 2 ? k0 : k1, *vo = P.passes % 2 ? v0 : v1;
        id_count_kernel<BITS><<<g, kETileNT, 0, s>>>(in, P.passes, (1u << P.bits) - 1u, P.n_tiles, ki, row_of, counts, done, touched);
        for (int p = 0; p < P.passes; ++p) {
            uint32_t* c = counts + (int64_t)p * P.n_tiles * D;
            uint32_t* next = p + 1 < P.passes ? c + P.n_tiles * D : nullptr;
            if (!fused) launch_next(id_prefix_kernel, D / 32, 256, 0, s, c, P.n_tiles, D, totals);
            auto pass = [&](auto first, auto whole) {
                auto k = id_scatter_kernel<A, BITS, decltype(first)::value, decltype(whole)::value && BITS == 8>;
                static bool asked[64];
                if (SM > 48 * 1024) allow_smem(k, device, SM, asked, "id sort shared memory");
                const Fill fill = p > 0 ? fills[p - 1] : Fill{};
                launch_next(k, g + fill.blocks, kETileNT, SM, s, ki, vi, ko, vo, n, P.n_tiles, P.bits * p, P.bits, c, totals, next, out, touched, fill);
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
    };
    if (P.wide)
        run(integral_constant<int, kWideBits>{});
    else
        run(integral_constant<int, 8>{});
    MFM_CHECK_LAUNCH("id sort launch");
}

}  // namespace mfm
