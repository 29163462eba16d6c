// embed.cu — latent rows as outputs: embedding lookup with scaling (single
// rows, or summed over the entries of sparse rows) and its gradient by sorted
// ids, over the whole table or the touched rows only.
//
// Everything here moves rows: a multiply and an add per value against 2 to 16
// bytes, so HBM bounds the large calls and latency (ids, then rows) the small
// ones. Rows are walked in 16-byte vectors by lane groups, several entries in
// flight per lane.
#include "embed_sort.cuh"

#include <algorithm>

namespace mfm {
namespace {

// ---------------------------------------------------------------- vectors --

// B bytes of T: 16, 8, or one value, the largest that every row begins on; sixteen
// are held raw.
template <class T, int B>
struct Lane {
    static constexpr int N = B > (int)sizeof(T) ? B / (int)sizeof(T) : 1;
    static constexpr bool WIDE = N * sizeof(T) == 16;
    using Few = Vec<T, WIDE ? 1 : N>;
    uint4 raw;
    Few few;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (WIDE)
            raw = *reinterpret_cast<const uint4*>(p);
        else
            few = *reinterpret_cast<const Few*>(p);
    }
    template <class A>
    __device__ __forceinline__ void get(A (&v)[N]) const {
        if constexpr (WIDE) {
            typename Arith<T>::type w[N];
            Pack<T>::unpack(raw, w);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = (A)w[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = widen<A>(few.v[j]);
        }
    }
};

// N values to `to` (aligned to N of them), each rounded once.
template <class O, class A, int N>
__device__ __forceinline__ void put(O* to, const A (&v)[N]) {
    constexpr int P = 16 / (int)sizeof(O);
    if constexpr (N == 1) {
        *to = narrow<O>(v[0]);
    } else if constexpr (N < P) {
        Vec<O, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = narrow<O>(v[j]);
        *reinterpret_cast<Vec<O, N>*>(to) = o;
    } else {
#pragma unroll
        for (int k = 0; k < N / P; ++k) {
            typename Arith<O>::type w[P];
#pragma unroll
            for (int j = 0; j < P; ++j) w[j] = v[k * P + j];
            *reinterpret_cast<uint4*>(to + k * P) = Pack<O>::pack(w);
        }
    }
}

// ---------------------------------------------------------------- lookup --

// out[t] = alpha scale[t] table[ids[t]], rows of at least 32 vectors: a warp per
// (row, piece of 32 U vectors), U vectors a lane in flight.
template <class T, class A, class O, class I, int B, int U>
__global__ void __launch_bounds__(256)
    embed_wide_kernel(const I* __restrict__ ids, int64_t n, const A* __restrict__ scale, A alpha,
                      const T* __restrict__ table, int64_t n_rows, int dv, int pieces, int64_t ld,
                      O* __restrict__ out, int64_t ld_out) {
    constexpr int N = Lane<T, B>::N;
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 32;
    const int64_t t = item / pieces;
    if (t >= n) return;
    const int j0 = (int)(item - t * pieces) * (32 * U) + (threadIdx.x & 31);
    const int64_t id = (int64_t)ids[t];
    const bool live = id >= 0 && id < n_rows;
    A f = alpha;
    if (scale) f *= scale[t];
    const T* from = table + (live ? id : 0) * ld;
    O* to = out + t * ld_out;
    Lane<T, B> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (live && j0 + u * 32 < dv) v[u].load(from + (int64_t)(j0 + u * 32) * N);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (j0 + u * 32 < dv) {
            A p[N];
            v[u].get(p);
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = live ? f * p[j] : A(0);
            put(to + (int64_t)(j0 + u * 32) * N, p);
        }
}

// The same for narrow or unaligned rows: one thread per vector (or value), U in
// flight, 256 apart.
template <class T, class A, class O, class I, int B, int U>
__global__ void __launch_bounds__(256)
    embed_rows_kernel(const I* __restrict__ ids, int64_t n, const A* __restrict__ scale, A alpha,
                      const T* __restrict__ table, int64_t n_rows, uint32_t dv, int64_t ld,
                      O* __restrict__ out, int64_t ld_out) {
    constexpr int N = Lane<T, B>::N;
    const int64_t first = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = first / dv;
    const uint32_t off0 = (uint32_t)(first - row0 * dv);
    Lane<T, B> v[U];
    A f[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t o = off0 + threadIdx.x + u * 256, r = o / dv;
        const int64_t row = row0 + r;
        live[u] = false;
        f[u] = alpha;
        if (row < n) {
            const int64_t id = (int64_t)ids[row];
            live[u] = id >= 0 && id < n_rows;
            if (live[u]) v[u].load(table + id * ld + (int64_t)(o - r * dv) * N);
            if (scale) f[u] *= scale[row];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t o = off0 + threadIdx.x + u * 256, r = o / dv;
        const int64_t row = row0 + r;
        if (row < n) {
            A p[N];
            v[u].get(p);
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = live[u] ? f[u] * p[j] : A(0);
            put(out + row * ld_out + (int64_t)(o - r * dv) * N, p);
        }
    }
}

// Bounds of a row's entries, limited to the entries there are.
__device__ __forceinline__ void row_bounds(const int64_t* indptr, int64_t b, int64_t n, int64_t& lo,
                                           int64_t& hi) {
    lo = indptr[b];
    hi = indptr[b + 1];
    lo = lo < 0 ? 0 : (lo > n ? n : lo);
    hi = hi < lo ? lo : (hi > n ? n : hi);
}

// out[b] = alpha sum_t scale[t] table[ids[t]]. EL x LV lanes per row: LV lanes hold
// the columns (a vector each; blockIdx.y walks them), EL take every EL-th entry, U
// entries a lane in flight; their parts are added by shuffles. Bound by the
// latency of the rows' gathers: 131072 rows of 36 entries, 16 float32 each in
// float64 arithmetic, 51 us at five blocks per SM (55 us at four, 75 us at six, which
// spill; 62 us with EL = 4; 83 us with eight entries a lane; 54 us with the ids held by
// every lane, 62 us with those fetched just before their rows). A row is one lane group's
// whatever its length: few rows of thousands of entries leave most of the GPU idle (10^6
// entries x 16 float32 in 27777 rows 27 us, in 1000 rows 111 us, in 100 rows 1 ms, in one
// row 81 ms; the gradient splits such runs, this sum does not).
template <class T, class A, class O, class I, int B, int LV, int EL>
__global__ void __launch_bounds__(256, 5)
    embed_sums_kernel(const I* __restrict__ ids, int64_t n, const int64_t* __restrict__ indptr,
                      int64_t n_out, const A* __restrict__ scale, A alpha,
                      const T* __restrict__ table, int64_t n_rows, int64_t d, int64_t ld,
                      O* __restrict__ out, int64_t ld_out) {
    constexpr int U = 4, G = LV * EL, N = Lane<T, B>::N;
    constexpr int E = U * EL, K = E > G ? E / G : 1;  // entries a round; ids a lane fetches of them
    const int lane = threadIdx.x % LV, gl = threadIdx.x % G, el = gl / LV;
    const int64_t b = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int64_t col = ((int64_t)blockIdx.y * LV + lane) * N;
    const bool in = b < n_out;
    int64_t lo = 0, hi = 0;
    if (in) row_bounds(indptr, b, n, lo, hi);
    A acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = A(0);
    // a lane fetches the round's entry gl (and every G-th behind it) and hands it
    // round; the next round's are on their way while a round's rows are
    int32_t id[K];
    A f[K];
    auto fetch = [&](int64_t e) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t at = e + gl + k * G;
            id[k] = -1;
            f[k] = A(1);
            if (gl + k * G < E && at < hi) {
                const int64_t i = (int64_t)ids[at];
                id[k] = i >= 0 && i < n_rows ? (int32_t)i : -1;
                if (scale) f[k] = scale[at];
            }
        }
    };
    fetch(lo);
    for (int64_t e = lo; __any_sync(0xffffffffu, e < hi); e += E) {
        Lane<T, B> v[U];
        A w[U];
        unsigned live = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int32_t i = __shfl_sync(0xffffffffu, id[u * EL / G], u * EL % G + el, G);
            w[u] = __shfl_sync(0xffffffffu, f[u * EL / G], u * EL % G + el, G);
            if (i >= 0 && col < d) {
                v[u].load(table + (int64_t)i * ld + col);
                live |= 1u << u;
            }
        }
        fetch(e + E);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live >> u & 1u) {
                A p[N];
                v[u].get(p);
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += w[u] * p[j];
            }
    }
#pragma unroll
    for (int o = G / 2; o >= LV; o >>= 1)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (in && el == 0 && col < d) {
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= alpha;
        put(out + b * ld_out + col, acc);
    }
}

// -------------------------------------------------------------- gradient --

// Sorted entries per lane group: short enough that a batch of a few thousand ids
// fills the GPU, long enough that the parts of runs cut by chunk bounds (two rows
// of sums a chunk) stay an eighth of the reading.
constexpr int kChunk = 16;
constexpr int kHeadTile = 4096;             // entries per block of chunk_heads_kernel
constexpr int kTileChunks = kHeadTile / kChunk;
constexpr int kMainNT = 128;

// base[c] = how many runs of equal real keys begin before chunk c within its tile
// of kHeadTile entries; tile_base[t] = how many before tile t, by the block that
// finishes last, and *count = all of them.
__global__ void __launch_bounds__(kTileChunks)
    chunk_heads_kernel(const uint32_t* keys, int64_t n, uint32_t pad_key, int64_t n_chunks,
                       uint32_t* base, uint32_t* tile_base, unsigned* done, int64_t* count) {
    after_previous();
    __shared__ uint32_t sm[kTileChunks / 32];
    __shared__ unsigned last;
    const int64_t c = (int64_t)blockIdx.x * kTileChunks + threadIdx.x, e0 = c * kChunk;
    uint32_t heads = 0;
    if (e0 < n) {
        uint32_t prev = e0 > 0 ? keys[e0 - 1] : pad_key;  // pad_key is no run
        uint32_t k[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) k[i] = e0 + i < n ? keys[e0 + i] : pad_key;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            heads += k[i] != pad_key && k[i] != prev ? 1u : 0u;
            prev = k[i];
        }
    }
    uint32_t all;
    const uint32_t ex = block_exclusive_scan<uint32_t, kTileChunks>(heads, sm, all);
    if (c < n_chunks) base[c] = ex;
    if (threadIdx.x == 0) {
        tile_base[blockIdx.x] = all;
        __threadfence();
        last = atomicAdd(done, 1u) == gridDim.x - 1 ? 1u : 0u;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    uint32_t carry = 0;
    for (unsigned b = 0; b < gridDim.x; b += kTileChunks) {
        const unsigned t = b + threadIdx.x;
        const uint32_t v = t < gridDim.x ? __ldcg(tile_base + t) : 0u;
        const uint32_t x = block_exclusive_scan<uint32_t, kTileChunks>(v, sm, all);
        if (t < gridDim.x) tile_base[t] = carry + x;
        carry += all;
    }
    if (threadIdx.x == 0) *count = carry;
}

// First places in the sorted keys whose keys are at least k0 and k1, k0 <= k1, by a
// whole warp: 32 probes a round for each.
__device__ __forceinline__ void warp_range(const uint32_t* keys, int64_t n, uint32_t k0, uint32_t k1,
                                           int64_t& first, int64_t& behind) {
    const int lane = threadIdx.x & 31;
    int64_t lo0 = 0, lo1 = 0, len0 = n, len1 = n;  // the answers are in [lo, lo + len]
    while (len0 > 0 || len1 > 0) {
        const int64_t s0 = (len0 + 31) / 32, s1 = (len1 + 31) / 32;
        const int64_t p0 = (lane + 1) * s0, p1 = (lane + 1) * s1;  // probes end the 32 parts
        const bool less0 = len0 > 0 && p0 <= len0 && keys[lo0 + p0 - 1] < k0;
        const bool less1 = len1 > 0 && p1 <= len1 && keys[lo1 + p1 - 1] < k1;
        const int n0 = __popc(__ballot_sync(0xffffffffu, less0)), n1 = __popc(__ballot_sync(0xffffffffu, less1));
        // n parts lie before the answer; it is in the next part, or at its last place
        lo0 += n0 * s0;
        lo1 += n1 * s1;
        const int64_t r0 = len0 - n0 * s0, r1 = len1 - n1 * s1;
        len0 = r0 < s0 - 1 ? (r0 > 0 ? r0 : 0) : s0 - 1;
        len1 = r1 < s1 - 1 ? (r1 > 0 ? r1 : 0) : s1 - 1;
        if (s0 == 0) len0 = 0;
        if (s1 == 0) len1 = 0;
    }
    first = lo0;
    behind = lo1;
}

struct KeysOut {  // the touched ids, of the ids' type; p NULL: not wanted
    void* p;
    int is64;
    __device__ __forceinline__ void put(int64_t at, int64_t key) const {
        if (is64)
            static_cast<int64_t*>(p)[at] = key;
        else
            static_cast<int32_t*>(p)[at] = (int32_t)key;
    }
};

template <class G, class T, class A, class O>
struct GradArgs {
    Entries in;
    const A* scale;
    A alpha;
    const G* grad;
    int64_t ld;
    const T* table;
    int64_t ld_table, d;
    O *d_table, *rows;
    KeysOut keys_out;
    int64_t* count;
    A* d_scale;
    // sorted entries, padded to whole chunks: key, gradient row, scale
    const uint32_t *keys, *srows;
    const A* scales;
    const int32_t* row_of;  // by position
    Fill fill, fill_late;  // the main kernel's part of the untouched rows, the last one's
    const uint32_t *base, *tile_base;
    A *part_head, *part_tail;
    int64_t n_chunks;
    unsigned reduce_blocks, scale_blocks, fill_blocks;  // of the main kernel
    int fill_per;                                       // rows per warp that fills
    unsigned cross_blocks;
    __device__ __forceinline__ int64_t runs_before(int64_t c) const {
        return (int64_t)tile_base[c / kTileChunks] + base[c];
    }
};

// One chunk of sorted entries x LV vectors of columns by one lane group: sums of
// scale grad[row], run by run. A run that lies in the chunk is written; the
// part of a run that began before goes to part_head[chunk], the part of one that
// goes on behind to part_tail[chunk] (all of it to part_head when both).
template <class G, class T, class A, class O, int B, int LV>
__device__ __forceinline__ void reduce_chunk(const GradArgs<G, T, A, O>& a, int64_t c, int64_t col,
                                             bool first_lane) {
    constexpr int U = 8, N = Lane<G, B>::N;
    const uint32_t pad_key = (uint32_t)a.in.n_rows;
    const int64_t n = a.in.n, e0 = c * kChunk, e1 = e0 + kChunk;
    uint32_t k[kChunk], row[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk / 4; ++i) {
        const uint4 x = reinterpret_cast<const uint4*>(a.keys + e0)[i], y = reinterpret_cast<const uint4*>(a.srows + e0)[i];
        k[4 * i] = x.x;
        k[4 * i + 1] = x.y;
        k[4 * i + 2] = x.z;
        k[4 * i + 3] = x.w;
        row[4 * i] = y.x;
        row[4 * i + 1] = y.y;
        row[4 * i + 2] = y.z;
        row[4 * i + 3] = y.w;
    }
    const uint32_t last = e0 > 0 ? a.keys[e0 - 1] : pad_key;
    const bool behind = e1 < n;
    const uint32_t next = behind ? a.keys[e1] : pad_key;
    uint32_t cur = k[0];
    if (cur == pad_key) return;  // padding sorts last
    bool before = e0 > 0 && last == cur;
    int64_t rank = a.rows ? a.runs_before(c) - (before ? 1 : 0) : 0;
    A acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = A(0);
    auto part = [&](A* to) {
        Vec<A, N> p;
#pragma unroll
        for (int j = 0; j < N; ++j) p.v[j] = acc[j];
        *reinterpret_cast<Vec<A, N>*>(to + c * a.d + col) = p;
    };
    auto finish = [&]() {  // a run ends inside the chunk
        if (before) {
            part(a.part_head);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] *= a.alpha;
            put((a.rows ? a.rows + rank * a.d : a.d_table + (int64_t)cur * a.d) + col, acc);
            if (a.keys_out.p && first_lane) a.keys_out.put(rank, cur);
        }
    };
#pragma unroll
    for (int b = 0; b < kChunk; b += U) {
        if (b > 0 && k[b] == pad_key) break;
        Lane<G, B> v[U];
        A f[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k[b + u] != pad_key) v[u].load(a.grad + (int64_t)row[b + u] * a.ld + col);
#pragma unroll
        for (int u = 0; u < U; ++u) f[u] = a.scales ? a.scales[e0 + b + u] : A(1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (cur != pad_key) {
                if (k[b + u] != cur) {
                    finish();
                    cur = k[b + u];
                    before = false;
                    ++rank;
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] = A(0);
                }
                if (cur != pad_key) {
                    A w[N];
                    v[u].get(w);
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += f[u] * w[j];
                }
            }
        }
    }
    if (cur == pad_key) return;
    if (behind && next == cur)  // the run goes on behind the chunk
        part(before ? a.part_head : a.part_tail);
    else
        finish();
}

// Zeros for the rows of the result that no run writes: table rows without an
// entry (a warp per `per` <= 32 rows; by the bits the sort left, or for a few ids by
// a search among the sorted keys), or the places behind the last touched row.
// Each row of the result is written once.
template <class G, class T, class A, class O>
__device__ __forceinline__ void fill_rest(const GradArgs<G, T, A, O>& a, unsigned block) {
    if (a.fill.touched) {
        fill_untouched(a.fill, block);
        return;
    }
    const int lane = threadIdx.x & 31, per = a.fill_per;
    const int64_t warp = (int64_t)block * (kMainNT / 32) + threadIdx.x / 32, warps = (int64_t)a.fill_blocks * (kMainNT / 32);
    const int64_t n = a.in.n, n_rows = a.in.n_rows, bytes = a.d * (int64_t)sizeof(O);
    char* const base = reinterpret_cast<char*>(a.rows ? a.rows : a.d_table);
    const bool vec = bytes % 16 == 0 && (uintptr_t)base % 16 == 0;
    const int64_t first = a.rows ? *a.count : 0, end = a.rows ? (n < n_rows ? n : n_rows) : n_rows;
    for (int64_t r0 = first + warp * per; r0 < end; r0 += warps * per) {
        const int rows = (int)(r0 + per < end ? per : end - r0);
        unsigned touched = 0;
        if (a.rows) {
            if (lane < rows) a.keys_out.put(r0 + lane, -1);
        } else {
            int64_t lo, hi;
            warp_range(a.keys, n, (uint32_t)r0, (uint32_t)(r0 + rows), lo, hi);
            for (int64_t i = lo + lane; i < hi; i += 32) touched |= 1u << (a.keys[i] - (uint32_t)r0);
            touched = __reduce_or_sync(0xffffffffu, touched);
        }
        clear_rows(base + r0 * bytes, bytes, rows, touched, vec);
    }
}

// d_scale[t] = alpha <grad[row(t)], table[ids[t]]> for kScaleEntries entries LV lanes
// apart, their loads in flight together.
constexpr int kScaleEntries = 4;

template <class G, class T, class A, class O, int B, int LV>
__device__ __forceinline__ void scale_entries(const GradArgs<G, T, A, O>& a, const int32_t* row_of,
                                              int64_t t0, int stride, int lane) {
    constexpr int N = Lane<G, B>::N, U = kScaleEntries;
    const T* v[U];
    const G* g[U];
    bool live[U];
    A acc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t t = t0 + u * stride;
        int64_t id = -1, row = -1;
        if (t < a.in.n) {
            id = a.in.ids[t];
            row = row_of ? (int64_t)row_of[t] : t;
        }
        live[u] = id >= 0 && id < a.in.n_rows && row >= 0;
        v[u] = a.table + (live[u] ? id : 0) * a.ld_table;
        g[u] = a.grad + (live[u] ? row : 0) * a.ld;
        acc[u] = A(0);
    }
    for (int64_t c = (int64_t)lane * N; c < a.d; c += LV * N) {
        Lane<G, B> x[U];
        // a float32 table with float64 gradients: half a vector
        using Y = std::conditional_t<sizeof(T) == sizeof(G), Lane<T, B>, Vec<T, N>>;
        Y y[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) {
                x[u].load(g[u] + c);
                if constexpr (sizeof(T) == sizeof(G))
                    y[u].load(v[u] + c);
                else
                    y[u] = ldg_vec<T, N>(v[u] + c);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) {
                A p[N], q[N];
                x[u].get(p);
                if constexpr (sizeof(T) == sizeof(G)) {
                    y[u].get(q);
                } else {
#pragma unroll
                    for (int j = 0; j < N; ++j) q[j] = widen<A>(y[u].v[j]);
                }
#pragma unroll
                for (int j = 0; j < N; ++j) acc[u] += p[j] * q[j];
            }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = LV / 2; o > 0; o >>= 1) acc[u] += __shfl_xor_sync(0xffffffffu, acc[u], o);
        const int64_t t = t0 + u * stride;
        if (lane == 0 && t < a.in.n) a.d_scale[t] = a.alpha * acc[u];
    }
}

// The gradient in one launch of three independent parts: blocks that sum chunks,
// blocks that take the scales' gradient, and blocks that fill. Filling is bound
// by HBM and the others by latency, so its blocks alternate with theirs.
template <class G, class T, class A, class O, int B, int LV>
__global__ void __launch_bounds__(kMainNT)
    embed_main_kernel(const GradArgs<G, T, A, O> a, int slabs) {
    after_previous();
    constexpr int N = Lane<G, B>::N, GR = kMainNT / LV;
    const int lane = threadIdx.x % LV, group = threadIdx.x / LV;
    const unsigned work = a.reduce_blocks + a.scale_blocks;
    const unsigned both = 2 * (work < a.fill_blocks ? work : a.fill_blocks);
    unsigned b = blockIdx.x;
    bool fill = false;
    if (b < both) {
        fill = b & 1;
        b >>= 1;
    } else {
        b -= both / 2;
        fill = work <= a.fill_blocks;
    }
    if (fill) {
        fill_rest(a, b);
    } else if (b < a.reduce_blocks) {
        const int64_t c = (int64_t)(b / slabs) * GR + group;
        const int64_t col = ((int64_t)(b % slabs) * LV + lane) * N;
        if (c < a.n_chunks && col < a.d) reduce_chunk<G, T, A, O, B, LV>(a, c, col, col == 0);
    } else {
        scale_entries<G, T, A, O, B, LV>(a, a.row_of, (int64_t)(b - a.reduce_blocks) * (GR * kScaleEntries) + group, GR, lane);
    }
}

// A few ids (at most kFewIds): one launch and no workspace. Every block sorts them
// for itself (2 us) and then sums runs, takes scales' gradients or fills, a lane
// group per run and LV vectors of columns. (66 entries into 1003 x 60: a sort, a
// main and a cross launch take 26 us a call, this one 18 us.)
template <class G, class T, class A, class O, int B, int LV>
__global__ void __launch_bounds__(kFewIds)
    embed_few_kernel(const GradArgs<G, T, A, O> a, int key_bits, int slabs) {
    constexpr int U = 8, N = Lane<G, B>::N, GR = kFewIds / LV;
    __shared__ BlockSort<kFewIds, 1> sort;
    __shared__ int32_t rows[kFewIds];      // by position
    __shared__ uint32_t key[kFewIds], row[kFewIds], run[kFewIds + 1];
    __shared__ A scale[kFewIds];
    const int t = threadIdx.x, lane = t % LV, group = t / LV, n = (int)a.in.n;
    const uint32_t pad_key = (uint32_t)a.in.n_rows;
    sort.run(a.in, key_bits, rows);
    bool live = false, head = false;
    if (t < n) {
        const uint2 e = sort.skv[t];
        live = e.x != pad_key;
        head = live && (t == 0 || sort.skv[t - 1].x != e.x);
        key[t] = e.x;
        row[t] = a.in.indptr ? (uint32_t)rows[e.y] : e.y;
        scale[t] = a.scale ? a.scale[e.y] : A(1);
    }
    uint32_t n_runs;
    const uint32_t rank = block_exclusive_scan<uint32_t, kFewIds>(head ? 1u : 0u, sort.scan_sm, n_runs);
    if (head) run[rank] = (uint32_t)t;
    const int n_live = __syncthreads_count(live);
    if (t == 0) run[n_runs] = (uint32_t)n_live;
    __syncthreads();
    if (blockIdx.x < a.reduce_blocks) {
        if (a.rows && blockIdx.x == 0 && t == 0) *a.count = n_runs;
        for (unsigned item = blockIdx.x * GR + group; item < n_runs * (unsigned)slabs; item += a.reduce_blocks * GR) {
            const unsigned r = item / (unsigned)slabs;
            const int64_t col = ((int64_t)(item % (unsigned)slabs) * LV + lane) * N;
            if (col >= a.d) continue;
            A acc[N];
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = A(0);
            const int end = (int)run[r + 1];
            for (int e = (int)run[r]; e < end; e += U) {
                Lane<G, B> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (e + u < end) v[u].load(a.grad + (int64_t)row[e + u] * a.ld + col);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (e + u < end) {
                        A w[N];
                        v[u].get(w);
#pragma unroll
                        for (int j = 0; j < N; ++j) acc[j] += scale[e + u] * w[j];
                    }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] *= a.alpha;
            const uint32_t k = key[run[r]];
            put((a.rows ? a.rows + (int64_t)r * a.d : a.d_table + (int64_t)k * a.d) + col, acc);
            if (a.keys_out.p && col == 0) a.keys_out.put(r, k);
        }
    } else if (blockIdx.x < a.reduce_blocks + a.scale_blocks) {
        scale_entries<G, T, A, O, B, LV>(a, a.in.indptr ? rows : nullptr,
                                         (int64_t)(blockIdx.x - a.reduce_blocks) * (GR * kScaleEntries) + group, GR, lane);
    } else {  // the rows that nothing touches
        const int wl = t & 31, per = a.fill_per;
        const int64_t warp = (int64_t)(blockIdx.x - a.reduce_blocks - a.scale_blocks) * (kFewIds / 32) + t / 32;
        const int64_t bytes = a.d * (int64_t)sizeof(O), cap = n < a.in.n_rows ? n : a.in.n_rows;
        char* const base = reinterpret_cast<char*>(a.rows ? a.rows : a.d_table);
        const bool vec = bytes % 16 == 0 && (uintptr_t)base % 16 == 0;
        const int64_t first = a.rows ? (int64_t)n_runs : 0, end = a.rows ? cap : a.in.n_rows;
        for (int64_t r0 = first + warp * per; r0 < end; r0 += (int64_t)a.fill_blocks * (kFewIds / 32) * per) {
            const int m = (int)(r0 + per < end ? per : end - r0);
            unsigned touched = 0;
            if (a.rows) {
                if (wl < m) a.keys_out.put(r0 + wl, -1);
            } else {
                for (int i = wl; i < n; i += 32) {
                    const int64_t at = (int64_t)key[i] - r0;
                    if (at >= 0 && at < m) touched |= 1u << at;
                }
                touched = __reduce_or_sync(0xffffffffu, touched);
            }
            clear_rows(base + r0 * bytes, bytes, m, touched, vec);
        }
    }
}

// The runs that cross chunks: the lane group of the chunk where one begins adds
// its parts in chunk order and writes the run; the block's groups share a run of
// more than kLongRun chunks (ids that occur in every row: one chunk per 16 rows).
constexpr int kLongRun = 16;

template <class G, class T, class A, class O, int B, int LV>
__global__ void __launch_bounds__(256)
    embed_cross_kernel(const GradArgs<G, T, A, O> a, int slabs) {
    after_previous();
    if (blockIdx.x >= a.cross_blocks) {
        fill_untouched(a.fill_late, blockIdx.x - a.cross_blocks);
        return;
    }
    constexpr int N = Lane<G, B>::N, GR = 256 / LV;
    __shared__ int64_t run_last[GR];  // last chunk of the run begun in the group's chunk, -1: none
    __shared__ int long_groups[GR], n_long;
    __shared__ A shared_part[256 * N];
    const int lane = threadIdx.x % LV, group = threadIdx.x / LV;
    const int64_t c0 = (int64_t)(blockIdx.x / slabs) * GR, c = c0 + group;
    const int64_t col = ((int64_t)(blockIdx.x % slabs) * LV + lane) * N;
    const uint32_t pad_key = (uint32_t)a.in.n_rows;
    if (threadIdx.x == 0) n_long = 0;
    __syncthreads();
    if (lane == 0) {
        int64_t last = -1;
        if (c + 1 < a.n_chunks) {
            // the keys at the chunk's bounds and the first keys of the chunks behind
            // it, where most runs end: all in flight
            const int64_t e0 = c * kChunk, e1 = e0 + kChunk;  // not the last chunk: e1 < n
            const uint32_t key = a.keys[e1 - 1], next = a.keys[e1], prev = e0 > 0 ? a.keys[e0 - 1] : pad_key;
            uint32_t ahead[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) ahead[i] = c + 2 + i < a.n_chunks ? a.keys[(c + 2 + i) * kChunk] : pad_key;
            if (key != pad_key && next == key && prev != key) {
                last = c + 1;
#pragma unroll
                for (int i = 0; i < 8; ++i) last += last == c + 1 + i && ahead[i] == key ? 1 : 0;
                for (int64_t r = c + 9; last == r && r - c <= kLongRun; r += 8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) ahead[i] = r + 1 + i < a.n_chunks ? a.keys[(r + 1 + i) * kChunk] : pad_key;
#pragma unroll
                    for (int i = 0; i < 8; ++i) last += last == r + i && ahead[i] == key ? 1 : 0;
                }
            }
        }
        run_last[group] = last;
        // which group's run is added first does not change any sum
        if (last - c > kLongRun) long_groups[atomicAdd(&n_long, 1)] = group;
    }
    __syncthreads();
    // the row of the run that crosses the end of a chunk
    auto place = [&](int64_t chunk, uint32_t key) {
        return a.rows ? a.runs_before(chunk + 1) - 1 : (int64_t)key;
    };
    auto write = [&](int64_t at, uint32_t key, A (&acc)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= a.alpha;
        put((a.rows ? a.rows : a.d_table) + at * a.d + col, acc);
        if (a.keys_out.p && col == 0) a.keys_out.put(at, key);
    };
    const bool in = col < a.d;
    const int64_t mine = run_last[group];
    if (mine >= 0 && mine - c <= kLongRun && in) {
        const uint32_t key = a.keys[c * kChunk + kChunk - 1];
        const int64_t at = place(c, key);
        const Vec<A, N> own = ldg_vec<A, N>(a.part_tail + c * a.d + col);
        A acc[N];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = own.v[j];
        for (int64_t k0 = c + 1; k0 <= mine; k0 += 8) {  // eight parts in flight
            Vec<A, N> p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k <= mine) p[k] = ldg_vec<A, N>(a.part_head + (k0 + k) * a.d + col);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k <= mine) {
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += p[k].v[j];
                }
        }
        write(at, key, acc);
    }
    for (int i = 0; i < n_long; ++i) {
        const int g = long_groups[i];
        const int64_t from = c0 + g;
        // the run's last chunk: chunks are probed 256 a round by their first key
        const uint32_t key = a.keys[from * kChunk + kChunk - 1];
        const int64_t at = place(from, key);
        int64_t last = run_last[g], end = a.n_chunks;  // in [last, end)
        while (end - last > 1) {
            const int64_t step = (end - last + 254) / 256;
            const int64_t p = last + (threadIdx.x + 1) * step;
            const int same = __syncthreads_count(p < end && a.keys[p * kChunk] == key);
            last += same * step;
            if (last + step < end) end = last + step;
        }
        A acc[N];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = A(0);
        if (in) {
#pragma unroll 8
            for (int64_t k = from + 1 + group; k <= last; k += GR) {
                const Vec<A, N> p = ldg_vec<A, N>(a.part_head + k * a.d + col);
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += p.v[j];
            }
            if (group == 0) {
                const Vec<A, N> p = ldg_vec<A, N>(a.part_tail + from * a.d + col);
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += p.v[j];
            }
        }
        // the groups' sums by a tree in shared memory
#pragma unroll
        for (int j = 0; j < N; ++j) shared_part[threadIdx.x * N + j] = acc[j];
        for (int w = GR / 2; w > 0; w >>= 1) {
            __syncthreads();
            if (group < w) {
#pragma unroll
                for (int j = 0; j < N; ++j) shared_part[threadIdx.x * N + j] += shared_part[(threadIdx.x + w * LV) * N + j];
            }
        }
        if (group == 0 && in) {
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = shared_part[threadIdx.x * N + j];
            write(at, key, acc);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------- launchers --

constexpr int64_t kMaxCount = INT32_MAX;

void check_embed(int dtype, const void* ids, int64_t n_entries, const int64_t* indptr,
                 int64_t n_out, int64_t n_rows, int64_t d) {
    if (dtype < MFM_DTYPE_F64 || dtype > MFM_DTYPE_F16)
        fail(MFM_ERR_INVALID, fmt("unknown dtype %d", dtype));
    if (n_entries < 0 || n_out < 0 || n_rows < 0)
        fail(MFM_ERR_INVALID, "negative embedding size");
    if (d < 1) fail(MFM_ERR_INVALID, "embedding width must be >= 1");
    if (n_entries > 0 && !ids) fail(MFM_ERR_INVALID, "ids must be provided");
    if (!indptr && n_out != n_entries)
        fail(MFM_ERR_INVALID, fmt("n_out %lld != n_entries %lld without indptr", (long long)n_out,
                                  (long long)n_entries));
    if (n_entries > kMaxCount || n_out > kMaxCount || n_rows > kMaxCount || d > kMaxCount)
        fail(MFM_ERR_UNSUPPORTED, "embedding sizes exceed the engine's 2^31-1 limit");
}

void check_pitch(const char* name, int64_t ld, int64_t d) {
    if (ld < d) fail(MFM_ERR_INVALID, fmt("row pitch of %s %lld < %lld", name, (long long)ld, (long long)d));
}

// f(T, A, O) of null pointers of the table, arithmetic and output-row types.
template <class F>
void with_embed_types(int dtype, F&& f) {
    switch (dtype) {
        case MFM_DTYPE_F64: f((double*)nullptr, (double*)nullptr, (double*)nullptr); break;
        case MFM_DTYPE_F32_F64: f((float*)nullptr, (double*)nullptr, (double*)nullptr); break;
        case MFM_DTYPE_F32: f((float*)nullptr, (float*)nullptr, (float*)nullptr); break;
        case MFM_DTYPE_BF16:
            f((__nv_bfloat16*)nullptr, (float*)nullptr, (__nv_bfloat16*)nullptr);
            break;
        default: f((__half*)nullptr, (float*)nullptr, (__half*)nullptr); break;
    }
}

// f(LV): lanes per row for dv vectors.
template <class F>
void with_lanes(int64_t dv, F&& f) {
    if (dv <= 1)
        f(std::integral_constant<int, 1>{});
    else if (dv <= 4)
        f(std::integral_constant<int, 4>{});
    else if (dv <= 8)
        f(std::integral_constant<int, 8>{});
    else if (dv <= 16)
        f(std::integral_constant<int, 16>{});
    else
        f(std::integral_constant<int, 32>{});
}

template <class P>
using Elem = std::remove_const_t<std::remove_pointer_t<std::remove_reference_t<P>>>;

template <class T, class A, class O, class I, int B>
void lookup_launch(int device, const I* ids, int64_t n, const int64_t* indptr, int64_t n_out,
                   const A* scale, A alpha, const T* table, int64_t n_rows, int64_t d, int64_t ld,
                   O* out, int64_t ld_out, cudaStream_t s) {
    constexpr int N = Lane<T, B>::N;
    const int64_t dv = d / N;
    const int64_t fill = (int64_t)sm_count(device) * 2048;  // threads at once
    if (indptr) {
        with_lanes(dv, [&](auto lv) {
            constexpr int LV = decltype(lv)::value, EL = LV >= 8 ? 1 : 8 / LV;
            const dim3 g((unsigned)ceil_div(n_out, 256 / (LV * EL)), (unsigned)ceil_div(dv, LV));
            embed_sums_kernel<T, A, O, I, B, LV, EL><<<g, 256, 0, s>>>(
                ids, n, indptr, n_out, scale, alpha, table, n_rows, d, ld, out, ld_out);
        });
    } else if (dv >= 32) {
        auto wide = [&](auto unroll) {
            constexpr int U = decltype(unroll)::value;
            const int64_t pieces = ceil_div(dv, 32 * U);
            embed_wide_kernel<T, A, O, I, B, U><<<(unsigned)ceil_div(n * pieces, 8), 256, 0, s>>>(
                ids, n, scale, alpha, table, n_rows, (int)dv, (int)pieces, ld, out, ld_out);
        };
        // fewer vectors a lane while the lanes do not fill the GPU
        if (n * dv >= 4 * fill && dv >= 128)
            wide(std::integral_constant<int, 4>{});
        else if (n * dv >= 2 * fill && dv >= 64)
            wide(std::integral_constant<int, 2>{});
        else
            wide(std::integral_constant<int, 1>{});
    } else {
        const int64_t total = n * dv;
        if (total <= fill)
            embed_rows_kernel<T, A, O, I, B, 1><<<(unsigned)ceil_div(total, 256), 256, 0, s>>>(
                ids, n, scale, alpha, table, n_rows, (uint32_t)dv, ld, out, ld_out);
        else
            embed_rows_kernel<T, A, O, I, B, 4><<<(unsigned)ceil_div(total, 1024), 256, 0, s>>>(
                ids, n, scale, alpha, table, n_rows, (uint32_t)dv, ld, out, ld_out);
    }
    MFM_CHECK_LAUNCH("embedding lookup launch");
}

// f(B) with the most bytes a lane that every row of T (and of a second type Q) begins on.
template <class T, class F>
void with_bytes(int64_t d, const void* p, int64_t ld, size_t q_size, const void* q, int64_t ld_q, F&& f) {
    auto fits = [&](int bytes) {
        const int n = bytes / (int)sizeof(T);
        return n >= 1 && d % n == 0 && vec_ok(p, ld, sizeof(T), n) &&
               vec_ok(q, ld_q, q_size, std::min<int>(n, 16 / (int)q_size));
    };
    if (fits(16))
        f(std::integral_constant<int, 16>{});
    else if (fits(8) && sizeof(T) < 8)
        f(std::integral_constant<int, 8>{});
    else
        f(std::integral_constant<int, 1>{});
}

// Workspace layout of the gradient, 256-byte aligned pieces.
struct GradWs {
    IdSortPlan sort;
    int64_t n_chunks = 0;
    size_t off_row = 0, off_scale = 0, off_base = 0, off_tile = 0, off_head = 0, off_tail = 0, off_bits = 0, bytes = 0;
    GradWs(int dtype, bool by_rows, int64_t n, int64_t n_rows, int64_t d) : sort(n, n_rows) {
        if (n <= kFewIds) return;  // none
        auto up = [](size_t b) { return (b + 255) / 256 * 256; };
        const size_t a = dtype == MFM_DTYPE_F64 || dtype == MFM_DTYPE_F32_F64 ? 8 : 4;
        n_chunks = ceil_div(n, kChunk);
        off_row = up((size_t)sort.words * 4 + 4);  // the block count is the last word
        off_scale = off_row + up((size_t)n * 4);
        off_base = off_scale + up((size_t)(n + kSortPad) * a);
        off_tile = off_base + up((size_t)n_chunks * 4);
        off_head = off_tile + up((size_t)ceil_div(n_chunks, kTileChunks) * 4);
        off_tail = off_head + up((size_t)n_chunks * d * a);
        off_bits = off_tail + up((size_t)n_chunks * d * a);
        bytes = off_bits + (by_rows || n <= kSmallSort ? 0 : up((size_t)ceil_div(n_rows, 32) * 4));
    }
};

template <class G, class T, class A, class O, int B>
void few_launch(int device, GradArgs<G, T, A, O>& a, cudaStream_t s) {
    const int64_t dv = a.d / Lane<G, B>::N, n = a.in.n, bytes = a.d * (int64_t)sizeof(O), sm = sm_count(device);
    with_lanes(dv, [&](auto lv) {
        constexpr int LV = decltype(lv)::value, GR = kFewIds / LV;
        const int64_t slabs = ceil_div(dv, LV), most = std::min(n, a.in.n_rows);
        a.reduce_blocks = (unsigned)std::min<int64_t>(ceil_div(most * slabs, GR), sm * 4);
        a.scale_blocks = a.d_scale ? (unsigned)ceil_div(n, GR * kScaleEntries) : 0u;
        a.fill_per = 32;
        while (a.fill_per > 1 && a.fill_per * bytes > 32768) a.fill_per /= 2;
        a.fill_blocks = (unsigned)std::min<int64_t>(
            ceil_div(a.rows ? most : a.in.n_rows, (int64_t)a.fill_per * (kFewIds / 32)), sm * 8);
        embed_few_kernel<G, T, A, O, B, LV><<<a.reduce_blocks + a.scale_blocks + a.fill_blocks, kFewIds, 0, s>>>(
            a, id_key_bits(a.in.n_rows), (int)slabs);
    });
    MFM_CHECK_LAUNCH("embedding gradient launch");
}

template <class G, class T, class A, class O, int B>
void grad_launch(int device, GradArgs<G, T, A, O>& a, const GradWs& W, char* ws, cudaStream_t s) {
    if (a.in.n <= kFewIds) {
        few_launch<G, T, A, O, B>(device, a, s);
        return;
    }
    constexpr int N = Lane<G, B>::N;
    const int64_t n = a.in.n, nc = W.n_chunks, dv = a.d / N;
    uint32_t* words = reinterpret_cast<uint32_t*>(ws);
    unsigned* done = words + W.sort.words;
    int32_t* row_of = a.in.indptr ? reinterpret_cast<int32_t*>(ws + W.off_row) : nullptr;
    SortedOut<A> sorted{};
    sorted.scale = a.scale;
    sorted.scales = reinterpret_cast<A*>(ws + W.off_scale);
    // a warp fills 32 rows, or fewer where the rows are long
    const int64_t bytes = a.d * (int64_t)sizeof(O), sm = sm_count(device);
    a.fill_per = 32;
    while (a.fill_per > 4 && a.fill_per * bytes > 32768) a.fill_per /= 2;
    // The untouched rows in parts: the launches behind the first pass take two shares
    // each, the main one, whose sums take bandwidth too, one (16384 x 2048 tokens into
    // 32000 rows: 81 us of kernels; 87 us with all of it in the main launch).
    Fill parts[6] = {};
    uint32_t* bits = nullptr;
    const bool late = nc > 1;
    if (a.d_table && n > kSmallSort) {
        bits = reinterpret_cast<uint32_t*>(ws + W.off_bits);
        const int early = W.sort.passes - 1, shares = 2 * early + 1 + (late ? 2 : 0);
        const int64_t groups = ceil_div(a.in.n_rows, 32);
        int64_t lo = 0;
        for (int i = 0, k = 0; i < early + 1 + (late ? 1 : 0); ++i) {
            k += i == early ? 1 : 2;
            const int64_t hi = std::min(a.in.n_rows, groups * k / shares * 32);
            const int64_t warps = ceil_div(hi - lo, (int64_t)a.fill_per);
            parts[i] = Fill{reinterpret_cast<char*>(a.d_table), bytes, lo, k == shares ? a.in.n_rows : hi, bits, a.fill_per, 0u};
            parts[i].blocks = (unsigned)std::min<int64_t>(ceil_div(warps, i == early ? kMainNT / 32 : 8), sm * (i == early ? 16 : 4));
            lo = hi;
        }
        a.fill = parts[early];
        if (late) a.fill_late = parts[early + 1];
    }
    sort_ids(device, W.sort, a.in, row_of, done, words, sorted, bits, parts, s);
    a.keys = sorted.keys;
    a.srows = sorted.rows;
    a.scales = a.scale ? sorted.scales : nullptr;
    a.row_of = row_of;
    a.n_chunks = nc;
    a.part_head = reinterpret_cast<A*>(ws + W.off_head);
    a.part_tail = reinterpret_cast<A*>(ws + W.off_tail);
    if (a.rows) {
        uint32_t* base = reinterpret_cast<uint32_t*>(ws + W.off_base);
        uint32_t* tiles = reinterpret_cast<uint32_t*>(ws + W.off_tile);
        launch_next(chunk_heads_kernel, (unsigned)ceil_div(nc, kTileChunks), kTileChunks, 0, s,
                    a.keys, n, (uint32_t)a.in.n_rows, nc, base, tiles, done, a.count);
        a.base = base;
        a.tile_base = tiles;
    }
    with_lanes(dv, [&](auto lv) {
        constexpr int LV = decltype(lv)::value;
        const int64_t slabs = ceil_div(dv, LV);
        a.reduce_blocks = (unsigned)(ceil_div(nc, kMainNT / LV) * slabs);
        a.scale_blocks = a.d_scale ? (unsigned)ceil_div(n, kMainNT / LV * kScaleEntries) : 0u;
        const int64_t rest = a.rows ? std::min(n, a.in.n_rows) : a.in.n_rows;
        a.fill_blocks = bits ? a.fill.blocks
                             : (unsigned)std::min<int64_t>(ceil_div(rest, (int64_t)a.fill_per * (kMainNT / 32)), sm * 16);
        launch_next(embed_main_kernel<G, T, A, O, B, LV>, a.reduce_blocks + a.scale_blocks + a.fill_blocks,
                    kMainNT, 0, s, a, (int)slabs);
        if (late) {
            a.cross_blocks = (unsigned)(ceil_div(nc, 256 / LV) * slabs);
            launch_next(embed_cross_kernel<G, T, A, O, B, LV>, a.cross_blocks + a.fill_late.blocks, 256, 0, s, a, (int)slabs);
        }
    });
    MFM_CHECK_LAUNCH("embedding gradient launch");
}

template <class G, class T, class A, class O>
void grad_entry(int device, GradArgs<G, T, A, O>& a, const GradWs& W, char* ws, cudaStream_t s) {
    const int64_t cap = std::min(a.in.n, a.in.n_rows);
    if (a.in.n == 0 || a.in.n_rows == 0 || a.in.n_out == 0) {  // nothing to add up
        auto set = [&](void* p, int value, size_t bytes) {
            if (p && bytes) MFM_CUDA(cudaMemsetAsync(p, value, bytes, s), "memset");
        };
        set(a.d_table, 0, (size_t)a.in.n_rows * a.d * sizeof(O));
        set(a.keys_out.p, 0xff, (size_t)cap * (a.keys_out.is64 ? 8 : 4));
        set(a.rows, 0, (size_t)cap * a.d * sizeof(O));
        set(a.count, 0, sizeof(int64_t));
        set(a.d_scale, 0, (size_t)a.in.n * sizeof(A));
        return;
    }
    const O* result = a.d_table ? a.d_table : a.rows;
    with_bytes<G>(a.d, a.grad, a.ld, sizeof(O), result, a.d, [&](auto bytes) {
        constexpr int B = decltype(bytes)::value, N = Lane<G, B>::N;
        // the table's rows may begin elsewhere
        if (N > 1 && a.d_scale && !vec_ok(a.table, a.ld_table, sizeof(T), N))
            grad_launch<G, T, A, O, 1>(device, a, W, ws, s);
        else
            grad_launch<G, T, A, O, B>(device, a, W, ws, s);
    });
}

}  // namespace
}  // namespace mfm

using namespace mfm;

extern "C" int mfm_embedding_lookup_device(int dtype, int device, int ids64, const void* ids,
                                           int64_t n_entries, const int64_t* indptr,
                                           int64_t n_out, const void* scale, double alpha,
                                           const void* table, int64_t n_rows, int64_t d,
                                           int64_t ld_table, void* out, int64_t ld_out,
                                           void* stream) {
    return guarded([&] {
        check_embed(dtype, ids, n_entries, indptr, n_out, n_rows, d);
        if (indptr && d > 65535 * 32)  // a grid's second axis, 32 values or more each
            fail(MFM_ERR_UNSUPPORTED, fmt("rows of %lld values are too long to be summed", (long long)d));
        if (n_out == 0) return;
        if ((n_rows > 0 && !table) || !out) fail(MFM_ERR_INVALID, "table and out must be provided");
        check_pitch("table", ld_table, d);
        check_pitch("out", ld_out, d);
        DeviceGuard g(device);
        with_embed_types(dtype, [&](auto* t, auto* a, auto* o) {
            using T = Elem<decltype(t)>;
            using A = Elem<decltype(a)>;
            using O = Elem<decltype(o)>;
            with_index_type(ids64, [&](auto* i) {
                using I = Elem<decltype(i)>;
                with_bytes<T>(d, table, ld_table, sizeof(O), out, ld_out, [&](auto bytes) {
                    lookup_launch<T, A, O, I, decltype(bytes)::value>(
                        device, (const I*)ids, n_entries, indptr, n_out, (const A*)scale, (A)alpha,
                        (const T*)table, n_rows, d, ld_table, (O*)out, ld_out, (cudaStream_t)stream);
                });
            });
        });
    });
}

extern "C" int64_t mfm_embedding_grad_workspace_bytes(int dtype, int by_rows, int64_t n_entries,
                                                      int64_t n_rows, int64_t d) {
    if (n_entries <= 0 || n_rows < 0 || d < 1 || n_entries > kMaxCount || n_rows > kMaxCount || d > kMaxCount)
        return 0;
    return (int64_t)GradWs(dtype, by_rows != 0, n_entries, n_rows, d).bytes;
}

extern "C" int mfm_embedding_grad_device(int dtype, int out_dtype, int device, int ids64,
                                         const void* ids, int64_t n_entries,
                                         const int64_t* indptr, int64_t n_out, const void* scale,
                                         double alpha, const void* grad, int64_t ld_grad,
                                         const void* table, int64_t ld_table, int64_t n_rows,
                                         int64_t d, void* d_table, void* keys, void* rows,
                                         int64_t* count, void* d_scale, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_embed(dtype, ids, n_entries, indptr, n_out, n_rows, d);
        const bool by_rows = keys || rows || count;
        if (by_rows ? (d_table || !keys || !rows || !count) : !d_table)
            fail(MFM_ERR_INVALID, "exactly one of d_table and (keys, rows, count) must be provided");
        const bool halves = dtype == MFM_DTYPE_BF16 || dtype == MFM_DTYPE_F16;
        const int own = dtype == MFM_DTYPE_F32_F64 ? MFM_DTYPE_F64 : dtype;
        if (out_dtype != own && !(halves && out_dtype == MFM_DTYPE_F32))
            fail(MFM_ERR_INVALID, fmt("out_dtype %d does not go with dtype %d", out_dtype, dtype));
        if (n_out > 0 && n_entries > 0) {
            if (!grad) fail(MFM_ERR_INVALID, "grad must be provided");
            check_pitch("grad", ld_grad, d);
        }
        if (d_scale && n_rows > 0 && n_entries > 0) {
            if (!table) fail(MFM_ERR_INVALID, "table must be provided for d_scale");
            check_pitch("table", ld_table, d);
        }
        DeviceGuard g(device);
        const GradWs W(dtype, by_rows, n_entries, n_rows, d);
        if (W.bytes > 0 && (!workspace || workspace_bytes < (int64_t)W.bytes))
            fail(MFM_ERR_INVALID, fmt("workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                                      (long long)W.bytes));
        if ((uintptr_t)workspace % 256) fail(MFM_ERR_INVALID, "workspace must be 256-byte aligned");
        with_embed_types(dtype, [&](auto* t, auto* a, auto* o) {
            using T = Elem<decltype(t)>;
            using A = Elem<decltype(a)>;
            using G = Elem<decltype(o)>;
            auto go = [&](auto* r) {
                using O = Elem<decltype(r)>;
                GradArgs<G, T, A, O> x{};
                x.in = Entries{Ids{ids, ids64}, n_entries, indptr, n_out, n_rows};
                x.scale = (const A*)scale;
                x.alpha = (A)alpha;
                x.grad = (const G*)grad;
                x.ld = ld_grad;
                x.table = (const T*)table;
                x.ld_table = ld_table;
                x.d = d;
                x.d_table = (O*)d_table;
                x.rows = (O*)rows;
                x.keys_out = KeysOut{keys, ids64};
                x.count = count;
                x.d_scale = (A*)d_scale;
                grad_entry(device, x, W, (char*)workspace, (cudaStream_t)stream);
            };
            if constexpr (sizeof(G) == 2) {
                if (out_dtype == MFM_DTYPE_F32) {
                    go((float*)nullptr);
                    return;
                }
            }
            go((G*)nullptr);
        });
    });
}
