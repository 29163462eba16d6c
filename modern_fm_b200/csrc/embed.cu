// embed.cu — latent rows as outputs: embedding lookup with scaling (single
// rows, or summed over the entries of sparse rows) and its gradient by sorted
// ids, over the whole table or the touched rows only.
#include "embed_sort.cuh"

#include <algorithm>

namespace mfm {
namespace {

// ---------------------------------------------------------------- lookup --

// out[t] = alpha scale[t] table[ids[t]]. One thread per vector of VEC elements,
// U of them in flight.
template <class T, class A, class O, class I, int VEC, int U>
__global__ void __launch_bounds__(256)
    embed_rows_kernel(const I* __restrict__ ids, int64_t n, const A* __restrict__ scale, A alpha,
                      const T* __restrict__ table, int64_t n_rows, uint32_t dv, int64_t ld,
                      O* __restrict__ out, int64_t ld_out) {
    const int64_t first = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = first / dv;
    const uint32_t off0 = (uint32_t)(first - row0 * dv);
    Vec<T, VEC> v[U];
    A f[U];
    int64_t row[U];
    uint32_t col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t o = off0 + threadIdx.x + u * 256;
        const uint32_t r = o / dv;
        row[u] = row0 + r;
        col[u] = (o - r * dv) * VEC;
        f[u] = A(0);
        if (row[u] < n) {
            const int64_t id = (int64_t)ids[row[u]];
            if (id >= 0 && id < n_rows) {
                v[u] = ldg_vec<T, VEC>(table + id * ld + col[u]);
                f[u] = alpha;
                if (scale) f[u] *= scale[row[u]];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[u].v[j] = narrow<T>(A(0));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (row[u] < n) {
            Vec<O, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = narrow<O>(f[u] * widen<A>(v[u].v[j]));
            *reinterpret_cast<Vec<O, VEC>*>(out + row[u] * ld_out + col[u]) = o;
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

// out[b] = alpha sum_t scale[t] table[ids[t]]: LV lanes per row, each a vector of
// VEC columns, four entries in flight; blockIdx.y walks the columns.
template <class T, class A, class O, class I, int VEC, int LV>
__global__ void __launch_bounds__(256)
    embed_sums_kernel(const I* __restrict__ ids, int64_t n, const int64_t* __restrict__ indptr,
                      int64_t n_out, const A* __restrict__ scale, A alpha,
                      const T* __restrict__ table, int64_t n_rows, int64_t d, int64_t ld,
                      O* __restrict__ out, int64_t ld_out) {
    constexpr int U = 4;
    const int lane = threadIdx.x % LV;
    const int64_t b = (int64_t)blockIdx.x * (256 / LV) + threadIdx.x / LV;
    const int64_t col = ((int64_t)blockIdx.y * LV + lane) * VEC;
    if (b >= n_out || col >= d) return;
    int64_t lo, hi;
    row_bounds(indptr, b, n, lo, hi);
    A acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = A(0);
    for (int64_t e = lo; e < hi; e += U) {
        Vec<T, VEC> v[U];
        A f[U];
        bool live[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            live[u] = false;
            f[u] = A(1);
            if (e + u < hi) {
                const int64_t id = (int64_t)ids[e + u];
                live[u] = id >= 0 && id < n_rows;
                if (scale) f[u] = scale[e + u];
                if (live[u]) v[u] = ldg_vec<T, VEC>(table + id * ld + col);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u])
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += f[u] * widen<A>(v[u].v[j]);
    }
    Vec<O, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.v[j] = narrow<O>(alpha * acc[j]);
    *reinterpret_cast<Vec<O, VEC>*>(out + b * ld_out + col) = o;
}

// -------------------------------------------------------------- gradient --

constexpr int kChunk = 32;  // sorted entries per lane group

// row_of[t] = the output row whose sum entry t belongs to, -1 for none.
__global__ void entry_rows_kernel(const int64_t* __restrict__ indptr, int64_t n_out, int64_t n,
                                  int32_t* __restrict__ row_of) {
    const int64_t stride = (int64_t)gridDim.x * blockDim.x / 32;
    for (int64_t b = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32; b < n_out; b += stride) {
        int64_t lo, hi;
        row_bounds(indptr, b, n, lo, hi);
        for (int64_t t = lo + (threadIdx.x & 31); t < hi; t += 32) row_of[t] = (int32_t)b;
    }
}

// heads[c] = how many runs of equal real keys begin in chunk c.
__global__ void chunk_heads_kernel(const uint32_t* __restrict__ keys, int64_t n, uint32_t pad_key,
                                   int64_t n_chunks, uint32_t* __restrict__ heads) {
    const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
    const int64_t e = c * kChunk + (threadIdx.x & 31);
    bool head = false;
    if (e < n) {
        const uint32_t k = keys[e];
        head = k != pad_key && (e == 0 || keys[e - 1] != k);
    }
    const unsigned m = __ballot_sync(0xffffffffu, head);
    if ((threadIdx.x & 31) == 0 && c < n_chunks) heads[c] = (uint32_t)__popc(m);
}

template <class O, class I>
struct GradOut {  // where a finished run goes
    O* table;          // (n_rows, d), or
    O* rows;           // (cap, d) by rank with
    I* keys;           // the ids
    const uint32_t* base;  // runs begun before each chunk
};

// One chunk of kChunk sorted entries x LV * VEC columns by one lane group: sums
// of scale[pos] grad[row], run by run. A run that lies in the chunk is
// written; the part of a run that began before goes to part_head[chunk], the
// part of one that goes on behind to part_tail[chunk] (all of it to part_head
// when both).
template <class G, class A, class O, class I, int VEC, int LV>
__global__ void __launch_bounds__(128)
    embed_reduce_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                        int64_t n, uint32_t pad_key, const int32_t* __restrict__ row_of,
                        const A* __restrict__ scale, A alpha, const G* __restrict__ grad,
                        int64_t ld, int64_t d, int64_t n_chunks, A* __restrict__ part_head,
                        A* __restrict__ part_tail, GradOut<O, I> out) {
    constexpr int U = 8;
    const int lane = threadIdx.x % LV;
    const int64_t c = (int64_t)blockIdx.x * (128 / LV) + threadIdx.x / LV;
    const int64_t col = ((int64_t)blockIdx.y * LV + lane) * VEC;
    if (c >= n_chunks || col >= d) return;
    const int64_t e0 = c * kChunk, e1 = e0 + kChunk < n ? e0 + kChunk : n;
    uint32_t cur = keys[e0];
    bool begun_before = e0 > 0 && keys[e0 - 1] == cur;
    uint32_t rank = out.rows ? out.base[c] - (begun_before ? 1u : 0u) : 0u;
    A acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = A(0);
    auto put = [&](uint32_t key) {  // a run ends inside the chunk
        if (begun_before) {
            Vec<A, VEC> p;
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.v[j] = acc[j];
            *reinterpret_cast<Vec<A, VEC>*>(part_head + c * d + col) = p;
        } else {
            Vec<O, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = narrow<O>(alpha * acc[j]);
            O* base = out.rows ? out.rows + (int64_t)rank * d : out.table + (int64_t)key * d;
            *reinterpret_cast<Vec<O, VEC>*>(base + col) = o;
        }
        if (out.keys && !begun_before && col == 0) out.keys[rank] = (I)key;
    };
    for (int64_t e = e0; e < e1; e += U) {
        uint32_t k[U];
        A f[U];
        Vec<G, VEC> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = pad_key;
            f[u] = A(1);
            if (e + u < e1) k[u] = keys[e + u];
            if (k[u] != pad_key) {
                const uint32_t p = pos[e + u];
                const int64_t row = row_of ? (int64_t)row_of[p] : (int64_t)p;
                if (scale) f[u] = scale[p];
                v[u] = ldg_vec<G, VEC>(grad + row * ld + col);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (e + u >= e1) break;
            if (k[u] != cur) {
                put(cur);
                cur = k[u];
                begun_before = false;
                ++rank;
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = A(0);
            }
            if (cur == pad_key) return;  // padding sorts last
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += f[u] * widen<A>(v[u].v[j]);
        }
    }
    if (e1 < n && keys[e1] == cur) {  // the run goes on behind the chunk
        Vec<A, VEC> p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.v[j] = acc[j];
        A* part = begun_before ? part_head : part_tail;
        *reinterpret_cast<Vec<A, VEC>*>(part + c * d + col) = p;
    } else {
        put(cur);
    }
}

// The runs that cross chunks: the lane group of the chunk where one begins adds
// its parts in chunk order and writes the run.
template <class A, class O, class I, int VEC, int LV>
__global__ void __launch_bounds__(128)
    embed_cross_kernel(const uint32_t* __restrict__ keys, int64_t n, uint32_t pad_key, A alpha,
                       int64_t d, int64_t n_chunks, const A* __restrict__ part_head,
                       const A* __restrict__ part_tail, GradOut<O, I> out) {
    const int lane = threadIdx.x % LV;
    const int64_t c = (int64_t)blockIdx.x * (128 / LV) + threadIdx.x / LV;
    const int64_t col = ((int64_t)blockIdx.y * LV + lane) * VEC;
    if (c + 1 >= n_chunks || col >= d) return;
    const int64_t e0 = c * kChunk, e1 = e0 + kChunk;  // not the last chunk: e1 < n
    const uint32_t key = keys[e1 - 1];
    if (key == pad_key || keys[e1] != key) return;
    if (e0 > 0 && keys[e0 - 1] == key) return;  // began before this chunk
    int64_t lo = e1, hi = n;  // first entry behind the run
    while (lo < hi) {
        const int64_t mid = lo + (hi - lo) / 2;
        if (keys[mid] > key)
            hi = mid;
        else
            lo = mid + 1;
    }
    const int64_t last = (lo - 1) / kChunk;
    Vec<A, VEC> acc = ldg_vec<A, VEC>(part_tail + c * d + col);
#pragma unroll 8
    for (int64_t k = c + 1; k <= last; ++k) {
        const Vec<A, VEC> p = ldg_vec<A, VEC>(part_head + k * d + col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc.v[j] += p.v[j];
    }
    const int64_t at = out.rows ? (int64_t)out.base[c + 1] - 1 : (int64_t)key;
    Vec<O, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.v[j] = narrow<O>(alpha * acc.v[j]);
    *reinterpret_cast<Vec<O, VEC>*>((out.rows ? out.rows : out.table) + at * d + col) = o;
    if (out.keys && col == 0) out.keys[at] = (I)key;
}

__global__ void run_count_kernel(const uint32_t* base, int64_t n_chunks, int64_t* count) {
    *count = base[n_chunks];
}

// d_scale[t] = alpha <grad[row(t)], table[ids[t]]>: one warp per entry.
template <class G, class T, class A, class I, int VEC>
__global__ void __launch_bounds__(256)
    embed_scale_kernel(const I* __restrict__ ids, int64_t n, const int32_t* __restrict__ row_of,
                       A alpha, const G* __restrict__ grad, int64_t ld, const T* __restrict__ table,
                       int64_t n_rows, int64_t ld_table, int64_t d, A* __restrict__ d_scale) {
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    if (t >= n) return;
    const int64_t id = (int64_t)ids[t], row = row_of ? (int64_t)row_of[t] : t;
    A acc = A(0);
    if (id >= 0 && id < n_rows && row >= 0)
        for (int64_t c = (int64_t)lane * VEC; c < d; c += 32 * VEC) {
            const Vec<G, VEC> g = ldg_vec<G, VEC>(grad + row * ld + c);
            const Vec<T, VEC> v = ldg_vec<T, VEC>(table + id * ld_table + c);
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc += widen<A>(g.v[j]) * widen<A>(v.v[j]);
        }
    acc = warp_sum(acc);
    if (lane == 0) d_scale[t] = alpha * acc;
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

// f(integral constant): lanes per row for dv vectors.
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
using Elem = std::remove_pointer_t<std::remove_reference_t<P>>;

template <class T, class A, class O, class I, int VEC>
void lookup_launch(int device, const I* ids, int64_t n, const int64_t* indptr, int64_t n_out,
                   const A* scale, A alpha, const T* table, int64_t n_rows, int64_t d, int64_t ld,
                   O* out, int64_t ld_out, cudaStream_t s) {
    const int64_t dv = d / VEC;
    if (!indptr) {
        const int64_t total = n * dv;
        if (total <= (int64_t)sm_count(device) * 2048)
            embed_rows_kernel<T, A, O, I, VEC, 1><<<(unsigned)ceil_div(total, 256), 256, 0, s>>>(
                ids, n, scale, alpha, table, n_rows, (uint32_t)dv, ld, out, ld_out);
        else
            embed_rows_kernel<T, A, O, I, VEC, 4><<<(unsigned)ceil_div(total, 1024), 256, 0, s>>>(
                ids, n, scale, alpha, table, n_rows, (uint32_t)dv, ld, out, ld_out);
    } else {
        with_lanes(dv, [&](auto lv) {
            constexpr int LV = decltype(lv)::value;
            const dim3 g((unsigned)ceil_div(n_out, 256 / LV), (unsigned)ceil_div(dv, LV));
            embed_sums_kernel<T, A, O, I, VEC, LV><<<g, 256, 0, s>>>(
                ids, n, indptr, n_out, scale, alpha, table, n_rows, d, ld, out, ld_out);
        });
    }
    MFM_CHECK_LAUNCH("embedding lookup launch");
}

// Workspace layout of the gradient, 256-byte aligned pieces.
struct GradWs {
    IdSortPlan sort;
    int64_t n_chunks = 0;
    size_t off_row = 0, off_base = 0, off_sums = 0, off_head = 0, off_tail = 0, bytes = 0;
    GradWs(int dtype, int64_t n, int64_t n_rows, int64_t d) : sort(n, n_rows) {
        auto up = [](size_t b) { return (b + 255) / 256 * 256; };
        const size_t a = dtype == MFM_DTYPE_F64 || dtype == MFM_DTYPE_F32_F64 ? 8 : 4;
        n_chunks = ceil_div(n, kChunk);
        off_row = up((size_t)sort.words * 4);
        off_base = off_row + up((size_t)n * 4);
        off_sums = off_base + up((size_t)(n_chunks + 1) * 4);
        off_head = off_sums + up((size_t)(ceil_div(n_chunks, kScanTile) + 2) * 4);
        off_tail = off_head + up((size_t)n_chunks * d * a);
        bytes = off_tail + up((size_t)n_chunks * d * a);
    }
};

template <class G, class T, class A, class O, class I>
struct GradArgs {
    int device;
    const I* ids;
    int64_t n;
    const int64_t* indptr;
    int64_t n_out;
    const A* scale;
    A alpha;
    const G* grad;
    int64_t ld;
    const T* table;
    int64_t ld_table, n_rows, d;
    O *d_table, *rows;
    I* keys;
    int64_t* count;
    A* d_scale;
    char* ws;
    cudaStream_t s;
};

template <class G, class T, class A, class O, class I, int VEC>
void grad_launch(const GradArgs<G, T, A, O, I>& a, const GradWs& W) {
    const uint32_t pad = (uint32_t)a.n_rows;
    int32_t* row_of = nullptr;
    if (a.indptr) {
        row_of = reinterpret_cast<int32_t*>(a.ws + W.off_row);
        MFM_CUDA(cudaMemsetAsync(row_of, 0xff, (size_t)a.n * 4, a.s), "memset");
        if (a.n_out > 0)
            entry_rows_kernel<<<warp_grid(a.device, a.n_out, 8, 8), 256, 0, a.s>>>(a.indptr, a.n_out, a.n, row_of);
    }
    if (a.d_scale) {
        const bool ok = vec_ok(a.table, a.ld_table, sizeof(T), VEC);
        const unsigned g = (unsigned)ceil_div(a.n, 8);
        if (ok)
            embed_scale_kernel<G, T, A, I, VEC><<<g, 256, 0, a.s>>>(a.ids, a.n, row_of, a.alpha, a.grad, a.ld, a.table, a.n_rows, a.ld_table, a.d, a.d_scale);
        else
            embed_scale_kernel<G, T, A, I, 1><<<g, 256, 0, a.s>>>(a.ids, a.n, row_of, a.alpha, a.grad, a.ld, a.table, a.n_rows, a.ld_table, a.d, a.d_scale);
    }
    const IdSorted S = sort_ids(W.sort, a.ids, row_of, a.n_rows, reinterpret_cast<uint32_t*>(a.ws), a.s);
    GradOut<O, I> out{a.d_table, a.rows, a.keys, nullptr};
    const int64_t nc = W.n_chunks;
    if (a.rows) {
        uint32_t* base = reinterpret_cast<uint32_t*>(a.ws + W.off_base);
        uint32_t* sums = reinterpret_cast<uint32_t*>(a.ws + W.off_sums);
        chunk_heads_kernel<<<(unsigned)ceil_div(nc, 8), 256, 0, a.s>>>(S.keys, a.n, pad, nc, base);
        const int64_t nb = ceil_div(nc, kScanTile);
        scan_reduce_kernel<uint32_t, uint32_t><<<(unsigned)nb, kScanNT, 0, a.s>>>(base, nc, sums);
        scan_sums_kernel<uint32_t><<<1, kScanNT, 0, a.s>>>(sums, nb);
        scan_apply_kernel<uint32_t, uint32_t><<<(unsigned)nb, kScanNT, 0, a.s>>>(base, nc, sums, base);
        run_count_kernel<<<1, 1, 0, a.s>>>(base, nc, a.count);
        out.base = base;
    }
    A* head = reinterpret_cast<A*>(a.ws + W.off_head);
    A* tail = reinterpret_cast<A*>(a.ws + W.off_tail);
    with_lanes(a.d / VEC, [&](auto lv) {
        constexpr int LV = decltype(lv)::value;
        const dim3 g((unsigned)ceil_div(nc, 128 / LV), (unsigned)ceil_div(a.d / VEC, LV));
        embed_reduce_kernel<G, A, O, I, VEC, LV><<<g, 128, 0, a.s>>>(
            S.keys, S.pos, a.n, pad, row_of, a.scale, a.alpha, a.grad, a.ld, a.d, nc, head, tail, out);
        embed_cross_kernel<A, O, I, VEC, LV><<<g, 128, 0, a.s>>>(S.keys, a.n, pad, a.alpha, a.d, nc, head, tail, out);
    });
    MFM_CHECK_LAUNCH("embedding gradient launch");
}

template <class G, class T, class A, class O, class I>
void grad_entry(const GradArgs<G, T, A, O, I>& a, const GradWs& W) {
    // rows of the result that nothing touches
    const int64_t cap = std::min(a.n, a.n_rows);
    if (a.d_table) MFM_CUDA(cudaMemsetAsync(a.d_table, 0, (size_t)a.n_rows * a.d * sizeof(O), a.s), "memset");
    if (a.keys) {
        MFM_CUDA(cudaMemsetAsync(a.keys, 0xff, (size_t)cap * sizeof(I), a.s), "memset");
        MFM_CUDA(cudaMemsetAsync(a.rows, 0, (size_t)cap * a.d * sizeof(O), a.s), "memset");
        MFM_CUDA(cudaMemsetAsync(a.count, 0, sizeof(int64_t), a.s), "memset");
    }
    if (a.n == 0) return;
    if (a.n_rows == 0 || a.n_out == 0) {  // nothing to add up
        if (a.d_scale) MFM_CUDA(cudaMemsetAsync(a.d_scale, 0, (size_t)a.n * sizeof(A), a.s), "memset");
        return;
    }
    constexpr int VEC = 16 / sizeof(G);
    if (vec_ok(a.grad, a.ld, sizeof(G), VEC) && vec_ok(a.d_table ? a.d_table : a.rows, a.d, sizeof(O), VEC))
        grad_launch<G, T, A, O, I, VEC>(a, W);
    else
        grad_launch<G, T, A, O, I, 1>(a, W);
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
                using I = std::remove_const_t<Elem<decltype(i)>>;
                constexpr int VEC = 16 / sizeof(T);
                auto go = [&](auto vec) {
                    lookup_launch<T, A, O, I, decltype(vec)::value>(
                        device, (const I*)ids, n_entries, indptr, n_out, (const A*)scale, (A)alpha,
                        (const T*)table, n_rows, d, ld_table, (O*)out, ld_out, (cudaStream_t)stream);
                };
                if (d % VEC == 0 && vec_ok(table, ld_table, sizeof(T), VEC) && vec_ok(out, ld_out, sizeof(O), VEC))
                    go(std::integral_constant<int, VEC>{});
                else
                    go(std::integral_constant<int, 1>{});
            });
        });
    });
}

extern "C" int64_t mfm_embedding_grad_workspace_bytes(int dtype, int64_t n_entries,
                                                      int64_t n_rows, int64_t d) {
    if (n_entries <= 0 || n_rows < 0 || d < 1 || n_entries > kMaxCount || n_rows > kMaxCount || d > kMaxCount)
        return 0;
    return (int64_t)GradWs(dtype, n_entries, n_rows, d).bytes;
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
        const GradWs W(dtype, n_entries, n_rows, d);
        if (n_entries > 0 && (!workspace || workspace_bytes < (int64_t)W.bytes))
            fail(MFM_ERR_INVALID, fmt("workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                                      (long long)W.bytes));
        if ((uintptr_t)workspace % 256) fail(MFM_ERR_INVALID, "workspace must be 256-byte aligned");
        with_embed_types(dtype, [&](auto* t, auto* a, auto* o) {
            using T = Elem<decltype(t)>;
            using A = Elem<decltype(a)>;
            using G = Elem<decltype(o)>;
            with_index_type(ids64, [&](auto* i) {
                using I = std::remove_const_t<Elem<decltype(i)>>;
                auto go = [&](auto* r) {
                    using O = Elem<decltype(r)>;
                    GradArgs<G, T, A, O, I> x{device, (const I*)ids, n_entries, indptr, n_out,
                                              (const A*)scale, (A)alpha, (const G*)grad, ld_grad,
                                              (const T*)table, ld_table, n_rows, d, (O*)d_table,
                                              (O*)rows, (I*)keys, count, (A*)d_scale,
                                              (char*)workspace, (cudaStream_t)stream};
                    grad_entry(x, W);
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
    });
}
