// features.hip -- rows of learned features: lookup in a shared table with the gradient by sorted index, layer norm.
//
// Both are bound by memory: a value is touched by a handful of operations, so the kernels are laid out for 16-byte packs,
// few passes over the data and enough bytes in flight.  All sums run in fp32 and in an order that depends on sizes, strides
// and alignment alone (no floating-point atomics): results are the same bit for bit from call to call.
#include "rows.h"

int e3_fail(hipError_t e, const char* what);
int launch_radix_sort_pairs(uint32_t* k0, uint32_t* k1, uint32_t* v0, uint32_t* v1, size_t n, int nbits,
                            uint32_t* scratch, uint32_t** keys_out, uint32_t** vals_out, hipStream_t s,
                            bool identity_payload, uint32_t* drop_count_dev, const uint32_t* n_dev, uint2* ranges_out,
                            uint32_t nranges, uint32_t* lpt_cnt, uint32_t* lpt_list);
#define LAUNCH_OK(name)                                       \
    do {                                                      \
        hipError_t _e = hipGetLastError();                    \
        if (_e != hipSuccess) return e3_fail(_e, name);       \
    } while (0)
// whether one launch takes that many workgroups: the threads past 2^32 would be cut off without an error
static inline bool grid_fits(size_t blocks, size_t threads) { return blocks < ((size_t)1 << 32) / threads; }

// ============================================================================================== embedding, forward
// out[i, :] = round(scale * table[index[i], :]).  An index below 0 stands for "no row" (zeros); one past the table gives a
// row of NaN -- an error that only the device sees, made visible without a wait.
// One thread moves several packs of the flat output (4 of 16 bytes, 8 of 4 or 8: a workgroup waits for the index, then for the
// row, and has to have enough behind that), a workgroup's packs are contiguous: every lane works whatever the row length, the
// stores are whole lines, and the rows of a pack-block are found by one division each.
template <typename T, int V>
struct EmbedPacks {
    static constexpr int N = V * (int)sizeof(T) == 16 ? 4 : 8;
};
template <bool STREAM, typename T, int V, typename I>
__global__ __launch_bounds__(256) void embed_fwd_kernel(size_t n, long long rows, uint32_t ppr /* packs per row */,
                                                        const I* __restrict__ index, const T* __restrict__ table, size_t stride, float scale,
                                                        T* __restrict__ out) {
    constexpr int PACKS = EmbedPacks<T, V>::N;
    const size_t total = n * (size_t)ppr, base = (size_t)blockIdx.x * (256 * PACKS);
    const size_t row0 = base / ppr;                                  // (uniform)
    const uint32_t rem0 = (uint32_t)(base - row0 * ppr);
    const uint32_t last = n - 1 - row0 < 0x7FFFFFFFu ? (uint32_t)(n - 1 - row0) : 0x7FFFFFFFu;
    const uint32_t count = total - base < 256 * PACKS ? (uint32_t)(total - base) : 256 * PACKS;
    index += row0;
    out += base * V;
    const uint32_t dq = 256 / ppr, dr = 256 - dq * ppr;              // one pack on to the next: one division for all
    uint32_t q = (rem0 + threadIdx.x) / ppr, c = rem0 + threadIdx.x - q * ppr;
    I id[PACKS];
    uint32_t col[PACKS];
    Pack<T, V> p[PACKS];
#pragma unroll
    for (int u = 0; u < PACKS; ++u) {
        col[u] = c;
        id[u] = index[q < last ? q : last];                          // (unconditional loads, all in flight)
        q += dq;
        c += dr;
        if (c >= ppr) {
            c -= ppr;
            ++q;
        }
    }
#pragma unroll
    for (int u = 0; u < PACKS; ++u) {
        if (id[u] >= 0 && id[u] < rows)
            p[u] = *reinterpret_cast<const Pack<T, V>*>(table + (size_t)(uint32_t)id[u] * stride + (size_t)col[u] * V);
    }
#pragma unroll
    for (int u = 0; u < PACKS; ++u) {
        const uint32_t at = (uint32_t)u * 256 + threadIdx.x;
        if (at >= count) continue;
        Pack<T, V> r;
#pragma unroll
        for (int j = 0; j < V; ++j)
            r.v[j] = id[u] < 0 ? (T)0.0f : (id[u] < rows ? (T)(scale * (float)p[u].v[j]) : (T)__builtin_nanf(""));
        put<STREAM, T, V>(out + (size_t)at * V, r);
    }
}

// Rows that are no multiple of 4 bytes (8 for fp32), or do not lie on such a boundary: a workgroup gathers EMBED_FLAT values one
// by one into LDS and stores them from there in packs; the indices of its rows wait in LDS too.  Bound by the issue of the
// single loads (408482 x 115 fp16 41 us; with an index and a store to every value 51 us; 21053 x 567 fp32 15 and 20 us).
constexpr int EMBED_FLAT = 4096;
template <bool STREAM, typename T, typename I>
__global__ __launch_bounds__(256) void embed_fwd_odd_kernel(size_t n, long long rows, uint32_t dim, const I* __restrict__ index,
                                                            const T* __restrict__ table, size_t stride, float scale, T* __restrict__ out) {
    constexpr int EACH = EMBED_FLAT / 256, BATCH = 8, N = Wide<T>::N;
    __shared__ words_t tile[EMBED_FLAT / N];
    __shared__ int ids[EMBED_FLAT + 2];                              // -1: zeros, ID_PAST: NaN
    constexpr int ID_PAST = 0x7FFFFFFF;
    T* values = reinterpret_cast<T*>(tile);
    const size_t total = n * (size_t)dim, base = (size_t)blockIdx.x * EMBED_FLAT;
    const size_t row0 = base / dim;                                  // (uniform)
    const uint32_t rem0 = (uint32_t)(base - row0 * dim);
    const uint32_t count = total - base < EMBED_FLAT ? (uint32_t)(total - base) : EMBED_FLAT;
    const uint32_t nids = (rem0 + count - 1) / dim + 1;
    for (uint32_t i = threadIdx.x; i < nids; i += 256) {
        const I id = index[row0 + i];
        ids[i] = id < 0 ? -1 : id < rows ? (int)id : ID_PAST;
    }
    __syncthreads();
    const uint32_t dq = 256 / dim, dr = 256 - dq * dim;
    uint32_t q = (rem0 + threadIdx.x) / dim, c = rem0 + threadIdx.x - q * dim;
#pragma unroll
    for (int b = 0; b < EACH; b += BATCH) {
        int id[BATCH];
        uint32_t v[BATCH];                                           // (a register each: halves of one would wait for each other)
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            id[u] = (uint32_t)(b + u) * 256 + threadIdx.x < count ? ids[q] : -1;
            const bool in = id[u] >= 0 && id[u] != ID_PAST;
            v[u] = reinterpret_cast<const Bits<T>*>(table)[in ? (size_t)(uint32_t)id[u] * stride + c : 0];      // (unconditional)
            q += dq;
            c += dr;
            if (c >= dim) {
                c -= dim;
                ++q;
            }
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
            values[(b + u) * 256 + threadIdx.x] = id[u] < 0 ? (T)0.0f : id[u] == ID_PAST ? (T)__builtin_nanf("") : (T)(scale * (float)bits_elem<T>(v[u]));
    }
    __syncthreads();
    out += base;
    const uint32_t packs = (reinterpret_cast<uintptr_t>(out) & 15) == 0 ? count / N : 0u;
    for (uint32_t i = threadIdx.x; i < packs; i += 256) put<STREAM, T, N>(out + (size_t)i * N, reinterpret_cast<const Pack<T, N>*>(tile)[i]);
    for (uint32_t i = packs * N + threadIdx.x; i < count; i += 256) out[i] = values[i];
}

template <bool STREAM, typename T, int V, typename I>
static int embed_fwd_launch(size_t n, size_t rows, size_t dim, const void* index, const void* table, size_t stride, float scale,
                            void* out, hipStream_t s) {
    const size_t ppr = dim / V, each = 256 * EmbedPacks<T, V>::N, blocks = (n * ppr + each - 1) / each;
    embed_fwd_kernel<STREAM, T, V, I><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(
        n, (long long)rows, (uint32_t)ppr, (const I*)index, (const T*)table, stride, scale, (T*)out);
    LAUNCH_OK("embed_fwd_kernel");
    return 0;
}
template <typename T, typename I>
static int embed_fwd_t(size_t n, size_t rows, size_t dim, const void* index, const void* table, size_t stride, int dtype,
                       float scale, void* out, hipStream_t s) {
    constexpr int N = Wide<T>::N;
    const bool large = n * dim * sizeof(T) > E3_STREAM_BYTES;
    if (rows == 0) table = index;                              // (no row is read; the odd kernel's loads need some address)
    auto fits = [&](size_t bytes) { return e3_rows_packs(table, stride, dim, dtype, bytes) && e3_rows_packs(out, dim, dim, dtype, bytes); };
    if (fits(16) && large) return embed_fwd_launch<true, T, N, I>(n, rows, dim, index, table, stride, scale, out, s);
    if (fits(16)) return embed_fwd_launch<false, T, N, I>(n, rows, dim, index, table, stride, scale, out, s);
    if (fits(8)) return embed_fwd_launch<false, T, N / 2, I>(n, rows, dim, index, table, stride, scale, out, s);
    if (N == 8 && fits(4)) return embed_fwd_launch<false, T, 2, I>(n, rows, dim, index, table, stride, scale, out, s);
    const size_t blocks = (n * dim + EMBED_FLAT - 1) / EMBED_FLAT;
    if (large) embed_fwd_odd_kernel<true, T, I><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(
        n, (long long)rows, (uint32_t)dim, (const I*)index, (const T*)table, stride, scale, (T*)out);
    else embed_fwd_odd_kernel<false, T, I><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(
        n, (long long)rows, (uint32_t)dim, (const I*)index, (const T*)table, stride, scale, (T*)out);
    LAUNCH_OK("embed_fwd_odd_kernel");
    return 0;
}

int e3_embedding_forward_impl(size_t n, size_t rows, size_t dim, const void* index, int index_bytes, const void* table,
                              size_t stride, int dtype, float scale, void* out, hipStream_t s) {
    // A launch ends before 2^32 threads (those past it are cut off without an error), so large results take several: 2^35 values
    // are at most 2^23 workgroups of 4096 values or more.  A slice is a multiple of 8 rows: `out` keeps its boundary.
    const size_t each = ((size_t)1 << 35) / dim / 8 * 8;
    for (size_t at = 0; at < n; at += each) {
        const size_t m = n - at < each ? n - at : each;
        const void* idx = reinterpret_cast<const char*>(index) + at * index_bytes;
        void* to = reinterpret_cast<char*>(out) + at * dim * e3_elem_bytes(dtype);
#define E3_FWD(T) (index_bytes == 8 ? embed_fwd_t<T, long long>(m, rows, dim, idx, table, stride, dtype, scale, to, s) \
                                    : embed_fwd_t<T, int>(m, rows, dim, idx, table, stride, dtype, scale, to, s))
        const int rc = dtype == E3_F32 ? E3_FWD(float) : dtype == E3_F16 ? E3_FWD(f16_t) : E3_FWD(bf16_t);
#undef E3_FWD
        if (rc) return rc;
    }
    return 0;
}

// ============================================================================================== embedding, gradient
// d_table[v, :] = round(scale * sum of d_out[i, :] over the positions i with index[i] == v, in the order of i).
// The positions are sorted by index (stable), so that a row's positions are one run of the sorted list; the list is cut
// into chunks of equal length, a group of lanes sums the rows of one chunk (times a slice of the columns), and
//   * a run inside a chunk is finished there,
//   * a run that crosses chunks leaves one fp32 partial row per chunk, which embed_join_kernel adds up in order,
//   * a table row without a position is cleared by further workgroups of the same launch (embed_zero), or with all others beside
//     the sort where one workgroup sorts.
// So a row that half of all positions share costs no more than rows with one position each.
constexpr uint32_t EMBED_NONE = 0xFFFFFFFFu;

__global__ __launch_bounds__(256) void embed_keys_kernel(size_t n, unsigned long long rows, const void* __restrict__ index,
                                                         int index_bytes, uint32_t* __restrict__ keys) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const unsigned long long id = (unsigned long long)load_index(index, i, index_bytes);   // (negative: beyond any row)
    keys[i] = id < rows ? (uint32_t)id : EMBED_NONE;
}

// first position of the sorted keys [lo, hi) that holds a key >= k
__device__ __forceinline__ uint32_t lower_bound_u32(const uint32_t* __restrict__ keys, uint32_t lo, uint32_t hi, uint32_t k) {
    while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < k) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T, int V>
__device__ __forceinline__ void embed_store(T* __restrict__ d_table, size_t dim, uint32_t row, size_t col, float scale,
                                            const float acc[V]) {
    Pack<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = (T)(scale * acc[j]);
    *reinterpret_cast<Pack<T, V>*>(d_table + (size_t)row * dim + col) = r;
}

// Clears table rows: a wave takes `per` rows from `first` on, each of its lanes knows whether one of them is to be cleared.
template <bool STREAM, typename T, int V>
__device__ __forceinline__ void embed_zero(bool empty, size_t first, uint32_t rows, uint32_t per, size_t dim, T* __restrict__ d_table) {
    const int lane = threadIdx.x & 63;
    unsigned long long todo = __ballot(empty);
    if (todo == 0ull) return;
    const uint32_t count = (uint32_t)__popcll(todo), mine = rows - first < per ? (uint32_t)(rows - first) : per;
    if (V == 1 && count == mine) {
        // none of the wave's rows is named (most waves of a large table): one stretch of memory, in 16-byte packs (with packs of
        // 4 or 8 bytes row by row is the quicker way: 44064 rows of 84 bf16 14 us, as one stretch 17)
        constexpr int N = Wide<T>::N;
        T* p = d_table + first * dim;
        const size_t total = (size_t)mine * dim;
        size_t head = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
        if (head > total) head = total;
        const size_t packs = (total - head) / N, tail = head + packs * N;
        Pack<T, N> z;
#pragma unroll
        for (int j = 0; j < N; ++j) z.v[j] = (T)0.0f;
        for (size_t i = lane; i < packs; i += 64) put<STREAM, T, N>(p + head + i * N, z);
        if ((size_t)lane < head) p[lane] = (T)0.0f;
        if (tail + lane < total) p[tail + lane] = (T)0.0f;
        return;
    }
    Pack<T, V> z;
#pragma unroll
    for (int j = 0; j < V; ++j) z.v[j] = (T)0.0f;
    if (dim < 64 * V) {                                    // short rows: a lane walks over the packs of all of them
        const uint32_t ppr = (uint32_t)(dim / V), dq = 64 / ppr, dr = 64 - dq * ppr;
        uint32_t r = (uint32_t)lane / ppr, c = (uint32_t)lane - r * ppr;
        T* p = d_table + first * dim;
        for (size_t i = lane; r < mine; i += 64) {
            if (todo >> r & 1ull) put<STREAM, T, V>(p + i * V, z);
            r += dq;
            c += dr;
            if (c >= ppr) {
                c -= ppr;
                ++r;
            }
        }
        return;
    }
    while (todo) {
        const int r = __builtin_ctzll(todo);
        todo &= todo - 1;
        T* row = d_table + (first + r) * dim;
        for (size_t col = (size_t)lane * V; col < dim; col += 64 * V) put<STREAM, T, V>(row + col, z);
    }
}

// Up to EMBED_TINY positions go in one launch and without a sort.  A workgroup stands for a position (times a slice of the
// columns): it lists the positions with the same index, in order, and sums their rows when its own is the first of them.  The
// groups of a workgroup share the list, their sums are added in order.  Further workgroups clear the rows that no position
// names.  (191 positions, 1580 rows of 802 fp32: 5 us; with a sort in every workgroup 18.)
constexpr uint32_t EMBED_TINY = 256;
template <typename T, int V, int G>
__global__ __launch_bounds__(256) void embed_tiny_kernel(uint32_t n, uint32_t rows, const void* __restrict__ index, int index_bytes,
                                                         uint32_t nslices, size_t dim, const T* __restrict__ d_out, size_t stride,
                                                         float scale, T* __restrict__ d_table, uint32_t sum_blocks, uint32_t zero_rows) {
    constexpr int PER = EMBED_TINY / 256, GROUPS = 256 / G, UNROLL = 8;
    __shared__ uint32_t list[EMBED_TINY], found[4 * PER];
    __shared__ float sums[256 * V];
    uint32_t key[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const uint32_t i = u * 256 + threadIdx.x;
        const unsigned long long id = (unsigned long long)load_index_flat(index, i < n ? i : n - 1, index_bytes);
        key[u] = i < n && id < rows ? (uint32_t)id : EMBED_NONE;
    }
    if (blockIdx.x >= sum_blocks) {
        const uint32_t row0 = (blockIdx.x - sum_blocks) * 4 * zero_rows;       // (4 * zero_rows <= 256 rows)
        list[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < PER; ++u)
            if (key[u] - row0 < 4 * zero_rows) list[key[u] - row0] = 1;        // (several threads: the same value)
        __syncthreads();
        const uint32_t lane = threadIdx.x & 63, mine = (threadIdx.x >> 6) * zero_rows;
        const bool empty = lane < zero_rows && (size_t)row0 + mine + lane < rows && list[mine + lane] == 0;
        const size_t first = (size_t)row0 + mine;
        if ((size_t)rows * dim * sizeof(T) > E3_STREAM_BYTES) embed_zero<true, T, V>(empty, first, rows, zero_rows, dim, d_table);
        else embed_zero<false, T, V>(empty, first, rows, zero_rows, dim, d_table);
        return;
    }
    const uint32_t own = blockIdx.x / nslices, slice = blockIdx.x - own * nslices;
    const unsigned long long id = (unsigned long long)load_index_flat(index, own, index_bytes);
    if (id >= rows) return;                                                    // (uniform)
    unsigned long long hit[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        hit[u] = __ballot(key[u] == (uint32_t)id);
        if ((threadIdx.x & 63) == 0) found[u * 4 + (threadIdx.x >> 6)] = (uint32_t)__popcll(hit[u]);
    }
    __syncthreads();
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w == (int)(threadIdx.x >> 6) && key[u] == (uint32_t)id)
                list[m + (uint32_t)__popcll(hit[u] & ((1ull << (threadIdx.x & 63)) - 1ull))] = u * 256 + threadIdx.x;
            m += found[u * 4 + w];
        }
    __syncthreads();
    if (list[0] != own) return;                                                // (uniform)
    const int g = threadIdx.x / G, lane = threadIdx.x % G;
    const size_t col = ((size_t)slice * G + lane) * V;
    const uint32_t lo = m * g / GROUPS, hi = m * (g + 1) / GROUPS;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    for (uint32_t b = lo; b < hi && col < dim; b += UNROLL) {
        Held<T, V> r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u].load(d_out + (size_t)list[b + u < hi ? b + u : hi - 1] * stride + col);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (b + u >= hi) break;
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += r[u].value(j);
        }
    }
    if (m > 1) {                                                               // (uniform)
#pragma unroll
        for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = acc[j];
        __syncthreads();
    }
    // (a list of one: the last group has it)
    if (m == 1 ? g != GROUPS - 1 : g != 0) return;
    if (col >= dim) return;
    if (m > 1)
        for (int k = 1; k < GROUPS; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += sums[(k * G + lane) * V + j];
    embed_store<T, V>(d_table, dim, (uint32_t)id, col, scale, acc);
}

// A group of G lanes sums one chunk of the sorted list, times a slice of G V columns, EMBED_UNROLL gathered rows in flight.
// Bound by the gather: 1M rows of 48 fp32 values into 4096 table rows 48 us (4.0 TB/s of gradient read), 8192 rows of 4096
// bf16 values into a cleared table of 32000 rows 33 us.
constexpr int EMBED_UNROLL = 8;
template <typename T, int V, int G>
__global__ __launch_bounds__(256) void embed_sum_kernel(const uint32_t* __restrict__ kept, const uint32_t* __restrict__ keys,
                                                        const uint32_t* __restrict__ pos, uint32_t chunk, uint32_t nchunks,
                                                        uint32_t nslices, size_t dim, const T* __restrict__ d_out,
                                                        size_t stride, float scale, T* __restrict__ d_table,
                                                        float* __restrict__ part, uint32_t sum_blocks, uint32_t rows,
                                                        uint32_t zero_rows) {
    const uint32_t n = *kept;
    if (blockIdx.x >= sum_blocks) {      // (in the same launch: the sums wait for their gathers, the stores do not)
        const size_t first = ((size_t)(blockIdx.x - sum_blocks) * 4 + (threadIdx.x >> 6)) * zero_rows;
        bool empty = false;                                 // (a lane looks one row up in the sorted keys)
        if ((threadIdx.x & 63) < zero_rows && first + (threadIdx.x & 63) < rows) {
            const uint32_t row = (uint32_t)first + (threadIdx.x & 63), at = lower_bound_u32(keys, 0, n, row);
            empty = at >= n || keys[at] != row;
        }
        if ((size_t)rows * dim * sizeof(T) > E3_STREAM_BYTES) embed_zero<true, T, V>(empty, first, rows, zero_rows, dim, d_table);
        else embed_zero<false, T, V>(empty, first, rows, zero_rows, dim, d_table);
        return;
    }
    const size_t unit = (size_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const uint32_t c = (uint32_t)(unit / nslices), slice = (uint32_t)(unit - (size_t)c * nslices);
    const size_t col = ((size_t)slice * G + threadIdx.x % G) * V;
    if (c >= nchunks || (size_t)c * chunk >= n || col >= dim) return;
    const uint32_t j0 = c * chunk, j1 = n - j0 < chunk ? n : j0 + chunk;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    uint32_t cur = keys[j0];
    bool from_before = j0 > 0 && keys[j0 - 1] == cur;       // the run in hand began in an earlier chunk
    for (uint32_t b = j0; b < j1; b += EMBED_UNROLL) {
        uint32_t k[EMBED_UNROLL];
        Held<T, V> r[EMBED_UNROLL];
#pragma unroll
        for (int u = 0; u < EMBED_UNROLL; ++u) {            // (entries behind the chunk read its last one and are not added)
            const uint32_t at = b + u < j1 ? b + u : j1 - 1;
            k[u] = keys[at];
            r[u].load(d_out + (size_t)pos[at] * stride + col);
        }
#pragma unroll
        for (int u = 0; u < EMBED_UNROLL; ++u) {
            if (b + u >= j1) break;
            if (k[u] != cur) {
                if (from_before) {
#pragma unroll
                    for (int j = 0; j < V; ++j) part[(size_t)(2 * c) * dim + col + j] = acc[j];
                } else {
                    embed_store<T, V>(d_table, dim, cur, col, scale, acc);
                }
                from_before = false;
                cur = k[u];
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += r[u].value(j);
        }
    }
    const bool goes_on = j1 < n && keys[j1] == cur;
    if (from_before || goes_on) {
        const size_t slot = from_before ? 2 * (size_t)c : 2 * (size_t)c + 1;
#pragma unroll
        for (int j = 0; j < V; ++j) part[slot * dim + col + j] = acc[j];
    } else {
        embed_store<T, V>(d_table, dim, cur, col, scale, acc);
    }
}

// Adds up the partials of the runs that cross chunks: slot 1 of the chunk a run starts in, slot 0 of the following ones.
// Workgroups of two kinds in one launch:
//   short runs   a group of 16 lanes takes a chunk (times a slice of 16 V columns) and adds up to JOIN_SHORT partials in order
//   long runs    a workgroup looks at JOIN_SHORT neighbouring chunks (times a slice of the columns, 16 at a time): only the
//                last run that starts among them can be longer than JOIN_SHORT partials; 64 groups of 16 lanes take a 64th
//                of them each, the 64 sums are added eight by eight
constexpr uint32_t JOIN_SHORT = 32;
// Whether a run starts in chunk c and goes on behind it; its key.
__device__ __forceinline__ bool embed_crossing(const uint32_t* __restrict__ keys, uint32_t n, uint32_t chunk, uint32_t c,
                                               uint32_t& key) {
    if ((size_t)(c + 1) * chunk >= n) return false;                      // nothing lies behind the chunk
    const uint32_t j0 = c * chunk, j1 = j0 + chunk, head = keys[j0], next = keys[j1], before = keys[j0 > 0 ? j0 - 1 : 0];
    key = keys[j1 - 1];
    return next == key && !(head == key && j0 > 0 && before == key);     // (it goes on, and did not begin earlier)
}
// Whether chunk c exists and begins with `key`: then it holds a partial of the run.
__device__ __forceinline__ bool embed_in_run(const uint32_t* __restrict__ keys, uint32_t n, uint32_t chunk, uint32_t c, uint32_t key) {
    return (size_t)c * chunk < n && keys[(size_t)c * chunk] == key;
}
template <typename T, int V>
__global__ __launch_bounds__(1024) void embed_join_kernel(const uint32_t* __restrict__ kept,
                                                          const uint32_t* __restrict__ keys, uint32_t chunk,
                                                          uint32_t nchunks, uint32_t short_blocks, uint32_t cols, size_t dim,
                                                          const float* __restrict__ part, float scale,
                                                          T* __restrict__ d_table) {
    __shared__ float sums[64][17];
    __shared__ uint32_t long_chunk, long_key;
    const uint32_t n = *kept;
    const int g = threadIdx.x >> 4, lane = threadIdx.x & 15;
    if (blockIdx.x < short_blocks) {
        const uint32_t nslices = (uint32_t)((dim + 16 * V - 1) / (16 * V));
        const size_t unit = (size_t)blockIdx.x * 64 + g;
        const uint32_t c = (uint32_t)(unit / nslices);
        const size_t col = ((unit - (size_t)c * nslices) * 16 + lane) * V;
        uint32_t key = 0;
        if (c >= nchunks || !embed_crossing(keys, n, chunk, c, key)) return;        // (the same for the whole group)
        // partials behind the first: chunks c + 1, c + 2, ... that begin with the key, 16 looked at together
        uint32_t m = 1;
        for (uint32_t k = 1; k <= JOIN_SHORT; k += 16) {
            const unsigned long long in = __ballot(embed_in_run(keys, n, chunk, c + k + lane, key));
            const uint32_t mine = (uint32_t)(in >> (threadIdx.x & 48)) & 0xFFFFu;
            m += (uint32_t)__popc(mine);
            if (mine != 0xFFFFu) break;
        }
        if (m > JOIN_SHORT || col >= dim) return;
        const Pack<float, V> p = *reinterpret_cast<const Pack<float, V>*>(part + (2 * (size_t)c + 1) * dim + col);
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = p.v[j];
#pragma unroll 4
        for (uint32_t k = 1; k < m; ++k) {
            const Pack<float, V> q = *reinterpret_cast<const Pack<float, V>*>(part + 2 * (size_t)(c + k) * dim + col);
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += q.v[j];
        }
        embed_store<T, V>(d_table, dim, key, col, scale, acc);
        return;
    }
    const uint32_t nparts = (uint32_t)((dim + cols - 1) / cols), unit = blockIdx.x - short_blocks;
    const uint32_t first = unit / nparts * JOIN_SHORT;
    if (threadIdx.x < 64) {
        const uint32_t c = first + threadIdx.x;
        uint32_t key = 0;
        const bool is_long = threadIdx.x < JOIN_SHORT && c < nchunks && embed_crossing(keys, n, chunk, c, key) &&
                             embed_in_run(keys, n, chunk, c + JOIN_SHORT, key);
        const unsigned long long hit = __ballot(is_long);                      // (one lane at most)
        if (threadIdx.x == 0 && hit == 0ull) long_chunk = 0xFFFFFFFFu;
        if (is_long) {
            long_chunk = c;
            long_key = key;
        }
    }
    __syncthreads();
    const uint32_t c = long_chunk;
    if (c == 0xFFFFFFFFu) return;                                              // (uniform)
    // partials: chunks from c on that belong to the run, the last one found by 64 probes at a time
    uint32_t in = c + JOIN_SHORT, out = nchunks;                               // `in` begins with the key, `out` does not
    while (out - in > 1) {
        const uint32_t step = (out - in - 1) / 64 + 1, at = in + 1 + (threadIdx.x & 63) * step;
        const unsigned long long hit = __ballot(at < out && embed_in_run(keys, n, chunk, at, long_key));
        const uint32_t k = (uint32_t)__popcll(hit);                            // (the run is contiguous: the first k probes)
        const uint32_t low = k ? in + 1 + (k - 1) * step : in, high = in + 1 + k * step;
        out = high < out && k < 64 ? high : out;
        in = low;
    }
    const uint32_t m = in - c + 1u;
    const uint32_t lo = (uint32_t)((unsigned long long)m * g / 64), hi = (uint32_t)((unsigned long long)m * (g + 1) / 64);
    const size_t col0 = (size_t)(unit % nparts) * cols, col1 = col0 + cols < dim ? col0 + cols : dim;
    for (size_t col = col0 + lane; col < col1 + lane; col += 16) {             // (every lane takes part in the barriers)
        float s = 0.0f;
        if (col < col1) {
#pragma unroll 8
            for (uint32_t k = lo; k < hi; ++k) s += part[(k == 0 ? 2 * (size_t)c + 1 : 2 * (size_t)(c + k)) * dim + col];
        }
        sums[g][lane] = s;
        __syncthreads();
        if (g < 8) {
            s = sums[8 * g][lane];
#pragma unroll
            for (int w = 1; w < 8; ++w) s += sums[8 * g + w][lane];
        }
        __syncthreads();
        if (g < 8) sums[g][lane] = s;
        __syncthreads();
        if (g == 0 && col < col1) {
#pragma unroll
            for (int w = 1; w < 8; ++w) s += sums[w][lane];
            d_table[(size_t)long_key * dim + col] = (T)(scale * s);
        }
        __syncthreads();
    }
}

// The lanes of a wave that hold the same digit of `bits` bits (up to 8).
__device__ __forceinline__ unsigned long long digit_peers(uint32_t d, int bits) {
    uint32_t lo = ~0u, hi = ~0u;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        if (b >= bits) break;
        const int bit = (int)(d << (31 - b)) >> 31;          // 0 or -1
        const unsigned long long bal = __ballot(bit < 0);
        lo &= ~((uint32_t)bal ^ (uint32_t)bit);
        hi &= ~((uint32_t)(bal >> 32) ^ (uint32_t)bit);
    }
    return (unsigned long long)hi << 32 | lo;
}

// Sorts up to 1024 * ITEMS positions by index in one workgroup (stable, 8 bits a pass): for few positions the launches of the
// general sort would cost more than everything else.  A wave owns 64 * ITEMS consecutive keys and ranks 64 at a time with
// ballots; the digits' counters of the 16 waves are joined by a prefix over waves and digits.  Indices outside the table get
// the key `rows`, so that they end up behind the others.
template <int ITEMS>
struct SmallSort {
    static constexpr int N = 1024 * ITEMS;
    uint32_t key[N];
    uint16_t pos[N], rank[N];
    uint32_t cnt[16][256];
    uint32_t wtot[4], valid;
};
// The other workgroups of the launch clear the table's gradient meanwhile, all of it (the sums then write the rows that have
// positions): gradient of 1328 positions, 23345 rows of 1571 fp32 36 us, 50 where the sums' launch clears the rows without one;
// lookup and gradient of 8192 positions, 32000 rows of 4096 bf16 106 and 113 us.
template <int ITEMS, typename I>
__global__ __launch_bounds__(1024) void embed_sort_small_kernel(uint32_t n, uint32_t rows, int passes, int bits,
                                                                const I* __restrict__ index, uint32_t* __restrict__ keys,
                                                                uint32_t* __restrict__ pos, uint32_t* __restrict__ kept,
                                                                uint16_t* __restrict__ table, size_t halves) {
    __shared__ SmallSort<ITEMS> L;
    if (blockIdx.x > 0) {
        size_t head = ((16 - (reinterpret_cast<uintptr_t>(table) & 15)) & 15) / 2;
        if (head > halves) head = halves;
        const size_t packs = (halves - head) / 8, tail = head + packs * 8, first = (size_t)(blockIdx.x - 1) * 4096 + threadIdx.x;
        Pack<f16_t, 8> z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z.v[j] = (f16_t)0.0f;
        f16_t* body = reinterpret_cast<f16_t*>(table + head);
        for (size_t i = first; i < packs; i += (size_t)(gridDim.x - 1) * 4096) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * 1024 < packs) put<false, f16_t, 8>(body + (i + u * 1024) * 8, z);
        }
        if (blockIdx.x == 1) {
            if (threadIdx.x < head) table[threadIdx.x] = 0;
            if (tail + threadIdx.x < halves) table[tail + threadIdx.x] = 0;
        }
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t base = (uint32_t)wave * (64 * ITEMS) + lane;
    const unsigned long long before = (1ull << lane) - 1ull;
    if (threadIdx.x == 0) L.valid = 0;
    __syncthreads();
    I id[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t at = base + i * 64;
        id[i] = index[at < n ? at : n - 1];
    }
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t at = base + i * 64;
        const bool ok = at < n && id[i] >= 0 && (long long)id[i] < (long long)rows;
        L.key[at] = ok ? (uint32_t)id[i] : rows;
        L.pos[at] = (uint16_t)at;
        mine += (uint32_t)__popcll(__ballot(ok));
    }
    if (lane == 0) atomicAdd(&L.valid, mine);
    const uint32_t mask = (1u << bits) - 1u;
    for (int pass = 0, shift = 0; pass < passes; ++pass, shift += bits) {
        for (int d = threadIdx.x; d < 16 * 256; d += 1024) L.cnt[d >> 8][d & 255] = 0;
        __syncthreads();
#pragma unroll 1
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t d = L.key[base + i * 64] >> shift & mask;
            const unsigned long long peers = digit_peers(d, bits);
            const uint32_t first = L.cnt[wave][d];
            wave_sync();
            if ((peers & before) == 0ull) L.cnt[wave][d] = first + (uint32_t)__popcll(peers);
            wave_sync();
            L.rank[base + i * 64] = (uint16_t)(first + (uint32_t)__popcll(peers & before));
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            uint32_t c[16], total = 0;
#pragma unroll
            for (int w = 0; w < 16; ++w) { c[w] = L.cnt[w][threadIdx.x]; total += c[w]; }
            uint32_t inc = total;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const uint32_t t = __shfl_up(inc, o, 64); if (lane >= o) inc += t; }
            if (lane == 63) L.wtot[wave] = inc;
            uint32_t run = inc - total;
#pragma unroll
            for (int w = 0; w < 16; ++w) { L.cnt[w][threadIdx.x] = run; run += c[w]; }
        }
        __syncthreads();
        uint32_t k[ITEMS], to[ITEMS];
        uint16_t p[ITEMS];
        const uint32_t t1 = L.wtot[0], t2 = t1 + L.wtot[1], t3 = t2 + L.wtot[2];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            k[i] = L.key[base + i * 64];
            p[i] = L.pos[base + i * 64];
            const uint32_t d = k[i] >> shift & mask, q = d >> 6;
            to[i] = L.cnt[wave][d] + L.rank[base + i * 64] + (q == 0 ? 0u : q == 1 ? t1 : q == 2 ? t2 : t3);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            L.key[to[i]] = k[i];
            L.pos[to[i]] = p[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t at = base + i * 64;
        if (at < n) {
            keys[at] = L.key[at];
            pos[at] = L.pos[at];
        }
    }
    if (threadIdx.x == 0) *kept = L.valid;
}

// More positions: passes of up to 8 bits over tiles of 1024 * ITEMS keys, two launches each.  The first counts the digits of
// every tile (and makes the keys); in the second every tile adds up the counts before its own (at most SORT_TILES of them, a
// kilobyte each: cheaper than a launch that scans them), ranks its keys, puts them in order in LDS and writes them out
// digit by digit.  1M positions of 12 bits: 37 us (the general sort with its seven launches 43), 60905 of 16 bits: 21 us (36),
// 372939 of 17 bits: 40 us (65).  Keys to a thread: 1 up to 128 tiles, then 2 up to 128 tiles, then 4, then 8; 560085
// positions took 12 us a scatter with 137 tiles of four, 14 with 69 tiles of eight, 372939 took 9 with 92 tiles and 10 with 183.
constexpr uint32_t SORT_TILES = 256;
__device__ __forceinline__ uint32_t sort_digit(uint32_t key, int shift, uint32_t mask) { return key >> shift & mask; }
template <int ITEMS, bool FIRST, typename I>
__global__ __launch_bounds__(1024) void embed_count_kernel(uint32_t n, uint32_t rows, int shift, uint32_t mask,
                                                           const I* __restrict__ index, uint32_t* __restrict__ keys,
                                                           uint32_t* __restrict__ counts, uint32_t* __restrict__ valid) {
    __shared__ uint32_t cnt[4][256], ok_count;
    for (int d = threadIdx.x; d < 4 * 256; d += 1024) cnt[d >> 8][d & 255] = 0;
    if (threadIdx.x == 0) ok_count = 0;
    __syncthreads();
    const uint32_t tile0 = blockIdx.x * (1024 * ITEMS);
    uint32_t k[ITEMS], ok = 0;
    if (FIRST) {
        I id[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t at = tile0 + i * 1024 + threadIdx.x;
            id[i] = index[at < n ? at : n - 1];
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t at = tile0 + i * 1024 + threadIdx.x;
            const bool in = id[i] >= 0 && (long long)id[i] < (long long)rows;
            k[i] = in ? (uint32_t)id[i] : rows;
            if (at < n) {
                keys[at] = k[i];
                ok += in ? 1u : 0u;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t at = tile0 + i * 1024 + threadIdx.x;
            k[i] = keys[at < n ? at : n - 1];
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (tile0 + i * 1024 + threadIdx.x < n) atomicAdd(&cnt[threadIdx.x >> 6 & 3][sort_digit(k[i], shift, mask)], 1u);
    if (FIRST) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) ok += __shfl_xor(ok, o, 64);
        if ((threadIdx.x & 63) == 0) atomicAdd(&ok_count, ok);
    }
    __syncthreads();
    if (threadIdx.x < 256) counts[blockIdx.x * 256 + threadIdx.x] =
        (cnt[0][threadIdx.x] + cnt[1][threadIdx.x]) + (cnt[2][threadIdx.x] + cnt[3][threadIdx.x]);
    if (FIRST && threadIdx.x == 0) valid[blockIdx.x] = ok_count;
}
// Exclusive prefix sum over 256 values, one per thread of the first four waves; every thread of the workgroup takes part.
__device__ __forceinline__ uint32_t prefix_256(uint32_t v, uint32_t* wave_totals) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const uint32_t t = __shfl_up(inc, o, 64); if (lane >= o) inc += t; }
    if (lane == 63 && wave < 4) wave_totals[wave] = inc;
    __syncthreads();
    uint32_t run = inc - v;
    for (int w = 0; w < wave && w < 4; ++w) run += wave_totals[w];
    return run;
}
template <int ITEMS>
struct SortTile {
    uint32_t key[1024 * ITEMS], pos[1024 * ITEMS];
    uint32_t cnt[16][256], all[256], before[256], to[256], wl[4], wg[4];
};
template <int ITEMS, bool FIRST>
__global__ __launch_bounds__(1024) void embed_scatter_kernel(uint32_t n, int shift, int bits, uint32_t tiles,
                                                             const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                             const uint32_t* __restrict__ counts, const uint32_t* __restrict__ valid,
                                                             uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out,
                                                             uint32_t* __restrict__ kept) {
    __shared__ SortTile<ITEMS> L;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t mask = (1u << bits) - 1u, tile0 = blockIdx.x * (1024 * ITEMS), base = tile0 + (uint32_t)wave * (64 * ITEMS) + lane;
    const unsigned long long before = (1ull << lane) - 1ull;
    uint32_t k[ITEMS], p[ITEMS], rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {                       // (behind the list: the largest digit, last of all)
        const uint32_t at = base + i * 64;
        k[i] = keys[at < n ? at : n - 1];
        p[i] = FIRST ? at : pos[at < n ? at : n - 1];
        if (at >= n) k[i] = 0xFFFFFFFFu;
    }
    for (int d = threadIdx.x; d < 16 * 256; d += 1024) L.cnt[d >> 8][d & 255] = 0;
    if (threadIdx.x < 256) L.all[threadIdx.x] = L.before[threadIdx.x] = 0;
    __syncthreads();
    if (4u * lane <= mask) {   // counts of the digits in all tiles, and in those before this one: four digits to a lane
        uint32_t all[4] = {0, 0, 0, 0}, less[4] = {0, 0, 0, 0};
        for (uint32_t t0 = wave; t0 < tiles; t0 += 16 * 8) {
            uint4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {                   // (a batch of loads in flight; behind the last tile the first again)
                const uint32_t t = t0 + 16 * u;
                v[u] = reinterpret_cast<const uint4*>(counts + (t < tiles ? t : t0) * 256)[lane];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t t = t0 + 16 * u;
                if (t >= tiles) break;
                const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    all[j] += x[j];
                    less[j] += t < blockIdx.x ? x[j] : 0u;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            atomicAdd(&L.all[4 * lane + j], all[j]);
            atomicAdd(&L.before[4 * lane + j], less[j]);
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t d = sort_digit(k[i], shift, mask);
        const unsigned long long peers = digit_peers(d, bits);
        const uint32_t first = L.cnt[wave][d];
        wave_sync();
        if ((peers & before) == 0ull) L.cnt[wave][d] = first + (uint32_t)__popcll(peers);
        wave_sync();
        rank[i] = first + (uint32_t)__popcll(peers & before);
    }
    __syncthreads();
    uint32_t c[16], local = 0, all = 0, less = 0;
    if (threadIdx.x < 256) {
#pragma unroll
        for (int w = 0; w < 16; ++w) { c[w] = L.cnt[w][threadIdx.x]; local += c[w]; }
        all = L.all[threadIdx.x];
        less = L.before[threadIdx.x];
    }
    uint32_t run = prefix_256(local, L.wl);
    const uint32_t start = prefix_256(all, L.wg) + less;
    if (threadIdx.x < 256) {
        L.to[threadIdx.x] = start - run;
#pragma unroll
        for (int w = 0; w < 16; ++w) { L.cnt[w][threadIdx.x] = run; run += c[w]; }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t at = L.cnt[wave][sort_digit(k[i], shift, mask)] + rank[i];
        L.key[at] = k[i];
        L.pos[at] = p[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t at = i * 1024 + threadIdx.x;
        if (tile0 + at >= n) continue;
        const uint32_t key = L.key[at], to = L.to[sort_digit(key, shift, mask)] + at;
        keys_out[to] = key;
        pos_out[to] = L.pos[at];
    }
    if (FIRST && blockIdx.x == 0 && wave == 15) {
        uint32_t m = 0;
        for (uint32_t t = lane; t < tiles; t += 64) m += valid[t];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) m += __shfl_xor(m, o, 64);
        if (lane == 0) *kept = m;
    }
}

constexpr size_t EMBED_SMALL = 16384;            // positions that one workgroup sorts
namespace {
struct EmbedScratch {
    uint32_t *key0, *key1, *pos0, *pos1, *kept, *sort;
    float* part;
    static uint32_t chunk(size_t n, size_t dim) {
        // Rows of a chunk: 128 where there is plenty of work, fewer where the groups would otherwise not fill the chip (each
        // group moves `chunk` row slices of at most 1 KB).
        uint32_t c = 128;
        while (c > 8 && (n / c) * ((dim + 511) / 512) < 4096) c >>= 1;
        return c;
    }
    static uint32_t chunks(size_t n, size_t dim) { return (uint32_t)((n + chunk(n, dim) - 1) / chunk(n, dim)); }
    static EmbedScratch from(char*& p, size_t n, size_t dim) {
        EmbedScratch s;
        const size_t m = n ? n : 1;
        s.key0 = carve<uint32_t>(p, m);
        s.key1 = carve<uint32_t>(p, m);
        s.pos0 = carve<uint32_t>(p, m);
        s.pos1 = carve<uint32_t>(p, m);
        s.kept = carve<uint32_t>(p, 1);
        const size_t general = sort_scratch_words(m), tiles = SORT_TILES * 257;
        s.sort = carve<uint32_t>(p, general > tiles ? general : tiles);
        s.part = carve<float>(p, m <= EMBED_TINY ? 1 : 2 * (size_t)chunks(m, dim) * dim);      // (few positions: no partials)
        return s;
    }
};

template <typename T, int V, int G>
int embed_sum_launch(const EmbedScratch& w, const uint32_t* keys, const uint32_t* pos, size_t n, size_t rows, size_t dim,
                     const void* d_out, size_t stride, float scale, void* d_table, const void* index, int index_bytes,
                     hipStream_t s) {
    const size_t nslices = (dim + (size_t)G * V - 1) / ((size_t)G * V);
    size_t per = 16384 / (dim * sizeof(T));                    // about 16 KB of table rows to a wave that clears them
    per = per < 1 ? 1 : (per > 64 ? 64 : per);
    const size_t zero_blocks = (rows + 4 * per - 1) / (4 * per);
    if (n <= EMBED_TINY) {
        const size_t blocks = n * nslices;
        if (!grid_fits(blocks + zero_blocks, 256)) return e3_fail(hipErrorInvalidValue, "e3dgs_embedding_backward: too many values");
        embed_tiny_kernel<T, V, G><<<dim3((unsigned)(blocks + zero_blocks)), dim3(256), 0, s>>>(
            (uint32_t)n, (uint32_t)rows, index, index_bytes, (uint32_t)nslices, dim, (const T*)d_out, stride, scale, (T*)d_table,
            (uint32_t)blocks, (uint32_t)per);
        LAUNCH_OK("embed_tiny_kernel");
        return 0;
    }
    const uint32_t chunk = EmbedScratch::chunk(n, dim), nchunks = EmbedScratch::chunks(n, dim);
    const size_t units = nslices * nchunks, blocks = (units + 256 / G - 1) / (256 / G);
    const size_t clears = n <= EMBED_SMALL ? 0 : zero_blocks;  // (the launch of the small sort has cleared the table)
    if (!grid_fits(blocks + clears, 256)) return e3_fail(hipErrorInvalidValue, "e3dgs_embedding_backward: too many values");
    embed_sum_kernel<T, V, G><<<dim3((unsigned)(blocks + clears)), dim3(256), 0, s>>>(
        w.kept, keys, pos, chunk, nchunks, (uint32_t)nslices, dim, (const T*)d_out, stride, scale, (T*)d_table, w.part,
        (uint32_t)blocks, (uint32_t)rows, (uint32_t)per);
    LAUNCH_OK("embed_sum_kernel");
    return 0;
}
template <typename T, int V>
int embed_join_launch(const EmbedScratch& w, const uint32_t* keys, size_t n, size_t dim, float scale, void* d_table,
                      hipStream_t s) {
    const uint32_t chunk = EmbedScratch::chunk(n, dim), nchunks = EmbedScratch::chunks(n, dim);
    if (nchunks <= 1) return 0;
    const size_t shorts = ((size_t)nchunks * ((dim + 16 * V - 1) / (16 * V)) + 63) / 64;
    // (columns of a workgroup of the second kind: 16 as long as that is not far more workgroups than the chip holds, most of
    // which find no long run: 5539 positions, 12 rows of 289 bf16 5.6 us, with 64 columns 14.4)
    const size_t groups = nchunks > JOIN_SHORT ? (nchunks + JOIN_SHORT - 1) / JOIN_SHORT : 0;
    const size_t cols = groups * ((dim + 15) / 16) <= 2048 ? 16 : 64, longs = groups * ((dim + cols - 1) / cols);
    if (!grid_fits(shorts + longs, 1024)) return e3_fail(hipErrorInvalidValue, "e3dgs_embedding_backward: too many values");
    embed_join_kernel<T, V><<<dim3((unsigned)(shorts + longs)), dim3(1024), 0, s>>>(w.kept, keys, chunk, nchunks, (uint32_t)shorts,
                                                                                  (uint32_t)cols, dim, w.part, scale, (T*)d_table);
    LAUNCH_OK("embed_join_kernel");
    return 0;
}

// Passes and bits of a digit (up to 8, the same in every pass) for the keys 0 .. rows: the key `rows` itself occurs.
void embed_digits(uint32_t rows, int& passes, int& bits) {
    int nbits = 1;
    while (rows >> nbits) ++nbits;
    passes = (nbits + 7) / 8;
    bits = (nbits + passes - 1) / passes;
}
template <typename I>
void embed_sort_small(uint32_t n, uint32_t rows, const I* index, uint32_t* keys, uint32_t* pos, uint32_t* kept, void* table,
                      size_t bytes, hipStream_t s) {
    int passes, bits;
    embed_digits(rows, passes, bits);
    const size_t need = (bytes + 65535) / 65536;               // 64 KB to a workgroup, at most one to each of the other CUs
    const dim3 blocks(1 + (unsigned)(need < 255 ? need : 255)), threads(1024);
#define E3_SMALL(ITEMS) \
    embed_sort_small_kernel<ITEMS, I><<<blocks, threads, 0, s>>>(n, rows, passes, bits, index, keys, pos, kept, (uint16_t*)table, bytes / 2)
    if (n <= 1024) E3_SMALL(1);
    else if (n <= 4096) E3_SMALL(4);
    else if (n <= 8192) E3_SMALL(8);
    else E3_SMALL(16);
#undef E3_SMALL
}
// The tiles' sort; keys / pos: where the result lies.
template <int ITEMS>
int embed_sort_tiles(const EmbedScratch& w, uint32_t n, uint32_t rows, const void* index, int index_bytes, uint32_t** keys,
                     uint32_t** pos, hipStream_t s) {
    int passes, bits;
    embed_digits(rows, passes, bits);
    const uint32_t tiles = (n + 1024 * ITEMS - 1) / (1024 * ITEMS), mask = (1u << bits) - 1u;
    uint32_t *counts = w.sort, *valid = w.sort + SORT_TILES * 256;
    uint32_t *k0 = w.key0, *k1 = w.key1, *p0 = w.pos0, *p1 = w.pos1;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
        if (pass > 0) embed_count_kernel<ITEMS, false, int><<<dim3(tiles), dim3(1024), 0, s>>>(n, rows, shift, mask, nullptr, k0, counts, valid);
        else if (index_bytes == 8) embed_count_kernel<ITEMS, true, long long><<<dim3(tiles), dim3(1024), 0, s>>>(n, rows, shift, mask, (const long long*)index, k0, counts, valid);
        else embed_count_kernel<ITEMS, true, int><<<dim3(tiles), dim3(1024), 0, s>>>(n, rows, shift, mask, (const int*)index, k0, counts, valid);
        LAUNCH_OK("embed_count_kernel");
        if (pass > 0) embed_scatter_kernel<ITEMS, false><<<dim3(tiles), dim3(1024), 0, s>>>(n, shift, bits, tiles, k0, p0, counts, valid, k1, p1, w.kept);
        else embed_scatter_kernel<ITEMS, true><<<dim3(tiles), dim3(1024), 0, s>>>(n, shift, bits, tiles, k0, nullptr, counts, valid, k1, p1, w.kept);
        LAUNCH_OK("embed_scatter_kernel");
        uint32_t* t = k0; k0 = k1; k1 = t;
        t = p0; p0 = p1; p1 = t;
    }
    *keys = k0;
    *pos = p0;
    return 0;
}

template <typename T>
int embed_bwd_t(size_t n, size_t rows, size_t dim, const void* index, int index_bytes, const void* d_out, size_t stride,
                int dtype, float scale, void* d_table, char* scratch, hipStream_t s) {
    EmbedScratch w = EmbedScratch::from(scratch, n, dim);
    uint32_t *keys = w.key0, *pos = w.pos0;
    int rc = 0;
    if (n > EMBED_TINY && n <= EMBED_SMALL) {
        const size_t bytes = rows * dim * sizeof(T);
        if (index_bytes == 8) embed_sort_small((uint32_t)n, (uint32_t)rows, (const long long*)index, keys, pos, w.kept, d_table, bytes, s);
        else embed_sort_small((uint32_t)n, (uint32_t)rows, (const int*)index, keys, pos, w.kept, d_table, bytes, s);
        LAUNCH_OK("embed_sort_small_kernel");
    } else if (n > EMBED_TINY && n <= SORT_TILES * 8192) {
#define E3_TILES(ITEMS) embed_sort_tiles<ITEMS>(w, (uint32_t)n, (uint32_t)rows, index, index_bytes, &keys, &pos, s)
        rc = n <= 128 * 1024 ? E3_TILES(1) : n <= 128 * 2048 ? E3_TILES(2) : n <= 256 * 4096 ? E3_TILES(4) : E3_TILES(8);
#undef E3_TILES
        if (rc) return rc;
    } else if (n > EMBED_TINY) {
        embed_keys_kernel<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s>>>(n, rows, index, index_bytes, w.key0);
        LAUNCH_OK("embed_keys_kernel");
        int nbits = 1;
        while (nbits < 32 && (rows - 1) >> nbits) ++nbits;
        rc = launch_radix_sort_pairs(w.key0, w.key1, w.pos0, w.pos1, n, nbits, w.sort, &keys, &pos, s, true, w.kept, nullptr,
                                     nullptr, 0, nullptr, nullptr);
        if (rc) return rc;
    }
    auto fits = [&](size_t bytes) { return e3_rows_packs(d_out, stride, dim, dtype, bytes) && e3_rows_packs(d_table, dim, dim, dtype, bytes); };
    constexpr int N = Wide<T>::N, HALF = N / 2, QUARTER = N == 8 ? 2 : 1;
#define E3_SUM(V, G) rc = embed_sum_launch<T, V, G>(w, keys, pos, n, rows, dim, d_out, stride, scale, d_table, index, index_bytes, s)
    if (fits(16)) {
        const size_t packs = dim / N;
        if (packs <= 4) E3_SUM(N, 4);
        else if (packs <= 8) E3_SUM(N, 8);
        else if (packs <= 16) E3_SUM(N, 16);
        else if (packs <= 32) E3_SUM(N, 32);
        else E3_SUM(N, 64);
    } else if (fits(8)) {
        if (dim / HALF <= 16) E3_SUM(HALF, 16);
        else if (dim / HALF <= 32) E3_SUM(HALF, 32);
        else E3_SUM(HALF, 64);
    } else if (N == 8 && fits(4)) {
        if (dim / QUARTER <= 4) E3_SUM(QUARTER, 4);
        else if (dim / QUARTER <= 16) E3_SUM(QUARTER, 16);
        else if (dim / QUARTER <= 32) E3_SUM(QUARTER, 32);
        else E3_SUM(QUARTER, 64);
    } else {
        if (dim <= 4) E3_SUM(1, 4);
        else if (dim <= 16) E3_SUM(1, 16);
        else if (dim <= 32) E3_SUM(1, 32);
        else E3_SUM(1, 64);
    }
#undef E3_SUM
    if (rc || n <= EMBED_TINY) return rc;
    // (partial rows start on 16-byte boundaries where dim is a multiple of 4)
    return dim % 4 == 0 && e3_rows_wide(d_table, dim, dim, dtype) ? embed_join_launch<T, 4>(w, keys, n, dim, scale, d_table, s)
                                                                 : embed_join_launch<T, 1>(w, keys, n, dim, scale, d_table, s);
}

__global__ __launch_bounds__(256) void fill_zero_kernel(size_t halves, uint16_t* __restrict__ out) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < halves; i += (size_t)gridDim.x * 256) out[i] = 0;
}
}  // namespace

size_t e3_embedding_scratch_bytes(size_t n, size_t dim) {
    char* p = nullptr;
    EmbedScratch::from(p, n, dim);
    return (size_t)p + 256;
}

int e3_embedding_backward_impl(size_t n, size_t rows, size_t dim, const void* index, int index_bytes, const void* d_out,
                               size_t stride, int dtype, float scale, void* d_table, char* scratch, hipStream_t s) {
    if (n == 0) {
        // no positions: clear the table's gradient with a kernel (a captured memset is not repeatable on every replay)
        const size_t bytes = rows * dim * e3_elem_bytes(dtype);
        const size_t blocks = (bytes / 2 + 255) / 256;
        fill_zero_kernel<<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s>>>(bytes / 2, (uint16_t*)d_table);
        LAUNCH_OK("fill_zero_kernel");
        return 0;
    }
    if (dtype == E3_F32) return embed_bwd_t<float>(n, rows, dim, index, index_bytes, d_out, stride, dtype, scale, d_table, scratch, s);
    if (dtype == E3_F16) return embed_bwd_t<f16_t>(n, rows, dim, index, index_bytes, d_out, stride, dtype, scale, d_table, scratch, s);
    return embed_bwd_t<bf16_t>(n, rows, dim, index, index_bytes, d_out, stride, dtype, scale, d_table, scratch, s);
}

// ============================================================================================== layer norm
// y = (x - mean) * rstd * weight + bias per row, mean and rstd = 1 / sqrt(var + eps) in fp32.  A row stays in the registers
// of its lanes between the statistics and the output (one pass over memory); the variance is the mean square of
// x - mean, not a difference of sums, so a row far from zero keeps its digits.
// Lanes per row: a group of 8 .. 64 lanes of one wave, or a workgroup of 256, 512 or 1024 threads for long rows
// (NormRow).
template <int G>
struct NormRow {      // sums over the lanes of a row
    static constexpr int THREADS = G > 256 ? G : 256;
    static constexpr int PER_BLOCK = THREADS / G;
    static __device__ __forceinline__ float sum(float v, float* lds) {
        if (G <= 64) return group_sum<(G <= 64 ? G : 64)>(v);
        v = group_sum<64>(v);
        const int wave = threadIdx.x >> 6;
        __syncthreads();                                    // (the previous use of `lds` has been read)
        if ((threadIdx.x & 63) == 0) lds[wave] = v;
        __syncthreads();
        float t = lds[0];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) t += lds[w];
        return t;
    }
};

// Parameters col, col + step, ... (N of them, `none` from dim on or without an array).  The branch on their type stands
// outside the loop, so that all loads are in flight together.
template <typename A, int N>
__device__ __forceinline__ void load_params(const A* __restrict__ p, int col, int step, int dim, float none, float v[N]) {
    A raw[N];
#pragma unroll
    for (int j = 0; j < N; ++j) raw[j] = p[col + j * step < dim ? col + j * step : dim - 1];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = col + j * step < dim ? (float)raw[j] : none;
}
template <int N>
__device__ __forceinline__ void load_affine(const void* __restrict__ p, int dtype, int col, int step, int dim, float none, float v[N]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = none;
    } else if (dtype == E3_F32) {
        load_params<float, N>(reinterpret_cast<const float*>(p), col, step, dim, none, v);
    } else if (dtype == E3_F16) {
        load_params<f16_t, N>(reinterpret_cast<const f16_t*>(p), col, step, dim, none, v);
    } else {
        load_params<bf16_t, N>(reinterpret_cast<const bf16_t*>(p), col, step, dim, none, v);
    }
}

// ... V neighbouring ones (col a multiple of V), in 16-byte loads where the array allows it
template <int V>
__device__ __forceinline__ void load_affine_pack(const void* __restrict__ p, int dtype, int col, int dim, float none, float v[V]) {
    if (V < 4 || !p || (reinterpret_cast<uintptr_t>(p) & 15) != 0 || (V == 4 && dtype != E3_F32)) {
        load_affine<V>(p, dtype, col, 1, dim, none, v);
        return;
    }
    if (col >= dim) col = 0;                              // (lanes behind the row: any value)
    if (dtype == E3_F32) {
        words_t q[V / 4 ? V / 4 : 1];
#pragma unroll
        for (int j = 0; j < V / 4; ++j) q[j] = reinterpret_cast<const words_t*>(reinterpret_cast<const float*>(p) + col)[j];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = word_elem<float>(q[j / 4], j % 4);
    } else {
        const words_t q = *reinterpret_cast<const words_t*>(reinterpret_cast<const uint16_t*>(p) + col);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = dtype == E3_F16 ? word_elem<f16_t>(q, j) : word_elem<bf16_t>(q, j);
    }
}

template <bool STREAM, typename T, int V, int G, int ITEMS>
__global__ __launch_bounds__(NormRow<G>::THREADS) void norm_fwd_kernel(size_t rows, int dim, const T* __restrict__ x,
                                                                       size_t stride, const void* __restrict__ weight,
                                                                       const void* __restrict__ bias, int affine_dtype,
                                                                       float eps, T* __restrict__ out,
                                                                       float* __restrict__ mean_out,
                                                                       float* __restrict__ rstd_out) {
    using R = NormRow<G>;
    __shared__ float lds[16];
    const int lane = threadIdx.x % G;
    float w[ITEMS][V], b[ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int col = (i * G + lane) * V;
        load_affine_pack<V>(weight, affine_dtype, col, dim, 1.0f, w[i]);
        load_affine_pack<V>(bias, affine_dtype, col, dim, 0.0f, b[i]);
    }
    const float len = (float)dim;                          // (divided by: its reciprocal would be rounded once more)
    const size_t step = (size_t)gridDim.x * R::PER_BLOCK;
    // (every lane of a wave, and every wave of a workgroup that shares a row, runs the same number of rounds)
    for (size_t base = (size_t)blockIdx.x * R::PER_BLOCK; base < rows; base += step) {
        const size_t row = base + threadIdx.x / G;
        const bool live = row < rows;
        float v[ITEMS][V], s = 0.0f;
        const T* xr = x + (live ? row : rows - 1) * stride;
        Held<T, V> xh[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {                   // (unconditional loads, all in flight)
            const int col = (i * G + lane) * V;
            xh[i].load(xr + (col < dim ? col : 0));
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool in = (i * G + lane) * V < dim;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = in ? xh[i].value(j) : 0.0f;
                s += v[i][j];
            }
        }
        const float mean = R::sum(s, lds) / len;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int col = (i * G + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] -= mean;
                if (col < dim) q = FMA(v[i][j], v[i][j], q);
            }
        }
        const float rstd = 1.0f / __builtin_sqrtf(R::sum(q, lds) / len + eps);
        if (!live) continue;
        if (lane == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int col = (i * G + lane) * V;
            if (col >= dim) continue;
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) r.v[j] = (T)FMA(v[i][j] * rstd, w[i][j], b[i][j]);
            put<STREAM, T, V>(out + row * (size_t)dim + col, r);
        }
    }
}

// Where the column sums go: one fp32 row pair per workgroup (norm_join_kernel adds them up), or straight to the results when
// there is only one workgroup.
struct NormSums {
    float* part;             // NULL: no column sums are wanted
    void *dweight, *dbias;
    int dtype;
    __device__ __forceinline__ void put(int dim, int which, int col, float v) const {
        if (gridDim.x > 1) {
            part[((size_t)blockIdx.x * 2 + which) * dim + col] = v;
            return;
        }
        void* out = which ? dbias : dweight;
        if (!out) return;
        if (dtype == E3_F32) reinterpret_cast<float*>(out)[col] = v;
        else if (dtype == E3_F16) reinterpret_cast<f16_t*>(out)[col] = (f16_t)v;
        else reinterpret_cast<bf16_t*>(out)[col] = (bf16_t)v;
    }
    // V neighbouring columns from a multiple of V on, in a row of a multiple of V
    template <int V>
    __device__ __forceinline__ void put_pack(int dim, int which, int col, const float v[V]) const {
        if (gridDim.x > 1) {
            constexpr int N = V < 4 ? V : 4;
#pragma unroll
            for (int j = 0; j < V; j += N) {
                Pack<float, N> p;
#pragma unroll
                for (int u = 0; u < N; ++u) p.v[u] = v[j + u];
                *reinterpret_cast<Pack<float, N>*>(part + ((size_t)blockIdx.x * 2 + which) * dim + col + j) = p;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) put(dim, which, col + j, v[j]);
    }
};

// Short rows whose length is no multiple of 16 bytes (or a few packs only), one behind the other: a workgroup moves `tile` rows
// at a time through LDS, in whole packs whatever the row length.  256 / tile lanes share a row there; each takes
// NORM_TILE_ITEMS of its values into registers, in one batch of LDS reads.  (200000 rows of 59 fp16 values: a lane per
// value straight from memory 38 us forward and 51 us backward, through LDS 15 us and 25 us.)
constexpr int NORM_TILE = 16384, NORM_TILE_PACKS = NORM_TILE / 16 / 256, NORM_TILE_ITEMS = 16;
// A tile on its way: loaded into registers while the tile before it is worked on, then put down in LDS.
template <typename T>
struct Tile {
    words_t in[NORM_TILE_PACKS];
    T single;
    __device__ __forceinline__ void load(const T* __restrict__ src, int elems) {
        const int packs = (int)(elems * sizeof(T) / 16), rest = packs * (16 / (int)sizeof(T));
        if (packs > 0) {                     // (uniform; the loads are unconditional and in flight together)
#pragma unroll
            for (int u = 0; u < NORM_TILE_PACKS; ++u) {
                const int i = u * 256 + threadIdx.x;
                in[u] = reinterpret_cast<const words_t*>(src)[i < packs ? i : packs - 1];
            }
        }
        if (rest + (int)threadIdx.x < elems) single = src[rest + threadIdx.x];
    }
    __device__ __forceinline__ void put_down(words_t* dst, int elems) const {
        const int packs = (int)(elems * sizeof(T) / 16), rest = packs * (16 / (int)sizeof(T));
#pragma unroll
        for (int u = 0; u < NORM_TILE_PACKS; ++u) {
            const int i = u * 256 + threadIdx.x;
            if (i < packs) dst[i] = in[u];
        }
        if (rest + (int)threadIdx.x < elems) reinterpret_cast<T*>(dst)[rest + threadIdx.x] = single;
    }
};
__device__ __forceinline__ int tile_count(size_t rows, size_t first, int tile) {
    return first >= rows ? 0 : rows - first < (size_t)tile ? (int)(rows - first) : tile;
}
template <typename T>
__device__ __forceinline__ void tile_store(T* __restrict__ dst, const words_t* src, int elems) {
    const int packs = (int)(elems * sizeof(T) / 16), rest = packs * (16 / (int)sizeof(T));
#pragma unroll
    for (int u = 0; u < NORM_TILE_PACKS; ++u) {
        const int i = u * 256 + threadIdx.x;
        if (i < packs) reinterpret_cast<words_t*>(dst)[i] = src[i];
    }
    if (rest + (int)threadIdx.x < elems) dst[rest + threadIdx.x] = reinterpret_cast<const T*>(src)[rest + threadIdx.x];
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <typename T>
__global__ __launch_bounds__(256) void norm_fwd_tile_kernel(size_t rows, int dim, int tile, const T* __restrict__ x,
                                                            const void* __restrict__ weight, const void* __restrict__ bias,
                                                            int affine_dtype, float eps, T* __restrict__ out,
                                                            float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    extern __shared__ words_t tile_mem[];
    const int LANES = 256 / tile, r = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    T* z = reinterpret_cast<T*>(tile_mem) + r * dim;
    float w[NORM_TILE_ITEMS], b[NORM_TILE_ITEMS];
    load_affine<NORM_TILE_ITEMS>(weight, affine_dtype, lane, LANES, dim, 1.0f, w);
    load_affine<NORM_TILE_ITEMS>(bias, affine_dtype, lane, LANES, dim, 0.0f, b);
    const float len = (float)dim;                          // (divided by: its reciprocal would be rounded once more)
    const size_t step = (size_t)gridDim.x * tile;
    size_t first = (size_t)blockIdx.x * tile;
    int n = tile_count(rows, first, tile);
    Tile<T> next;
    next.load(x + first * dim, n * dim);
    for (; first < rows; first += step, n = tile_count(rows, first, tile)) {
        next.put_down(tile_mem, n * dim);
        __syncthreads();
        if (first + step < rows) next.load(x + (first + step) * dim, tile_count(rows, first + step, tile) * dim);
        const bool live = r < n;
        float v[NORM_TILE_ITEMS], s = 0.0f, q = 0.0f;
        Held<T, 1> zh[NORM_TILE_ITEMS];
#pragma unroll
        for (int i = 0; i < NORM_TILE_ITEMS; ++i) zh[i].load(z + (i * LANES + lane < dim ? i * LANES + lane : 0));
#pragma unroll
        for (int i = 0; i < NORM_TILE_ITEMS; ++i) {
            v[i] = live && i * LANES + lane < dim ? zh[i].value(0) : 0.0f;
            s += v[i];
        }
        const float mean = lanes_sum(s, LANES) / len;
#pragma unroll
        for (int i = 0; i < NORM_TILE_ITEMS; ++i) {
            v[i] -= mean;
            if (i * LANES + lane < dim) q = FMA(v[i], v[i], q);
        }
        const float rstd = 1.0f / __builtin_sqrtf(lanes_sum(q, LANES) / len + eps);
        if (live) {
#pragma unroll
            for (int i = 0; i < NORM_TILE_ITEMS; ++i) {
                const int c = i * LANES + lane;
                if (c < dim) z[c] = (T)FMA(v[i] * rstd, w[i], b[i]);
            }
            if (lane == 0) {
                if (mean_out) mean_out[first + r] = mean;
                if (rstd_out) rstd_out[first + r] = rstd;
            }
        }
        __syncthreads();
        tile_store(out + first * dim, tile_mem, n * dim);
        __syncthreads();
    }
}

// Its gradient; a lane keeps the column sums of its values over all tiles of the workgroup.
template <typename T, int ITEMS>
__global__ __launch_bounds__(256) void norm_bwd_tile_kernel(size_t rows, int dim, int tile, const T* __restrict__ dy,
                                                            const T* __restrict__ x, const void* __restrict__ weight,
                                                            int affine_dtype, const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                            const NormSums out_sums) {
    extern __shared__ words_t tile_mem[];
    const int LANES = 256 / tile, r = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const int tile_packs = (int)((tile * dim * (int)sizeof(T) + 15) / 16);
    T* z = reinterpret_cast<T*>(tile_mem) + r * dim;
    const T* gr = reinterpret_cast<const T*>(tile_mem + tile_packs) + r * dim;
    float w[ITEMS], dw[ITEMS], db[ITEMS];
    load_affine<ITEMS>(weight, affine_dtype, lane, LANES, dim, 1.0f, w);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) dw[i] = db[i] = 0.0f;
    const float len = (float)dim;                          // (divided by: its reciprocal would be rounded once more)
    const size_t step = (size_t)gridDim.x * tile;
    size_t first = (size_t)blockIdx.x * tile;
    int n = tile_count(rows, first, tile);
    Tile<T> next_x, next_dy;
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto load = [&](size_t at, int count) {
        next_x.load(x + at * dim, count * dim);
        next_dy.load(dy + at * dim, count * dim);
        if (r < count) {
            next_mean = mean_in[at + r];
            next_rstd = rstd_in[at + r];
        }
    };
    load(first, n);
    for (; first < rows; first += step, n = tile_count(rows, first, tile)) {
        const bool live = r < n;
        const float mean = live ? next_mean : 0.0f, rstd = live ? next_rstd : 0.0f;
        next_x.put_down(tile_mem, n * dim);
        next_dy.put_down(tile_mem + tile_packs, n * dim);
        __syncthreads();
        if (first + step < rows) load(first + step, tile_count(rows, first + step, tile));
        float h[ITEMS], g[ITEMS], s1 = 0.0f, s2 = 0.0f;
        // (16 values: all LDS reads first, 100000 x 300 bf16 87 us, value by value 99; with 8 values that would cost a workgroup of the
        // CU its registers, 748061 x 65 fp16 152 us value by value, 235 so)
        if constexpr (ITEMS > 8) {
            Held<T, 1> zh[ITEMS], gh[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = i * LANES + lane < dim ? i * LANES + lane : 0;
                zh[i].load(z + c);
                gh[i].load(gr + c);
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const bool in = live && i * LANES + lane < dim;
                h[i] = in ? zh[i].value(0) : mean;
                g[i] = in ? gh[i].value(0) : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = i * LANES + lane;
                const bool in = live && c < dim;
                h[i] = in ? (float)z[c] : mean;
                g[i] = in ? (float)gr[c] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            h[i] = (h[i] - mean) * rstd;
            dw[i] = FMA(g[i], h[i], dw[i]);
            db[i] += g[i];
            g[i] *= w[i];
            s1 += g[i];
            s2 = FMA(g[i], h[i], s2);
        }
        s1 = lanes_sum(s1, LANES) / len;
        s2 = lanes_sum(s2, LANES) / len;
        if (dx) {
            if (live) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const int c = i * LANES + lane;
                    if (c < dim) z[c] = (T)((g[i] - s1 - h[i] * s2) * rstd);
                }
            }
            __syncthreads();
            tile_store(dx + first * dim, tile_mem, n * dim);
        }
        __syncthreads();
    }
    if (!out_sums.part) return;
    // the sums of the lanes that hold the same columns, in order: first within a wave, then over the waves through LDS
    __shared__ float sums[2][4][32 * ITEMS];
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        float a = dw[i], c = db[i];
        for (int o = LANES; o < 64; o <<= 1) {
            a += __shfl_xor(a, o, 64);
            c += __shfl_xor(c, o, 64);
        }
        if (wl < LANES) {
            sums[0][wave][i * LANES + wl] = a;
            sums[1][wave][i * LANES + wl] = c;
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < dim; c += 256) {
        out_sums.put(dim, 0, c, ((sums[0][0][c] + sums[0][1][c]) + sums[0][2][c]) + sums[0][3][c]);
        out_sums.put(dim, 1, c, ((sums[1][0][c] + sums[1][1][c]) + sums[1][2][c]) + sums[1][3][c]);
    }
}

// Rows longer than the registers of a workgroup hold: the row is read three times (the second and third time from cache).
template <typename T, int V>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(size_t rows, size_t dim, const T* __restrict__ x, size_t stride,
                                                             const void* __restrict__ weight, const void* __restrict__ bias,
                                                             int affine_dtype, float eps, T* __restrict__ out,
                                                             float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    using R = NormRow<1024>;
    __shared__ float lds[16];
    const float len = (float)dim;                          // (divided by: its reciprocal would be rounded once more)
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * stride;
        float s = 0.0f;
        for (size_t col = (size_t)threadIdx.x * V; col < dim; col += 1024 * V) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(xr + col);
#pragma unroll
            for (int j = 0; j < V; ++j) s += (float)p.v[j];
        }
        const float mean = R::sum(s, lds) / len;
        float q = 0.0f;
        for (size_t col = (size_t)threadIdx.x * V; col < dim; col += 1024 * V) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(xr + col);
#pragma unroll
            for (int j = 0; j < V; ++j) { const float d = (float)p.v[j] - mean; q = FMA(d, d, q); }
        }
        const float rstd = 1.0f / __builtin_sqrtf(R::sum(q, lds) / len + eps);
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
        for (size_t col = (size_t)threadIdx.x * V; col < dim; col += 1024 * V) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(xr + col);
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j)
                r.v[j] = (T)FMA(((float)p.v[j] - mean) * rstd, weight ? load_elem(weight, col + j, affine_dtype) : 1.0f,
                                bias ? load_elem(bias, col + j, affine_dtype) : 0.0f);
            *reinterpret_cast<Pack<T, V>*>(out + row * dim + col) = r;
        }
    }
}

// Gradient.  With h = (x - mean) * rstd and g = dy * weight:  dx = rstd * (g - mean(g) - h * mean(g h)),
// dweight = sum over the rows of dy h, dbias = sum of dy.  The column sums stay in registers while a workgroup walks over
// its rows, are added up over the workgroup's groups in LDS, and leave one fp32 row pair per workgroup, which
// norm_join_kernel adds up.
template <bool STREAM, typename T, int V, int G, int ITEMS>
__global__ __launch_bounds__(NormRow<G>::THREADS) void norm_bwd_kernel(size_t rows, int dim, const T* __restrict__ dy,
                                                                       size_t dy_stride, const T* __restrict__ x,
                                                                       size_t stride, const void* __restrict__ weight,
                                                                       int affine_dtype, const float* __restrict__ mean_in,
                                                                       const float* __restrict__ rstd_in,
                                                                       T* __restrict__ dx, const NormSums sums) {
    using R = NormRow<G>;
    __shared__ float lds[16];
    __shared__ float cols[R::PER_BLOCK > 1 ? R::THREADS * ITEMS * V : 1];
    const int lane = threadIdx.x % G;
    float w[ITEMS][V], dw[ITEMS][V], db[ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int col = (i * G + lane) * V;
        load_affine_pack<V>(weight, affine_dtype, col, dim, 1.0f, w[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
    }
    const float len = (float)dim;                          // (divided by: its reciprocal would be rounded once more)
    const size_t step = (size_t)gridDim.x * R::PER_BLOCK;
    for (size_t base = (size_t)blockIdx.x * R::PER_BLOCK; base < rows; base += step) {
        const size_t row = base + threadIdx.x / G;
        const bool live = row < rows;
        const size_t at = live ? row : rows - 1;
        const float mean = live ? mean_in[row] : 0.0f, rstd = live ? rstd_in[row] : 0.0f;
        float h[ITEMS][V], g[ITEMS][V], s1 = 0.0f, s2 = 0.0f;
        // All loads first, unconditional, where a thread has four packs or more (4096 x 8192 bf16 44 us, pack by pack 52); with
        // two of them the other waves hide the latency (8192 x 4096 bf16 42 us, 45 so), and 16 values in 1024 threads leave no
        // registers for it.
        if constexpr (ITEMS >= 4 && !(G == 1024 && ITEMS * V == 16)) {
            Held<T, V> xh[ITEMS], dh[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int col = (i * G + lane) * V < dim ? (i * G + lane) * V : 0;
                xh[i].load(x + at * stride + col);
                dh[i].load(dy + at * dy_stride + col);
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const bool in = live && (i * G + lane) * V < dim;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    h[i][j] = in ? xh[i].value(j) : mean;
                    g[i][j] = in ? dh[i].value(j) : 0.0f;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int col = (i * G + lane) * V;
                if (live && col < dim) {
                    Held<T, V> p, d;
                    p.load(x + row * stride + col);
                    d.load(dy + row * dy_stride + col);
#pragma unroll
                    for (int j = 0; j < V; ++j) { h[i][j] = p.value(j); g[i][j] = d.value(j); }
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) { h[i][j] = mean; g[i][j] = 0.0f; }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[i][j] = (h[i][j] - mean) * rstd;
                dw[i][j] = FMA(g[i][j], h[i][j], dw[i][j]);
                db[i][j] += g[i][j];
                g[i][j] *= w[i][j];
                s1 += g[i][j];
                s2 = FMA(g[i][j], h[i][j], s2);
            }
        s1 = R::sum(s1, lds) / len;
        s2 = R::sum(s2, lds) / len;
        if (!live || !dx) continue;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int col = (i * G + lane) * V;
            if (col >= dim) continue;
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) r.v[j] = (T)((g[i][j] - s1 - h[i][j] * s2) * rstd);
            put<STREAM, T, V>(dx + row * (size_t)dim + col, r);
        }
    }
    if (!sums.part) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float(&a)[ITEMS][V] = which ? db : dw;
        if (R::PER_BLOCK > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) cols[(threadIdx.x / G) * (G * ITEMS * V) + (i * G + lane) * V + j] = a[i][j];
            __syncthreads();
            for (int col = threadIdx.x; col < dim; col += R::THREADS) {
                float s = cols[col];
                for (int k = 1; k < R::PER_BLOCK; ++k) s += cols[k * (G * ITEMS * V) + col];
                sums.put(dim, which, col, s);
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int col = (i * G + lane) * V;
                if (col < dim) sums.template put_pack<V>(dim, which, col, a[i]);
            }
        }
    }
}

// dx of rows longer than the registers hold
template <typename T, int V>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(size_t rows, size_t dim, const T* __restrict__ dy,
                                                             size_t dy_stride, const T* __restrict__ x, size_t stride,
                                                             const void* __restrict__ weight, int affine_dtype,
                                                             const float* __restrict__ mean_in,
                                                             const float* __restrict__ rstd_in, T* __restrict__ dx) {
    using R = NormRow<1024>;
    __shared__ float lds[16];
    const float len = (float)dim;                          // (divided by: its reciprocal would be rounded once more)
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * stride, *dr = dy + row * dy_stride;
        const float mean = mean_in[row], rstd = rstd_in[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (size_t col = (size_t)threadIdx.x * V; col < dim; col += 1024 * V) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(xr + col), d = *reinterpret_cast<const Pack<T, V>*>(dr + col);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g = (float)d.v[j] * (weight ? load_elem(weight, col + j, affine_dtype) : 1.0f);
                s1 += g;
                s2 = FMA(g, ((float)p.v[j] - mean) * rstd, s2);
            }
        }
        s1 = R::sum(s1, lds) / len;
        s2 = R::sum(s2, lds) / len;
        for (size_t col = (size_t)threadIdx.x * V; col < dim; col += 1024 * V) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(xr + col), d = *reinterpret_cast<const Pack<T, V>*>(dr + col);
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g = (float)d.v[j] * (weight ? load_elem(weight, col + j, affine_dtype) : 1.0f);
                r.v[j] = (T)((g - s1 - ((float)p.v[j] - mean) * rstd * s2) * rstd);
            }
            *reinterpret_cast<Pack<T, V>*>(dx + row * dim + col) = r;
        }
    }
}
// ... and their column sums: a thread per column, a workgroup per 256 columns and slice of the rows
template <typename T>
__global__ __launch_bounds__(256) void norm_cols_kernel(size_t rows, size_t dim, const T* __restrict__ dy, size_t dy_stride,
                                                        const T* __restrict__ x, size_t stride,
                                                        const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                        float* __restrict__ part) {
    const size_t col = (size_t)blockIdx.y * 256 + threadIdx.x;
    if (col >= dim) return;
    float dw = 0.0f, db = 0.0f;
#pragma unroll 4
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float g = (float)dy[row * dy_stride + col];
        dw = FMA(g, ((float)x[row * stride + col] - mean_in[row]) * rstd_in[row], dw);
        db += g;
    }
    part[(size_t)blockIdx.x * 2 * dim + col] = dw;
    part[(size_t)blockIdx.x * 2 * dim + dim + col] = db;
}

// dweight and dbias = sums over the workgroups' partial rows: 64 columns to a workgroup, wave w takes the w-th sixteenth of
// the rows, the sixteen sums are added in order.
__global__ __launch_bounds__(1024) void norm_join_kernel(uint32_t nparts, size_t dim, const float* __restrict__ part,
                                                         int affine_dtype, void* __restrict__ dweight,
                                                         void* __restrict__ dbias) {
    __shared__ float sums[16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const size_t col = (size_t)blockIdx.x * 64 + lane;                  // 0 .. 2 dim
    const uint32_t lo = (uint32_t)((unsigned long long)nparts * wave / 16);
    const uint32_t hi = (uint32_t)((unsigned long long)nparts * (wave + 1) / 16);
    float s = 0.0f;
    if (col < 2 * dim) {
#pragma unroll 8
        for (uint32_t k = lo; k < hi; ++k) s += part[(size_t)k * 2 * dim + col];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= 2 * dim) return;
    s = sums[0][lane];
#pragma unroll
    for (int w = 1; w < 16; ++w) s += sums[w][lane];
    void* out = col < dim ? dweight : dbias;
    if (!out) return;
    const size_t at = col < dim ? col : col - dim;
    if (affine_dtype == E3_F32) reinterpret_cast<float*>(out)[at] = s;
    else if (affine_dtype == E3_F16) reinterpret_cast<f16_t*>(out)[at] = (f16_t)s;
    else reinterpret_cast<bf16_t*>(out)[at] = (bf16_t)s;
}

namespace {
// Workgroups of 256 CUs that are resident together.  Long rows are spread over no more than that, each the same number of
// rows: more workgroups fetch the parameters again, and the last ones leave most of the chip idle (forward, 4096 x 8192 bf16
// with 4096 workgroups 55 us, 1024 52 us, 768 = all resident 40 us; 30 us with a row's loads all in flight).
template <typename K>
size_t resident_blocks(K kernel, int threads) {
    int n = 0;
    const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, reinterpret_cast<const void*>(kernel), threads, 0);
    if (e != hipSuccess) (void)hipGetLastError();          // (its own error alone is taken back)
    return e == hipSuccess && n > 0 ? (size_t)n * 256 : 256;
}
unsigned even_blocks(size_t need, size_t most) {
    const size_t rounds = (need + most - 1) / most;
    return (unsigned)((need + rounds - 1) / rounds);
}
// workgroups of a launch over `rows` rows: enough to fill 256 CUs several times over, each with a few rows of its own
unsigned norm_blocks(size_t rows, int per_block, size_t most) {
    const size_t need = (rows + per_block - 1) / per_block;
    return (unsigned)(need < most ? need : most);
}
// ... of the gradient: what one workgroup does in four rounds goes to one, which saves the launch that would join the sums (10
// rows of 64 values with autograd around it: 66 us of host time with the second launch, 61 us without; a round takes about
// 1.5 us, the launch 2.5 us on the GPU and 4 us on the host).  Beyond 256 workgroups each takes four rounds before there are
// more of them: their partial sums cost as much as their rows (1000 x 1446 bf16 with a workgroup per row 27 us, so 22; 500 x 4096
// bf16 32 and 25 us).
unsigned norm_bwd_blocks(size_t rows, int per_block, size_t most) {
    const size_t need = (rows + per_block - 1) / per_block;
    if (need <= 4) return 1u;
    const size_t blocks = need <= 256 ? need : need / 4 < 256 ? 256 : need / 4;
    // (a workgroup per row: the same number of rounds for all; otherwise there are many rounds, and 1024 partial sums are
    // joined faster than 962)
    return per_block == 1 ? even_blocks(need, blocks < most ? blocks : most) : (unsigned)(blocks < most ? blocks : most);
}
// (a row of more than NORM_HELD values is never held in registers, whatever its type and boundary: its column sums come from
// norm_cols_kernel, in NORM_LONG_PARTS partial rows)
constexpr size_t NORM_FWD_BLOCKS = 4096, NORM_BWD_BLOCKS = 1024, NORM_TILE_BLOCKS = 1024, NORM_LONG_PARTS = 64, NORM_HELD = 16384;

struct NormArgs {
    size_t rows, dim, x_stride, dy_stride;
    const void *x, *dy, *weight, *bias;
    int affine_dtype;
    float eps;
    void *out, *dx, *dweight, *dbias;
    float *mean, *rstd, *part;
    hipStream_t s;
};

NormSums norm_sums(const NormArgs& a) { return {a.part, a.dweight, a.dbias, a.affine_dtype}; }

template <typename T, int V, int G, int ITEMS>
int norm_fwd_launch(const NormArgs& a) {
    const dim3 threads(NormRow<G>::THREADS);
    static const size_t most = resident_blocks(norm_fwd_kernel<false, T, V, G, ITEMS>, NormRow<G>::THREADS);
    const dim3 blocks(G < 256 ? norm_blocks(a.rows, NormRow<G>::PER_BLOCK, NORM_FWD_BLOCKS) : even_blocks(a.rows, most));
#define E3_NORM(S)                                                                                                            \
    norm_fwd_kernel<(S), T, V, G, ITEMS><<<blocks, threads, 0, a.s>>>(a.rows, (int)a.dim, (const T*)a.x, a.x_stride, a.weight, \
                                                                  a.bias, a.affine_dtype, a.eps, (T*)a.out, a.mean, a.rstd)
    constexpr bool WIDE = V == Wide<T>::N;
    if (WIDE && a.rows * a.dim * sizeof(T) > E3_STREAM_BYTES) E3_NORM(WIDE);
    else E3_NORM(false);
#undef E3_NORM
    LAUNCH_OK("norm_fwd_kernel");
    return 0;
}
template <typename T, int V, int G, int ITEMS>
int norm_bwd_launch(const NormArgs& a, uint32_t& nparts) {
    static const size_t most = resident_blocks(norm_bwd_kernel<false, T, V, G, ITEMS>, NormRow<G>::THREADS);
    nparts = norm_bwd_blocks(a.rows, NormRow<G>::PER_BLOCK, G < 256 || most > NORM_BWD_BLOCKS ? NORM_BWD_BLOCKS : most);
    const dim3 blocks(nparts), threads(NormRow<G>::THREADS);
#define E3_NORM(S)                                                                                                            \
    norm_bwd_kernel<(S), T, V, G, ITEMS><<<blocks, threads, 0, a.s>>>(a.rows, (int)a.dim, (const T*)a.dy, a.dy_stride,          \
                                                                  (const T*)a.x, a.x_stride, a.weight, a.affine_dtype,       \
                                                                  a.mean, a.rstd, (T*)a.dx, norm_sums(a))
    constexpr bool WIDE = V == Wide<T>::N;
    if (WIDE && a.rows * a.dim * sizeof(T) > E3_STREAM_BYTES) E3_NORM(WIDE);
    else E3_NORM(false);
#undef E3_NORM
    LAUNCH_OK("norm_bwd_kernel");
    if (nparts == 1) nparts = 0;
    return 0;
}
// Values of a row to a lane.  The gradient keeps five arrays of them in registers: 8 while 32 lanes are enough for the row.
int norm_tile_items(size_t dim, bool backward) { return backward && dim <= 256 ? 8 : NORM_TILE_ITEMS; }

// Rows of a tile, or 0 where the tile kernels do not apply: rows that do not lie one behind the other from a 16-byte boundary
// on, rows past 32 lanes of NORM_TILE_ITEMS values, and those that a group of lanes reads in packs as well (5 packs or
// more).  256 / the lanes of a row, with more lanes to it when the launch would not fill the chip otherwise; at least 8 rows,
// so that every tile begins on a 16-byte boundary.
int norm_tile_rows(const NormArgs& a, size_t bytes, bool backward) {
    size_t lanes = 1;
    while (lanes * norm_tile_items(a.dim, backward) < a.dim) lanes <<= 1;
    if (lanes > 32 || a.x_stride != a.dim || (a.dim * bytes % 16 == 0 && a.dim * bytes / 16 >= 5)) return 0;
    uintptr_t any = reinterpret_cast<uintptr_t>(a.x);
    if (!backward) any |= reinterpret_cast<uintptr_t>(a.out);
    else {
        if (a.dy_stride != a.dim) return 0;
        any |= reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.dx);
    }
    if (any & 15) return 0;
    while (lanes < 32 && lanes < a.dim && a.rows < 256 / lanes * 512) lanes <<= 1;
    return (int)(256 / lanes);
}
template <typename T>
int norm_fwd_tile(const NormArgs& a, int tile) {
    const size_t lds = (tile * a.dim * sizeof(T) + 15) / 16 * 16;
    norm_fwd_tile_kernel<T><<<dim3(norm_blocks(a.rows, tile, NORM_TILE_BLOCKS)), dim3(256), lds, a.s>>>(
        a.rows, (int)a.dim, tile, (const T*)a.x, a.weight, a.bias, a.affine_dtype, a.eps, (T*)a.out, a.mean, a.rstd);
    LAUNCH_OK("norm_fwd_tile_kernel");
    return 0;
}
template <typename T>
int norm_bwd_tile(const NormArgs& a, int tile, uint32_t& nparts) {
    const size_t lds = 2 * ((tile * a.dim * sizeof(T) + 15) / 16 * 16);
    // (16 values to a lane: two workgroups fit a CU, and no more are launched: 30112 x 483 fp32 37 us, with 1024 workgroups 44)
    nparts = norm_bwd_blocks(a.rows, tile, norm_tile_items(a.dim, true) > 8 ? NORM_TILE_BLOCKS / 2 : NORM_TILE_BLOCKS);
#define E3_TILE_BWD(ITEMS)                                                                                                    \
    norm_bwd_tile_kernel<T, ITEMS><<<dim3(nparts), dim3(256), lds, a.s>>>(a.rows, (int)a.dim, tile, (const T*)a.dy,           \
                                                                        (const T*)a.x, a.weight, a.affine_dtype, a.mean,     \
                                                                        a.rstd, (T*)a.dx, norm_sums(a))
    if (norm_tile_items(a.dim, true) == 8) E3_TILE_BWD(8);
    else E3_TILE_BWD(NORM_TILE_ITEMS);
#undef E3_TILE_BWD
    LAUNCH_OK("norm_bwd_tile_kernel");
    if (nparts == 1) nparts = 0;
    return 0;
}
template <typename T, int V>
int norm_fwd_again(const NormArgs& a) {
    const unsigned blocks = (unsigned)(a.rows < 2048 ? a.rows : 2048);
    norm_fwd_long_kernel<T, V><<<dim3(blocks), dim3(1024), 0, a.s>>>(a.rows, a.dim, (const T*)a.x, a.x_stride, a.weight,
                                                                    a.bias, a.affine_dtype, a.eps, (T*)a.out, a.mean, a.rstd);
    LAUNCH_OK("norm_fwd_long_kernel");
    return 0;
}
// Rows of more than 256 packs (V values each, 16, 8 or 4 bytes or a single one): workgroups of 256 threads up to 1024 packs, of
// 512 or 1024 threads up to 16384 values (8192 single ones); longer rows are read again for every step.  Held in registers / read
// again: 2000 x 16384 bf16 31 / 85 us, 4096 x 4588 bf16 29 / 66 us, 300 x 16384 fp32 11 / 24 us, 2000 x 4097 bf16 23 / 29 us.
template <typename T, int V>
int norm_fwd_long(const NormArgs& a) {
    const size_t packs = a.dim / V;
    constexpr int MORE = V < 8 ? 4 : 2, MOST = V < 4 ? 8 : MORE;
    if constexpr (V != 2) {                                // (packs of two values: only rows of more than 512 values)
        if (packs <= 256) return norm_fwd_launch<T, V, 64, 4>(a);
    }
    if (packs <= 512) return norm_fwd_launch<T, V, 256, 2>(a);
    if (packs <= 1024) return norm_fwd_launch<T, V, 256, 4>(a);
    if (packs <= 2048) return norm_fwd_launch<T, V, 512, 4>(a);
    if constexpr (MORE > 2) {
        if (packs <= 1024 * MORE) return norm_fwd_launch<T, V, 1024, MORE>(a);
    }
    if constexpr (MOST > MORE) {
        if (packs <= 1024 * MOST) return norm_fwd_launch<T, V, 1024, MOST>(a);
    }
    return norm_fwd_again<T, V>(a);
}
template <typename T, int V>
int norm_fwd_v(const NormArgs& a) {
    const size_t packs = a.dim / V;
    if (packs <= 8) return norm_fwd_launch<T, V, 8, 1>(a);
    if (packs <= 16) return norm_fwd_launch<T, V, 16, 1>(a);
    if (packs <= 32) return norm_fwd_launch<T, V, 32, 1>(a);
    if (packs <= 64) return norm_fwd_launch<T, V, 64, 1>(a);
    if (packs <= 128) return norm_fwd_launch<T, V, 64, 2>(a);
    return norm_fwd_long<T, V>(a);
}
template <typename T>
int norm_fwd_t(const NormArgs& a, int dtype) {
    constexpr int N = Wide<T>::N;
    auto fits = [&](size_t bytes) { return e3_rows_packs(a.x, a.x_stride, a.dim, dtype, bytes) && e3_rows_packs(a.out, a.dim, a.dim, dtype, bytes); };
    if (const int tile = norm_tile_rows(a, sizeof(T), false)) return norm_fwd_tile<T>(a, tile);
    if (fits(16)) return norm_fwd_v<T, N>(a);
    if (a.dim > 512 && fits(8)) return norm_fwd_long<T, N / 2>(a);
    if (a.dim > 512 && N == 8 && fits(4)) return norm_fwd_long<T, N == 8 ? 2 : 1>(a);
    return norm_fwd_v<T, 1>(a);
}
// The gradient, which keeps five arrays of the row, up to 16384 values where there are rows enough to make up for the partial
// sums of the workgroups: 2000 x 16384 bf16 57 us (read again: 123), 4096 x 4588 bf16 50 us (90), 113 x 4588 bf16 11 us (15);
// with 16 values to a thread 300 x 16384 fp32 took 47 us (38).
// nparts: how many partial sums there are for norm_join_kernel, 0: the results are written
template <typename T, int V>
int norm_bwd_long(const NormArgs& a, uint32_t& nparts) {
    const size_t packs = a.dim / V;
    constexpr int MORE = V < 8 ? 4 : 2, MOST = V < 4 ? 8 : MORE;
    static_assert(1024 * MOST * V <= NORM_HELD, "e3_layer_norm_scratch_bytes");
    if constexpr (V != 2) {
        if (packs <= 256) return norm_bwd_launch<T, V, 256, 1>(a, nparts);
    }
    if (packs <= 512) return norm_bwd_launch<T, V, 256, 2>(a, nparts);
    if (packs <= 1024) return norm_bwd_launch<T, V, 256, 4>(a, nparts);
    if (packs <= 2048) return norm_bwd_launch<T, V, V == 8 ? 512 : 1024, V == 8 ? 4 : 2>(a, nparts);
    [[maybe_unused]] const size_t most = a.rows >= 1024 || V == 1 ? 1024 * MOST : 8192 / V;
    if constexpr (MORE > 2) {
        if (packs <= 1024 * MORE && packs <= most) return norm_bwd_launch<T, V, 1024, MORE>(a, nparts);
    }
    if constexpr (MOST > MORE) {
        if (packs <= most) return norm_bwd_launch<T, V, 1024, MOST>(a, nparts);
    }
    if (a.dx) {
        const unsigned blocks = (unsigned)(a.rows < 2048 ? a.rows : 2048);
        norm_bwd_long_kernel<T, V><<<dim3(blocks), dim3(1024), 0, a.s>>>(a.rows, a.dim, (const T*)a.dy, a.dy_stride,
                                                                        (const T*)a.x, a.x_stride, a.weight,
                                                                        a.affine_dtype, a.mean, a.rstd, (T*)a.dx);
        LAUNCH_OK("norm_bwd_long_kernel");
    }
    if (a.part) {
        nparts = (uint32_t)(a.rows < NORM_LONG_PARTS ? a.rows : NORM_LONG_PARTS);
        norm_cols_kernel<T><<<dim3(nparts, (unsigned)((a.dim + 255) / 256)), dim3(256), 0, a.s>>>(
            a.rows, a.dim, (const T*)a.dy, a.dy_stride, (const T*)a.x, a.x_stride, a.mean, a.rstd, a.part);
        LAUNCH_OK("norm_cols_kernel");
    }
    return 0;
}
template <typename T, int V>
int norm_bwd_v(const NormArgs& a, uint32_t& nparts) {
    const size_t packs = a.dim / V;
    if (packs <= 8) return norm_bwd_launch<T, V, 8, 1>(a, nparts);
    if (packs <= 16) return norm_bwd_launch<T, V, 16, 1>(a, nparts);
    if (packs <= 32) return norm_bwd_launch<T, V, 32, 1>(a, nparts);
    if (packs <= 64) return norm_bwd_launch<T, V, 64, 1>(a, nparts);
    if (packs <= 128) return norm_bwd_launch<T, V, 64, 2>(a, nparts);
    return norm_bwd_long<T, V>(a, nparts);
}
template <typename T>
int norm_bwd_t(const NormArgs& a, int dtype) {
    constexpr int N = Wide<T>::N;
    uint32_t nparts = 0;
    int rc = 0;
    auto fits = [&](size_t bytes) {
        return e3_rows_packs(a.x, a.x_stride, a.dim, dtype, bytes) && e3_rows_packs(a.dy, a.dy_stride, a.dim, dtype, bytes) &&
               (!a.dx || e3_rows_packs(a.dx, a.dim, a.dim, dtype, bytes));
    };
    if (const int tile = norm_tile_rows(a, sizeof(T), true)) rc = norm_bwd_tile<T>(a, tile, nparts);
    else if (fits(16)) rc = norm_bwd_v<T, N>(a, nparts);
    else if (a.dim > 512 && fits(8)) rc = norm_bwd_long<T, N / 2>(a, nparts);
    else if (a.dim > 512 && N == 8 && fits(4)) rc = norm_bwd_long<T, N == 8 ? 2 : 1>(a, nparts);
    else rc = norm_bwd_v<T, 1>(a, nparts);
    if (rc || !a.part || nparts == 0) return rc;
    norm_join_kernel<<<dim3((unsigned)((2 * a.dim + 63) / 64)), dim3(1024), 0, a.s>>>(nparts, a.dim, a.part, a.affine_dtype,
                                                                                    a.dweight, a.dbias);
    LAUNCH_OK("norm_join_kernel");
    return 0;
}
}  // namespace

int e3_layer_norm_forward_impl(size_t rows, size_t dim, const void* x, size_t x_stride, int dtype, const void* weight,
                               const void* bias, int affine_dtype, float eps, void* out, float* mean, float* rstd,
                               hipStream_t s) {
    if (rows == 0) return 0;
    NormArgs a{};
    a.rows = rows; a.dim = dim; a.x = x; a.x_stride = x_stride; a.weight = weight; a.bias = bias;
    a.affine_dtype = affine_dtype; a.eps = eps; a.out = out; a.mean = mean; a.rstd = rstd; a.s = s;
    if (dtype == E3_F32) return norm_fwd_t<float>(a, dtype);
    return dtype == E3_F16 ? norm_fwd_t<f16_t>(a, dtype) : norm_fwd_t<bf16_t>(a, dtype);
}

size_t e3_layer_norm_scratch_bytes(size_t rows, size_t dim) {
    const size_t most = dim > NORM_HELD ? NORM_LONG_PARTS : NORM_BWD_BLOCKS;
    return (rows < most ? (rows ? rows : 1) : most) * 2 * dim * sizeof(float) + 256;
}

int e3_layer_norm_backward_impl(size_t rows, size_t dim, const void* dy, size_t dy_stride, const void* x, size_t x_stride,
                                int dtype, const void* weight, int affine_dtype, const float* mean, const float* rstd,
                                void* dx, void* dweight, void* dbias, char* scratch, hipStream_t s) {
    NormArgs a{};
    a.rows = rows; a.dim = dim; a.x = x; a.x_stride = x_stride; a.dy = dy; a.dy_stride = dy_stride; a.weight = weight;
    a.affine_dtype = affine_dtype; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.dx = dx;
    a.dweight = dweight; a.dbias = dbias; a.s = s;
    a.part = dweight || dbias ? reinterpret_cast<float*>(scratch) : nullptr;
    if (rows == 0) {
        if (!a.part) return 0;
        norm_join_kernel<<<dim3((unsigned)((2 * dim + 63) / 64)), dim3(1024), 0, s>>>(0, dim, a.part, affine_dtype, dweight, dbias);
        LAUNCH_OK("norm_join_kernel");
        return 0;
    }
    if (dtype == E3_F32) return norm_bwd_t<float>(a, dtype);
    return dtype == E3_F16 ? norm_bwd_t<f16_t>(a, dtype) : norm_bwd_t<bf16_t>(a, dtype);
}
