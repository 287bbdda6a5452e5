// distill.hip -- distillation from a teacher's best scores: value and gradient.
//
//   q = softmax over the teacher's listed classes (teacher / T),  p = softmax over all classes (logits / T)
//   row = T^2 * sum_k q_k (log q_k - log p[index_k]),   d row / d logits_j = T (p_j - sum of q_k with index_k == j)
//
// An entry counts when its index is >= 0 and its teacher score above -infinity; a row without such an entry has no label:
// it adds nothing, gets a zero gradient and is not counted in the mean.  An index past the classes makes the row NaN.
// The kernels read the scores once per pass with a running maximum and sum (fp32), the exponentials are the hardware's exp2
// of (z - max) * log2(e) / T: the difference is formed first, so that neither masks of the type's lowest value nor their
// scaling overflow.  Bound by memory: the scores are read once by the value and once by the gradient, which writes as much.
//
// Two layouts: rows of classes (class stride 1) and planes of classes (row stride 1, as the rasteriser lays an image out).
//   long rows             a wave or a workgroup to a row; value and gradient together keep the row in registers
//   short rows, planes    a workgroup takes some rows at a time through LDS, where planes become rows
//   many pixels of planes with a short list: a lane takes neighbouring pixels and walks over the planes
#include "rows.h"

int e3_fail(hipError_t e, const char* what);
#define LAUNCH_OK(name)                                       \
    do {                                                      \
        hipError_t _e = hipGetLastError();                    \
        if (_e != hipSuccess) return e3_fail(_e, name);       \
    } while (0)

namespace {
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int DISTILL_MAX_K = 1024;              // entries of a row's label (E3DGS_DISTILL_MAX_K)
constexpr int DISTILL_PLANES = 256;              // classes of the plane layout, and entries of its labels
constexpr unsigned DISTILL_BLOCKS = 4096;        // workgroups = partial sums of a launch

struct DistillArgs {
    size_t rows, k, row_stride, class_stride;
    uint32_t classes;
    const void* logits;
    const void *teacher, *index;
    size_t t_row, t_entry, i_row, i_entry;
    int dtype, teacher_dtype, index_bytes, reduction;
    float temperature;
    float2* stats;          // per row: (maximum, 1 / sum of exp2((z - max) c)); (0, 0): no label
    float* row_loss;
    float2* part;           // per workgroup: (sum of the rows, labelled rows as a float's bits)
    const float* weight;    // gradient: weight of a row (one for all, or with `none` one per row), times *scale
    const float* scale;
    void* grad;
    size_t g_row, g_class;
    float *loss, *weight_out;   // the value and the weight of a row, written by the only workgroup of a launch
    bool planes_wide;       // the planes of the scores (and of the gradient) can be moved in 16-byte packs
    const uint32_t* counts; // partial counts of the labelled rows (a value formed with its gradient)
    uint32_t ncounts;
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

// (max, sum) of a softmax: the pair of two disjoint parts
__device__ __forceinline__ void soft_merge(float& m, float& s, float m2, float s2, float c) {
    const float M = fmaxf(m, m2);
    s = s * (m == M ? 1.0f : exp2_hw((m - M) * c)) + s2 * (m2 == M ? 1.0f : exp2_hw((m2 - M) * c));
    m = M;
}
template <int V>
__device__ __forceinline__ void soft_add(float& m, float& s, const float z[V], float c) {
    float M = m;
#pragma unroll
    for (int j = 0; j < V; ++j) M = fmaxf(M, z[j]);
    if (M != m) s *= exp2_hw((m - M) * c);            // (nothing summed yet: 0 * 0)
    m = M;
    const float off = M == -__builtin_inff() ? 0.0f : M;
#pragma unroll
    for (int j = 0; j < V; ++j) s += exp2_hw((z[j] - off) * c);
}


// ---- labels.  An entry is listed when its index is >= 0 and its score above -infinity.
struct Label {
    float top, inv;          // largest listed score; 1 / sum of exp2((t - top) c)
    bool any, broken;        // an entry is listed; a listed one names a class past the end
};
constexpr int ID_BROKEN = 0x7FFFFFFF;
__device__ __forceinline__ float entry_score(const DistillArgs& a, size_t row, size_t k, long long& id) {
    id = load_index_flat(a.index, row * a.i_row + k * a.i_entry, a.index_bytes);
    const float t = load_elem_flat(a.teacher, row * a.t_row + k * a.t_entry, a.teacher_dtype);
    return id < 0 ? -__builtin_inff() : t;
}
// the class of an entry as it is kept in LDS: -1 not listed, ID_BROKEN past the end
__device__ __forceinline__ int entry_class(const DistillArgs& a, float t, long long id) {
    return t == -__builtin_inff() ? -1 : id >= (long long)a.classes ? ID_BROKEN : (int)id;
}

// The label of a row, worked out by one wave: classes and weights exp2((t - top) c) of all entries to LDS.
__device__ __forceinline__ Label wave_label(const DistillArgs& a, size_t row, float c, int* ids, float* ws) {
    const int lane = threadIdx.x & 63;
    float top = -__builtin_inff(), sum = 0.0f, flags = 0.0f;
    for (int k = lane; k < (int)a.k; k += 64) {
        long long id;
        const float t = entry_score(a, row, k, id);
        const int cls = entry_class(a, t, id);
        ids[k] = cls;
        ws[k] = t;
        if (cls < 0) continue;
        flags = fmaxf(flags, cls == ID_BROKEN ? 2.0f : 1.0f);
        top = fmaxf(top, t);                                        // (a NaN score makes the sum NaN)
    }
    Label l;
    l.top = top = group_max<64>(top);
    flags = group_max<64>(flags);
    for (int k = lane; k < (int)a.k; k += 64) {
        const float w = ids[k] < 0 ? 0.0f : exp2_hw((ws[k] - top) * c);
        ws[k] = w;
        sum += w;
    }
    sum = group_sum<64>(sum);
    l.inv = 1.0f / sum;
    l.any = flags > 0.0f;
    l.broken = flags > 1.5f;
    wave_sync();
    return l;
}
// whether a row has a listed entry; every lane of a wave gets the answer
__device__ __forceinline__ bool wave_any(const DistillArgs& a, size_t row) {
    bool any = false;
    for (int k = threadIdx.x & 63; k < (int)a.k; k += 64) {
        long long id;
        any |= entry_score(a, row, k, id) != -__builtin_inff();
    }
    return __ballot(any) != 0ull;
}
// Sum over the entries of q (log q - log p), with log p = (z - m) / T - log s; one lane's entries, `score(k)` gives z.
template <typename F>
__device__ __forceinline__ float label_value(const DistillArgs& a, size_t row, const Label& l, const int* ids, const float* ws,
                                             int first, int step, float m, float s, float rt, F score) {
    float d = 0.0f;
    const float rest = (log2_hw(l.inv) + log2_hw(s)) * LN2;
    for (int k = first; k < (int)a.k; k += step) {
        if (ids[k] < 0) continue;
        if (ids[k] == ID_BROKEN) { d = __builtin_nanf(""); continue; }
        const float q = ws[k] * l.inv;
        if (q == 0.0f) continue;
        long long id;
        const float t = entry_score(a, row, k, id);
        d += q * (((t - l.top) - (score(ids[k]) - m)) * rt + rest);
    }
    return d;
}
// Weight of the class of entry k: all its entries added up in order; 0 entries before k name it (else false).
__device__ __forceinline__ bool class_weight(const DistillArgs& a, const int* ids, const float* ws, int k, float& w) {
    const int id = ids[k];
    if (id < 0 || id == ID_BROKEN) return false;
    w = ws[k];
    int same = 0;
#pragma unroll 4
    for (int j = 0; j < (int)a.k; ++j) same += ids[j] == id ? 1 : 0;
    if (same == 1) return true;
    w = 0.0f;
    bool first = true;
    for (int j = 0; j < (int)a.k; ++j) {
        if (ids[j] != id) continue;
        first &= j >= k;
        w += ws[j];
    }
    return first;
}

// ---- sums over a launch
// Number of labelled rows; one thread's share.  Where the entries of a row lie next to each other they are read by as many
// neighbouring lanes as there are entries (a power of two, at most a wave), and the row counts for the first of them; where
// neighbouring rows do (planes), a lane takes a row.
__device__ __forceinline__ uint32_t count_rows(const DistillArgs& a, size_t thread, size_t threads) {
    int lanes = a.i_entry == 1 ? 64 : 1;
    while (lanes > 1 && lanes > (int)a.k) lanes >>= 1;
    const int lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 63) & ~(lanes - 1);
    const unsigned long long mine = (lanes == 64 ? ~0ull : (1ull << lanes) - 1ull) << group;
    uint32_t n = 0;
    const size_t step = threads / lanes, rounds = (a.rows + step - 1) / step;
    for (size_t i = 0; i < rounds; ++i) {                 // (the same number of rounds for every lane of a wave)
        const size_t row = i * step + thread / lanes;
        unsigned long long any = 0ull;
        for (int k0 = 0; k0 < (int)a.k; k0 += lanes) {    // (most rows are decided by their first entries)
            long long id;
            const bool in = row < a.rows && k0 + lane < (int)a.k;
            any |= __ballot(in && entry_score(a, row, k0 + lane, id) != -__builtin_inff());
            if (lanes == 1 && any == ~0ull) break;
        }
        if (lane == 0 && (any & mine) != 0ull) ++n;
    }
    return n;
}
template <int THREADS>
__device__ __forceinline__ uint32_t block_sum_u32(uint32_t n, uint32_t* lds) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = n;
    __syncthreads();
    n = lds[0];
    for (int w = 1; w < THREADS / 64; ++w) n += lds[w];
    __syncthreads();
    return n;
}
constexpr int COUNT_BLOCKS = 1024;
__global__ __launch_bounds__(256) void distill_count_kernel(const DistillArgs a, uint32_t* __restrict__ counts) {
    __shared__ uint32_t lds[4];
    const uint32_t n = block_sum_u32<256>(count_rows(a, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256), lds);
    if (threadIdx.x == 0) counts[blockIdx.x] = n;
}
// Weight of a row for a kernel that forms the gradient with the value: 1 / labelled rows for the mean, from the partial
// counts of distill_count_kernel, or counted by the only workgroup of the launch.
template <int THREADS>
__device__ __forceinline__ float row_weight(const DistillArgs& a, uint32_t* lds) {
    if (a.reduction != 1 || a.rows == 1) return 1.0f;
    uint32_t n = 0;
    if (a.counts) {
        for (uint32_t i = threadIdx.x; i < a.ncounts; i += THREADS) n += a.counts[i];
    } else {
        n = count_rows(a, threadIdx.x, THREADS);
    }
    n = block_sum_u32<THREADS>(n, lds);
    return 1.0f / (float)(n ? n : 1u);
}
__device__ __forceinline__ void store_loss(const DistillArgs& a, double total, unsigned long long count) {
    const double weight = a.reduction == 1 ? 1.0 / (double)(count ? count : 1) : 1.0;
    a.loss[0] = (float)(total * weight);
    if (a.weight_out) *a.weight_out = (float)weight;
}
// Adds up what the workgroup's threads hold (in a fixed tree): one pair per workgroup, or the result itself when there is
// only one.
template <int THREADS>
__device__ __forceinline__ void store_part(const DistillArgs& a, float total, uint32_t count, float* lds) {
    total = group_sum<64>(total);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) count += __shfl_xor(count, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { lds[2 * (threadIdx.x >> 6)] = total; lds[2 * (threadIdx.x >> 6) + 1] = __uint_as_float(count); }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < THREADS / 64; ++w) { total += lds[2 * w]; count += __float_as_uint(lds[2 * w + 1]); }
    if (gridDim.x == 1) store_loss(a, total, count);
    else a.part[blockIdx.x] = make_float2(total, __uint_as_float(count));
}

// ---- long rows: a wave (G = 64) or a workgroup of G threads to a row
// A row of `n` elements at p as single elements up to the first 16-byte boundary, packs, and single elements behind the
// last pack: [0, head) and [tail, n) are singles.
struct Cut {
    uint32_t head, packs, tail, singles;
    __device__ __forceinline__ uint32_t single(uint32_t e) const { return e < head ? e : tail + (e - head); }
};
template <typename T, int V>
__device__ __forceinline__ Cut cut_row(const T* p, uint32_t n) {
    Cut r;
    if (V == 1) { r.head = 0; r.packs = n; r.tail = n; r.singles = 0; return r; }
    const uint32_t off = (uint32_t)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    r.head = off ? V - off : 0;
    if (r.head > n) r.head = n;
    r.packs = (n - r.head) / V;
    r.tail = r.head + r.packs * V;
    r.singles = n - r.packs * V;
    return r;
}

// LDS of a workgroup of the row kernels: a label per row, the waves' (max, sum), the label's summary
template <int G, int WORKGROUP = (G > 256 ? G : 256)>
struct RowsLds {
    static constexpr int THREADS = WORKGROUP;
    static constexpr int ROWS = THREADS / G;
    int ids[ROWS][DISTILL_MAX_K];
    float ws[ROWS][DISTILL_MAX_K];
    float ms[2 * THREADS / 64];
    Label label;
};
// (max, sum) over the lanes of a row.  Workgroup rows: ONE barrier (the caller keeps another between two uses).
template <int G>
__device__ __forceinline__ void row_soft(float& m, float& s, float c, float* ms) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
        soft_merge(m, s, m2, s2, c);
    }
    if (G == 64) return;
    if ((threadIdx.x & 63) == 0) { ms[2 * (threadIdx.x >> 6)] = m; ms[2 * (threadIdx.x >> 6) + 1] = s; }
    __syncthreads();
    m = ms[0];
    s = ms[1];
#pragma unroll
    for (int w = 1; w < G / 64; ++w) soft_merge(m, s, ms[2 * w], ms[2 * w + 1], c);
}
template <int G>
__device__ __forceinline__ void row_sync() {      // orders the row's stores before and behind this point
    if (G == 64) wave_sync();
    else __syncthreads();
}

constexpr int SOFT_UNROLL = 4;
template <typename T, int V, int G>
__global__ __launch_bounds__(RowsLds<G>::THREADS) void distill_fwd_rows_kernel(const DistillArgs a) {
    __shared__ RowsLds<G> L;
    const int lane = threadIdx.x % G, slot = threadIdx.x / G;
    const bool labeller = G == 64 || threadIdx.x < 64;
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    float total = 0.0f;
    uint32_t count = 0;
    for (size_t row = (size_t)blockIdx.x * RowsLds<G>::ROWS + slot; row < a.rows; row += (size_t)gridDim.x * RowsLds<G>::ROWS) {
        if (!wave_any(a, row)) {                          // (the same answer in every wave of the row: it is not read)
            if (lane == 0) {
                a.stats[row] = make_float2(0.0f, 0.0f);
                if (a.row_loss) a.row_loss[row] = 0.0f;
            }
            continue;
        }
        const T* z = reinterpret_cast<const T*>(a.logits) + row * a.row_stride;
        float m = -__builtin_inff(), s = 0.0f;
        const Cut cut = cut_row<T, V>(z, a.classes);
        for (uint32_t e = lane; e < cut.singles; e += G) {
            const float v = (float)z[cut.single(e)];
            soft_add<1>(m, s, &v, c);
        }
        const Pack<T, V>* zp = reinterpret_cast<const Pack<T, V>*>(z + cut.head);
        for (uint32_t i = lane; i < cut.packs; i += SOFT_UNROLL * G) {      // (a batch of loads, unconditional)
            Pack<T, V> p[SOFT_UNROLL];
#pragma unroll
            for (int u = 0; u < SOFT_UNROLL; ++u) p[u] = zp[i + u * G < cut.packs ? i + u * G : i];
            if (i - lane + SOFT_UNROLL * G <= cut.packs) {                  // (the same for all lanes)
                float v[SOFT_UNROLL * V];
#pragma unroll
                for (int u = 0; u < SOFT_UNROLL; ++u)
#pragma unroll
                    for (int j = 0; j < V; ++j) v[u * V + j] = (float)p[u].v[j];
                soft_add<SOFT_UNROLL * V>(m, s, v, c);
                continue;
            }
#pragma unroll
            for (int u = 0; u < SOFT_UNROLL; ++u) {
                if (i + u * G >= cut.packs) break;
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = (float)p[u].v[j];
                soft_add<V>(m, s, v, c);
            }
        }
        row_soft<G>(m, s, c, L.ms);
        if (labeller) {
            const Label l = wave_label(a, row, c, L.ids[slot], L.ws[slot]);
            float d = label_value(a, row, l, L.ids[slot], L.ws[slot], threadIdx.x & 63, 64, m, s, rt,
                                  [&](int id) { return (float)z[id]; });
            d = group_sum<64>(d) * (a.temperature * a.temperature);
            if (lane == 0) {
                a.stats[row] = make_float2(m, l.broken ? __builtin_nanf("") : 1.0f / s);
                if (a.row_loss) a.row_loss[row] = d;
                total += d;
                ++count;
            }
        }
        if (G > 64) __syncthreads();                      // (L.ms has been read)
    }
    store_part<RowsLds<G>::THREADS>(a, total, count, L.ms);
}

// The listed classes of a row again, from the full-precision value: one lane per class (its first entry).
template <typename T>
__device__ __forceinline__ void patch_row(const DistillArgs& a, const Label& l, const int* ids, const float* ws, const T* z,
                                          T* g, float m, float inv, float f, float c) {
    for (int k = threadIdx.x & 63; k < (int)a.k; k += 64) {
        float w;
        if (class_weight(a, ids, ws, k, w)) g[ids[k]] = (T)(f * (exp2_hw(((float)z[ids[k]] - m) * c) * inv - w * l.inv));
    }
}

template <bool STREAM, typename T, int V, int G>
__global__ __launch_bounds__(RowsLds<G>::THREADS) void distill_bwd_rows_kernel(const DistillArgs a) {
    __shared__ RowsLds<G> L;
    const int lane = threadIdx.x % G, slot = threadIdx.x / G;
    const bool labeller = G == 64 || threadIdx.x < 64;
    const float c = LOG2E / a.temperature;
    const float f_all = a.temperature * (a.weight ? *a.weight : 1.0f);
    for (size_t row = (size_t)blockIdx.x * RowsLds<G>::ROWS + slot; row < a.rows; row += (size_t)gridDim.x * RowsLds<G>::ROWS) {
        const float2 st = a.stats[row];
        const bool any = st.y != 0.0f;
        const T* z = reinterpret_cast<const T*>(a.logits) + row * a.row_stride;
        T* g = reinterpret_cast<T*>(a.grad) + row * a.g_row;
        const float f = f_all * (a.scale ? a.scale[a.reduction == 0 ? row : 0] : 1.0f), fi = f * st.y;
        const Cut cut = cut_row<T, V>(g, a.classes);
        for (uint32_t e = lane; e < cut.singles; e += G) {
            const uint32_t col = cut.single(e);
            g[col] = any ? (T)(exp2_hw(((float)z[col] - st.x) * c) * fi) : (T)0.0f;
        }
        const Pack<T, V>* zp = reinterpret_cast<const Pack<T, V>*>(z + cut.head);
        Pack<T, V>* gp = reinterpret_cast<Pack<T, V>*>(g + cut.head);
        if (!any) {
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) r.v[j] = (T)0.0f;
            for (uint32_t i = lane; i < cut.packs; i += G) gp[i] = r;
            continue;                                     // (the same in every wave of the row)
        }
        for (uint32_t i = lane; i < cut.packs; i += SOFT_UNROLL * G) {      // (a batch of loads, then the stores)
            Pack<T, V> p[SOFT_UNROLL];
#pragma unroll
            for (int u = 0; u < SOFT_UNROLL; ++u) p[u] = zp[i + u * G < cut.packs ? i + u * G : i];
#pragma unroll
            for (int u = 0; u < SOFT_UNROLL; ++u) {
                if (i + u * G >= cut.packs) break;
                Pack<T, V> r;
#pragma unroll
                for (int j = 0; j < V; ++j) r.v[j] = (T)(exp2_hw(((float)p[u].v[j] - st.x) * c) * fi);
                put<STREAM, T, V>(reinterpret_cast<T*>(gp + i + u * G), r);
            }
        }
        row_sync<G>();
        if (labeller) {
            const Label l = wave_label(a, row, c, L.ids[slot], L.ws[slot]);
            patch_row<T>(a, l, L.ids[slot], L.ws[slot], z, g, st.x, st.y, f, c);
            wave_sync();
        }
    }
}

// Value and gradient in one pass: the row stays in the registers of its workgroup (ITEMS packs to a thread) between the
// statistics and the gradient, so the scores are read once and the gradient is written once.
template <bool STREAM, typename T, int V, int G, int ITEMS>
__global__ __launch_bounds__(G) void distill_both_rows_kernel(const DistillArgs a) {
    __shared__ RowsLds<G, G> L;
    const int lane = threadIdx.x;
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    const float f = a.temperature * row_weight<G>(a, reinterpret_cast<uint32_t*>(L.ms));
    float total = 0.0f;
    uint32_t count = 0;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* z = reinterpret_cast<const T*>(a.logits) + row * a.row_stride;
        T* g = reinterpret_cast<T*>(a.grad) + row * a.g_row;
        const Cut cut = cut_row<T, V>(z, a.classes);
        const char* zp = reinterpret_cast<const char*>(z + cut.head);      // (a uniform base and 32-bit offsets: one register
        char* gp = reinterpret_cast<char*>(g + cut.head);                  // per address instead of two)
        if (!wave_any(a, row)) {                          // (the same in every wave: the row is not read)
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) r.v[j] = (T)0.0f;
            for (uint32_t i = lane; i < cut.packs; i += G) *reinterpret_cast<Pack<T, V>*>(gp + i * 16u) = r;
            if (lane < (int)cut.singles) g[cut.single(lane)] = (T)0.0f;
            if (lane == 0 && a.row_loss) a.row_loss[row] = 0.0f;
            continue;
        }
        // (the label first, by the first wave alone: the other waves' loads are on their way meanwhile)
        Label l;
        if (threadIdx.x < 64) l = wave_label(a, row, c, L.ids[0], L.ws[0]);
        words_t p[ITEMS];
        uint32_t at = lane;
        forget(at);                                       // (offsets are formed where they are used rather than kept)
#pragma unroll
        for (int u = 0; u < ITEMS; ++u)                   // (behind the row's last pack: that pack again, not used)
            p[u] = *reinterpret_cast<const words_t*>(zp + (at + u * G < cut.packs ? at + u * G : cut.packs - 1) * 16u);
        const bool has_single = lane < (int)cut.singles;  // (at most 2 V - 2 of them, fewer than a wave)
        const float single = has_single ? (float)z[cut.single(lane)] : 0.0f;
        float m = has_single ? single : -__builtin_inff();
#pragma unroll
        for (int u = 0; u < ITEMS; ++u)
            if ((uint32_t)(lane + u * G) < cut.packs) {
#pragma unroll
                for (int j = 0; j < V; ++j) m = fmaxf(m, word_elem<T>(p[u], j));
            }
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) forget(p[u]);
        const float off = m == -__builtin_inff() ? 0.0f : m;
        float s = has_single ? exp2_hw((single - off) * c) : 0.0f;
#pragma unroll
        for (int u = 0; u < ITEMS; ++u)
            if ((uint32_t)(lane + u * G) < cut.packs) {
#pragma unroll
                for (int j = 0; j < V; ++j) s += exp2_hw((word_elem<T>(p[u], j) - off) * c);
            }
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) forget(p[u]);
        row_soft<G>(m, s, c, L.ms);
        if (threadIdx.x < 64) {
            float d = label_value(a, row, l, L.ids[0], L.ws[0], lane, 64, m, s, rt, [&](int id) { return (float)z[id]; });
            d = group_sum<64>(d) * (a.temperature * a.temperature);
            if (lane == 0) {
                if (a.row_loss) a.row_loss[row] = d;
                total += d;
                ++count;
                L.label = l;
            }
        }
        const float inv = 1.0f / s, fi = f * inv;
        forget(at);
#pragma unroll
        for (int u = 0; u < ITEMS; ++u)
            if (at + u * G < cut.packs) {
                Pack<T, V> r;
#pragma unroll
                for (int j = 0; j < V; ++j) r.v[j] = (T)(exp2_hw((word_elem<T>(p[u], j) - m) * c) * fi);
                put<STREAM, T, V>(reinterpret_cast<T*>(gp + (at + u * G) * 16u), r);
            }
        if (has_single) g[cut.single(lane)] = (T)(exp2_hw((single - m) * c) * fi);
        __syncthreads();
        if (L.label.broken) {                             // (uniform; rare: an index past the classes)
            for (uint32_t i = lane; i < a.classes; i += G) g[i] = (T)__builtin_nanf("");
        } else if (threadIdx.x < 64) {
            patch_row<T>(a, l, L.ids[0], L.ws[0], z, g, m, inv, f, c);
        }
        if (threadIdx.x < 64) wave_sync();
    }
    store_part<G>(a, total, count, L.ms);
}

// ---- short rows, one behind the other, and planes: a workgroup takes `tile` rows at a time through LDS, so that memory is moved
// in whole packs whatever the row length, and planes are turned into rows; 256 / tile lanes work on a row there.
constexpr int TILE_BYTES = 32768, TILE_LABEL_BYTES = 24576, TILE_PACKS = TILE_BYTES / 16 / 256;
constexpr int VALUE = 1, GRADIENT = 2;
__host__ __device__ constexpr size_t tile_lds(size_t tile, size_t pitch, size_t k, size_t bytes) {
    return (tile * pitch * bytes + 15) / 16 * 16 + tile * k * 12;
}
// A tile between memory and LDS, as it lies ...
template <typename T>
__device__ __forceinline__ void tile_in(const T* __restrict__ src, words_t* mem, int elems) {
    const int packs = (int)(elems * sizeof(T) / 16), rest = packs * (16 / (int)sizeof(T));
    if (packs > 0) {                     // (uniform; the loads are unconditional and in flight together)
        words_t in[TILE_PACKS];
#pragma unroll
        for (int u = 0; u < TILE_PACKS; ++u) {
            const int i = u * 256 + threadIdx.x;
            in[u] = reinterpret_cast<const words_t*>(src)[i < packs ? i : packs - 1];
        }
#pragma unroll
        for (int u = 0; u < TILE_PACKS; ++u) {
            const int i = u * 256 + threadIdx.x;
            if (i < packs) mem[i] = in[u];
        }
    }
    if (rest + (int)threadIdx.x < elems) reinterpret_cast<T*>(mem)[rest + threadIdx.x] = src[rest + threadIdx.x];
}
template <typename T>
__device__ __forceinline__ void tile_out(T* __restrict__ dst, const words_t* mem, int elems) {
    const int packs = (int)(elems * sizeof(T) / 16), rest = packs * (16 / (int)sizeof(T));
#pragma unroll
    for (int u = 0; u < TILE_PACKS; ++u) {
        const int i = u * 256 + threadIdx.x;
        if (i < packs) reinterpret_cast<words_t*>(dst)[i] = mem[i];
    }
    if (rest + (int)threadIdx.x < elems) dst[rest + threadIdx.x] = reinterpret_cast<const T*>(mem)[rest + threadIdx.x];
}
// ... and from and to planes: V neighbouring pixels of a class to a thread, spread over the V rows of the tile (`pitch`
// elements apart, an odd number: neighbouring pixels lie in different banks).
template <typename T, int V, int TILE>
__device__ __forceinline__ void planes_in(const T* __restrict__ src, size_t stride, T* rows, int pitch, int n, int classes) {
    constexpr int PARTS = TILE / V, UN = 4;
    for (int i0 = threadIdx.x; i0 < classes * PARTS; i0 += 256 * UN) {
        Pack<T, V> in[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int i = i0 + u * 256, j = i / PARTS, r = i % PARTS * V;      // (unconditional loads: others again)
            in[u] = *reinterpret_cast<const Pack<T, V>*>(src + (size_t)(j < classes ? j : classes - 1) * stride + (r < n ? r : 0));
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int i = i0 + u * 256, j = i / PARTS, r = i % PARTS * V;
            if (j < classes && r < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) rows[(r + v) * pitch + j] = in[u].v[v];
            }
        }
    }
}
template <typename T, int V, int TILE>
__device__ __forceinline__ void planes_out(T* __restrict__ dst, size_t stride, const T* rows, int pitch, int n, int classes) {
    constexpr int PARTS = TILE / V;
    for (int i = threadIdx.x; i < classes * PARTS; i += 256) {
        const int j = i / PARTS, r = i % PARTS * V;
        if (r >= n) continue;
        Pack<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) out.v[v] = rows[(r + v) * pitch + j];
        *reinterpret_cast<Pack<T, V>*>(dst + (size_t)j * stride + r) = out;
    }
}

template <bool PLANES, typename T, int MODE, int LANES>
__global__ __launch_bounds__(256) void distill_tile_kernel(const DistillArgs a) {
    constexpr int tile = 256 / LANES;
    extern __shared__ words_t tile_mem[];
    __shared__ float lds[16];
    T* rows = reinterpret_cast<T*>(tile_mem);
    const int C = (int)a.classes, pitch = PLANES ? C | 1 : C;
    float* ts = reinterpret_cast<float*>(tile_mem + ((size_t)tile * pitch * sizeof(T) + 15) / 16);
    int* ids = reinterpret_cast<int*>(ts + tile * (int)a.k);
    float* ws = reinterpret_cast<float*>(ids + tile * (int)a.k);
    const int K = (int)a.k, r = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    float f_all = a.temperature;
    if (MODE == GRADIENT) f_all *= a.weight ? *a.weight : 1.0f;
    if (MODE == (VALUE | GRADIENT)) f_all *= row_weight<256>(a, reinterpret_cast<uint32_t*>(lds));
    float total = 0.0f;
    uint32_t count = 0;
    T* z = rows + r * pitch;
    int* id = ids + r * K;
    float *t = ts + r * K, *w = ws + r * K;
    for (size_t first = (size_t)blockIdx.x * tile; first < a.rows; first += (size_t)gridDim.x * tile) {
        const int n = a.rows - first < (size_t)tile ? (int)(a.rows - first) : tile;
        constexpr int V = Wide<T>::N <= tile ? Wide<T>::N : 1;
        const bool wide = a.planes_wide && n % V == 0;
        if (!PLANES) tile_in(reinterpret_cast<const T*>(a.logits) + first * C, tile_mem, n * C);
        else if (wide) planes_in<T, V, tile>(reinterpret_cast<const T*>(a.logits) + first, a.class_stride, rows, pitch, n, C);
        else planes_in<T, 1, tile>(reinterpret_cast<const T*>(a.logits) + first, a.class_stride, rows, pitch, n, C);
        // (planes: the labels lie as planes too, neighbouring lanes read neighbouring pixels; rows: the lanes of a row read it)
        if (PLANES) {
#pragma unroll 2
            for (int e = threadIdx.x; e < K * tile; e += 256) {
                const int k = e / tile, er = e % tile;
                if (er >= n) continue;
                long long index;
                const float score = entry_score(a, first + er, k, index);
                ts[er * K + k] = score;
                ids[er * K + k] = entry_class(a, score, index);
            }
        } else if (r < n) {
#pragma unroll 1
            for (int k = lane; k < K; k += LANES) {
                long long index;
                t[k] = entry_score(a, first + r, k, index);
                id[k] = entry_class(a, t[k], index);
            }
        }
        __syncthreads();
        const size_t row = first + r;
        const bool live = r < n;
        // the label (the lanes of a row are neighbours in one wave: no barrier)
        Label l;
        float flags = 0.0f, sum = 0.0f;
        l.top = -__builtin_inff();
        if (live)
            for (int k = lane; k < K; k += LANES) {
                if (id[k] < 0) continue;
                flags = fmaxf(flags, id[k] == ID_BROKEN ? 2.0f : 1.0f);
                l.top = fmaxf(l.top, t[k]);
            }
        flags = group_max<LANES>(flags);
        l.top = group_max<LANES>(l.top);
        l.any = flags > 0.0f;
        l.broken = flags > 1.5f;
        if (live)
            for (int k = lane; k < K; k += LANES) {
                w[k] = id[k] < 0 ? 0.0f : exp2_hw((t[k] - l.top) * c);
                sum += w[k];
            }
        sum = group_sum<LANES>(sum);
        l.inv = 1.0f / sum;
        wave_sync();
        float m = -__builtin_inff(), s = 0.0f, inv = 0.0f;
        if (MODE & VALUE) {
            if (live && l.any) {
                int col = lane;
                for (; col + 7 * LANES < C; col += 8 * LANES) {
                    float v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) v[u] = (float)z[col + u * LANES];
                    soft_add<8>(m, s, v, c);
                }
                for (; col < C; col += LANES) {
                    const float v = (float)z[col];
                    soft_add<1>(m, s, &v, c);
                }
            }
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) {
                const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
                soft_merge(m, s, m2, s2, c);
            }
            inv = l.broken ? __builtin_nanf("") : 1.0f / s;
            float d = 0.0f;
            if (live && l.any) {
                const float more = (log2_hw(l.inv) + log2_hw(s)) * LN2;
                for (int k = lane; k < K; k += LANES) {
                    if (id[k] < 0) continue;
                    if (id[k] == ID_BROKEN) d = __builtin_nanf("");
                    else if (w[k] * l.inv != 0.0f) d += w[k] * l.inv * (((t[k] - l.top) - ((float)z[id[k]] - m)) * rt + more);
                }
            }
            d = group_sum<LANES>(d);
            d *= a.temperature * a.temperature;
            if (live && lane == 0) {
                if (!(MODE & GRADIENT)) a.stats[row] = l.any ? make_float2(m, inv) : make_float2(0.0f, 0.0f);
                if (a.row_loss) a.row_loss[row] = d;
                total += d;
                count += l.any ? 1u : 0u;
            }
        } else if (live) {
            const float2 st = a.stats[row];
            m = st.x;
            inv = st.y;
        }
        if (MODE & GRADIENT) {
            float f = f_all;
            if (MODE == GRADIENT && a.scale && live) f *= a.scale[a.reduction == 0 ? row : 0];
            const float fi = f * inv;
            // (the listed classes' values first, while the scores are still there: they wait in t)
            if (live && l.any)
                for (int k = lane; k < K; k += LANES) {
                    if (id[k] < 0 || id[k] == ID_BROKEN) continue;
                    const int cls = id[k];
                    float q = w[k];
                    int same = 0;
#pragma unroll 4
                    for (int j = 0; j < K; ++j) same += id[j] == cls ? 1 : 0;
                    if (same > 1) {                     // the class is listed more than once: its weights in order
                        q = 0.0f;
                        for (int j = 0; j < K; ++j) q += id[j] == cls ? w[j] : 0.0f;
                    }
                    t[k] = f * (exp2_hw(((float)z[id[k]] - m) * c) * inv - q * l.inv);
                }
            wave_sync();
            if (live)
#pragma unroll 8
                for (int col = lane; col < C; col += LANES) z[col] = l.any ? (T)(exp2_hw(((float)z[col] - m) * c) * fi) : (T)0.0f;
            wave_sync();
            if (live && l.any)      // (entries of the same class hold the same value)
                for (int k = lane; k < K; k += LANES)
                    if (id[k] >= 0 && id[k] != ID_BROKEN) z[id[k]] = (T)t[k];
            __syncthreads();
            if (!PLANES) tile_out(reinterpret_cast<T*>(a.grad) + first * C, tile_mem, n * C);
            else if (wide) planes_out<T, V, tile>(reinterpret_cast<T*>(a.grad) + first, a.g_class, rows, pitch, n, C);
            else planes_out<T, 1, tile>(reinterpret_cast<T*>(a.grad) + first, a.g_class, rows, pitch, n, C);
        }
        __syncthreads();
    }
    if (MODE & VALUE) store_part<256>(a, total, count, lds);
}

// ---- planes, short lists: P neighbouring pixels to a lane, their labels in registers (KR entries each: the class of an entry
// is compared with every class that goes by, which is cheaper than LDS up to 8 entries and leaves the occupancy to the
// loads: P * sizeof(T) bytes per lane and load).
template <int KR>
struct PixelLabel {
    float q[KR];       // weight of the entry's class, at its first entry (0 elsewhere)
    int id[KR];        // its class, or -1
    float qlogq;
    bool any, broken;
};
template <int KR>
__device__ __forceinline__ void pixel_label(const DistillArgs& a, size_t row, float c, float rt, PixelLabel<KR>& l) {
    float t[KR], top = -__builtin_inff(), sum = 0.0f;
    l.any = l.broken = false;
    l.qlogq = 0.0f;
#pragma unroll
    for (int k = 0; k < KR; ++k) {
        const size_t at = k < (int)a.k ? k : a.k - 1;               // (unconditional loads, all in flight)
        const long long id = load_index_flat(a.index, row * a.i_row + at * a.i_entry, a.index_bytes);
        t[k] = load_elem_flat(a.teacher, row * a.t_row + at * a.t_entry, a.teacher_dtype);
        l.id[k] = id >= (long long)a.classes ? 0x7FFFFFFF : id < 0 || k >= (int)a.k ? -1 : (int)id;
    }
#pragma unroll
    for (int k = 0; k < KR; ++k) {
        if (t[k] == -__builtin_inff()) l.id[k] = -1;
        if (l.id[k] < 0) continue;
        l.any = true;
        l.broken |= l.id[k] == 0x7FFFFFFF;
        top = fmaxf(top, t[k]);
    }
#pragma unroll
    for (int k = 0; k < KR; ++k) {
        l.q[k] = l.id[k] < 0 ? 0.0f : exp2_hw((t[k] - top) * c);
        sum += l.q[k];
    }
    const float inv = l.any ? 1.0f / sum : 0.0f, rest = l.any ? log2_hw(inv) * LN2 : 0.0f;
#pragma unroll
    for (int k = 0; k < KR; ++k) {
        l.q[k] *= inv;
        if (l.q[k] != 0.0f) l.qlogq += l.q[k] * ((t[k] - top) * rt + rest);
    }
#pragma unroll
    for (int k = 0; k < KR; ++k)        // the same class again: its weight goes to the first entry
#pragma unroll
        for (int j = k + 1; j < KR; ++j)
            if (l.id[k] >= 0 && l.id[j] == l.id[k]) {
                l.q[k] += l.q[j];
                l.id[j] = -1;
            }
}

constexpr int WIDE_BATCH = 8;
template <typename T, int P>
struct WideBatch {
    Pack<T, P> v[WIDE_BATCH];
    __device__ __forceinline__ void load(const T* __restrict__ z, uint32_t first, uint32_t classes, size_t stride) {
#pragma unroll
        for (int u = 0; u < WIDE_BATCH; ++u) {
            const uint32_t j = first + u < classes ? first + u : classes - 1;
            v[u] = *reinterpret_cast<const Pack<T, P>*>(z + (size_t)j * stride);
        }
    }
};

template <typename T, int P, int KR>
__global__ __launch_bounds__(256) void distill_fwd_wide_kernel(const DistillArgs a) {
    __shared__ float lds[16];
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    float total = 0.0f;
    uint32_t count = 0;
    for (size_t row = ((size_t)blockIdx.x * 256 + threadIdx.x) * P; row < a.rows; row += (size_t)gridDim.x * 256 * P) {
        const T* z = reinterpret_cast<const T*>(a.logits) + row;
        WideBatch<T, P> next;
        next.load(z, 0, a.classes, a.class_stride);
        PixelLabel<KR> l[P];
        bool some = false;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            pixel_label<KR>(a, row + p, c, rt, l[p]);
            some |= l[p].any;
        }
        float m[P], s[P], zk[P][KR];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            m[p] = -__builtin_inff();
            s[p] = 0.0f;
#pragma unroll
            for (int k = 0; k < KR; ++k) zk[p][k] = 0.0f;
        }
        for (uint32_t j = 0; some && j < a.classes; j += WIDE_BATCH) {
            const WideBatch<T, P> b = next;
            if (j + WIDE_BATCH < a.classes) next.load(z, j + WIDE_BATCH, a.classes, a.class_stride);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                float v[WIDE_BATCH], M = m[p];
#pragma unroll
                for (int u = 0; u < WIDE_BATCH; ++u) {
                    v[u] = j + u < a.classes ? (float)b.v[u].v[p] : -__builtin_inff();
                    M = fmaxf(M, v[u]);
#pragma unroll
                    for (int k = 0; k < KR; ++k) zk[p][k] = l[p].id[k] == (int)(j + u) ? v[u] : zk[p][k];
                }
                const float off = M == -__builtin_inff() ? 0.0f : M;
                s[p] *= exp2_hw((m[p] - off) * c);
                m[p] = M;
#pragma unroll
                for (int u = 0; u < WIDE_BATCH; ++u) s[p] += exp2_hw((v[u] - off) * c);
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float d = 0.0f;
            float2 st = make_float2(0.0f, 0.0f);
            if (l[p].any) {
                // sum of q = 1:  sum q (log q - log p) = qlogq - sum q (z - m) / T + log s
                float qz = 0.0f;
#pragma unroll
                for (int k = 0; k < KR; ++k)
                    if (l[p].id[k] >= 0 && l[p].q[k] != 0.0f) qz += l[p].q[k] * (zk[p][k] - m[p]);
                d = (l[p].qlogq - qz * rt + log2_hw(s[p]) * LN2) * (a.temperature * a.temperature);
                if (l[p].broken) d = __builtin_nanf("");
                st = make_float2(m[p], l[p].broken ? __builtin_nanf("") : 1.0f / s[p]);
                ++count;
            }
            a.stats[row + p] = st;
            if (a.row_loss) a.row_loss[row + p] = d;
            total += d;
        }
    }
    store_part<256>(a, total, count, lds);
}

template <bool STREAM, typename T, int P, int KR>
__global__ __launch_bounds__(256) void distill_bwd_wide_kernel(const DistillArgs a) {
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    const float f_all = a.temperature * (a.weight ? *a.weight : 1.0f);
    for (size_t row = ((size_t)blockIdx.x * 256 + threadIdx.x) * P; row < a.rows; row += (size_t)gridDim.x * 256 * P) {
        T* g = reinterpret_cast<T*>(a.grad) + row;
        const T* z = reinterpret_cast<const T*>(a.logits) + row;
        float2 st[P];
        bool some = false;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            st[p] = a.stats[row + p];
            some |= st[p].y != 0.0f;
        }
        if (!some) {
            Pack<T, P> r;
#pragma unroll
            for (int p = 0; p < P; ++p) r.v[p] = (T)0.0f;
            for (uint32_t j = 0; j < a.classes; ++j) *reinterpret_cast<Pack<T, P>*>(g + (size_t)j * a.g_class) = r;
            continue;
        }
        WideBatch<T, P> next;
        next.load(z, 0, a.classes, a.class_stride);
        PixelLabel<KR> l[P];
        float f[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            pixel_label<KR>(a, row + p, c, rt, l[p]);
            f[p] = f_all * (a.scale ? a.scale[a.reduction == 0 ? row + p : 0] : 1.0f);
        }
        for (uint32_t j = 0; j < a.classes; j += WIDE_BATCH) {
            const WideBatch<T, P> b = next;
            if (j + WIDE_BATCH < a.classes) next.load(z, j + WIDE_BATCH, a.classes, a.class_stride);
#pragma unroll
            for (int u = 0; u < WIDE_BATCH; ++u) {
                if (j + u >= a.classes) break;
                Pack<T, P> r;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    float q = 0.0f;
#pragma unroll
                    for (int k = 0; k < KR; ++k) q = l[p].id[k] == (int)(j + u) ? l[p].q[k] : q;
                    const float d = f[p] * (exp2_hw(((float)b.v[u].v[p] - st[p].x) * c) * st[p].y - q);
                    r.v[p] = st[p].y == 0.0f ? (T)0.0f : (T)d;
                }
                put<STREAM, T, P>(g + (size_t)(j + u) * a.g_class, r);
            }
        }
    }
}

// the value from the workgroups' partial sums
__global__ __launch_bounds__(1024) void distill_join_kernel(const DistillArgs a, uint32_t nparts) {
    __shared__ double sums[16];
    __shared__ unsigned long long counts[16];
    double s = 0.0;
    unsigned long long n = 0;
    for (uint32_t i = threadIdx.x; i < nparts; i += 1024) {
        s += (double)a.part[i].x;
        n += __float_as_uint(a.part[i].y);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { s += __shfl_xor(s, o, 64); n += __shfl_xor(n, o, 64); }
    if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = s; counts[threadIdx.x >> 6] = n; }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) { s += sums[w]; n += counts[w]; }
    store_loss(a, s, n);
}

bool planes_layout(size_t row_stride, size_t class_stride) { return class_stride != 1 && row_stride == 1; }

unsigned distill_blocks(size_t rows, int per_block) {
    const size_t need = (rows + per_block - 1) / per_block;
    return (unsigned)(need < DISTILL_BLOCKS ? need : DISTILL_BLOCKS);
}

// Rows of a tile: as many as fit (a power of two, so that a lane count of 256 / tile stays inside a wave), fewer when the
// launch would not fill the chip otherwise.  0: the rows do not lie one behind the other from a 16-byte boundary on, or
// fewer than 8 fit.
int tile_rows(const DistillArgs& a, bool gradient) {
    const bool planes = planes_layout(a.row_stride, a.class_stride);
    const size_t b = e3_elem_bytes(a.dtype), pitch = planes ? a.classes | 1 : a.classes;
    if (!planes) {
        if (a.row_stride != a.classes || (reinterpret_cast<uintptr_t>(a.logits) & 15) != 0) return 0;
        if (gradient && (a.g_row != a.classes || (reinterpret_cast<uintptr_t>(a.grad) & 15) != 0)) return 0;
    }
    size_t t = 256;
    while (t >= 8 && (t * pitch * b > TILE_BYTES || t * a.k * 12 > TILE_LABEL_BYTES)) t >>= 1;
    // All rows in one workgroup where a lane has up to 28 of a row's classes: there is nothing to join (value and gradient of 16 x
    // 64 7.1 us, with two workgroups 9.5; 60 x 100 8.4 and 10.4 us; 128 x 64, 32 classes to a lane, 12.9 and 10.0 us).
    size_t one = 8;
    while (one < a.rows) one <<= 1;
    if (one <= t && a.classes * one <= 256 * 28) return (int)one;
    while (t > 8 && a.rows < t * 512) t >>= 1;
    return t >= 8 ? (int)t : 0;
}
template <bool PLANES, typename T, int MODE>
int distill_tile_launch(const DistillArgs& a, int tile, unsigned blocks, hipStream_t s) {
    const size_t lds = tile_lds(tile, PLANES ? a.classes | 1 : a.classes, a.k, sizeof(T));
    if (tile == 256) distill_tile_kernel<PLANES, T, MODE, 1><<<dim3(blocks), dim3(256), lds, s>>>(a);
    else if (tile == 128) distill_tile_kernel<PLANES, T, MODE, 2><<<dim3(blocks), dim3(256), lds, s>>>(a);
    else if (tile == 64) distill_tile_kernel<PLANES, T, MODE, 4><<<dim3(blocks), dim3(256), lds, s>>>(a);
    else if (tile == 32) distill_tile_kernel<PLANES, T, MODE, 8><<<dim3(blocks), dim3(256), lds, s>>>(a);
    else if (tile == 16) distill_tile_kernel<PLANES, T, MODE, 16><<<dim3(blocks), dim3(256), lds, s>>>(a);
    else distill_tile_kernel<PLANES, T, MODE, 32><<<dim3(blocks), dim3(256), lds, s>>>(a);
    LAUNCH_OK("distill_tile_kernel");
    return 0;
}
// whether n neighbouring pixels of every plane can be moved at once
template <typename T>
bool planes_wide(const void* p, size_t stride, size_t rows, size_t n) {
    return rows % n == 0 && stride % n == 0 && (reinterpret_cast<uintptr_t>(p) & (n * sizeof(T) - 1)) == 0;
}
template <typename T, int MODE>
int distill_tile(DistillArgs a, int tile, unsigned& blocks, hipStream_t s) {
    blocks = distill_blocks(a.rows, tile);
    if (!planes_layout(a.row_stride, a.class_stride)) return distill_tile_launch<false, T, MODE>(a, tile, blocks, s);
    constexpr size_t V = Wide<T>::N;
    a.planes_wide = planes_wide<T>(a.logits, a.class_stride, V, V) && (!(MODE & GRADIENT) || planes_wide<T>(a.grad, a.g_class, V, V));
    return distill_tile_launch<true, T, MODE>(a, tile, blocks, s);
}

template <typename T, int V, int G>
int distill_rows_launch(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
    blocks = distill_blocks(a.rows, RowsLds<G>::ROWS);
    const dim3 threads(RowsLds<G>::THREADS);
    if (!backward) {
        if constexpr (V > 1) distill_fwd_rows_kernel<T, V, G><<<dim3(blocks), threads, 0, s>>>(a);      // (rows_wide)
    } else if (V > 1 && a.rows * a.classes * sizeof(T) > E3_STREAM_BYTES) distill_bwd_rows_kernel<(V > 1), T, V, G><<<dim3(blocks), threads, 0, s>>>(a);
    else distill_bwd_rows_kernel<false, T, V, G><<<dim3(blocks), threads, 0, s>>>(a);
    LAUNCH_OK("distill_rows_kernel");
    return 0;
}
// Lanes of a long row: a wave for as long as the rows fill the chip that way (every workgroup of a row waits for the slowest
// wave and for the label: value of 25061 x 2653 fp16 95 us with 256 threads to a row, 54 with a wave; 10000 x 9000 bf16 53 and
// 44 us, its gradient 61 and 64), 256 threads beyond, 1024 threads for the gradient of long rows and where there are fewer rows
// than CUs (value of 4096 x 32000 bf16 118 us with 1024 threads, 54 with 256; of 100 x 128000 15 and 18 us; gradient of
// 2000 x 128000 186 and 207 us).
template <typename T, int V>
int distill_rows(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
    const size_t bytes = a.classes * sizeof(T);
    if (a.classes <= 2048 || (a.rows >= 1024 && bytes <= (backward ? 16384 : 32768))) return distill_rows_launch<T, V, 64>(a, backward, blocks, s);
    if (a.classes <= 16384 || (!backward && a.rows >= 256)) return distill_rows_launch<T, V, 256>(a, backward, blocks, s);
    return distill_rows_launch<T, V, 1024>(a, backward, blocks, s);
}

// Packs need the scores and their gradient to lie the same way to a 16-byte boundary in every row.
template <typename T>
bool rows_wide(const DistillArgs& a, bool gradient) {
    if (!gradient) return true;
    return ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0 &&
           (a.row_stride * sizeof(T)) % 16 == (a.g_row * sizeof(T)) % 16;
}

template <typename T>
bool grad_streams(const DistillArgs& a) { return a.rows * a.classes * sizeof(T) > E3_STREAM_BYTES; }

// pixels per lane: 4 for the gradient; 2 for the value, whose registers (the scores of the label's entries) would leave two
// waves to a SIMD with 4 (64 fp32 planes of 1920 x 1080: 173 us with 4, 157 us with 2); 1 where the planes do not lie on
// such boundaries
template <typename T, int P, int KR>
int distill_wide_fwd(const DistillArgs& a, unsigned& blocks, hipStream_t s) {
    blocks = distill_blocks(a.rows, 256 * P);
    distill_fwd_wide_kernel<T, P, KR><<<dim3(blocks), dim3(256), 0, s>>>(a);
    LAUNCH_OK("distill_fwd_wide_kernel");
    return 0;
}
template <typename T, int P, int KR>
int distill_wide_bwd(const DistillArgs& a, hipStream_t s) {
    if (P > 1 && grad_streams<T>(a)) distill_bwd_wide_kernel<(P > 1), T, P, KR><<<dim3(distill_blocks(a.rows, 256 * P)), dim3(256), 0, s>>>(a);
    else distill_bwd_wide_kernel<false, T, P, KR><<<dim3(distill_blocks(a.rows, 256 * P)), dim3(256), 0, s>>>(a);
    LAUNCH_OK("distill_bwd_wide_kernel");
    return 0;
}
// Planes go pixel by pixel (labels in registers, several pixels to a lane) where the list is short and there are enough pixels
// to fill the chip that way; through tiles otherwise.  Value and gradient, by pixel / by tiles: 16384 x 200 fp32 84 / 24 us,
// 65536 x 200 bf16 84 / 36 us, 262144 x 20 fp32 37 / 37 us, 262144 x 200 bf16 98 / 118 us, 2073600 x 64 fp32 359 / 419 us.
constexpr size_t PIXELS = 262144;
bool planes_by_pixel(const DistillArgs& a) { return a.k <= 8 && a.rows >= PIXELS; }

template <typename T>
int distill_t(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
    if (planes_layout(a.row_stride, a.class_stride) && planes_by_pixel(a)) {
        if (!backward) {
            if (planes_wide<T>(a.logits, a.class_stride, a.rows, 2))
                return a.k <= 4 ? distill_wide_fwd<T, 2, 4>(a, blocks, s) : distill_wide_fwd<T, 2, 8>(a, blocks, s);
            return a.k <= 4 ? distill_wide_fwd<T, 1, 4>(a, blocks, s) : distill_wide_fwd<T, 1, 8>(a, blocks, s);
        }
        if (planes_wide<T>(a.logits, a.class_stride, a.rows, 4) && planes_wide<T>(a.grad, a.g_class, a.rows, 4))
            return a.k <= 4 ? distill_wide_bwd<T, 4, 4>(a, s) : distill_wide_bwd<T, 4, 8>(a, s);
        return a.k <= 4 ? distill_wide_bwd<T, 1, 4>(a, s) : distill_wide_bwd<T, 1, 8>(a, s);
    }
    if (const int tile = tile_rows(a, backward))
        return backward ? distill_tile<T, GRADIENT>(a, tile, blocks, s) : distill_tile<T, VALUE>(a, tile, blocks, s);
    return rows_wide<T>(a, backward) ? distill_rows<T, Wide<T>::N>(a, backward, blocks, s) : distill_rows<T, 1>(a, backward, blocks, s);
}
int distill_any(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
    if (a.dtype == E3_F32) return distill_t<float>(a, backward, blocks, s);
    if (a.dtype == E3_F16) return distill_t<f16_t>(a, backward, blocks, s);
    return distill_t<bf16_t>(a, backward, blocks, s);
}

// Value and gradient in one pass over the scores.  blocks = 0: no such kernel for these (the caller runs both passes): planes
// pixel by pixel, rows too long for the registers of a workgroup, short rows that do not lie one behind the other.
template <typename T>
int distill_both_t(DistillArgs a, uint32_t* counts, unsigned& blocks, hipStream_t s) {
    constexpr int V = Wide<T>::N;
    blocks = 0;
    if (planes_layout(a.row_stride, a.class_stride) && planes_by_pixel(a)) return 0;
    const int tile = tile_rows(a, true);
    const size_t packs = a.classes / V;
    if (!tile && (a.classes * sizeof(T) <= 4096 || packs > 16384 || !rows_wide<T>(a, true))) return 0;
    blocks = distill_blocks(a.rows, tile ? tile : 1);
    // a wave to a row of up to 16 KB where the rows fill the chip that way (50000 x 2500 bf16: with 256 threads 293 us)
    const bool wave_rows = !tile && a.rows >= 1024 && packs <= 1024;
    if (a.reduction == 1 && blocks > 1 && (wave_rows || a.rows * a.k > 4096)) {      // (fewer are counted by every workgroup for itself)
        const size_t need = (a.rows * (a.i_entry == 1 ? a.k : 1) + 255) / 256;
        a.counts = counts;
        a.ncounts = (uint32_t)(need < COUNT_BLOCKS ? need : COUNT_BLOCKS);
        distill_count_kernel<<<dim3(a.ncounts), dim3(256), 0, s>>>(a, counts);
        LAUNCH_OK("distill_count_kernel");
    }
    if (tile) return distill_tile<T, VALUE | GRADIENT>(a, tile, blocks, s);
#define E3_BOTH(G, ITEMS)                                                                                          \
    if (grad_streams<T>(a)) distill_both_rows_kernel<true, T, V, G, ITEMS><<<dim3(blocks), dim3(G), 0, s>>>(a);    \
    else distill_both_rows_kernel<false, T, V, G, ITEMS><<<dim3(blocks), dim3(G), 0, s>>>(a)
    if (wave_rows && packs <= 512) { E3_BOTH(64, 8); }
    else if (wave_rows) { E3_BOTH(64, 16); }
    else if (packs <= 1024) { E3_BOTH(256, 4); }
    else if (packs <= 2048) { E3_BOTH(256, 8); }
    else if (packs <= 4096) { E3_BOTH(256, 16); }
    else if (packs <= 8192) { E3_BOTH(1024, 8); }
    else { E3_BOTH(1024, 16); }
#undef E3_BOTH
    LAUNCH_OK("distill_both_rows_kernel");
    return 0;
}
int distill_both(const DistillArgs& a, uint32_t* counts, unsigned& blocks, hipStream_t s) {
    if (a.dtype == E3_F32) return distill_both_t<float>(a, counts, blocks, s);
    if (a.dtype == E3_F16) return distill_both_t<f16_t>(a, counts, blocks, s);
    return distill_both_t<bf16_t>(a, counts, blocks, s);
}
DistillArgs distill_args(size_t rows, size_t classes, size_t k, const void* logits, size_t row_stride, size_t class_stride,
                         int dtype, const void* teacher, size_t t_row, size_t t_entry, int teacher_dtype, const void* index,
                         size_t i_row, size_t i_entry, int index_bytes, float temperature, int reduction) {
    DistillArgs a{};
    a.rows = rows; a.classes = (uint32_t)classes; a.k = k; a.logits = logits; a.row_stride = row_stride;
    a.class_stride = class_stride; a.dtype = dtype; a.teacher = teacher; a.t_row = t_row; a.t_entry = t_entry;
    a.teacher_dtype = teacher_dtype; a.index = index; a.i_row = i_row; a.i_entry = i_entry; a.index_bytes = index_bytes;
    a.temperature = temperature; a.reduction = reduction;
    return a;
}
}  // namespace

bool e3_distill_layout_ok(size_t rows, size_t classes, size_t k, size_t row_stride, size_t class_stride) {
    if (class_stride == 1 || rows == 1) return class_stride == 1;
    return row_stride == 1 && classes <= (size_t)DISTILL_PLANES && k <= (size_t)DISTILL_PLANES;
}
size_t e3_distill_scratch_bytes(size_t rows) {
    (void)rows;
    return DISTILL_BLOCKS * sizeof(float2) + COUNT_BLOCKS * sizeof(uint32_t) + 256;
}

int e3_distill_forward_impl(size_t rows, size_t classes, size_t k, const void* logits, size_t row_stride,
                            size_t class_stride, int dtype, const void* teacher, size_t t_row, size_t t_entry,
                            int teacher_dtype, const void* index, size_t i_row, size_t i_entry, int index_bytes,
                            float temperature, int reduction, float* stats, float* row_loss, float* loss, void* grad,
                            size_t g_row, size_t g_class, char* scratch, hipStream_t s) {
    DistillArgs a = distill_args(rows, classes, k, logits, row_stride, class_stride, dtype, teacher, t_row, t_entry,
                                 teacher_dtype, index, i_row, i_entry, index_bytes, temperature, reduction);
    a.stats = reinterpret_cast<float2*>(stats);
    a.row_loss = row_loss;
    a.loss = loss;
    a.weight_out = rows > 0 ? stats + 2 * rows : nullptr;
    a.part = reinterpret_cast<float2*>(scratch);
    uint32_t* counts = reinterpret_cast<uint32_t*>(a.part + DISTILL_BLOCKS);
    unsigned blocks = 0;
    int rc = 0;
    if (grad) {
        a.grad = grad;
        a.g_row = g_row;
        a.g_class = g_class;
        if (rows > 0) rc = distill_both(a, counts, blocks, s);
        if (rc) return rc;
    }
    const bool both = blocks > 0;
    if (!both && rows > 0) rc = distill_any(a, false, blocks, s);
    if (rc) return rc;
    if (blocks != 1) {
        distill_join_kernel<<<dim3(1), dim3(1024), 0, s>>>(a, blocks);
        LAUNCH_OK("distill_join_kernel");
    }
    if (!grad || both || rows == 0) return 0;
    a.weight = a.weight_out;
    return distill_any(a, true, blocks, s);
}

int e3_distill_backward_impl(size_t rows, size_t classes, size_t k, const void* logits, size_t row_stride,
                             size_t class_stride, int dtype, const void* teacher, size_t t_row, size_t t_entry,
                             int teacher_dtype, const void* index, size_t i_row, size_t i_entry, int index_bytes,
                             float temperature, int reduction, const float* stats, const float* d_loss, void* grad, size_t g_row, size_t g_class, hipStream_t s) {
    if (rows == 0) return 0;
    DistillArgs a = distill_args(rows, classes, k, logits, row_stride, class_stride, dtype, teacher, t_row, t_entry,
                                 teacher_dtype, index, i_row, i_entry, index_bytes, temperature, reduction);
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    a.weight = stats + 2 * rows;
    a.scale = d_loss;
    a.grad = grad;
    a.g_row = g_row;
    a.g_class = g_class;
    unsigned blocks = 0;
    return distill_any(a, true, blocks, s);
}
