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
// Two layouts: rows of classes (class stride 1; a workgroup or a group of lanes takes a row) and planes of classes (row
// stride 1, as the rasteriser lays an image out; a lane takes a pixel and walks over the planes).
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
constexpr int DISTILL_PLANES = 256;              // classes of the plane layout: one label column per pixel in LDS
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


// ---- the label of a row, worked out by a group of lanes (lane, G): entries lane, lane + G, ...
struct Label {
    float top, inv;          // largest listed score; 1 / sum of exp2((t - top) c)
    bool any, broken;
};
__device__ __forceinline__ float entry_score(const DistillArgs& a, size_t row, size_t k, long long& id) {
    id = load_index(a.index, row * a.i_row + k * a.i_entry, a.index_bytes);
    return id < 0 ? -__builtin_inff() : load_elem(a.teacher, row * a.t_row + k * a.t_entry, a.teacher_dtype);
}
// reductions over the lanes of a row: a group of one wave, or the whole workgroup (G > 64)
template <int G>
struct Lanes {
    static constexpr int THREADS = G > 256 ? G : 256;
    static constexpr int ROWS = THREADS / G;
    static constexpr int WAVES = G > 64 ? G / 64 : 1;
    static __device__ __forceinline__ float sum(float v, float* lds) {
        v = group_sum<(G < 64 ? G : 64)>(v);
        if (G <= 64) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += lds[w];
        return v;
    }
    static __device__ __forceinline__ float max(float v, float* lds) {
        v = group_max<(G < 64 ? G : 64)>(v);
        if (G <= 64) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v = fmaxf(v, lds[w]);
        return v;
    }
    static __device__ __forceinline__ void soft(float& m, float& s, float c, float* lds) {
#pragma unroll
        for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) {
            const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
            soft_merge(m, s, m2, s2, c);
        }
        if (G <= 64) return;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { lds[2 * (threadIdx.x >> 6)] = m; lds[2 * (threadIdx.x >> 6) + 1] = s; }
        __syncthreads();
        m = lds[0];
        s = lds[1];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) soft_merge(m, s, lds[2 * w], lds[2 * w + 1], c);
    }
    // what a lane stored before is seen by the row's lanes behind this point, and stores behind it land later
    static __device__ __forceinline__ void sync() {
        if (G <= 64) wave_sync();
        else __syncthreads();
    }
};

template <int G>
__device__ __forceinline__ Label row_label(const DistillArgs& a, size_t row, bool live, int lane, float c, float* lds) {
    Label l;
    float top = -__builtin_inff(), sum = 0.0f, flags = 0.0f;          // flags: 1 a listed entry, 2 a broken one
    if (live)
        for (size_t k = lane; k < a.k; k += G) {
            long long id;
            const float t = entry_score(a, row, k, id);
            if (t == -__builtin_inff()) continue;
            flags = fmaxf(flags, id >= (long long)a.classes ? 2.0f : 1.0f);
            top = fmaxf(top, t);                                        // (a NaN score makes the sum NaN)
        }
    flags = Lanes<G>::max(flags, lds);
    top = Lanes<G>::max(top, lds);
    l.any = flags > 0.0f;
    l.broken = flags > 1.5f;
    if (live && l.any)
        for (size_t k = lane; k < a.k; k += G) {
            long long id;
            const float t = entry_score(a, row, k, id);
            if (t != -__builtin_inff()) sum += exp2_hw((t - top) * c);
        }
    sum = Lanes<G>::sum(sum, lds);
    l.top = top;
    l.inv = 1.0f / sum;
    return l;
}

// A row of `n` elements at p as single elements up to the first 16-byte boundary, packs, and single elements behind the
// last pack: [0, head) and [tail, n) are singles.
struct Cut {
    uint32_t head, packs, tail;
};
template <typename T, int V>
__device__ __forceinline__ Cut cut_row(const T* p, uint32_t n) {
    Cut r;
    if (V == 1) { r.head = 0; r.packs = n; r.tail = n; return r; }
    const uint32_t off = (uint32_t)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    r.head = off ? V - off : 0;
    if (r.head > n) r.head = n;
    r.packs = (n - r.head) / V;
    r.tail = r.head + r.packs * V;
    return r;
}

// Sum of a value over the workgroup's rows (lane 0 of each group holds one), one pair per workgroup.
template <int ROWS, int G>
__device__ __forceinline__ void store_part(float total, uint32_t count, float2* part, float* lds) {
    __syncthreads();
    if (threadIdx.x % G == 0) { lds[2 * (threadIdx.x / G)] = total; lds[2 * (threadIdx.x / G) + 1] = __uint_as_float(count); }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int r = 1; r < ROWS; ++r) { total += lds[2 * r]; count += __float_as_uint(lds[2 * r + 1]); }
        part[blockIdx.x] = make_float2(total, __uint_as_float(count));
    }
}

constexpr int SOFT_UNROLL = 4;
template <typename T, int V, int G>
__global__ __launch_bounds__(Lanes<G>::THREADS) void distill_fwd_rows_kernel(const DistillArgs a) {
    using L = Lanes<G>;
    __shared__ float lds[64];
    const int lane = threadIdx.x % G;
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    float total = 0.0f;
    uint32_t count = 0;
    for (size_t base = (size_t)blockIdx.x * L::ROWS; base < a.rows; base += (size_t)gridDim.x * L::ROWS) {
        const size_t row = base + threadIdx.x / G;
        const bool live = row < a.rows;
        const Label l = row_label<G>(a, row, live, lane, c, lds);
        const T* z = reinterpret_cast<const T*>(a.logits) + row * a.row_stride;
        float m = -__builtin_inff(), s = 0.0f;
        if (live && l.any) {                             // (a row without a label is not read)
            const Cut cut = cut_row<T, V>(z, a.classes);
            if (V > 1) {
                const uint32_t singles = cut.head + (a.classes - cut.tail);
                for (uint32_t e = lane; e < singles; e += G) {
                    const float v = (float)z[e < cut.head ? e : cut.tail + (e - cut.head)];
                    soft_add<1>(m, s, &v, c);
                }
            }
            const Pack<T, V>* zp = reinterpret_cast<const Pack<T, V>*>(z + cut.head);
            uint32_t i = lane;
            for (; i + (SOFT_UNROLL - 1) * G < cut.packs; i += SOFT_UNROLL * G) {
                Pack<T, V> p[SOFT_UNROLL];
#pragma unroll
                for (int u = 0; u < SOFT_UNROLL; ++u) p[u] = zp[i + u * G];
                float v[SOFT_UNROLL * V];
#pragma unroll
                for (int u = 0; u < SOFT_UNROLL; ++u)
#pragma unroll
                    for (int j = 0; j < V; ++j) v[u * V + j] = (float)p[u].v[j];
                soft_add<SOFT_UNROLL * V>(m, s, v, c);
            }
            for (; i < cut.packs; i += G) {
                const Pack<T, V> p = zp[i];
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = (float)p.v[j];
                soft_add<V>(m, s, v, c);
            }
        }
        L::soft(m, s, c, lds);
        // sum of q (log q - log p) over the entries: log q = (t - top) / T + log inv,  log p = (z - m) / T - log s
        float d = 0.0f;
        if (live && l.any) {
            const float rest = (log2_hw(l.inv) + log2_hw(s)) * LN2;
            for (size_t k = lane; k < a.k; k += G) {
                long long id;
                const float t = entry_score(a, row, k, id);
                if (t == -__builtin_inff()) continue;
                const float q = exp2_hw((t - l.top) * c) * l.inv;
                if (id >= (long long)a.classes) d = __builtin_nanf("");
                else if (q != 0.0f) d += q * (((t - l.top) - ((float)z[id] - m)) * rt + rest);
            }
        }
        d = L::sum(d, lds) * (a.temperature * a.temperature);
        if (!live || lane != 0) continue;
        a.stats[row] = l.any ? make_float2(m, l.broken ? __builtin_nanf("") : 1.0f / s) : make_float2(0.0f, 0.0f);
        if (a.row_loss) a.row_loss[row] = d;
        total += d;
        count += l.any ? 1u : 0u;
    }
    store_part<L::ROWS, G>(total, count, a.part, lds);
}

template <typename T, int V, int G>
__global__ __launch_bounds__(Lanes<G>::THREADS) void distill_bwd_rows_kernel(const DistillArgs a) {
    using L = Lanes<G>;
    __shared__ float lds[64];
    const int lane = threadIdx.x % G;
    const float c = LOG2E / a.temperature;
    const float f_all = a.temperature * (a.weight ? *a.weight : 1.0f);
    for (size_t base = (size_t)blockIdx.x * L::ROWS; base < a.rows; base += (size_t)gridDim.x * L::ROWS) {
        const size_t row = base + threadIdx.x / G;
        const bool live = row < a.rows;
        const float2 st = live ? a.stats[row] : make_float2(0.0f, 0.0f);
        const bool any = st.y != 0.0f;
        const T* z = reinterpret_cast<const T*>(a.logits) + row * a.row_stride;
        T* g = reinterpret_cast<T*>(a.grad) + row * a.g_row;
        const float f = f_all * (a.scale ? a.scale[a.reduction == 0 && live ? row : 0] : 1.0f), fi = f * st.y;
        if (live) {
            const Cut cut = cut_row<T, V>(g, a.classes);
            if (V > 1) {
                const uint32_t singles = cut.head + (a.classes - cut.tail);
                for (uint32_t e = lane; e < singles; e += G) {
                    const uint32_t col = e < cut.head ? e : cut.tail + (e - cut.head);
                    g[col] = any ? (T)(exp2_hw(((float)z[col] - st.x) * c) * fi) : (T)0.0f;
                }
            }
            const Pack<T, V>* zp = reinterpret_cast<const Pack<T, V>*>(z + cut.head);
            Pack<T, V>* gp = reinterpret_cast<Pack<T, V>*>(g + cut.head);
            if (any) {
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
                        gp[i + u * G] = r;
                    }
                }
            } else {
                Pack<T, V> r;
#pragma unroll
                for (int j = 0; j < V; ++j) r.v[j] = (T)0.0f;
                for (uint32_t i = lane; i < cut.packs; i += G) gp[i] = r;
            }
        }
        // the listed classes again, from the full-precision value: one lane per class (its first entry)
        const Label l = row_label<G>(a, row, live && any, lane, c, lds);
        L::sync();
        if (live && any)
            for (size_t k = lane; k < a.k; k += G) {
                long long id, other;
                float t = entry_score(a, row, k, id);
                if (t == -__builtin_inff() || id >= (long long)a.classes) continue;
                float q = 0.0f;
                bool first = true;
                for (size_t j = 0; j < a.k; ++j) {
                    t = entry_score(a, row, j, other);
                    if (other != id || t == -__builtin_inff()) continue;
                    if (j < k) first = false;
                    q += exp2_hw((t - l.top) * c) * l.inv;
                }
                if (first) g[id] = (T)(f * (exp2_hw(((float)z[id] - st.x) * c) * st.y - q));
            }
        L::sync();
    }
}

// ---- planes: a lane takes a pixel; its label is a column of `classes` weights in LDS (only its own lane touches it)
struct PlaneLabel {
    float top, inv, qlogq;
    bool any, broken;
};
// Adds the weights of a pixel's label to its column.
__device__ __forceinline__ PlaneLabel plane_label(const DistillArgs& a, size_t row, float c, float rt, float* col) {
    PlaneLabel l;
    float top = -__builtin_inff(), sum = 0.0f;
    l.any = l.broken = false;
    for (size_t k = 0; k < a.k; ++k) {
        long long id;
        const float t = entry_score(a, row, k, id);
        if (t == -__builtin_inff()) continue;
        l.any = true;
        l.broken |= id >= (long long)a.classes;
        top = fmaxf(top, t);
    }
    l.top = top;
    l.inv = l.qlogq = 0.0f;
    if (!l.any) return l;
    for (size_t k = 0; k < a.k; ++k) {
        long long id;
        const float t = entry_score(a, row, k, id);
        if (t != -__builtin_inff()) sum += exp2_hw((t - top) * c);
    }
    l.inv = 1.0f / sum;
    const float rest = log2_hw(l.inv) * LN2;
    for (size_t k = 0; k < a.k; ++k) {
        long long id;
        const float t = entry_score(a, row, k, id);
        if (t == -__builtin_inff() || id >= (long long)a.classes) continue;
        const float q = exp2_hw((t - top) * c) * l.inv;
        if (q != 0.0f) l.qlogq += q * ((t - top) * rt + rest);
        col[(size_t)id * 64] += q;
    }
    return l;
}
__device__ __forceinline__ void plane_clear(const DistillArgs& a, size_t row, float* col) {
    for (size_t k = 0; k < a.k; ++k) {
        const long long id = load_index(a.index, row * a.i_row + k * a.i_entry, a.index_bytes);
        if (id >= 0 && id < (long long)a.classes) col[(size_t)id * 64] = 0.0f;
    }
}

// The planes go by in batches: the loads of the next batch are in flight while one is worked on (a lane's label takes
// 4 bytes of LDS per class, so that few waves fit a CU and each has to keep many loads in flight).
constexpr int PLANE_BATCH = 16;
template <typename T>
struct PlaneBatch {
    T v[PLANE_BATCH];
    __device__ __forceinline__ void load(const T* __restrict__ z, uint32_t first, uint32_t classes, size_t stride) {
#pragma unroll
        for (int u = 0; u < PLANE_BATCH; ++u) {          // (the last plane again behind the last one: never used)
            const uint32_t j = first + u < classes ? first + u : classes - 1;
            v[u] = z[(size_t)j * stride];
        }
    }
};

template <typename T>
__global__ __launch_bounds__(64) void distill_fwd_planes_kernel(const DistillArgs a) {
    extern __shared__ float cols[];
    const int lane = threadIdx.x;
    float* col = cols + lane;
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    for (uint32_t j = 0; j < a.classes; ++j) col[j * 64] = 0.0f;
    float total = 0.0f;
    uint32_t count = 0;
    for (size_t row = (size_t)blockIdx.x * 64 + lane; row < a.rows; row += (size_t)gridDim.x * 64) {
        const T* z = reinterpret_cast<const T*>(a.logits) + row;
        PlaneBatch<T> next;
        next.load(z, 0, a.classes, a.class_stride);
        const PlaneLabel l = plane_label(a, row, c, rt, col);
        if (!l.any) {
            a.stats[row] = make_float2(0.0f, 0.0f);
            if (a.row_loss) a.row_loss[row] = 0.0f;
            continue;
        }
        float m = -__builtin_inff(), s = 0.0f;
        float qz = 0.0f, qs = 0.0f;              // sum of q (z - m) and of q over the classes so far
        for (uint32_t j = 0; j < a.classes; j += PLANE_BATCH) {
            const PlaneBatch<T> b = next;
            if (j + PLANE_BATCH < a.classes) next.load(z, j + PLANE_BATCH, a.classes, a.class_stride);
            float v[PLANE_BATCH], M = m;
#pragma unroll
            for (int u = 0; u < PLANE_BATCH; ++u) {
                v[u] = j + u < a.classes ? (float)b.v[u] : -__builtin_inff();
                M = fmaxf(M, v[u]);
            }
            if (M != m) {
                s *= exp2_hw((m - M) * c);
                if (qs != 0.0f) qz += qs * (m - M);
                m = M;
            }
            const float off = M == -__builtin_inff() ? 0.0f : M;
#pragma unroll
            for (int u = 0; u < PLANE_BATCH; ++u) {
                const float d = v[u] - off, q = j + u < a.classes ? col[(j + u) * 64] : 0.0f;
                s += exp2_hw(d * c);
                qz += q != 0.0f ? q * d : 0.0f;              // (a class that is switched off has d = -inf)
                qs += q;
            }
        }
        // sum of q = 1:  sum q (log q - log p) = qlogq - sum q (z - m) / T + log s
        float d = l.qlogq - qz * rt + log2_hw(s) * LN2;
        if (l.broken) d = __builtin_nanf("");
        d *= a.temperature * a.temperature;
        a.stats[row] = make_float2(m, l.broken ? __builtin_nanf("") : 1.0f / s);
        if (a.row_loss) a.row_loss[row] = d;
        total += d;
        ++count;
        plane_clear(a, row, col);
    }
    total = group_sum<64>(total);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) count += __shfl_xor(count, o, 64);
    if (lane == 0) a.part[blockIdx.x] = make_float2(total, __uint_as_float(count));
}

template <typename T>
__global__ __launch_bounds__(64) void distill_bwd_planes_kernel(const DistillArgs a) {
    extern __shared__ float cols[];
    const int lane = threadIdx.x;
    float* col = cols + lane;
    const float rt = 1.0f / a.temperature, c = LOG2E * rt;
    const float f_all = a.temperature * (a.weight ? *a.weight : 1.0f);
    for (uint32_t j = 0; j < a.classes; ++j) col[j * 64] = 0.0f;
    for (size_t row = (size_t)blockIdx.x * 64 + lane; row < a.rows; row += (size_t)gridDim.x * 64) {
        const float2 st = a.stats[row];
        T* g = reinterpret_cast<T*>(a.grad) + row;
        if (st.y == 0.0f) {
            for (uint32_t j = 0; j < a.classes; ++j) g[(size_t)j * a.g_class] = (T)0.0f;
            continue;
        }
        const T* z = reinterpret_cast<const T*>(a.logits) + row;
        PlaneBatch<T> next;
        next.load(z, 0, a.classes, a.class_stride);
        const float f = f_all * (a.scale ? a.scale[a.reduction == 0 ? row : 0] : 1.0f);
        plane_label(a, row, c, rt, col);
        for (uint32_t j = 0; j < a.classes; j += PLANE_BATCH) {
            const PlaneBatch<T> b = next;
            if (j + PLANE_BATCH < a.classes) next.load(z, j + PLANE_BATCH, a.classes, a.class_stride);
#pragma unroll
            for (int u = 0; u < PLANE_BATCH; ++u)
                if (j + u < a.classes)
                    g[(size_t)(j + u) * a.g_class] = (T)(f * (exp2_hw(((float)b.v[u] - st.x) * c) * st.y - col[(j + u) * 64]));
        }
        plane_clear(a, row, col);
    }
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
        const long long id = load_index(a.index, row * a.i_row + at * a.i_entry, a.index_bytes);
        t[k] = load_elem(a.teacher, row * a.t_row + at * a.t_entry, a.teacher_dtype);
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
    total = group_sum<64>(total);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) count += __shfl_xor(count, o, 64);
    store_part<4, 64>(total, count, a.part, lds);
}

template <typename T, int P, int KR>
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
                *reinterpret_cast<Pack<T, P>*>(g + (size_t)(j + u) * a.g_class) = r;
            }
        }
    }
}

// loss[0] = sum of the partial sums (over the labelled rows for the mean), loss[1] = the weight of a row
__global__ __launch_bounds__(1024) void distill_join_kernel(uint32_t nparts, const float2* __restrict__ part, int reduction,
                                                            float* __restrict__ loss) {
    __shared__ double sums[16];
    __shared__ unsigned long long counts[16];
    double s = 0.0;
    unsigned long long n = 0;
    for (uint32_t i = threadIdx.x; i < nparts; i += 1024) {
        s += (double)part[i].x;
        n += __float_as_uint(part[i].y);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { s += __shfl_xor(s, o, 64); n += __shfl_xor(n, o, 64); }
    if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = s; counts[threadIdx.x >> 6] = n; }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) { s += sums[w]; n += counts[w]; }
    const double weight = reduction == 1 ? 1.0 / (double)(n ? n : 1) : 1.0;
    loss[0] = (float)(s * weight);
    loss[1] = (float)weight;
}

bool planes_layout(size_t row_stride, size_t class_stride) { return class_stride != 1 && row_stride == 1; }

unsigned distill_blocks(size_t rows, int per_block) {
    const size_t need = (rows + per_block - 1) / per_block;
    return (unsigned)(need < DISTILL_BLOCKS ? need : DISTILL_BLOCKS);
}

// Lanes of a row: 16 for a few classes, a wave up to some thousand, a workgroup beyond that.
int row_lanes(size_t classes) { return classes <= 64 ? 16 : classes <= 2048 ? 64 : classes <= 16384 ? 256 : 1024; }

template <typename T, int V>
int distill_rows(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
#define E3_ROWS(G)                                                                                            \
    {                                                                                                         \
        blocks = distill_blocks(a.rows, Lanes<G>::ROWS);                                                      \
        if (backward) distill_bwd_rows_kernel<T, V, G><<<dim3(blocks), dim3(Lanes<G>::THREADS), 0, s>>>(a);   \
        else distill_fwd_rows_kernel<T, V, G><<<dim3(blocks), dim3(Lanes<G>::THREADS), 0, s>>>(a);            \
    }
    switch (row_lanes(a.classes)) {
        case 16: E3_ROWS(16) break;
        case 64: E3_ROWS(64) break;
        case 256: E3_ROWS(256) break;
        default: E3_ROWS(1024)
    }
#undef E3_ROWS
    LAUNCH_OK("distill_rows_kernel");
    return 0;
}

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
    distill_bwd_wide_kernel<T, P, KR><<<dim3(distill_blocks(a.rows, 256 * P)), dim3(256), 0, s>>>(a);
    LAUNCH_OK("distill_bwd_wide_kernel");
    return 0;
}
// whether P neighbouring pixels of every plane can be moved at once
template <typename T>
bool planes_wide(const void* p, size_t stride, size_t rows, size_t n) {
    return rows % n == 0 && stride % n == 0 && (reinterpret_cast<uintptr_t>(p) & (n * sizeof(T) - 1)) == 0;
}

template <typename T>
int distill_t(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
    if (planes_layout(a.row_stride, a.class_stride)) {
        if (a.k <= 8) {
            if (!backward) {
                if (planes_wide<T>(a.logits, a.class_stride, a.rows, 2))
                    return a.k <= 4 ? distill_wide_fwd<T, 2, 4>(a, blocks, s) : distill_wide_fwd<T, 2, 8>(a, blocks, s);
                return a.k <= 4 ? distill_wide_fwd<T, 1, 4>(a, blocks, s) : distill_wide_fwd<T, 1, 8>(a, blocks, s);
            }
            if (planes_wide<T>(a.logits, a.class_stride, a.rows, 4) && planes_wide<T>(a.grad, a.g_class, a.rows, 4))
                return a.k <= 4 ? distill_wide_bwd<T, 4, 4>(a, s) : distill_wide_bwd<T, 4, 8>(a, s);
            return a.k <= 4 ? distill_wide_bwd<T, 1, 4>(a, s) : distill_wide_bwd<T, 1, 8>(a, s);
        }
        const size_t lds = (size_t)a.classes * 64 * sizeof(float);
        blocks = distill_blocks(a.rows, 64);
        if (backward) distill_bwd_planes_kernel<T><<<dim3(blocks), dim3(64), lds, s>>>(a);
        else distill_fwd_planes_kernel<T><<<dim3(blocks), dim3(64), lds, s>>>(a);
        LAUNCH_OK("distill_planes_kernel");
        return 0;
    }
    // packs need the scores and their gradient to lie the same way to a 16-byte boundary in every row
    const uintptr_t zp = reinterpret_cast<uintptr_t>(a.logits), gp = reinterpret_cast<uintptr_t>(backward ? a.grad : a.logits);
    const size_t gr = backward ? a.g_row : a.row_stride;
    const bool wide = zp % sizeof(T) == 0 && ((zp ^ gp) & 15) == 0 && (a.row_stride * sizeof(T)) % 16 == (gr * sizeof(T)) % 16;
    return wide ? distill_rows<T, Wide<T>::N>(a, backward, blocks, s) : distill_rows<T, 1>(a, backward, blocks, s);
}

int distill_any(const DistillArgs& a, bool backward, unsigned& blocks, hipStream_t s) {
    if (a.dtype == E3_F32) return distill_t<float>(a, backward, blocks, s);
    if (a.dtype == E3_F16) return distill_t<f16_t>(a, backward, blocks, s);
    return distill_t<bf16_t>(a, backward, blocks, s);
}
}  // namespace

bool e3_distill_layout_ok(size_t rows, size_t classes, size_t row_stride, size_t class_stride) {
    return class_stride == 1 || rows == 1 ? class_stride == 1 : row_stride == 1 && classes <= (size_t)DISTILL_PLANES;
}
size_t e3_distill_scratch_bytes(size_t rows) {
    (void)rows;
    return DISTILL_BLOCKS * sizeof(float2) + 256;
}

int e3_distill_forward_impl(size_t rows, size_t classes, size_t k, const void* logits, size_t row_stride,
                            size_t class_stride, int dtype, const void* teacher, size_t t_row, size_t t_entry,
                            int teacher_dtype, const void* index, size_t i_row, size_t i_entry, int index_bytes,
                            float temperature, int reduction, float* stats, float* row_loss, float* loss, char* scratch,
                            hipStream_t s) {
    DistillArgs a{};
    a.rows = rows; a.classes = (uint32_t)classes; a.k = k; a.logits = logits; a.row_stride = row_stride;
    a.class_stride = class_stride; a.dtype = dtype; a.teacher = teacher; a.t_row = t_row; a.t_entry = t_entry;
    a.teacher_dtype = teacher_dtype; a.index = index; a.i_row = i_row; a.i_entry = i_entry; a.index_bytes = index_bytes;
    a.temperature = temperature; a.reduction = reduction; a.stats = reinterpret_cast<float2*>(stats);
    a.row_loss = row_loss; a.part = reinterpret_cast<float2*>(scratch);
    unsigned blocks = 0;
    if (rows > 0) {
        const int rc = distill_any(a, false, blocks, s);
        if (rc) return rc;
    }
    if (!loss) return 0;
    distill_join_kernel<<<dim3(1), dim3(1024), 0, s>>>(blocks, a.part, reduction, loss);
    LAUNCH_OK("distill_join_kernel");
    return 0;
}

int e3_distill_backward_impl(size_t rows, size_t classes, size_t k, const void* logits, size_t row_stride,
                             size_t class_stride, int dtype, const void* teacher, size_t t_row, size_t t_entry,
                             int teacher_dtype, const void* index, size_t i_row, size_t i_entry, int index_bytes,
                             float temperature, int reduction, const float* stats, const float* loss, const float* d_loss,
                             void* grad, size_t g_row, size_t g_class, hipStream_t s) {
    if (rows == 0) return 0;
    DistillArgs a{};
    a.rows = rows; a.classes = (uint32_t)classes; a.k = k; a.logits = logits; a.row_stride = row_stride;
    a.class_stride = class_stride; a.dtype = dtype; a.teacher = teacher; a.t_row = t_row; a.t_entry = t_entry;
    a.teacher_dtype = teacher_dtype; a.index = index; a.i_row = i_row; a.i_entry = i_entry; a.index_bytes = index_bytes;
    a.temperature = temperature; a.reduction = reduction; a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    a.weight = loss ? loss + 1 : nullptr; a.scale = d_loss; a.grad = grad; a.g_row = g_row; a.g_class = g_class;
    unsigned blocks = 0;
    return distill_any(a, true, blocks, s);
}
