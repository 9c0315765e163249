// Whole rows of logits: their top entries with the row's softmax statistics (gvk_top_logits), and the divergence of a row's
// softmax from a teacher's list of logits with its gradient (gvk_distill, gvk_distill_grad); include/gvk.h.
//
// With m = max_j z_j, S = sum_j exp((z_j - m) / T), p_j = exp((z_j - m) / T) / S and the teacher's probabilities q_e of its
// list (candidate i_e, logit t_e):
//     q_e   = exp((t_e - mt) / T) / St,  mt and St those of the list, or of the teacher's whole row where its statistics are given
//     loss  = sum_e q_e (log q_e - log p_{i_e})
//     dz_j  = w / T * (Q p_j - sum_{e: i_e = j} q_e),  Q = sum_e q_e
// All of it is bound by HBM: a row is read once for m and S, and once more where it does not stay on the chip.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "gvk.h"
#include "gvk_internal.h"
#include "gvk_rows.hpp"

namespace {

using namespace gvk_rows;

constexpr float kInfinity = __builtin_inff();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// what exp((z - m) / T) subtracts: 0 where a row has nothing above minus infinity (its exponentials are then all 0, not NaN)
__device__ __forceinline__ float reference_of(float largest) { return largest == -kInfinity ? 0.0f : largest; }

// ---- the top of a row ---------------------------------------------------------------------------------------------------------
// Entries are ordered by (logit, lower candidate first): one 64-bit key, unique in a row, so whatever order candidates are
// collected in, the answer is the same.  A slice of a row lives in the registers of a workgroup.  The largest of every thread's
// elements gives a bound: of each wave's 64 such maxima the ceil(k / waves)-th largest, and of those the least.  At least k
// elements reach it, and only a few more than k do (16384 normal logits, k = 64: about 90), so they fit in LDS and are ranked by
// counting.  Rows that defeat the bound (all logits equal, NaN) take the exact way: a bisection of the key, bit by bit.

constexpr int kTopThreads = 256, kTopWaves = kTopThreads / 64, kTopBuffer = 2048;
constexpr int kMergeThreads = 512;

__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;  // NaN above everything: it shows
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float of_ordered(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return (uint64_t)ordered(x) << 32 | (uint32_t)~index; }

// the rank-th largest (1-based) of the 64 values a wave holds, its lowest 16 bits cut off: a bound that `rank` of them reach
__device__ __forceinline__ uint32_t wave_bound(uint32_t value, int rank) {
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t trial = bound | 1u << bit;
        if (__popcll(__ballot(value >= trial)) >= rank) bound = trial;
    }
    return bound;
}

struct top_shared {
    uint64_t keys[kTopBuffer];
    uint32_t bound[kMergeThreads / 64];
    float reduce[kMergeThreads / 64];
    uint32_t count, exact;
};

// keys[0 .. count) -> the k largest in order, by counting the larger ones
template<int THREADS, class Write>
__device__ __forceinline__ void write_ranked(const top_shared &s, uint32_t count, uint32_t k, Write write) {
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
        const uint64_t key = s.keys[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; j++) rank += s.keys[j] > key;
        if (rank < k) write(rank, key);
    }
}

// The least threshold found, from the highest bit down, that at least `want` keys reach and that leaves no more than fit the
// buffer; count_reaching(threshold) counts over the workgroup.  All 64 bits end at the want-th largest key itself.
template<class Count>
__device__ __forceinline__ uint64_t exact_threshold(uint32_t want, Count count_reaching) {
    uint64_t threshold = 0;
    for (int bit = 63; bit >= 0; bit--) {
        const uint64_t trial = threshold | 1ull << bit;
        const uint32_t count = count_reaching(trial);
        if (count < want) continue;
        threshold = trial;
        if (count <= (uint32_t)kTopBuffer) break;
    }
    return threshold;
}

template<int THREADS>
__device__ __forceinline__ uint32_t block_count(uint32_t v, top_shared &s) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) v += __shfl_xor((int)v, step);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.bound[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; i++) v += s.bound[i];
    return v;
}

struct top_output {
    float *values;
    int32_t *index;
    float *stats;      // [rows][2] or null
    uint64_t *lists;   // [rows][slices][capacity] (more than one slice)
    uint32_t *counts;  // [rows][slices]
    float2 *partial;   // [rows][slices]
};

// One slice of one row: U chunks to a thread, in registers.
template<class T, int U>
__global__ void __launch_bounds__(kTopThreads) top_kernel(const T *logits, int64_t stride, int64_t first_row, uint32_t slices, int64_t num_col, uint32_t k,
                                                          uint32_t capacity, float scale, top_output out) {
    constexpr int E = per_chunk<T>::value;
    __shared__ top_shared s;
    const int64_t row = first_row + blockIdx.x / slices;
    const uint32_t slice = blockIdx.x % slices;
    const chunked_row<T> z(logits + row * stride, num_col);
    const int64_t chunk0 = (int64_t)slice * U * kTopThreads;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = z.load(chunk0 + u * kTopThreads + threadIdx.x);
    if (threadIdx.x == 0) s.count = 0, s.exact = 0;

    float largest = -kInfinity;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < E; i++) largest = fmaxf(largest, x[i]);
    }
    const uint32_t wave_share = (k + kTopWaves - 1) / kTopWaves;
    const uint32_t bound = wave_bound(ordered(largest), (int)wave_share);
    if ((threadIdx.x & 63) == 0) s.bound[threadIdx.x >> 6] = bound;
    const float m = block_max<kTopThreads>(largest, s.reduce);  // its barriers publish the bounds too
    uint32_t least = s.bound[0];
#pragma unroll
    for (int w = 1; w < kTopWaves; w++) least = min(least, s.bound[w]);
    // cut bits may make a NaN of minus infinity's key
    const float tau = least <= 0x007fffffu ? -kInfinity : of_ordered(least);
    const float base = reference_of(m);
    float sum = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        unpack<T>(raw[u], x);
        const int64_t at = z.first(chunk0 + u * kTopThreads + threadIdx.x);
#pragma unroll
        for (int i = 0; i < E; i++) {
            sum += exp2_fast((x[i] - base) * scale);
            if (x[i] >= tau && at + i >= 0 && at + i < num_col) {
                const uint32_t place = atomicAdd(&s.count, 1u);
                if (place < (uint32_t)kTopBuffer) s.keys[place] = key_of(x[i], (uint32_t)(at + i));
            }
        }
    }
    sum = block_sum<kTopThreads>(sum, s.reduce);
    uint32_t count = s.count;  // behind the barriers of the sum
    if (count > (uint32_t)kTopBuffer || sum != sum) {
        const int64_t begin = max((int64_t)0, z.first(chunk0)), end = min(num_col, z.first(chunk0 + (int64_t)U * kTopThreads));
        const uint32_t want = (uint32_t)min((int64_t)k, max((int64_t)0, end - begin));
        auto each = [&](auto visit) {
#pragma unroll 1
            for (int u = 0; u < U; u++) {
                uint4 r = raw[0];
#pragma unroll
                for (int v = 1; v < U; v++)
                    if (v == u) r = raw[v];
                float x[E];
                unpack<T>(r, x);
                const int64_t at = z.first(chunk0 + u * kTopThreads + threadIdx.x);
#pragma unroll
                for (int i = 0; i < E; i++)
                    if (at + i >= 0 && at + i < num_col) visit(key_of(x[i], (uint32_t)(at + i)));
            }
        };
        const uint64_t threshold = exact_threshold(want, [&](uint64_t trial) {
            uint32_t mine = 0;
            each([&](uint64_t key) { mine += key >= trial; });
            return block_count<kTopThreads>(mine, s);
        });
        __syncthreads();
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        each([&](uint64_t key) {
            if (key >= threshold) {
                const uint32_t place = atomicAdd(&s.count, 1u);
                if (place < (uint32_t)kTopBuffer) s.keys[place] = key;
            }
        });
        __syncthreads();
        count = min(s.count, (uint32_t)kTopBuffer);
    }
    if (slices == 1) {
        write_ranked<kTopThreads>(s, count, k, [&](uint32_t rank, uint64_t key) {
            out.values[row * k + rank] = of_ordered((uint32_t)(key >> 32));
            out.index[row * k + rank] = (int32_t)~(uint32_t)key;
        });
        if (out.stats && threadIdx.x == 0) out.stats[2 * row] = m, out.stats[2 * row + 1] = logf(sum);
        return;
    }
    const uint64_t list = (uint64_t)blockIdx.x;
    uint64_t *keys = out.lists + list * capacity;
    if (count <= capacity) {
        for (uint32_t i = threadIdx.x; i < count; i += kTopThreads) keys[i] = s.keys[i];
    } else {
        write_ranked<kTopThreads>(s, count, k, [&](uint32_t rank, uint64_t key) { keys[rank] = key; });
        count = k;
    }
    if (threadIdx.x == 0) out.counts[list] = count, out.partial[list] = make_float2(m, sum);
}

// The lists of a row's slices -> its top entries and statistics.
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(int64_t first_row, uint32_t slices, uint32_t k, uint32_t log_capacity, float scale, top_output out) {
    __shared__ top_shared s;
    const int64_t row = first_row + blockIdx.x;
    const uint64_t list0 = (uint64_t)blockIdx.x * slices;
    const uint64_t *keys = out.lists + (list0 << log_capacity);
    const uint32_t *counts = out.counts + list0;
    const uint64_t total = (uint64_t)slices << log_capacity;
    const uint32_t mask = (1u << log_capacity) - 1;
    auto each = [&](auto visit) {
        for (uint64_t i = threadIdx.x; i < total; i += kMergeThreads)
            if ((uint32_t)(i & mask) < counts[i >> log_capacity]) visit(keys[i]);
    };
    if (threadIdx.x == 0) s.count = 0;
    uint32_t largest = 0;
    each([&](uint64_t key) { largest = max(largest, (uint32_t)(key >> 32)); });
    const uint32_t bound = wave_bound(largest, (int)((k + kMergeThreads / 64 - 1) / (kMergeThreads / 64)));
    if ((threadIdx.x & 63) == 0) s.bound[threadIdx.x >> 6] = bound;
    float m = -kInfinity, sum = 0;
    for (uint32_t i = threadIdx.x; i < slices; i += kMergeThreads) m = fmaxf(m, out.partial[list0 + i].x);
    m = block_max<kMergeThreads>(m, s.reduce);
    const float base = reference_of(m);
    for (uint32_t i = threadIdx.x; i < slices; i += kMergeThreads) {
        const float2 p = out.partial[list0 + i];
        if (p.x > -kInfinity || p.y != p.y) sum += p.y * exp2_fast((reference_of(p.x) - base) * scale);  // not a slice of nothing but masks
    }
    sum = block_sum<kMergeThreads>(sum, s.reduce);
    uint32_t least = s.bound[0];
#pragma unroll
    for (int w = 1; w < kMergeThreads / 64; w++) least = min(least, s.bound[w]);
    each([&](uint64_t key) {
        if ((uint32_t)(key >> 32) >= least) {
            const uint32_t place = atomicAdd(&s.count, 1u);
            if (place < (uint32_t)kTopBuffer) s.keys[place] = key;
        }
    });
    __syncthreads();
    uint32_t count = s.count;
    if (count > (uint32_t)kTopBuffer) {
        const uint64_t threshold = exact_threshold(k, [&](uint64_t trial) {
            uint32_t mine = 0;
            each([&](uint64_t key) { mine += key >= trial; });
            return block_count<kMergeThreads>(mine, s);
        });
        __syncthreads();
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        each([&](uint64_t key) {
            if (key >= threshold) {
                const uint32_t place = atomicAdd(&s.count, 1u);
                if (place < (uint32_t)kTopBuffer) s.keys[place] = key;
            }
        });
        __syncthreads();
        count = min(s.count, (uint32_t)kTopBuffer);
    }
    write_ranked<kMergeThreads>(s, count, k, [&](uint32_t rank, uint64_t key) {
        out.values[row * k + rank] = of_ordered((uint32_t)(key >> 32));
        out.index[row * k + rank] = (int32_t)~(uint32_t)key;
    });
    if (out.stats && threadIdx.x == 0) out.stats[2 * row] = m, out.stats[2 * row + 1] = logf(sum);
}

// ---- a teacher's list and a student's row -----------------------------------------------------------------------------------

constexpr int kMaxList = GVK_MAX_DISTILL_LIST;

struct distill_input {
    const void *logits;
    int64_t stride, num_col;
    const int32_t *index;          // [rows][k], -1: no entry
    const float *teacher;          // [rows][k]
    const float *teacher_stats;    // [rows][2] or null
    const float *weight;           // [rows] or null
    uint32_t k;
    float temperature, scale;      // scale = log2(e) / temperature
};

struct distill_output {
    float *loss, *stats;
    void *grad;
    int64_t grad_stride;
    float2 *partial;  // [rows][slices]
    float *listed;    // [rows][k]: the student's logits of the list (the gradient may lie over the logits)
};

struct list_shared {
    int32_t index[kMaxList];  // -1 where the list has no entry
    float q[kMaxList];
    float reduce[16];
    uint32_t bad, any;
};

// The list of a row into LDS: q_e of its entries; returns Q, and log St and mt through the pointers.  An index outside the row makes
// the row's answer NaN: it shows, and nothing is read or written out of bounds.
template<int THREADS>
__device__ __forceinline__ float load_list(const distill_input &in, int64_t row, list_shared &s, float *log_total, float *reference) {
    if (threadIdx.x == 0) s.bad = 0, s.any = 0;
    __syncthreads();
    const int32_t *index = in.index + row * in.k;
    const float *teacher = in.teacher + row * in.k;
    float largest = -kInfinity;
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {
        const int32_t i = index[e];
        const float t = teacher[e];
        const bool inside = i >= 0 && i < in.num_col;
        if (!inside && i != -1) s.bad = 1;
        const bool entry = inside && !(t == -kInfinity);
        s.index[e] = entry ? i : -1;
        s.q[e] = t;
        if (entry) largest = fmaxf(largest, t), s.any = 1;
    }
    float mt, lt, inverse = 1;
    if (in.teacher_stats) {
        mt = in.teacher_stats[2 * row], lt = in.teacher_stats[2 * row + 1];
    } else {
        mt = reference_of(block_max<THREADS>(largest, s.reduce));
        float sum = 0;
        for (uint32_t e = threadIdx.x; e < in.k; e += THREADS)
            if (s.index[e] >= 0) sum += expf((s.q[e] - mt) / in.temperature);
        sum = block_sum<THREADS>(sum, s.reduce);
        lt = logf(sum);
        inverse = 1.0f / sum;
    }
    float q = 0;
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {
        float mine = 0;
        if (s.index[e] >= 0) {
            const float shifted = (s.q[e] - mt) / in.temperature;
            mine = in.teacher_stats ? expf(shifted - lt) : expf(shifted) * inverse;
        }
        s.q[e] = mine;
        q += mine;
    }
    q = block_sum<THREADS>(q, s.reduce);
    *log_total = lt, *reference = mt;
    return s.bad ? __builtin_nanf("") : q;
}

// the row's loss; logit(e) is the student's logit of entry e
template<int THREADS, class Logit>
__device__ __forceinline__ float list_loss(const distill_input &in, int64_t row, list_shared &s, float q_total, float log_total, float reference, float m,
                                           float log_sum, Logit logit) {
    const float *teacher = in.teacher + row * in.k;
    float sum = 0;
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {
        const float q = s.q[e];
        if (s.index[e] < 0 || q == 0) continue;  // 0 log 0 = 0
        const float log_q = (teacher[e] - reference) / in.temperature - log_total;
        const float log_p = (logit(e) - m) / in.temperature - log_sum;
        sum += q * (log_q - log_p);
    }
    sum = block_sum<THREADS>(sum, s.reduce);
    if (q_total != q_total) return q_total;
    return m == -kInfinity && log_sum == log_sum ? 0.0f : sum;
}

// What the gradient of elements [begin, begin + SIZE) takes from the list: a bit per element that has an entry, and there the
// sum of its entries' q (in the list's order, so that an index that occurs twice gives the same answer every time).
template<int SIZE>
struct listed_slice {
    uint32_t bits[SIZE / 32 + 1];
    float q[SIZE];
};

template<int THREADS, int SIZE>
__device__ __forceinline__ void mark_listed(const distill_input &in, const list_shared &s, int64_t begin, listed_slice<SIZE> &l) {
    for (int i = threadIdx.x; i < SIZE / 32 + 1; i += THREADS) l.bits[i] = 0;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {
        const int32_t i = s.index[e];
        if (i < begin || i >= begin + SIZE) continue;
        bool first = true;
        float q = s.q[e];
        for (uint32_t other = 0; other < in.k; other++) {
            if (s.index[other] != i) continue;
            if (other < e) first = false;
            if (other > e) q += s.q[other];
        }
        if (!first) continue;
        l.q[i - begin] = q;
        atomicOr(&l.bits[(i - begin) >> 5], 1u << ((i - begin) & 31));
    }
    __syncthreads();
}

// Nothing to learn from a row without entries, whatever its logits hold, nor from one whose candidates are all masked.
__device__ __forceinline__ bool learns_nothing(const list_shared &s, float m, float sum) { return !s.bad && (!s.any || (m == -kInfinity && sum == sum)); }

// gradient of a chunk: p_factor = w Q / (T S), q_factor = w / T
template<class T, int SIZE>
__device__ __forceinline__ void chunk_gradient(const uint4 raw, int place, float base, float scale, float p_factor, float q_factor, bool nothing,
                                               const listed_slice<SIZE> &l, float g[per_chunk<T>::value]) {
    constexpr int E = per_chunk<T>::value;
    float x[E];
    unpack<T>(raw, x);
#pragma unroll
    for (int i = 0; i < E; i++) g[i] = nothing ? 0.0f : exp2_fast((x[i] - base) * scale) * p_factor;
    // a chunk's place in the slice is a multiple of E, E divides 32: its bits lie in one word
    const uint32_t mine = l.bits[place >> 5] >> (place & 31) & ((1u << E) - 1);
    if (mine && !nothing) {
#pragma unroll
        for (int i = 0; i < E; i++)
            if (mine >> i & 1) g[i] -= l.q[place + i] * q_factor;
    }
}

// Rows that fit a workgroup's registers: read once, written once, one launch.  U chunks to a thread.
template<class T, int THREADS, int U, bool GRAD>
__global__ void __launch_bounds__(THREADS) distill_row_kernel(distill_input in, distill_output out, int64_t first_row) {
    constexpr int E = per_chunk<T>::value, SIZE = THREADS * U * E;
    __shared__ list_shared s;
    __shared__ listed_slice<GRAD ? SIZE : 32> l;
    const int64_t row = first_row + blockIdx.x;
    const chunked_row<T> z((const T *)in.logits + row * in.stride, in.num_col);
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = z.load(u * THREADS + threadIdx.x);
    float log_total, reference;
    float q_total = load_list<THREADS>(in, row, s, &log_total, &reference);
    float largest = -kInfinity;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < E; i++) largest = fmaxf(largest, x[i]);
    }
    const float m = block_max<THREADS>(largest, s.reduce), base = reference_of(m);
    float sum = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < E; i++) sum += exp2_fast((x[i] - base) * in.scale);
    }
    sum = block_sum<THREADS>(sum, s.reduce);
    const float log_sum = logf(sum);
    const float loss = list_loss<THREADS>(in, row, s, q_total, log_total, reference, m, log_sum, [&](uint32_t e) { return to_float(z.row[s.index[e]]); });
    if (threadIdx.x == 0) {
        out.loss[row] = loss;
        out.stats[2 * row] = m, out.stats[2 * row + 1] = log_sum;
    }
    if constexpr (GRAD) {
        const float q_factor = (in.weight ? in.weight[row] : 1.0f) / in.temperature;
        const bool nothing = learns_nothing(s, m, sum);
        const float p_factor = q_factor * q_total / sum;
        mark_listed<THREADS, SIZE>(in, s, -z.lead, l);
        T *grad = (T *)out.grad + row * out.grad_stride;
        const bool wide = (uintptr_t)grad % 16 == (uintptr_t)z.row % 16;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int place = (u * THREADS + (int)threadIdx.x) * E;
            float g[E];
            chunk_gradient<T, SIZE>(raw[u], place, base, in.scale, p_factor, q_factor, nothing, l, g);
            store_chunk<T>(grad, (int64_t)place - z.lead, in.num_col, wide, g);
        }
    }
}

constexpr int kSliceThreads = 256, kSliceElements = 8192;

template<class T>
constexpr int slice_chunks() {
    return kSliceElements / kSliceThreads / per_chunk<T>::value;
}

// longer rows, first launch: max and sum of a slice, and the student's logits of the list's entries in it
template<class T>
__global__ void __launch_bounds__(kSliceThreads) distill_partial_kernel(distill_input in, distill_output out, int64_t first_row, uint32_t slices) {
    constexpr int E = per_chunk<T>::value, U = slice_chunks<T>();
    __shared__ float reduce[kSliceThreads / 64];
    const int64_t row = first_row + blockIdx.x / slices;
    const uint32_t slice = blockIdx.x % slices;
    const chunked_row<T> z((const T *)in.logits + row * in.stride, in.num_col);
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = z.load((int64_t)(slice * (uint64_t)U + u) * kSliceThreads + threadIdx.x);
    if (out.listed) {
        const int64_t begin = z.first((int64_t)slice * (U * kSliceThreads));
        for (uint32_t e = threadIdx.x; e < in.k; e += kSliceThreads) {
            const int64_t i = in.index[row * in.k + e];
            if (i >= 0 && i < in.num_col && i >= begin && i < begin + kSliceElements) out.listed[(uint64_t)(blockIdx.x / slices) * in.k + e] = to_float(z.row[i]);
        }
    }
    float largest = -kInfinity;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < E; i++) largest = fmaxf(largest, x[i]);
    }
    const float m = block_max<kSliceThreads>(largest, reduce), base = reference_of(m);
    float sum = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < E; i++) sum += exp2_fast((x[i] - base) * in.scale);
    }
    sum = block_sum<kSliceThreads>(sum, reduce);
    if (threadIdx.x == 0) out.partial[blockIdx.x] = make_float2(m, sum);
}

// max and sum of a row from those of its slices
template<int THREADS>
__device__ __forceinline__ void join_slices(const float2 *partial, uint32_t slices, float scale, float *shared, float *m_out, float *sum_out) {
    float m = -kInfinity, sum = 0;
    for (uint32_t i = threadIdx.x; i < slices; i += THREADS) m = fmaxf(m, partial[i].x);
    m = block_max<THREADS>(m, shared);
    const float base = reference_of(m);
    for (uint32_t i = threadIdx.x; i < slices; i += THREADS) {
        const float2 p = partial[i];
        if (p.x > -kInfinity || p.y != p.y) sum += p.y * exp2_fast((reference_of(p.x) - base) * scale);
    }
    *sum_out = block_sum<THREADS>(sum, shared);
    *m_out = m;
}

// longer rows, the loss alone
template<class T>
__global__ void __launch_bounds__(kSliceThreads) distill_finish_kernel(distill_input in, distill_output out, int64_t first_row, uint32_t slices) {
    __shared__ list_shared s;
    const int64_t row = first_row + blockIdx.x;
    float log_total, reference, m, sum;
    const float q_total = load_list<kSliceThreads>(in, row, s, &log_total, &reference);
    join_slices<kSliceThreads>(out.partial + (uint64_t)blockIdx.x * slices, slices, in.scale, s.reduce, &m, &sum);
    const float log_sum = logf(sum);
    const T *z = (const T *)in.logits + row * in.stride;
    const float loss = list_loss<kSliceThreads>(in, row, s, q_total, log_total, reference, m, log_sum, [&](uint32_t e) { return to_float(z[s.index[e]]); });
    if (threadIdx.x == 0) {
        out.loss[row] = loss;
        out.stats[2 * row] = m, out.stats[2 * row + 1] = log_sum;
    }
}

// the gradient of a slice; with LOSS the statistics come from the partial results and slice 0 writes the row's loss, else they are given
template<class T, bool LOSS>
__global__ void __launch_bounds__(kSliceThreads) distill_grad_kernel(distill_input in, distill_output out, int64_t first_row, uint32_t slices) {
    constexpr int E = per_chunk<T>::value, U = slice_chunks<T>();
    __shared__ list_shared s;
    __shared__ listed_slice<kSliceElements> l;
    const int64_t row = first_row + blockIdx.x / slices;
    const uint32_t slice = blockIdx.x % slices;
    const chunked_row<T> z((const T *)in.logits + row * in.stride, in.num_col);
    const int64_t chunk0 = (int64_t)slice * (U * kSliceThreads);
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = z.load(chunk0 + u * kSliceThreads + threadIdx.x);
    float log_total, reference, m, sum;
    const float q_total = load_list<kSliceThreads>(in, row, s, &log_total, &reference);
    if constexpr (LOSS) {
        const uint32_t local = blockIdx.x / slices;
        join_slices<kSliceThreads>(out.partial + (uint64_t)local * slices, slices, in.scale, s.reduce, &m, &sum);
        if (slice == 0) {
            const float log_sum = logf(sum);
            const float loss = list_loss<kSliceThreads>(in, row, s, q_total, log_total, reference, m, log_sum,
                                                        [&](uint32_t e) { return out.listed[(uint64_t)local * in.k + e]; });
            if (threadIdx.x == 0) {
                out.loss[row] = loss;
                out.stats[2 * row] = m, out.stats[2 * row + 1] = log_sum;
            }
        }
    } else {
        m = out.stats[2 * row];
        sum = expf(out.stats[2 * row + 1]);
    }
    const float base = reference_of(m), q_factor = (in.weight ? in.weight[row] : 1.0f) / in.temperature;
    const bool nothing = learns_nothing(s, m, sum);
    const float p_factor = q_factor * q_total / sum;
    mark_listed<kSliceThreads, kSliceElements>(in, s, z.first(chunk0), l);
    T *grad = (T *)out.grad + row * out.grad_stride;
    const bool wide = (uintptr_t)grad % 16 == (uintptr_t)z.row % 16;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int place = (u * kSliceThreads + (int)threadIdx.x) * E;
        float g[E];
        chunk_gradient<T, kSliceElements>(raw[u], place, base, in.scale, p_factor, q_factor, nothing, l, g);
        store_chunk<T>(grad, z.first(chunk0) + place, in.num_col, wide, g);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------

constexpr int64_t kMaxGroups = 1 << 21;  // workgroups of a launch; more rows take more launches

size_t size_of(int dtype) { return dtype == GVK_F32 ? 4 : 2; }

int launched(const char *who) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? GVK_OK : gvk_fail(GVK_EHIP, "%s: %s", who, hipGetErrorString(err));
}

int check_logits(const char *who, int dtype, const void *logits, int64_t num_row, int64_t num_col, int64_t stride) {
    if (dtype != GVK_F32 && dtype != GVK_BF16 && dtype != GVK_F16) return gvk_fail(GVK_EINVAL, "%s: unknown type %d", who, dtype);
    if (num_row < 0 || num_col < 0 || num_col > 0x7fffffff) return gvk_fail(GVK_EINVAL, "%s: %lld rows of %lld logits", who, (long long)num_row, (long long)num_col);
    if (num_row > 1 && stride < num_col) return gvk_fail(GVK_EINVAL, "%s: rows of %lld logits with a stride of %lld", who, (long long)num_col, (long long)stride);
    if (num_row && num_col && !logits) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    if ((uintptr_t)logits % size_of(dtype)) return gvk_fail(GVK_EINVAL, "%s: logits are not aligned to their type", who);
    return GVK_OK;
}

int check_temperature(const char *who, float temperature, float *scale) {
    *scale = (float)(1.4426950408889634 / (double)temperature);
    if (!(temperature > 0) || !isfinite(temperature) || !isfinite(*scale) || !(*scale > 0))
        return gvk_fail(GVK_EINVAL, "%s: the temperature must be a positive finite number, not %g", who, (double)temperature);
    return GVK_OK;
}

// slices a row of num_col takes wherever in 16 bytes it begins
int64_t slices_of(int64_t num_col, int64_t slice, int per_chunk) { return (num_col + per_chunk - 1 + slice - 1) / slice; }

constexpr int64_t kTopSlice = 16384, kTopSmallSlice = 4096;

struct top_plan {
    int64_t slice, slices;
    int log_capacity;
    size_t bytes;
};

top_plan plan_top(int dtype, int64_t num_row, int64_t num_col, int k) {
    const int per_chunk = 16 / (int)size_of(dtype);
    top_plan p;
    p.slice = kTopSlice;
    p.slices = slices_of(num_col, p.slice, per_chunk);
    if (p.slices > 1 && num_row * p.slices < 512) {  // few rows: more, smaller slices, to reach every CU
        p.slice = kTopSmallSlice;
        p.slices = slices_of(num_col, p.slice, per_chunk);
    } else if (slices_of(num_col, kTopSmallSlice, per_chunk) == 1) {
        p.slice = kTopSmallSlice, p.slices = 1;
    }
    p.log_capacity = 6;
    while ((1 << p.log_capacity) < 2 * k) p.log_capacity++;
    p.bytes = p.slices > 1 ? (size_t)num_row * p.slices * ((8ull << p.log_capacity) + sizeof(float2) + sizeof(uint32_t)) : 0;
    return p;
}

template<class T>
void launch_top(hipStream_t stream, const top_plan &p, const T *logits, int64_t stride, int64_t first_row, int64_t num_row, int64_t num_col, int k, float scale,
                const top_output &out) {
    constexpr int E = per_chunk<T>::value, kLarge = kTopSlice / kTopThreads / E, kSmall = kTopSmallSlice / kTopThreads / E;
    const dim3 grid((unsigned)(num_row * p.slices));
    if (p.slice == kTopSlice)
        hipLaunchKernelGGL((top_kernel<T, kLarge>), grid, dim3(kTopThreads), 0, stream, logits, stride, first_row, (uint32_t)p.slices, num_col, (uint32_t)k, 1u << p.log_capacity, scale, out);
    else
        hipLaunchKernelGGL((top_kernel<T, kSmall>), grid, dim3(kTopThreads), 0, stream, logits, stride, first_row, (uint32_t)p.slices, num_col, (uint32_t)k, 1u << p.log_capacity, scale, out);
    if (p.slices > 1)
        hipLaunchKernelGGL(merge_kernel, dim3((unsigned)num_row), dim3(kMergeThreads), 0, stream, first_row, (uint32_t)p.slices, (uint32_t)k, (uint32_t)p.log_capacity, scale, out);
}

constexpr int64_t kRowElements = 16384;  // a row that a workgroup of 1024 threads holds

int64_t distill_slices(int dtype, int64_t num_col) { return slices_of(num_col, kSliceElements, 16 / (int)size_of(dtype)); }

bool one_launch(int dtype, int64_t num_col) { return slices_of(num_col, kRowElements, 16 / (int)size_of(dtype)) <= 1; }

template<class T, bool GRAD>
void launch_rows(hipStream_t stream, const distill_input &in, const distill_output &out, int64_t first, unsigned rows) {
    constexpr int E = per_chunk<T>::value;
    const int64_t need = in.num_col + E - 1;
#define GVK_ROWS(THREADS, ELEMENTS) \
    hipLaunchKernelGGL((distill_row_kernel<T, THREADS, ELEMENTS / THREADS / E, GRAD>), dim3(rows), dim3(THREADS), 0, stream, in, out, first)
    if (need <= 2048) GVK_ROWS(256, 2048);
    else if (need <= 8192) GVK_ROWS(512, 8192);
    else GVK_ROWS(1024, 16384);
#undef GVK_ROWS
}

template<class T>
void launch_distill(hipStream_t stream, const distill_input &in, distill_output out, int64_t num_row, int64_t slices, bool one) {
    const int64_t step = one ? kMaxGroups : (kMaxGroups / slices > 0 ? kMaxGroups / slices : 1);
    const bool loss = out.loss != nullptr;
    const distill_output all = out;
    for (int64_t first = 0; first < num_row; first += step) {
        const unsigned rows = (unsigned)(num_row - first < step ? num_row - first : step);
        if (one) {
            if (out.grad) launch_rows<T, true>(stream, in, out, first, rows);
            else launch_rows<T, false>(stream, in, out, first, rows);
            continue;
        }
        const dim3 grid(rows * (unsigned)slices), block(kSliceThreads);
        if (all.partial) out.partial = all.partial + first * slices;
        if (all.listed) out.listed = all.listed + first * in.k;
        if (loss) hipLaunchKernelGGL((distill_partial_kernel<T>), grid, block, 0, stream, in, out, first, (uint32_t)slices);
        if (!out.grad) hipLaunchKernelGGL((distill_finish_kernel<T>), dim3(rows), block, 0, stream, in, out, first, (uint32_t)slices);
        else if (loss) hipLaunchKernelGGL((distill_grad_kernel<T, true>), grid, block, 0, stream, in, out, first, (uint32_t)slices);
        else hipLaunchKernelGGL((distill_grad_kernel<T, false>), grid, block, 0, stream, in, out, first, (uint32_t)slices);
    }
}

int check_distill(const char *who, int dtype, const void *logits, int64_t num_row, int64_t num_col, int64_t stride, int k, const int32_t *index,
                  const float *teacher, const float *stats, const void *grad, int64_t grad_stride) {
    const int rc = check_logits(who, dtype, logits, num_row, num_col, stride);
    if (rc != GVK_OK) return rc;
    if (num_col < 1) return gvk_fail(GVK_EINVAL, "%s: rows without logits", who);
    if (k < 1 || k > kMaxList) return gvk_fail(GVK_EINVAL, "%s: a list holds 1 to %d entries, not %d", who, kMaxList, k);
    if (num_row == 0) return GVK_OK;
    if (!index || !teacher || !stats) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    if (grad) {
        if ((uintptr_t)grad % size_of(dtype)) return gvk_fail(GVK_EINVAL, "%s: grad is not aligned to its type", who);
        if (num_row > 1 && grad_stride < num_col) return gvk_fail(GVK_EINVAL, "%s: rows of %lld gradients with a stride of %lld", who, (long long)num_col, (long long)grad_stride);
        // over the logits, element for element, or apart from them
        const uintptr_t z0 = (uintptr_t)logits, g0 = (uintptr_t)grad;
        const uintptr_t z1 = z0 + ((uintptr_t)(num_row - 1) * stride + num_col) * size_of(dtype), g1 = g0 + ((uintptr_t)(num_row - 1) * grad_stride + num_col) * size_of(dtype);
        if (z0 < g1 && g0 < z1 && !(z0 == g0 && (stride == grad_stride || num_row == 1)))
            return gvk_fail(GVK_EINVAL, "%s: grad overlaps the logits (it may be them, or lie apart)", who);
    }
    return GVK_OK;
}

}  // namespace

extern "C" size_t gvk_top_logits_workspace(int dtype, int64_t num_row, int64_t num_col, int k) {
    if ((dtype != GVK_F32 && dtype != GVK_BF16 && dtype != GVK_F16) || num_row < 1 || num_col < 1 || num_col > 0x7fffffff || k < 1 || k > GVK_MAX_TOP) return 0;
    return plan_top(dtype, num_row, num_col, k).bytes;
}

extern "C" int gvk_top_logits(void *stream, int dtype, const void *logits, int64_t num_row, int64_t num_col, int64_t stride, int k, float temperature, float *values,
                              int32_t *index, float *stats, void *workspace, size_t workspace_bytes) {
    const char *who = "gvk_top_logits";
    int rc = check_logits(who, dtype, logits, num_row, num_col, stride);
    if (rc != GVK_OK) return rc;
    float scale;
    if ((rc = check_temperature(who, temperature, &scale)) != GVK_OK) return rc;
    if (k < 1 || k > GVK_MAX_TOP || k > num_col)
        return gvk_fail(GVK_EINVAL, "%s: the top %d of %lld logits (a call gives 1 to %d, and no more than a row has)", who, k, (long long)num_col, GVK_MAX_TOP);
    if (num_row == 0) return GVK_OK;
    if (!values || !index) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    const top_plan p = plan_top(dtype, num_row, num_col, k);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 16))
        return gvk_fail(GVK_EINVAL, "%s: needs a workspace of %zu bytes on a multiple of 16, %zu given", who, p.bytes, workspace ? workspace_bytes : (size_t)0);
    const int64_t step = kMaxGroups / p.slices > 0 ? kMaxGroups / p.slices : 1;
    const size_t lists = (size_t)num_row * p.slices;
    for (int64_t first = 0; first < num_row; first += step) {
        const int64_t rows = num_row - first < step ? num_row - first : step;
        top_output out = {values, index, stats, nullptr, nullptr, nullptr};
        if (p.bytes) {
            const size_t at = (size_t)first * p.slices;
            out.lists = (uint64_t *)workspace + (at << p.log_capacity);
            out.partial = (float2 *)((uint64_t *)workspace + (lists << p.log_capacity)) + at;
            out.counts = (uint32_t *)((float2 *)((uint64_t *)workspace + (lists << p.log_capacity)) + lists) + at;
        }
        if (dtype == GVK_F32) launch_top((hipStream_t)stream, p, (const float *)logits, stride, first, rows, num_col, k, scale, out);
        else if (dtype == GVK_BF16) launch_top((hipStream_t)stream, p, (const __bf16 *)logits, stride, first, rows, num_col, k, scale, out);
        else launch_top((hipStream_t)stream, p, (const _Float16 *)logits, stride, first, rows, num_col, k, scale, out);
    }
    return launched(who);
}

extern "C" size_t gvk_distill_workspace(int dtype, int64_t num_row, int64_t num_col, int k) {
    if ((dtype != GVK_F32 && dtype != GVK_BF16 && dtype != GVK_F16) || num_row < 1 || num_col < 1 || num_col > 0x7fffffff || k < 1 || k > kMaxList) return 0;
    if (one_launch(dtype, num_col)) return 0;
    return (size_t)num_row * ((size_t)distill_slices(dtype, num_col) * sizeof(float2) + (size_t)k * sizeof(float));
}

extern "C" int gvk_distill(void *stream, int dtype, const void *logits, int64_t num_row, int64_t num_col, int64_t stride, int k, const int32_t *index,
                           const float *teacher, const float *teacher_stats, float temperature, const float *weight, float *loss, float *stats, void *grad,
                           int64_t grad_stride, void *workspace, size_t workspace_bytes) {
    const char *who = "gvk_distill";
    int rc = check_distill(who, dtype, logits, num_row, num_col, stride, k, index, teacher, stats, grad, grad_stride);
    if (rc != GVK_OK) return rc;
    float scale;
    if ((rc = check_temperature(who, temperature, &scale)) != GVK_OK) return rc;
    if (num_row == 0) return GVK_OK;
    if (!loss) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    const size_t need = gvk_distill_workspace(dtype, num_row, num_col, k);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return gvk_fail(GVK_EINVAL, "%s: needs a workspace of %zu bytes on a multiple of 16, %zu given", who, need, workspace ? workspace_bytes : (size_t)0);
    const int64_t slices = distill_slices(dtype, num_col);
    const distill_input in = {logits, stride, num_col, index, teacher, teacher_stats, weight, (uint32_t)k, temperature, scale};
    distill_output out = {loss, stats, grad, grad_stride, nullptr, nullptr};
    if (need) out.partial = (float2 *)workspace, out.listed = grad ? (float *)((float2 *)workspace + (size_t)num_row * slices) : nullptr;
    const bool one = need == 0;
    if (dtype == GVK_F32) launch_distill<float>((hipStream_t)stream, in, out, num_row, slices, one);
    else if (dtype == GVK_BF16) launch_distill<__bf16>((hipStream_t)stream, in, out, num_row, slices, one);
    else launch_distill<_Float16>((hipStream_t)stream, in, out, num_row, slices, one);
    return launched(who);
}

extern "C" int gvk_distill_grad(void *stream, int dtype, const void *logits, int64_t num_row, int64_t num_col, int64_t stride, int k, const int32_t *index,
                                const float *teacher, const float *teacher_stats, float temperature, const float *weight, const float *stats, void *grad,
                                int64_t grad_stride) {
    const char *who = "gvk_distill_grad";
    int rc = check_distill(who, dtype, logits, num_row, num_col, stride, k, index, teacher, stats, grad, grad_stride);
    if (rc != GVK_OK) return rc;
    float scale;
    if ((rc = check_temperature(who, temperature, &scale)) != GVK_OK) return rc;
    if (num_row == 0) return GVK_OK;
    if (!grad) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    const distill_input in = {logits, stride, num_col, index, teacher, teacher_stats, weight, (uint32_t)k, temperature, scale};
    const distill_output out = {nullptr, const_cast<float *>(stats), grad, grad_stride, nullptr, nullptr};
    const int64_t slices = distill_slices(dtype, num_col);
    if (dtype == GVK_F32) launch_distill<float>((hipStream_t)stream, in, out, num_row, slices, false);
    else if (dtype == GVK_BF16) launch_distill<__bf16>((hipStream_t)stream, in, out, num_row, slices, false);
    else launch_distill<_Float16>((hipStream_t)stream, in, out, num_row, slices, false);
    return launched(who);
}
