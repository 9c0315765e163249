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
// collected in, the answer is the same.  A slice of a row (16384 logits) lives in the registers of a workgroup.  Every thread takes
// the largest of its elements (of each quarter of them for k above 128); of a wave's 64 (256) such maxima the ceil(k / waves)-th
// largest, and of those the least, is a bound that at least k elements reach, and only a few more than k do (normal logits,
// k = 64: about 85).  Every lane marks those of its own, a bit each, and puts the chunks they are in into LDS; then they are packed, one
// addition to the count for a wave.  One slice: they are ranked by counting.  More: they go to a list, and one workgroup per row does the
// same with the lists.  Rows that defeat the bound (all logits equal, NaN) take the exact way: a bisection of the key, bit by bit.
// Seven instructions an element, the exponential at a quarter of the rate: 512 x 1M f32 377 us (5.4 TB/s, what reading a row's slices reaches), 1024 x 1M bf16
// 395 (5.2 TB/s), of those 21 the lists; calls in a row — one by itself, before the clock is up, takes 470.  When it was chosen, collecting elements one
// by one as they are met took 450 and 565 against 382 and 490: four instructions each, and an atomic a round.
constexpr int kTopThreads = 256, kTopWaves = kTopThreads / 64, kMergeThreads = 512, kMergeWaves = kMergeThreads / 64;
constexpr uint32_t kPacked = 1024;  // keys a workgroup packs
constexpr uint32_t kKept = 4;       // chunks of a thread kept in LDS; more are read again from memory

__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;  // NaN above everything: it shows
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float of_ordered(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return (uint64_t)ordered(x) << 32 | (uint32_t)~index; }

__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// the rank-th largest (1-based) of the 64 * N values a wave holds, its lowest 16 bits cut off: a bound that `rank` of them reach (0: not
// that many do)
template<int N>
__device__ __forceinline__ uint32_t wave_bound(const uint32_t (&value)[N], int rank) {
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t trial = bound | 1u << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; i++) count += __popcll(__ballot(value[i] >= trial));
        if (count >= rank) bound = trial;
    }
    return bound;
}

template<int WAVES>
struct top_shared {
    uint64_t packed[kPacked + 8];
    uint32_t count;  // of packed keys, beyond what fits, so that it is known
    uint32_t bound[WAVES];
    float reduce[WAVES], sum[WAVES];
};

// Lanes with a key of a wave append it.
template<int WAVES>
__device__ __forceinline__ void append(top_shared<WAVES> &s, bool mine, uint64_t key) {
    const uint64_t all = __ballot(mine);
    uint32_t base = 0;
    if ((threadIdx.x & 63) == 0) base = atomicAdd(&s.count, (uint32_t)__popcll(all));
    base = __builtin_amdgcn_readfirstlane(base);
    const uint32_t place = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
    if (mine && place < kPacked) s.packed[place] = key;
}

// the packed keys -> the k largest in order, by counting the larger ones
template<int WAVES, class Write>
__device__ __forceinline__ void write_ranked(top_shared<WAVES> &s, uint32_t count, uint32_t k, Write write) {
    if (threadIdx.x < 8) s.packed[count + threadIdx.x] = 0;  // whole eights
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += WAVES * 64) {
        const uint64_t key = s.packed[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; j += 8) {
#pragma unroll
            for (int u = 0; u < 8; u++) rank += s.packed[j + u] > key;
        }
        if (rank < k) write(rank, key);
    }
}

template<int WAVES>
__device__ __forceinline__ uint32_t block_count(uint32_t v, top_shared<WAVES> &s) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) v += __shfl_xor((int)v, step);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.bound[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) v += s.bound[i];
    return v;
}

// The exact way.  The least threshold found, from the highest bit down, that at least `want` keys reach and no more than can be packed; all
// 64 bits end at the want-th largest key itself.  Then those keys, packed.
template<int WAVES, class Each>
__device__ __forceinline__ uint32_t collect_exactly(top_shared<WAVES> &s, uint32_t want, Each each) {
    uint64_t threshold = 0;
    for (int bit = 63; bit >= 0; bit--) {
        const uint64_t trial = threshold | 1ull << bit;
        uint32_t reached = 0;
        each([&](bool valid, uint64_t key) { reached += valid && key >= trial; });
        reached = block_count(reached, s);
        if (reached < want) continue;
        threshold = trial;
        if (reached <= kPacked) break;
    }
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    each([&](bool valid, uint64_t key) { append(s, valid && key >= threshold, key); });
    __syncthreads();
    return min(s.count, kPacked);
}

// For each of N parts of a thread's elements one of them, as large as comes cheap: the largest, or — bf16, compared two at a time as 16-bit
// whole numbers — the largest where any is positive (or a NaN, which hides it), else some element.
template<class T>
constexpr bool representative_is_largest() { return !__is_same(T, __bf16); }

template<class T, int U, int N>
__device__ __forceinline__ void representatives(const uint4 (&raw)[U], float (&part)[N]) {
    constexpr int E = per_chunk<T>::value;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) part[i] = -kInfinity;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[E];
            unpack<T>(raw[u], x);
#pragma unroll
            for (int i = 0; i < E; i++) part[(u * E + i) * N / (U * E)] = fmaxf(part[(u * E + i) * N / (U * E)], x[i]);
        }
    } else {
        typedef short pair_bits __attribute__((ext_vector_type(2)));
        typedef _Float16 pair_f16 __attribute__((ext_vector_type(2)));
        uint32_t best[N];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t word[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                constexpr int words = U * 4 / N;
                const int p = (u * 4 + i) / words;
                if ((u * 4 + i) % words == 0) best[p] = word[i];
                else if constexpr (__is_same(T, __bf16))
                    best[p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair_bits, best[p]), __builtin_bit_cast(pair_bits, word[i])));
                else
                    best[p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair_f16, best[p]), __builtin_bit_cast(pair_f16, word[i])));
            }
        }
#pragma unroll
        for (int p = 0; p < N; p++) {
            T t[2];
            __builtin_memcpy(t, &best[p], 4);
            part[p] = fmaxf(to_float(t[0]), to_float(t[1]));
        }
    }
}

// The same for bf16 parts that hold nothing positive, where signed whole numbers stand in reverse: as unsigned ones the largest is the least.
// With their least elements in place of the largest nearly everything reaches the bound and the exact way follows: top 64 of 1024 x 1M bf16 from
// N(-10, 2) 5740 us against 414, log-probabilities around -14 6650 against 474; a wave asks for it only where its bound would not be
// positive (N(0, 2): 473 us, 476 without the question).
template<int U, int N>
__device__ __forceinline__ void negative_representatives(const uint4 (&raw)[U], float (&part)[N]) {
    typedef unsigned short pair_bits __attribute__((ext_vector_type(2)));
    constexpr int words = U * 4 / N;
    uint32_t least[N];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t word[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = (u * 4 + i) / words;
            if ((u * 4 + i) % words == 0) least[p] = word[i];
            else least[p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(pair_bits, least[p]), __builtin_bit_cast(pair_bits, word[i])));
        }
    }
#pragma unroll
    for (int p = 0; p < N; p++) {
        __bf16 t[2];
        __builtin_memcpy(t, &least[p], 4);
        if (!(part[p] >= 0)) part[p] = fmaxf(to_float(t[0]), to_float(t[1]));
    }
}

struct top_output {
    float *values;
    int32_t *index;
    float *stats;      // [rows][2] or null
    uint64_t *lists;   // [rows][slices][capacity] (more than one slice)
    uint32_t *counts;  // [rows][slices]
    float2 *partial;   // [rows][slices]
};

// One slice of one row: U chunks to a thread, in registers; N maxima to a thread.
template<class T, int U, int N>
__global__ void __launch_bounds__(kTopThreads) top_kernel(const T *logits, int64_t stride, int64_t first_row, uint32_t slices, int64_t num_col, uint32_t k,
                                                          uint32_t capacity, float scale, top_output out) {
    constexpr int E = per_chunk<T>::value;
    __shared__ top_shared<kTopWaves> s;
    __shared__ uint4 kept[kKept][kTopThreads];
    const int64_t row = first_row + blockIdx.x / slices;
    const uint32_t slice = blockIdx.x % slices, wave = threadIdx.x >> 6;
    const chunked_row<T> z(logits + row * stride, num_col);
    // slices of equal length, in whole cache lines: a short last one would give few maxima and a poor bound
    const int64_t chunks = z.chunks(), share = ((chunks + slices - 1) / slices + 7) & ~(int64_t)7;
    const int64_t chunk0 = min(chunks, share * slice), chunk1 = min(chunks, chunk0 + share);
    const auto load = [&](int u) {
        const int64_t chunk = chunk0 + u * kTopThreads + threadIdx.x;
        return z.load(chunk < chunk1 ? chunk : chunks);  // the one behind the last reads as minus infinity
    };
    uint4 raw[U];
    z.template load<U, kTopThreads>(raw, chunk0, chunk1);
    float part[N];
    representatives<T>(raw, part);
    const int rank = (int)((k + kTopWaves - 1) / kTopWaves);
    if constexpr (!representative_is_largest<T>()) {
        int positive = 0;
#pragma unroll
        for (int i = 0; i < N; i++) positive += __popcll(__ballot(part[i] >= 0));
        if (positive < rank) negative_representatives(raw, part);  // the wave's bound is one of these
    }
    float largest = part[0];
    uint32_t part_ordered[N];
#pragma unroll
    for (int i = 0; i < N; i++) part_ordered[i] = ordered(part[i]), largest = fmaxf(largest, part[i]);
    const uint32_t bound = wave_bound(part_ordered, rank);
    largest = wave_max(largest);
    if ((threadIdx.x & 63) == 0) s.bound[wave] = bound, s.reduce[wave] = largest;
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    float m = s.reduce[0];
    uint32_t least = s.bound[0];
#pragma unroll
    for (int w = 1; w < kTopWaves; w++) least = min(least, s.bound[w]), m = fmaxf(m, s.reduce[w]);
    // A hair below the bound, so that what reaches it lies above, 0 and -0 alike.  Without a bound (cut bits may make a NaN of minus
    // infinity's key) the exact way follows.
    const bool bounded = least > 0x0080ffffu;
    const float below = uniform(of_ordered((bounded ? least : 0x80000000u) - 16)), base = uniform(reference_of(m));
    float sum = 0;
    // What reaches the bound: a bit per element, and the chunk it is in goes to LDS (registers take no index), a few of a thread's.  What lies outside the row is minus infinity and does not; a NaN, and infinity less
    // infinity, are NaN in the sum too and take the exact way.
    constexpr int kWords = (U * E + 31) / 32;
    uint32_t hits[kWords] = {}, chunk_hits = 0, chunk_place = threadIdx.x;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[E];
        // 16-bit logits are unpacked again, rather than kept unpacked: 78 registers, not 152 (when it was chosen, 1024 x 1M bf16: 577 us against 631)
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(raw[u].x), "+v"(raw[u].y), "+v"(raw[u].z), "+v"(raw[u].w), "+v"(sum));
        else asm volatile("" : "+v"(sum), "+v"(hits[0]), "+v"(hits[kWords - 1]));
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < E; i++) {
            sum += exp2_fast((x[i] - base) * scale);
            uint32_t &word = hits[(u * E + i) / 32];
            word = __builtin_amdgcn_alignbit(word, __float_as_uint(below - x[i]), 31);  // the sign's bit, from below
        }
        if (hits[u * E / 32] & ((1u << E) - 1)) {
            if (u < (int)kKept || chunk_place < kKept * kTopThreads) (&kept[0][0])[chunk_place] = raw[u];
            chunk_place += kTopThreads, chunk_hits |= 1u << u;
        }
    }
    // Where the elements stand in LDS and in the slice is packed: one addition to the workgroup's count for a wave.
    uint32_t mine = 0;
#pragma unroll
    for (int w = 0; w < kWords; w++) mine += __popc(hits[w]);
    uint32_t place = wave_scan(mine);
    uint32_t before = 0;
    if ((threadIdx.x & 63) == 63) before = atomicAdd(&s.count, place);
    place += (uint32_t)__builtin_amdgcn_readlane((int)before, 63) - mine;
#pragma unroll
    for (int w = 0; w < kWords; w++) {
        while (hits[w]) {
            const uint32_t first = __clz(hits[w]), e = w * 32 + first - (32 - min(32, U * E - w * 32)), u = e / E;  // the word's bits end with its lowest
            hits[w] &= ~(0x80000000u >> first);
            const uint32_t slot = __popc(chunk_hits & ((1u << u) - 1));
            if (place < kPacked) s.packed[place] = (uint64_t)(slot < kKept ? ((slot * kTopThreads + threadIdx.x) * E + e % E) : ~0u) << 32 | ((u * kTopThreads + threadIdx.x) * E + e % E);
            place++;
        }
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) s.sum[wave] = sum;  // not s.reduce: a slower wave may still read its maxima there
    __syncthreads();
    sum = s.sum[0];
#pragma unroll
    for (int w = 1; w < kTopWaves; w++) sum += s.sum[w];
    uint32_t count = s.count;
    if (count > kPacked || sum != sum || !bounded) {
        const int64_t begin = max((int64_t)0, z.first(chunk0)), end = min(num_col, z.first(chunk1));
        count = collect_exactly(s, (uint32_t)min((int64_t)k, max((int64_t)0, end - begin)), [&](auto visit) {
#pragma unroll 1
            for (int u = 0; u < U; u++) {  // read again: registers take no index
                float x[E];
                unpack<T>(load(u), x);
                const int64_t at = z.first(chunk0 + u * kTopThreads + threadIdx.x);
#pragma unroll
                for (int i = 0; i < E; i++) visit(at + i >= 0 && at + i < end, key_of(x[i], (uint32_t)(at + i)));
            }
        });
        if constexpr (!representative_is_largest<T>()) {  // a NaN among a thread's elements hides their largest
            float largest = -kInfinity;
#pragma unroll 1
            for (int u = 0; u < U; u++) {
                float x[E];
                unpack<T>(load(u), x);
#pragma unroll
                for (int i = 0; i < E; i++) largest = fmaxf(largest, x[i]);
            }
            m = block_max<kTopThreads>(largest, s.reduce);
        }
    } else {
        const T *const elements = reinterpret_cast<const T *>(kept);
        for (uint32_t i = threadIdx.x; i < count; i += kTopThreads) {
            const uint64_t it = s.packed[i];
            const uint32_t at = (uint32_t)z.first(chunk0) + (uint32_t)it, from = (uint32_t)(it >> 32);
            s.packed[i] = key_of(to_float(from == ~0u ? z.row[at] : elements[from]), at);
        }
    }
    if (slices == 1) {
        write_ranked(s, count, k, [&](uint32_t rank, uint64_t key) {
            out.values[row * k + rank] = of_ordered((uint32_t)(key >> 32));
            out.index[row * k + rank] = (int32_t)~(uint32_t)key;
        });
        if (out.stats && threadIdx.x == 0) out.stats[2 * row] = m, out.stats[2 * row + 1] = logf(sum);
        return;
    }
    const uint64_t list = (uint64_t)blockIdx.x;
    uint64_t *const keys = out.lists + list * capacity;
    if (count <= capacity) {
        for (uint32_t i = threadIdx.x; i < count; i += kTopThreads) keys[i] = s.packed[i];
    } else {
        write_ranked(s, count, k, [&](uint32_t rank, uint64_t key) { keys[rank] = key; });
        count = k;
    }
    if (threadIdx.x == 0) out.counts[list] = count, out.partial[list] = make_float2(m, sum);
}

// The lists of a row's slices -> its top entries and statistics.  CACHED keys to a thread hold all the lists, which are read once;
// the lists' 64-entry pieces are dealt to the waves in turn, from another wave on every time (a list's last pieces are emptier than its
// first).  CACHED 0: a wave takes every eighth list, several at a time, and reads them twice.  The bound is the k-th largest of all threads'
// largest keys.
template<int CACHED>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(int64_t first_row, uint32_t slices, uint32_t k, uint32_t log_capacity, float scale, top_output out) {
    __shared__ top_shared<kMergeWaves> s;
    __shared__ uint32_t maxima[kMergeThreads];
    const int64_t row = first_row + blockIdx.x;
    const uint64_t list0 = (uint64_t)blockIdx.x * slices;
    const uint64_t *const keys = out.lists + (list0 << log_capacity);
    const uint32_t *const counts = out.counts + list0;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, slots = slices << log_capacity;
    uint64_t cached[CACHED ? CACHED : 1] = {};  // no key is 0
    if constexpr (CACHED > 0) {
        uint32_t length[CACHED];
        const auto slot = [&](uint32_t r) { return r * kMergeThreads + ((wave + r) % kMergeWaves) * 64 + lane; };
#pragma unroll
        for (int r = 0; r < CACHED; r++) length[r] = slot(r) < slots ? counts[slot(r) >> log_capacity] : 0;
#pragma unroll
        for (int r = 0; r < CACHED; r++)
            if ((slot(r) & ((1u << log_capacity) - 1)) < length[r]) cached[r] = keys[slot(r)];
    }
    const auto each = [&](auto visit) {
        if constexpr (CACHED > 0) {
#pragma unroll
            for (int r = 0; r < CACHED; r++)
                if (r * kMergeThreads < slots) visit(cached[r] != 0, cached[r]);
            return;
        }
        constexpr int kTogether = 4;
        for (uint32_t l = wave; l < slices; l += kMergeWaves * kTogether) {
            uint32_t count[kTogether], longest = 0;
#pragma unroll
            for (int t = 0; t < kTogether; t++) {
                count[t] = l + t * kMergeWaves < slices ? counts[l + t * kMergeWaves] : 0;
                longest = max(longest, count[t]);
            }
            for (uint32_t j = lane; j < ((longest + 63) & ~63u); j += 64) {
                uint64_t key[kTogether];
#pragma unroll
                for (int t = 0; t < kTogether; t++) key[t] = j < count[t] ? keys[((uint64_t)(l + t * kMergeWaves) << log_capacity) + j] : 0;
#pragma unroll
                for (int t = 0; t < kTogether; t++) visit(j < count[t], key[t]);
            }
        }
    };
    if (threadIdx.x == 0) s.count = 0;
    const float2 part = threadIdx.x < slices ? out.partial[list0 + threadIdx.x] : make_float2(-kInfinity, 0.0f);
    uint32_t largest = 0;
    each([&](bool valid, uint64_t key) {
        if (valid) largest = max(largest, (uint32_t)(key >> 32));
    });
    maxima[threadIdx.x] = largest;
    float m = part.x, sum = 0;
    for (uint32_t i = threadIdx.x + kMergeThreads; i < slices; i += kMergeThreads) m = fmaxf(m, out.partial[list0 + i].x);
    m = block_max<kMergeThreads>(m, s.reduce);  // its barriers publish the maxima too
    const float base = reference_of(m);
    for (uint32_t i = threadIdx.x; i < slices; i += kMergeThreads) {
        const float2 p = i == threadIdx.x ? part : out.partial[list0 + i];
        if (p.x > -kInfinity || p.y != p.y) sum += p.y * exp2_fast((reference_of(p.x) - base) * scale);  // not a slice of nothing but masks
    }
    uint32_t all[kMergeWaves];
#pragma unroll
    for (int i = 0; i < kMergeWaves; i++) all[i] = maxima[i * 64 + lane];
    const uint32_t least = wave_bound(all, (int)k);
    each([&](bool valid, uint64_t key) {
        const bool reaches = valid && (uint32_t)(key >> 32) >= least;
        if (__any(reaches)) append(s, reaches, key);
    });
    sum = block_sum<kMergeThreads>(sum, s.reduce);  // its barriers publish the keys and their count
    uint32_t count = s.count;
    if (count > kPacked) count = collect_exactly(s, k, each);
    write_ranked(s, count, k, [&](uint32_t rank, uint64_t key) {
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
    // workspace of rows longer than a workgroup holds
    float2 *partial;   // [rows][slices]: max and sum
    float4 *factors;   // [rows]: what the exponent subtracts, w Q / (T S), 0 (16 bytes: one load, and what follows stays aligned), 1 where there is nothing to learn
    int32_t *index;    // [rows][k]: candidates with a share of q, each once; -1: none
    float *q;          // [rows][k]: w q / T
};

template<int THREADS>
struct list_shared {
    alignas(16) int32_t index[kMaxList];  // -1 where the list has no entry
    float q[kMaxList];        // first the logits, then the probabilities
    float largest[THREADS / 64], listed[THREADS / 64], sum[THREADS / 64], listed_sum[THREADS / 64], q_total[THREADS / 64], loss[THREADS / 64];
    uint32_t bad[THREADS / 64], any[THREADS / 64], repeated[THREADS / 64];
};

struct row_answer {
    float m, sum, log_sum, q_total, loss;
    bool nothing, repeated;
};

// A row and its list, by a workgroup: three reductions of two numbers each, three barriers.
//   largest() / sum(base)   a thread's part of max z and of S
//   seen(i)                 whether candidate i was listed before (by an entry that got there first)
//   logit(i)                z_i
//   place(e, i)             called for every entry and its candidate, before the last barrier
// An index outside the row makes the row's answer NaN: it shows, and nothing is read or written out of bounds.  Nothing is to be
// learned from a row without entries, whatever its logits hold, nor from one whose candidates are all masked: loss and gradient 0.
template<int THREADS, class Largest, class Sum, class Seen, class Logit, class Place>
__device__ __forceinline__ row_answer solve_row(const distill_input &in, int64_t row, list_shared<THREADS> &s, Largest largest, Sum sum, Seen seen, Logit logit, Place place) {
    constexpr int WAVES = THREADS / 64;
    const uint32_t wave = threadIdx.x >> 6;
    const bool first_lane = (threadIdx.x & 63) == 0;
    const int32_t *const index = in.index + row * in.k;
    const float *const teacher = in.teacher + row * in.k;
    bool bad = false, any = false, repeated = false;
    float t_largest = -kInfinity;
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {
        const int32_t i = index[e];
        const float t = teacher[e];
        const bool inside = i >= 0 && i < in.num_col, entry = inside && !(t == -kInfinity);
        bad |= !inside && i != -1;
        any |= entry;
        s.index[e] = entry ? i : -1;
        s.q[e] = t;
        if (entry) t_largest = fmaxf(t_largest, t);
    }
    float mine = wave_max(largest());
    t_largest = wave_max(t_largest);
    bad = __any(bad), any = __any(any);
    if (first_lane) s.largest[wave] = mine, s.listed[wave] = t_largest, s.bad[wave] = bad, s.any[wave] = any;
    __syncthreads();
    row_answer r;
    r.m = s.largest[0], t_largest = s.listed[0];
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        r.m = fmaxf(r.m, s.largest[w]), t_largest = fmaxf(t_largest, s.listed[w]);
        bad |= s.bad[w] != 0, any |= s.any[w] != 0;
    }
    const float mt = in.teacher_stats ? in.teacher_stats[2 * row] : reference_of(t_largest);
    float t_sum = 0;
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {  // a thread's own entries
        const int32_t i = s.index[e];
        if (i < 0) continue;
        repeated |= seen(i);
        if (!in.teacher_stats) t_sum += expf((s.q[e] - mt) / in.temperature);
    }
    mine = wave_sum(sum(reference_of(r.m)));
    t_sum = wave_sum(t_sum);
    repeated = __any(repeated);
    if (first_lane) s.sum[wave] = mine, s.listed_sum[wave] = t_sum, s.repeated[wave] = repeated;
    __syncthreads();
    r.sum = s.sum[0], t_sum = s.listed_sum[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) r.sum += s.sum[w], t_sum += s.listed_sum[w];
#pragma unroll
    for (int w = 0; w < WAVES; w++) repeated |= s.repeated[w] != 0;
    r.log_sum = logf(r.sum), r.repeated = repeated;
    const float lt = in.teacher_stats ? in.teacher_stats[2 * row + 1] : logf(t_sum), inverse = 1.0f / t_sum;
    float q_total = 0, loss = 0;
    for (uint32_t e = threadIdx.x; e < in.k; e += THREADS) {
        const int32_t i = s.index[e];
        float q = 0;
        if (i >= 0) {
            const float shifted = (s.q[e] - mt) / in.temperature;
            q = in.teacher_stats ? expf(shifted - lt) : expf(shifted) * inverse;
            if (!(q == 0)) loss += q * ((shifted - lt) - ((logit(i) - r.m) / in.temperature - r.log_sum));  // 0 log 0 = 0
            place(e, i);
        }
        s.q[e] = q;
        q_total += q;
    }
    q_total = wave_sum(q_total), loss = wave_sum(loss);
    if (first_lane) s.q_total[wave] = q_total, s.loss[wave] = loss;
    __syncthreads();
    r.q_total = s.q_total[0], r.loss = s.loss[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) r.q_total += s.q_total[w], r.loss += s.loss[w];
    r.nothing = !bad && (!any || (r.m == -kInfinity && r.sum == r.sum));
    if (bad) r.q_total = r.loss = __builtin_nanf("");
    if (r.nothing) r.loss = 0;
    return r;
}

// Where a candidate is listed more than once: the sum of its entries' q to the first of them, in the list's order, so that the answer is
// the same every time.  write(e, i, q): q for the first, the others get none.
template<int THREADS, class Write>
__device__ __forceinline__ void join_repeated(uint32_t k, const list_shared<THREADS> &s, Write write) {
    for (uint32_t e = threadIdx.x; e < k; e += THREADS) {
        const int32_t i = s.index[e];
        if (i < 0) continue;
        bool first = true;
        float q = s.q[e];
        for (uint32_t at = 0; at < k; at += 4) {
            const int4 four = *reinterpret_cast<const int4 *>(s.index + at);
            const int32_t index[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (index[u] != i || at + u >= k) continue;
                if (at + u < e) first = false;
                if (at + u > e) q += s.q[at + u];
            }
        }
        if (first) write(e, i, q);
    }
}

// What the gradient of a stretch of elements takes from the list: a bit per element that has a share, and which entry of the list holds it.
template<int SIZE>
struct listed_slice {
    uint32_t bits[SIZE / 32 + 1];
    uint16_t share[SIZE];
};

// gradient of a chunk: p_factor = w Q / (T S); share(place) is subtracted where the list has one
template<class T, class Share>
__device__ __forceinline__ void chunk_gradient(const uint4 raw, int place, float base, float scale, float p_factor, bool nothing, const uint32_t *bits, Share share,
                                               float g[per_chunk<T>::value]) {
    constexpr int E = per_chunk<T>::value;
    float x[E];
    unpack<T>(raw, x);
#pragma unroll
    for (int i = 0; i < E; i++) g[i] = nothing ? 0.0f : exp2_fast((x[i] - base) * scale) * p_factor;
    // a chunk's place in the stretch is a multiple of E, E divides 32: its bits lie in one word
    const uint32_t mine = bits[place >> 5] >> (place & 31) & ((1u << E) - 1);
    if (mine && !nothing) {
#pragma unroll
        for (int i = 0; i < E; i++)
            if (mine >> i & 1) g[i] -= share(place + i);
    }
}

// Rows that fit a workgroup's registers: read once, written once, one launch.  U chunks to a thread.  What bounds many rows is how many of them
// a CU holds (they wait for their loads and three barriers each): few threads with many chunks, builds near the row's length, the
// list's entries by their 16-bit place.  4000 x 10312 bf16, k = 64, a step: 38 us (44 where lists name candidates twice); 1024 threads, 16384 elements and
// shares of 32 bits, when it was chosen: 89.  4000 x 16000 f32 98 (5.2 TB/s) against 134; a few rows are no slower (50 x 10312 f32: 9.4).
template<class T, int THREADS, int U, bool GRAD>
__global__ void __launch_bounds__(THREADS) distill_row_kernel(distill_input in, distill_output out, int64_t first_row) {
    constexpr int E = per_chunk<T>::value, SIZE = THREADS * U * E;
    __shared__ list_shared<THREADS> s;
    __shared__ listed_slice<GRAD ? SIZE : 32> l;
    const int64_t row = first_row + blockIdx.x;
    const chunked_row<T> z((const T *)in.logits + row * in.stride, in.num_col);
    uint4 raw[U];
    z.template load<U, THREADS>(raw, 0, z.chunks());
    if constexpr (GRAD)
        for (int i = threadIdx.x; i < SIZE / 32 + 1; i += THREADS) l.bits[i] = 0;
    const row_answer r = solve_row<THREADS>(
        in, row, s,
        [&] {
            float largest = -kInfinity;
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[E];
                unpack<T>(raw[u], x);
#pragma unroll
                for (int i = 0; i < E; i++) largest = fmaxf(largest, x[i]);
            }
            return largest;
        },
        [&](float base) {
            float sum = 0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[E];
                unpack<T>(raw[u], x);
#pragma unroll
                for (int i = 0; i < E; i++) sum += exp2_fast((x[i] - base) * in.scale);
            }
            return sum;
        },
        [&](int32_t i) {
            if constexpr (!GRAD) return false;
            const int at = i + z.lead;
            const uint32_t bit = 1u << (at & 31);
            return (atomicOr(&l.bits[at >> 5], bit) & bit) != 0;
        },
        [&](int32_t i) { return to_float(z.row[i]); },
        [&](uint32_t e, int32_t i) {
            if constexpr (GRAD) l.share[i + z.lead] = (uint16_t)e;
        });
    if (threadIdx.x == 0) {
        out.loss[row] = r.loss;
        out.stats[2 * row] = r.m, out.stats[2 * row + 1] = r.log_sum;
    }
    if constexpr (GRAD) {
        if (r.repeated) {
            // in place: of a candidate's entries only the first one's q changes, and no other thread reads that
            join_repeated(in.k, s, [&](uint32_t e, int32_t i, float q) { s.q[e] = q, l.share[i + z.lead] = (uint16_t)e; });
            __syncthreads();
        }
        const float base = reference_of(r.m), q_factor = (in.weight ? in.weight[row] : 1.0f) / in.temperature, p_factor = q_factor * r.q_total / r.sum;
        T *grad = (T *)out.grad + row * out.grad_stride;
        const bool wide = (uintptr_t)grad % 16 == (uintptr_t)z.row % 16;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int place = (u * THREADS + (int)threadIdx.x) * E;
            float g[E];
            chunk_gradient<T>(raw[u], place, base, in.scale, p_factor, r.nothing, l.bits, [&](int at) { return s.q[l.share[at]] * q_factor; }, g);
            store_chunk<T>(grad, (int64_t)place - z.lead, in.num_col, wide, g);
        }
    }
}

// Longer rows, in slices: max and sum of every slice; then, a workgroup per row, those joined and the list; then the gradient of every
// slice, with nothing left to do per row but to find the slice's entries.
// Slices of 4096 / 8192 / 16384 logits: the loss of 500 x 99991 f16 25.3 / 24.1 / 25.8 us, the step of 512 x 1M bf16 577 / 581 / 562, of 256 x 1M f32
// 577 / 554 / 561, of 300 x 40000 f32 39.0 / 38.2 / 42.7, of 300 x 20000 bf16 25.6 / 28.0 / 32.2.
constexpr int kSliceThreads = 256, kSliceElements = 8192;

template<class T>
constexpr int slice_chunks() {
    return kSliceElements / kSliceThreads / per_chunk<T>::value;
}

template<class T>
__global__ void __launch_bounds__(kSliceThreads) distill_partial_kernel(distill_input in, distill_output out, int64_t first_row, uint32_t slices) {
    constexpr int E = per_chunk<T>::value, U = slice_chunks<T>();
    __shared__ float reduce[kSliceThreads / 64];
    const int64_t row = first_row + blockIdx.x / slices;
    const uint32_t slice = blockIdx.x % slices;
    const chunked_row<T> z((const T *)in.logits + row * in.stride, in.num_col);
    uint4 raw[U];
    z.template load<U, kSliceThreads>(raw, (int64_t)slice * (U * kSliceThreads), z.chunks());
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

// Candidates of a list, hashed, to find out whether one is listed twice.
constexpr uint32_t kSeen = 4 * kMaxList;

template<class T, bool GIVEN>
__global__ void __launch_bounds__(kSliceThreads) distill_finish_kernel(distill_input in, distill_output out, int64_t first_row, uint32_t slices) {
    __shared__ list_shared<kSliceThreads> s;
    __shared__ int32_t table[kSeen];
    const int64_t row = first_row + blockIdx.x, local = blockIdx.x;
    const float2 *const partial = out.partial + local * slices;
    const T *const z = (const T *)in.logits + row * in.stride;
    if (out.grad)
        for (uint32_t i = threadIdx.x; i < kSeen; i += kSliceThreads) table[i] = -1;
    const row_answer r = solve_row<kSliceThreads>(
        in, row, s,
        [&] {
            if constexpr (GIVEN) return out.stats[2 * row];
            float m = -kInfinity;
            for (uint32_t i = threadIdx.x; i < slices; i += kSliceThreads) m = fmaxf(m, partial[i].x);
            return m;
        },
        [&](float base) {
            if constexpr (GIVEN) return threadIdx.x == 0 ? expf(out.stats[2 * row + 1]) : 0.0f;
            float sum = 0;
            for (uint32_t i = threadIdx.x; i < slices; i += kSliceThreads) {
                const float2 p = partial[i];
                if (p.x > -kInfinity || p.y != p.y) sum += p.y * exp2_fast((reference_of(p.x) - base) * in.scale);  // not a slice of nothing but masks
            }
            return sum;
        },
        [&](int32_t i) {
            if (!out.grad) return false;
            for (uint32_t at = (uint32_t)i * 2654435761u >> 20;; at++) {  // 12 bits; at most a quarter of the places are taken
                const int32_t was = atomicCAS(&table[at % kSeen], -1, i);
                if (was == -1) return false;
                if (was == i) return true;
            }
        },
        [&](int32_t i) { return GIVEN ? 0.0f : to_float(z[i]); }, [](uint32_t, int32_t) {});
    if (!GIVEN && threadIdx.x == 0) {
        out.loss[row] = r.loss;
        out.stats[2 * row] = r.m, out.stats[2 * row + 1] = r.log_sum;
    }
    if (!out.grad) return;
    const float q_factor = (in.weight ? in.weight[row] : 1.0f) / in.temperature;
    if (threadIdx.x == 0) out.factors[local] = make_float4(reference_of(r.m), q_factor * r.q_total / r.sum, 0.0f, r.nothing ? 1.0f : 0.0f);
    int32_t *const index = out.index + local * in.k;
    float *const q = out.q + local * in.k;
    for (uint32_t e = threadIdx.x; e < in.k; e += kSliceThreads) index[e] = r.repeated ? -1 : s.index[e], q[e] = s.q[e] * q_factor;
    if (r.repeated) join_repeated(in.k, s, [&](uint32_t e, int32_t i, float sum) { index[e] = i, q[e] = sum * q_factor; });  // a thread's own entries again
}

template<class T>
__global__ void __launch_bounds__(kSliceThreads) distill_grad_kernel(distill_input in, distill_output out, int64_t first_row, uint32_t slices) {
    constexpr int E = per_chunk<T>::value, U = slice_chunks<T>();
    __shared__ listed_slice<kSliceElements> l;
    const int64_t local = blockIdx.x / slices, row = first_row + local;
    const uint32_t slice = blockIdx.x % slices;
    const chunked_row<T> z((const T *)in.logits + row * in.stride, in.num_col);
    const int64_t chunk0 = (int64_t)slice * (U * kSliceThreads), begin = z.first(chunk0);
    uint4 raw[U];
    z.template load<U, kSliceThreads>(raw, chunk0, z.chunks());
    const float4 f = out.factors[local];
    for (int i = threadIdx.x; i < kSliceElements / 32 + 1; i += kSliceThreads) l.bits[i] = 0;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < in.k; e += kSliceThreads) {
        const int64_t at = out.index[local * in.k + e] - begin;
        if (out.index[local * in.k + e] < 0 || at < 0 || at >= kSliceElements) continue;
        l.share[at] = (uint16_t)e;
        atomicOr(&l.bits[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    T *grad = (T *)out.grad + row * out.grad_stride;
    const bool wide = (uintptr_t)grad % 16 == (uintptr_t)z.row % 16;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int place = (u * kSliceThreads + (int)threadIdx.x) * E;
        float g[E];
        chunk_gradient<T>(raw[u], place, f.x, in.scale, f.y, f.w != 0, l.bits, [&](int at) { return out.q[local * in.k + l.share[at]]; }, g);
        store_chunk<T>(grad, begin + place, in.num_col, wide, g);
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

// Slices of 8192 / 16384 logits: top 64 of 1024 x 1M bf16 515 / 414 us, of 16 x 1M bf16 40 / 21.7, top 10 of 1000 x 10312 f32 26 / 12.7 (a row is then
// two slices, two launches); top 100 of 333 x 99991 f32 goes the other way, 37 / 41, and 64 of 1000 x 20000 f32, 35.6 / 40.
constexpr int64_t kTopSlice = 16384, kTopStep = 4096;

struct top_plan {
    int64_t slice, slices;  // a row of one slice takes the shortest build that holds it
    int log_capacity;
    size_t bytes;
};

top_plan plan_top(int dtype, int64_t num_row, int64_t num_col, int k) {
    const int per_chunk = 16 / (int)size_of(dtype);
    top_plan p;
    p.slices = slices_of(num_col, kTopSlice, per_chunk);
    p.slice = kTopSlice;
    while (p.slices == 1 && p.slice > kTopStep && slices_of(num_col, p.slice - kTopStep, per_chunk) == 1) p.slice -= kTopStep;
    p.log_capacity = 6;
    while ((1 << p.log_capacity) < 2 * k) p.log_capacity++;
    p.bytes = p.slices > 1 ? (size_t)num_row * p.slices * ((8ull << p.log_capacity) + sizeof(float2) + sizeof(uint32_t)) : 0;
    return p;
}

template<class T>
void launch_top(hipStream_t stream, const top_plan &p, const T *logits, int64_t stride, int64_t first_row, int64_t num_row, int64_t num_col, int k, float scale,
                const top_output &out) {
    constexpr int kChunks = kTopStep / kTopThreads / per_chunk<T>::value;
    const dim3 grid((unsigned)(num_row * p.slices));
    // One / four maxima to a thread, 333 x 99991 f32: k = 72 39.6 / 40.4 us, 100 41.4 / 42.7, 128 48.6 / 43.8, 200 69.6 / 47.2; 512 x 1M bf16 k = 128
    // 223 / 228; 333 x 99991 bf16 k = 256 228 / 41 (too many reach the bound then).
#define GVK_TOP(STEPS)                                                                                                                                              \
    if (k <= 128)                                                                                                                                                  \
        hipLaunchKernelGGL((top_kernel<T, STEPS * kChunks, 1>), grid, dim3(kTopThreads), 0, stream, logits, stride, first_row, (uint32_t)p.slices, num_col, (uint32_t)k, \
                           1u << p.log_capacity, scale, out);                                                                                                      \
    else                                                                                                                                                           \
        hipLaunchKernelGGL((top_kernel<T, STEPS * kChunks, 4>), grid, dim3(kTopThreads), 0, stream, logits, stride, first_row, (uint32_t)p.slices, num_col, (uint32_t)k, \
                           1u << p.log_capacity, scale, out)
    if (p.slice == kTopStep) GVK_TOP(1);
    else if (p.slice == 2 * kTopStep) GVK_TOP(2);
    else if (p.slice == 3 * kTopStep) GVK_TOP(3);
    else GVK_TOP(4);
#undef GVK_TOP
    if (p.slices > 1) {
        const int64_t slots = p.slices << p.log_capacity;
        const dim3 rows((unsigned)num_row);
#define GVK_MERGE(CACHED) \
    hipLaunchKernelGGL((merge_kernel<CACHED>), rows, dim3(kMergeThreads), 0, stream, first_row, (uint32_t)p.slices, (uint32_t)k, (uint32_t)p.log_capacity, scale, out)
        if (slots <= 16 * kMergeThreads) GVK_MERGE(16);
        else if (slots <= 32 * kMergeThreads) GVK_MERGE(32);
        else GVK_MERGE(0);
#undef GVK_MERGE
    }
}

constexpr int64_t kRowElements = 16384;  // what the largest build of launch_rows holds: a row of 16381 f32 or 16377 16-bit logits, wherever it begins

int64_t distill_slices(int dtype, int64_t num_col) { return slices_of(num_col, kSliceElements, 16 / (int)size_of(dtype)); }

bool one_launch(int dtype, int64_t num_col) { return slices_of(num_col, kRowElements, 16 / (int)size_of(dtype)) <= 1; }

template<class T, bool GRAD>
void launch_rows(hipStream_t stream, const distill_input &in, const distill_output &out, int64_t first, unsigned rows) {
    constexpr int E = per_chunk<T>::value;
    const int64_t need = in.num_col + E - 1;
#define GVK_ROWS(THREADS, ELEMENTS) \
    hipLaunchKernelGGL((distill_row_kernel<T, THREADS, ELEMENTS / THREADS / E, GRAD>), dim3(rows), dim3(THREADS), 0, stream, in, out, first)
    if (need <= 2048) GVK_ROWS(256, 2048);
    else if (need <= 4096) GVK_ROWS(256, 4096);
    else if (need <= 6144) GVK_ROWS(256, 6144);
    else if (need <= 8192) GVK_ROWS(512, 8192);
    else if (need <= 12288) GVK_ROWS(512, 12288);
    else GVK_ROWS(512, 16384);
#undef GVK_ROWS
}

// bytes of a row's workspace: factors first, so that every part is aligned whatever the number of slices and entries
size_t distill_row_bytes(int64_t slices, int k) { return sizeof(float4) + (size_t)slices * sizeof(float2) + (size_t)k * (sizeof(int32_t) + sizeof(float)); }

template<class T>
void launch_distill(hipStream_t stream, const distill_input &in, distill_output out, int64_t num_row, int64_t slices, void *workspace) {
    if (!workspace) {
        for (int64_t first = 0; first < num_row; first += kMaxGroups) {
            const unsigned rows = (unsigned)(num_row - first < kMaxGroups ? num_row - first : kMaxGroups);
            if (out.grad) launch_rows<T, true>(stream, in, out, first, rows);
            else launch_rows<T, false>(stream, in, out, first, rows);
        }
        return;
    }
    const int64_t step = kMaxGroups / slices > 0 ? kMaxGroups / slices : 1;
    out.factors = (float4 *)workspace;
    out.partial = (float2 *)(out.factors + num_row);
    out.index = (int32_t *)(out.partial + num_row * slices);
    out.q = (float *)(out.index + num_row * in.k);
    const bool given = !out.loss;
    for (int64_t first = 0; first < num_row; first += step) {
        const unsigned rows = (unsigned)(num_row - first < step ? num_row - first : step);
        const dim3 grid(rows * (unsigned)slices), block(kSliceThreads);
        if (given) {
            hipLaunchKernelGGL((distill_finish_kernel<T, true>), dim3(rows), block, 0, stream, in, out, first, (uint32_t)slices);
        } else {
            hipLaunchKernelGGL((distill_partial_kernel<T>), grid, block, 0, stream, in, out, first, (uint32_t)slices);
            hipLaunchKernelGGL((distill_finish_kernel<T, false>), dim3(rows), block, 0, stream, in, out, first, (uint32_t)slices);
        }
        if (out.grad) hipLaunchKernelGGL((distill_grad_kernel<T>), grid, block, 0, stream, in, out, first, (uint32_t)slices);
    }
}

int launch_distill_of(const char *who, int dtype, hipStream_t stream, const distill_input &in, const distill_output &out, int64_t num_row, void *workspace) {
    const int64_t slices = distill_slices(dtype, in.num_col);
    if (dtype == GVK_F32) launch_distill<float>(stream, in, out, num_row, slices, workspace);
    else if (dtype == GVK_BF16) launch_distill<__bf16>(stream, in, out, num_row, slices, workspace);
    else launch_distill<_Float16>(stream, in, out, num_row, slices, workspace);
    return launched(who);
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
    return (size_t)num_row * distill_row_bytes(distill_slices(dtype, num_col), k);
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
    return launch_distill_of(who, dtype, (hipStream_t)stream, {logits, stride, num_col, index, teacher, teacher_stats, weight, (uint32_t)k, temperature, scale},
                             {loss, stats, grad, grad_stride, nullptr, nullptr, nullptr, nullptr}, num_row, need ? workspace : nullptr);
}

extern "C" size_t gvk_distill_grad_workspace(int dtype, int64_t num_row, int64_t num_col, int k) {
    if ((dtype != GVK_F32 && dtype != GVK_BF16 && dtype != GVK_F16) || num_row < 1 || num_col < 1 || num_col > 0x7fffffff || k < 1 || k > kMaxList) return 0;
    return (size_t)num_row * distill_row_bytes(distill_slices(dtype, num_col), k);
}

extern "C" int gvk_distill_grad(void *stream, int dtype, const void *logits, int64_t num_row, int64_t num_col, int64_t stride, int k, const int32_t *index,
                                const float *teacher, const float *teacher_stats, float temperature, const float *weight, const float *stats, void *grad,
                                int64_t grad_stride, void *workspace, size_t workspace_bytes) {
    const char *who = "gvk_distill_grad";
    int rc = check_distill(who, dtype, logits, num_row, num_col, stride, k, index, teacher, stats, grad, grad_stride);
    if (rc != GVK_OK) return rc;
    float scale;
    if ((rc = check_temperature(who, temperature, &scale)) != GVK_OK) return rc;
    if (num_row == 0) return GVK_OK;
    if (!grad) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    const size_t need = gvk_distill_grad_workspace(dtype, num_row, num_col, k);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
        return gvk_fail(GVK_EINVAL, "%s: needs a workspace of %zu bytes on a multiple of 16, %zu given", who, need, workspace ? workspace_bytes : (size_t)0);
    return launch_distill_of(who, dtype, (hipStream_t)stream, {logits, stride, num_col, index, teacher, teacher_stats, weight, (uint32_t)k, temperature, scale},
                             {nullptr, const_cast<float *>(stats), grad, grad_stride, nullptr, nullptr, nullptr, nullptr}, num_row, workspace);
}
