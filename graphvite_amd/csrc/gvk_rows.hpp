// Device code shared by the kernels over whole rows of logits or embeddings (gvk_blocks.hip, gvk_logits.hip): the three
// element types, a row seen as aligned 16-byte chunks, reductions over a workgroup.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gvk_rows {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }

// rounded once, to nearest even
template<class T>
__device__ __forceinline__ T from_float(float x) { return (T)x; }

template<class T>
struct per_chunk {
    static constexpr int value = 16 / (int)sizeof(T);
};

// A row of n elements as chunks of 16 bytes on multiples of 16 bytes: chunk c holds elements c * E - lead ... + E, those in
// front of the row and behind it read as minus infinity.  Rows may start anywhere (an odd stride of 16-bit numbers): only
// the first and the last chunk are read element by element, nothing outside the row is touched.
template<class T>
struct chunked_row {
    static constexpr int E = per_chunk<T>::value;
    const T *row;
    int64_t n;
    int lead;

    __device__ __forceinline__ chunked_row(const T *row, int64_t n) : row(row), n(n), lead((int)((uintptr_t)row % 16 / sizeof(T))) {}
    __device__ __forceinline__ int64_t chunks() const { return (n + lead + E - 1) / E; }
    __device__ __forceinline__ int64_t first(int64_t chunk) const { return chunk * E - lead; }
    __device__ __forceinline__ uint4 load(int64_t chunk) const {
        const int64_t at = first(chunk);
        if (at >= 0 && at + E <= n) return *reinterpret_cast<const uint4 *>(row + at);
        uint4 raw;
        T t[E];
#pragma unroll
        for (int i = 0; i < E; i++) t[i] = at + i >= 0 && at + i < n ? row[at + i] : (T)(-__builtin_inff());
        __builtin_memcpy(&raw, t, 16);
        return raw;
    }
    // U chunks to a thread, THREADS apart, from chunk0 on: those at chunk1 and behind read as minus infinity.  Only the first and the last can
    // lie across the row's ends, unless the slice is shorter than that: the others are asked for without a question each (when it was chosen, top 64 of
    // 512 x 1M f32: 385 us against 450).
    template<int U, int THREADS>
    __device__ __forceinline__ void load(uint4 (&raw)[U], int64_t chunk0, int64_t chunk1) const {
        const auto checked = [&](int u) {
            const int64_t chunk = chunk0 + u * THREADS + threadIdx.x;
            return load(chunk < chunk1 ? chunk : chunks());
        };
        const int64_t last = chunk0 + (U - 1) * THREADS;
        if (U > 1 && last <= chunk1 && first(last) <= n) {
            const uint4 *const from = reinterpret_cast<const uint4 *>(row + first(chunk0)) + threadIdx.x;
            if (chunk0 > 0 || lead == 0) raw[0] = from[0];
            else raw[0] = checked(0);
#pragma unroll
            for (int u = 1; u + 1 < U; u++) raw[u] = from[u * THREADS];
            raw[U - 1] = checked(U - 1);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = checked(u);
        }
    }
};

template<class T>
__device__ __forceinline__ void unpack(const uint4 raw, float x[per_chunk<T>::value]) {
    T t[per_chunk<T>::value];
    __builtin_memcpy(t, &raw, 16);
#pragma unroll
    for (int i = 0; i < per_chunk<T>::value; i++) x[i] = to_float(t[i]);
}

// chunk `at` (its first element's index) of a row of n elements <- x; the row shares its lead with the row that x came from
// where `wide`, else every element is stored by itself
template<class T>
__device__ __forceinline__ void store_chunk(T *row, int64_t at, int64_t n, bool wide, const float x[per_chunk<T>::value]) {
    constexpr int E = per_chunk<T>::value;
    T t[E];
#pragma unroll
    for (int i = 0; i < E; i++) t[i] = from_float<T>(x[i]);
    if (wide && at >= 0 && at + E <= n) {
        uint4 raw;
        __builtin_memcpy(&raw, t, 16);
        *reinterpret_cast<uint4 *>(row + at) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < E; i++)
            if (at + i >= 0 && at + i < n) row[at + i] = t[i];
    }
}

// what the lanes of a wave wrote to LDS is there for its other lanes (LDS works in order for a wave: this binds the compiler)
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// max / sum over a wave, every lane gets it: four steps inside rows of 16 lanes by DPP, two across them
template<int CONTROL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}

template<class Op>
__device__ __forceinline__ float wave_reduce(float v, Op op) {
    v = op(v, dpp<0xb1>(v));   // quad_perm [1 0 3 2]
    v = op(v, dpp<0x4e>(v));   // quad_perm [2 3 0 1]
    v = op(v, dpp<0x141>(v));  // row_half_mirror
    v = op(v, dpp<0x140>(v));  // row_mirror
    v = op(v, __shfl_xor(v, 16));
    return op(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}

__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, [](float a, float b) { return a + b; });
}

// the sum of a wave's lanes up to and with this one: inside rows of 16, then across them
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

// max / sum over a workgroup of THREADS threads, every thread gets it; `shared` holds THREADS / 64 floats.  Fixed order.
template<int THREADS>
__device__ __forceinline__ float block_max(float v, float *shared) {
    v = wave_max(v);
    __syncthreads();  // the last use of `shared` is over
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; i++) v = fmaxf(v, shared[i]);
    return v;
}

template<int THREADS>
__device__ __forceinline__ float block_sum(float v, float *shared) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; i++) v += shared[i];
    return v;
}

}  // namespace gvk_rows
