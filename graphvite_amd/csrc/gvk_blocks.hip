// Logits of query rows against a whole table of candidates held in 8 bits: gvk_block_quantize, gvk_block_dequantize,
// gvk_block_logits (include/gvk.h).
//
//   table      x[n][c] = value[n][c] * 2^(exponent[n][c / 128] - 127),  value in e4m3 (one byte), exponent one byte per block of
//              128 columns of a row: the least power of two that brings the block's largest magnitude to 448 or below.  A power of
//              two costs e4m3 nothing (its relative step is the same at every scale) and multiplies exactly.
//   logits     z[m][n] = sum_c q[m][c] * x[n][c],  q quantised by the same rule on the way in.
//
// Which matrix instruction: every e4m3 value times its power of two is a bf16 number, exactly, and the product of two of them
// is a float, exactly; the bf16 instruction adds those with an error of float sums (measured: 1.4e-8 of the result's norm
// over 128 columns).  The 8-bit instructions, with or without scales, align the products of a step to its largest one and
// drop what lies below: 1.5e-5 of the norm on normal rows, 5e-5 on rows that use e4m3's whole range (measured, all four
// shapes alike).  That is a sum in fewer than 32 bits, so the table is read in 8 bits, widened in registers by
// v_cvt_scalef32_pk_bf16_fp8 (two values an instruction, the scale applied in it) and multiplied in bf16.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gvk.h"
#include "gvk_internal.h"
#include "gvk_rows.hpp"

namespace {

using gvk_rows::from_float;
using gvk_rows::to_float;
using gvk_rows::wave_fence;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlockColumns = 128;

// exponent byte of a block from the bits of its largest magnitude (448 = 1.75 * 2^8); 255 marks a block that holds NaN or infinity
__device__ __forceinline__ uint32_t exponent_of(uint32_t largest) {
    if (largest >= 0x7f800000u) return 255;
    if (largest == 0) return 127;
    const int e = (int)(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(e, 0);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the largest of a half wave (32 lanes: one block of columns, four to a lane), of numbers below 2^31
__device__ __forceinline__ uint32_t half_wave_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));   // quad_perm [1 0 3 2]
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));   // quad_perm [2 3 0 1]
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // row_half_mirror
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));  // row_mirror
    return max(v, (uint32_t)__shfl_xor((int)v, 16));
}

// four e4m3 bytes of x * 2^(127 - exponent), rounded to nearest even; NaN bytes where the block is marked
__device__ __forceinline__ uint32_t quantise4(const float x[4], uint32_t exponent) {
    const int shift = 127 - (int)exponent;
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(x[0], shift), ldexpf(x[1], shift), 0, false);
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(x[2], shift), ldexpf(x[3], shift), packed, true);
    return exponent == 255 ? 0x7f7f7f7fu : (uint32_t)packed;
}

// columns [column, column + 4) of a row as floats, zero behind its end
template<class T>
__device__ __forceinline__ void load4(const T *row, int column, int dim, bool wide, float out[4]) {
    if (wide && column + 4 <= dim) {
        if constexpr (sizeof(T) == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(row + column);
            out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(row + column);
            const T *t = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int i = 0; i < 4; i++) out[i] = to_float(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = column + i < dim ? to_float(row[column + i]) : 0.0f;
    }
}

// One half wave per (row, block): every value is read and written once, HBM bound.
template<class T>
__global__ void __launch_bounds__(256) quantize_kernel(const T *rows, int64_t row_stride, bool wide, uint32_t num_row, int dim, int blocks,
                                                       int padded, uint8_t *values, int64_t value_stride, uint8_t *exponents) {
    for (uint64_t item = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32; item < (uint64_t)num_row * blocks; item += (uint64_t)gridDim.x * 8) {
        const uint32_t row = (uint32_t)(item / blocks), block = (uint32_t)(item % blocks);
        const int column = (int)block * kBlockColumns + (threadIdx.x & 31) * 4;
        float x[4];
        load4(rows + (int64_t)row * row_stride, column, dim, wide, x);
        const uint32_t exponent = exponent_of(half_wave_max(max(max(magnitude(x[0]), magnitude(x[1])), max(magnitude(x[2]), magnitude(x[3])))));
        if (column < padded) *reinterpret_cast<uint32_t *>(values + (int64_t)row * value_stride + column) = quantise4(x, exponent);
        if ((threadIdx.x & 31) == 0) exponents[item] = (uint8_t)exponent;
    }
}

template<class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t *values, int64_t value_stride, const uint8_t *exponents, uint32_t num_row,
                                                         int dim, int blocks, T *rows, int64_t row_stride, bool wide) {
    for (uint64_t item = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32; item < (uint64_t)num_row * blocks; item += (uint64_t)gridDim.x * 8) {
        const uint32_t row = (uint32_t)(item / blocks), block = (uint32_t)(item % blocks);
        const int column = (int)block * kBlockColumns + (threadIdx.x & 31) * 4;
        if (column >= dim) continue;
        const int packed = *reinterpret_cast<const int *>(values + (int64_t)row * value_stride + column);  // padded to 16 columns
        const int shift = (int)exponents[item] - 127;
        const float x[4] = {ldexpf(__builtin_amdgcn_cvt_f32_fp8(packed, 0), shift), ldexpf(__builtin_amdgcn_cvt_f32_fp8(packed, 1), shift),
                            ldexpf(__builtin_amdgcn_cvt_f32_fp8(packed, 2), shift), ldexpf(__builtin_amdgcn_cvt_f32_fp8(packed, 3), shift)};
        T *out = rows + (int64_t)row * row_stride + column;
        if (wide && column + 4 <= dim) {
            T t[4] = {from_float<T>(x[0]), from_float<T>(x[1]), from_float<T>(x[2]), from_float<T>(x[3])};
            if constexpr (sizeof(T) == 4)
                *reinterpret_cast<float4 *>(out) = *reinterpret_cast<const float4 *>(t);
            else
                *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(t);
        } else {
            for (int i = 0; i < 4 && column + i < dim; i++) out[i] = from_float<T>(x[i]);
        }
    }
}

// ---- the product ------------------------------------------------------------------------------------------------------------
// v_mfma_f32_16x16x32_bf16 with the TABLE as its first operand: a lane then ends with four consecutive candidates of one query
// (n = 4 * (lane / 16) + r, m = lane % 16) and stores them at once.
// Inside a block of 128 columns the order of the columns is free as long as both operands agree.  Lane group g = lane / 16 takes
// columns j * 64 + g * 16 .. + 16 for j = 0, 1 — sixteen consecutive bytes of a table row — and step s = 2 j + h of
// the four 32-column steps multiplies the half h of them.
// Queries are laid out once as the fragments of that order: [block][16-row tile][step][lane][8] bf16, 4 KB per tile and block,
// so that a wave reads a fragment as one contiguous KB, from LDS without bank conflicts.

constexpr int kFragment = 512;  // bf16 numbers of a (tile, block, step)

// the place of query column c (inside its block) of row m (inside its tile)
__device__ __forceinline__ int fragment_place(int m, int c) {
    const int j = c >> 6, g = (c >> 4) & 3, h = (c >> 3) & 1;
    return (2 * j + h) * kFragment + (g * 16 + m) * 8 + (c & 7);
}

// the four columns x of query row m, quantised, as bf16 fragments (every e4m3 value times its power of two is a bf16 number)
__device__ __forceinline__ void put_fragment(__bf16 *tile, int m, int c, const float x[4]) {
    const uint32_t exponent = exponent_of(half_wave_max(max(max(magnitude(x[0]), magnitude(x[1])), max(magnitude(x[2]), magnitude(x[3])))));
    const uint32_t packed = quantise4(x, exponent);
    const float scale = __uint_as_float(exponent << 23);
    const bf16x2 low = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(packed, scale, false);
    const bf16x2 high = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(packed, scale, true);
    uint2 both = {__builtin_bit_cast(uint32_t, low), __builtin_bit_cast(uint32_t, high)};
    *reinterpret_cast<uint2 *>(tile + fragment_place(m, c)) = both;
}

// queries -> fragments [blocks][tiles][4][64][8]; the last tile holds the last sixteen queries (moved), or zeros behind the last one
template<class T>
__global__ void __launch_bounds__(256) fragment_kernel(const T *query, int64_t query_stride, bool wide, uint32_t num_query, uint32_t tiles, int dim,
                                                       int blocks, bool moved, __bf16 *fragments) {
    const uint32_t item = blockIdx.x * 8 + threadIdx.x / 32;  // (row, block)
    const uint32_t row = item / blocks, block = item % blocks;
    if (row >= tiles * 16) return;
    const int c = (threadIdx.x & 31) * 4;
    float x[4] = {0, 0, 0, 0};
    const uint32_t from = moved && row / 16 == tiles - 1 ? num_query - 16 + row % 16 : row;
    if (from < num_query) load4(query + (int64_t)from * query_stride, (int)block * kBlockColumns + c, dim, wide, x);
    put_fragment(fragments + ((size_t)block * tiles + row / 16) * 4 * kFragment, row % 16, c, x);
}

// the lane, made where it is asked for: neither it nor what is made of it is kept in registers all along
__device__ __forceinline__ int lane_here() {
    int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
    asm volatile("" : "+v"(lane));
    return lane;
}

// until this wave's global loads have arrived, those into LDS among them (s_waitcnt vmcnt(0))
__device__ __forceinline__ void wait_for_loads() {
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
}

// the same for all but the last COUNT loads and stores (vmcnt(COUNT), its two high bits apart)
template<int COUNT>
__device__ __forceinline__ void wait_for_loads_before() {
    static_assert(COUNT > 0 && COUNT < 64);
    __builtin_amdgcn_s_waitcnt(0x0f70 | (COUNT & 15) | COUNT >> 4 << 14);
    asm volatile("" ::: "memory");
}

// __syncthreads() but for what is on its way from or to memory: this wave's use of LDS is over (lgkmcnt(0)), then everyone's
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// sixteen bytes of a table row -> the two bf16 operands of steps 2 j and 2 j + 1
__device__ __forceinline__ void widen(const uint4 raw, float scale, bf16x8 out[2]) {
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const bf16x2 low = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[2 * h + i], scale, false);
            const bf16x2 high = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[2 * h + i], scale, true);
            out[h][4 * i] = low[0], out[h][4 * i + 1] = low[1], out[h][4 * i + 2] = high[0], out[h][4 * i + 3] = high[1];
        }
    }
}

// 16 queries x 64 candidates of a wave -> logits.  A lane holds 4 x 4 consecutive candidates of one query (acc[i]: candidates
// 16 i + 4 (lane / 16) ...): stored as they are, an instruction would write 16 rows, 32 or 64 bytes in each.  They turn in the wave's
// own LDS (rows padded by 16 bytes: no bank conflicts), and an instruction then writes 16 bytes a lane along 4 or 8 rows, 256 or 128
// bytes in each — measured with the stores alone, 777 x 99991 f16: 29 us against 63, 1024 x 1M f32: 745 against 797.  Rows may begin
// anywhere: this hardware stores 16 bytes at any address (aligned ones would take 27 us of those 29).
template<class T>
struct wave_turn {
    static constexpr int pitch = 64 * (int)sizeof(T) + 16;
    uint4 bytes[16 * pitch / 16];
};

template<bool WHOLE, class T>
__device__ __forceinline__ void store_turned(wave_turn<T> &turn, T *logits, int64_t logit_stride, uint32_t m0, uint32_t num_query, uint32_t n0, uint32_t num_row,
                                             const f32x4 acc[4]) {
    constexpr int E = 16 / (int)sizeof(T), lanes = 64 / E, rows = 64 / lanes;  // lanes to a row's 64 candidates, rows to an instruction
    const int lane = lane_here();
    char *const bytes = reinterpret_cast<char *>(turn.bytes);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        T t[4] = {from_float<T>(acc[i][0]), from_float<T>(acc[i][1]), from_float<T>(acc[i][2]), from_float<T>(acc[i][3])};
        __builtin_memcpy(__builtin_assume_aligned(bytes + (lane & 15) * wave_turn<T>::pitch + (i * 16 + (lane >> 4) * 4) * (int)sizeof(T), 4 * sizeof(T)), t, sizeof(t));
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < 16 / rows; i++) {
        const int row = i * rows + lane / lanes, column = lane % lanes * E;
        const uint4 raw = *reinterpret_cast<const uint4 *>(bytes + row * wave_turn<T>::pitch + column * (int)sizeof(T));
        const uint32_t m = m0 + row, n = n0 + column;
        T *const out = logits + (int64_t)m * logit_stride + n;
        if constexpr (WHOLE) {
            __builtin_memcpy(out, &raw, 16);
            continue;
        }
        if (m >= num_query) continue;
        if (n + E <= num_row) {
            __builtin_memcpy(out, &raw, 16);
        } else {
            T t[E];
            __builtin_memcpy(t, &raw, 16);
            for (int r = 0; r < E; r++)
                if (n + r < num_row) out[r] = t[r];
        }
    }
    wave_fence();  // the next tile turns in the same place
}

// logits [m][n .. n + 4) of one lane
template<class T>
__device__ __forceinline__ void store4(T *row, uint32_t n, uint32_t num_row, const f32x4 z) {
    T t[4] = {from_float<T>(z[0]), from_float<T>(z[1]), from_float<T>(z[2]), from_float<T>(z[3])};
    if (n + 4 <= num_row) {
        __builtin_memcpy(row + n, t, sizeof(t));
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < num_row) row[n + r] = t[r];
    }
}

struct table_view {
    const uint8_t *values, *exponents;
    int64_t value_stride;
    uint32_t num_row;
    int blocks, padded;  // padded: columns a row holds, dim rounded up to 16
};

// A wave's 64 rows of a table, four tiles of sixteen, as it walks along the columns.  Rows behind the last one are the last one (read, never
// stored); for columns behind a row's end the block's last sixteen are read, and the queries' fragments are zero there: no branch and no mask, so
// that nothing waits for a load before it is used.
// The matrix operand of a tile is 16 rows x 64 bytes; read as that, a load touches 16 cache lines by half and asks the L2 for each
// twice.  So the two loads of a tile and block take whole lines, eight rows each: lane (r, g) of L0 holds row r % 8, sixteen bytes at
// 16 g (r < 8) or 64 + 16 g (r >= 8), of L1 the same of row 8 + r % 8; halves of sixteen lanes change places (a DPP move) to make the
// operands of it.  When it was chosen, 4096 x 65536 x d512, bf16: 388 -> 338 us together with the order of the workgroups, 1 x 1M x d512: 115 -> 102 us.
//
// A strip of 256 may end before its last waves begin, and a wave's 64 rows may end inside: both read the table's last row instead, and
// nothing of what they compute from it is stored.
constexpr __host__ __device__ uint32_t first_in_table(uint32_t first, uint32_t num_row) { return first < num_row ? first : num_row - 1; }
constexpr __host__ __device__ uint32_t row_of_wave(uint32_t row, uint32_t first, uint32_t num_row) {
    return row < num_row - 1 - first ? row : num_row - 1 - first;
}
constexpr bool strips_stay_inside(uint32_t num_row) {
    for (uint32_t wave = 0; wave < 256; wave += 64) {
        const uint32_t first = first_in_table((num_row - 1) / 256 * 256 + wave, num_row);
        for (uint32_t row = 0; row < 64; row++)
            if (first >= num_row || row_of_wave(row, first, num_row) >= num_row - first) return false;
    }
    return true;
}
static_assert(strips_stay_inside(1) && strips_stay_inside(64) && strips_stay_inside(65) && strips_stay_inside(256) && strips_stay_inside(257) &&
                  strips_stay_inside(448) && strips_stay_inside(449) && strips_stay_inside(0x7fffff00u),
              "a wave reads rows of the table only");

struct table_rows {
    const uint8_t *values, *exponents;  // of the strip's first row: the same for the wave
    uint32_t at[4][2], exponent[4];
    int padded, column;

    __device__ __forceinline__ table_rows(const table_view &t, uint32_t first) : padded(t.padded) {
        column = ((threadIdx.x & 63) >> 4) * 16 + (threadIdx.x & 8) * 8;
        move(t, first);
    }
    __device__ __forceinline__ void move(const table_view &t, uint32_t first) {
        const int lane = threadIdx.x & 63;
        first = __builtin_amdgcn_readfirstlane(first_in_table(first, t.num_row));
        values = t.values + (int64_t)first * t.value_stride, exponents = t.exponents + (size_t)first * t.blocks;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            at[i][0] = row_of_wave(i * 16u + (lane & 7), first, t.num_row) * (uint32_t)t.value_stride;
            at[i][1] = row_of_wave(i * 16u + 8 + (lane & 7), first, t.num_row) * (uint32_t)t.value_stride;
            exponent[i] = row_of_wave(i * 16u + (lane & 15), first, t.num_row) * t.blocks;
        }
    }
    // L0 or L1 of tile i
    __device__ __forceinline__ uint4 load(int i, int block, int half) const {
        const int c = block * kBlockColumns + column;
        return *reinterpret_cast<const uint4 *>(values + (at[i][half] + (uint32_t)min(c, padded - 16)));
    }
    __device__ __forceinline__ uint32_t exponent_byte(int i, int block) const { return exponents[exponent[i] + block]; }
    struct place {};
    __device__ __forceinline__ place at_block(int) const { return {}; }
    __device__ __forceinline__ uint4 load(place, int i, int block, int half) const { return load(i, block, half); }
    __device__ __forceinline__ uint32_t exponent_byte(place, int i, int block) const { return exponent_byte(i, block); }
    __device__ __forceinline__ float scale(int i, int block) const { return __uint_as_float(exponent_byte(i, block) << 23); }
};

// The same where all 64 rows are there: the wave's own address and one offset of the lane's serve them all.
struct whole_rows {
    const uint8_t *values, *exponents;
    int64_t stride;
    int blocks, padded;

    __device__ __forceinline__ whole_rows(const table_view &t, uint32_t first) : stride(t.value_stride), blocks(t.blocks), padded(t.padded) { move(t, first); }
    __device__ __forceinline__ void move(const table_view &t, uint32_t first) {
        first = __builtin_amdgcn_readfirstlane(first);
        values = t.values + (int64_t)first * stride, exponents = t.exponents + (size_t)first * blocks;
    }
    struct place {
        uint32_t value, exponent;
    };
    __device__ __forceinline__ place at_block(int block) const {
        const int lane = lane_here();
        return {(uint32_t)((lane & 7) * (int)stride + min(block * kBlockColumns + (lane >> 4) * 16 + (lane & 8) * 8, padded - 16)), (uint32_t)((lane & 15) * blocks)};
    }
    __device__ __forceinline__ uint4 load(const place &p, int i, int, int half) const {
        return *reinterpret_cast<const uint4 *>(values + (i * 16 + half * 8) * stride + p.value);
    }
    __device__ __forceinline__ uint32_t exponent_byte(const place &p, int i, int block) const { return (exponents + (size_t)(i * 16) * blocks + block)[p.exponent]; }
};

template<int BANKS>
__device__ __forceinline__ uint32_t take_turned(uint32_t keep, uint32_t from) {  // lanes of BANKS take the lane eight places on in their sixteen
    return (uint32_t)__builtin_amdgcn_update_dpp((int)keep, (int)from, 0x128, 0xf, BANKS, false);
}

// L0, L1 -> columns 0 ... 63 and 64 ... 127 of the sixteen rows, lane (r, g) holding row r, sixteen bytes at 16 g
__device__ __forceinline__ void change_places(uint4 &l0, uint4 &l1) {
    const uint4 a = l0, b = l1;
    l0 = uint4{take_turned<0xc>(a.x, b.x), take_turned<0xc>(a.y, b.y), take_turned<0xc>(a.z, b.z), take_turned<0xc>(a.w, b.w)};
    l1 = uint4{take_turned<0x3>(b.x, a.x), take_turned<0x3>(b.y, a.y), take_turned<0x3>(b.z, a.z), take_turned<0x3>(b.w, a.w)};
}

// up to 16 queries: the table is read once and that bounds it.  Each workgroup lays the queries out for itself (no launch
// before this one) and walks over strips of 64 candidates per wave.  1 x 1M x d128, f32: 22 us (6.0 TB/s), 16 x 1M 31 (6.2).
// A tile is what its lanes hold, hence 16 queries.  Blocks, against the kernels for many queries with a launch before them: 1 x 10312 x d128
// 7.1 us against 11.2; d512 8.8 against 11.5, 1 x 100003 13.8 against 15.4, 16 x 100003 16.2 against 16.1, 16 x 1M 122 against 119; with eight
// blocks (d1024) every workgroup's laying out costs more than the launch: 1 x 100003 26 against 23.5, 16 x 100003 30.5 against 25.
constexpr int kFewBlocks = 4;  // 512 columns: 16 KB of fragments

template<class Q, class T>
__global__ void __launch_bounds__(256) few_queries_kernel(const Q *query, int64_t query_stride, bool query_wide, uint32_t num_query, int dim,
                                                          table_view table, T *logits, int64_t logit_stride) {
    __shared__ __bf16 fragments[kFewBlocks * 4 * kFragment];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int item = threadIdx.x / 32; item < 16 * table.blocks; item += 8) {
        const int row = item % 16, block = item / 16, c = (threadIdx.x & 31) * 4;
        float x[4] = {0, 0, 0, 0};
        if (row < (int)num_query) load4(query + row * query_stride, block * kBlockColumns + c, dim, query_wide, x);
        put_fragment(fragments + block * 4 * kFragment, row, c, x);
    }
    __syncthreads();
    const uint32_t strips = (table.num_row + 63) / 64;
    for (uint32_t strip = blockIdx.x * 4 + wave; strip < strips; strip += gridDim.x * 4) {
        f32x4 acc[4] = {};
        const table_rows rows(table, strip * 64);
        for (int block = 0; block < table.blocks; block++) {
            uint4 raw[4][2];
            float scale[4];
#pragma unroll
            for (int i = 0; i < 4; i++) raw[i][0] = rows.load(i, block, 0), raw[i][1] = rows.load(i, block, 1), scale[i] = rows.scale(i, block);
#pragma unroll
            for (int i = 0; i < 4; i++) change_places(raw[i][0], raw[i][1]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                bf16x8 b[2];
#pragma unroll
                for (int h = 0; h < 2; h++) b[h] = *reinterpret_cast<const bf16x8 *>(fragments + (block * 4 + 2 * j + h) * kFragment + lane * 8);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    bf16x8 a[2];
                    widen(raw[i][j], scale[i], a);
#pragma unroll
                    for (int h = 0; h < 2; h++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[h], b[h], acc[i], 0, 0, 0);
                }
            }
        }
        const uint32_t m = lane & 15;
        if (m < num_query) {
#pragma unroll
            for (int i = 0; i < 4; i++) store4(logits + (int64_t)m * logit_stride, strip * 64 + i * 16 + (lane >> 4) * 4, table.num_row, acc[i]);
        }
    }
}

// up to 128 columns, 256 candidates and 17 queries or more: what moves is the answer, and the table once.  A wave widens 64 candidates into
// registers and walks over the queries' tiles, whose fragments (4 KB each, the same for every wave) come through L1: sixteen matrix
// instructions and 64 x 16 logits a step; the four waves of a workgroup put theirs side by side in LDS and store 256 candidates of a row
// at once.  Loads and stores of a wave come back in order, so what is loaded behind stores waits until those are in memory: the next
// tile's fragments are asked for before this tile's logits are stored, and nothing on the way is conditional, so that the wait is for
// the loads alone (the last tile and the last strip are moved back to end with the rows: some logits are computed twice, to the
// same bits).
// Rows that begin anywhere share cache lines with their neighbours' stores, and a line written in parts by two L2s, or twice by one, costs
// memory a read as well: hence the wide stores, and an XCD takes an eighth of the candidates, in order, the parts of a strip one after
// the other (777 x 99991 f16 on eight outputs in turn: 64 us with 64 candidates of a row at once and strips dealt over the XCDs, 49 with
// the strips in order, 45 with 256 candidates; 777 x 99968, whose rows begin on lines: 40).
// 1024 x 1M x d128: f32 816 us, bf16 436; when it was chosen, without the table's loads 773 and 395, the stores alone 745 and 380 in any order of them:
// the write rate of rows (5.5 TB/s) bounds it, and reads between the writes cost more than their bytes.  Waves that stay and walk over
// strips with the queries in LDS: 882 and 476.
// 16 queries x 256 candidates of a workgroup on their way from the waves' registers to memory
template<class T>
struct group_turn {
    static constexpr int pitch = 256 * (int)sizeof(T) + 16;
    uint4 bytes[2][16 * pitch / 16];
};

// ALONE: no launch before this one; a part is one or two tiles, and every workgroup lays out its own.
template<bool ALONE, class Q, class T>
__global__ void __launch_bounds__(256, ALONE ? 3 : 4) narrow_kernel(const Q *query, int64_t query_stride, bool query_wide, int dim, const __bf16 *fragments, uint32_t tiles,
                                                                    uint32_t num_query, uint32_t parts, table_view table, T *logits, int64_t logit_stride) {
    __shared__ group_turn<T> turns;
    __shared__ __bf16 own[ALONE ? 2 * 4 * kFragment : 8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t part = turn % parts, strip = xcd * (gridDim.x / 8 / parts) + turn / parts;
    if ((uint64_t)strip * 256 >= table.num_row) return;
    const uint32_t first = min(strip * 256, table.num_row - 256);
    const uint32_t begin = (uint32_t)((uint64_t)tiles * part / parts), end = (uint32_t)((uint64_t)tiles * (part + 1) / parts);
    const whole_rows rows(table, first + wave * 64);
    const auto place = rows.at_block(0);
    uint4 raw[4][2];
    uint32_t exponent[4];
#pragma unroll
    for (int i = 0; i < 4; i++) raw[i][0] = rows.load(place, i, 0, 0), raw[i][1] = rows.load(place, i, 0, 1), exponent[i] = rows.exponent_byte(place, i, 0);
    if constexpr (ALONE) {
        for (uint32_t item = threadIdx.x / 32; item < (end - begin) * 16; item += 8) {  // a half wave takes a row, four columns to a lane
            const uint32_t tile = begin + item / 16, c = (threadIdx.x & 31) * 4;
            float x[4];
            load4(query + (int64_t)(min(tile * 16, num_query - 16) + item % 16) * query_stride, (int)c, dim, query_wide, x);
            put_fragment(own + item / 16 * 4 * kFragment, item % 16, c, x);
        }
        __syncthreads();
    }
    bf16x8 a[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float scale = __uint_as_float(exponent[i] << 23);
        change_places(raw[i][0], raw[i][1]);
        widen(raw[i][0], scale, a[i]), widen(raw[i][1], scale, a[i] + 2);
    }
    bf16x8 b[4];
    const auto fetch = [&](uint32_t tile) {
        const bf16x8 *const at = reinterpret_cast<const bf16x8 *>(ALONE ? own : fragments) + (size_t)(ALONE ? tile - begin : tile) * 4 * 64 + lane;
#pragma unroll
        for (int s = 0; s < 4; s++) b[s] = at[s * 64];
    };
    constexpr int E = 16 / (int)sizeof(T), lanes = 256 / E, rows_at_once = 64 / lanes;  // lanes to a row, rows to an instruction of a wave
    fetch(begin);
    wait_for_loads();
    for (uint32_t tile = begin; tile < end; tile++) {
        f32x4 acc[4] = {};
#pragma unroll
        for (int s = 0; s < 4; s++) {
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][s], b[s], acc[i], 0, 0, 0);
        }
        fetch(min(tile + 1, end - 1));
        char *const bytes = reinterpret_cast<char *>(turns.bytes[tile & 1]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            T t[4] = {from_float<T>(acc[i][0]), from_float<T>(acc[i][1]), from_float<T>(acc[i][2]), from_float<T>(acc[i][3])};
            __builtin_memcpy(__builtin_assume_aligned(bytes + (lane & 15) * group_turn<T>::pitch + (wave * 64 + i * 16 + (lane >> 4) * 4) * (int)sizeof(T), 4 * sizeof(T)), t, sizeof(t));
        }
        __syncthreads();
        const uint32_t m0 = min(tile * 16, num_query - 16);
#pragma unroll
        for (int i = 0; i < 4 / rows_at_once; i++) {
            const int row = wave * 4 + i * rows_at_once + lane / lanes, column = lane % lanes * E;
            const uint4 raw = *reinterpret_cast<const uint4 *>(bytes + row * group_turn<T>::pitch + column * (int)sizeof(T));
            __builtin_memcpy(logits + (int64_t)(m0 + row) * logit_stride + first + column, &raw, 16);
        }
    }
}

// more columns: a workgroup makes 256 candidates x 16 * TILES queries, 64 candidates to a wave, the queries' fragments of a block of columns
// in LDS, those of the next block and its table rows on their way meanwhile: asked for at the block's start, the scheduler kept from
// moving them behind the matrix instructions, and first touched when the block is over.  Workgroups stay and take one such square after
// the other: while the last block of one is multiplied the first of the next is on its way, and the logits are stored behind those loads.
// 4096 x 65536 x d512 bf16 264 to 282 us from run to run (1040 to 975 TFLOP/s; the library's bf16 product of that shape 307), f32 323; a launch
// per square, with loads where the scheduler put them: 325 and 367 in the same runs.  d2048: 915 us, 1201 TFLOP/s; a shorter row pays for its
// stores, which a CU's other workgroup overlaps with its own products in part.
// Odd numbers of blocks change the buffers' roles from square to square, which takes a build with two squares to a turn.
template<int TILES>
constexpr int staying_groups() {  // to a CU: what registers and LDS allow
    return TILES <= 2 ? 3 : 2;
}

template<int TILES, class T, bool WHOLE, bool ODD>
__global__ void __launch_bounds__(256, staying_groups<TILES>()) logits_kernel(const __bf16 *fragments, uint32_t tiles, uint32_t num_query, table_view table,
                                                                              T *logits, int64_t logit_stride) {
    // two objects, not one array: the compiler then knows that reading one does not wait for what is on its way into the other
    constexpr int kTurns = 4 * (int)sizeof(wave_turn<T>) / 16, kStaged = TILES * 256 > kTurns ? TILES * 256 : kTurns;
    __shared__ uint4 even[kStaged], odd[kStaged];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // An XCD's workgroups take squares of up to 8 parts x 8 strips in turn, the strips first: its L2 holds what the 64 of them read.
    const uint32_t parts = (tiles + TILES - 1) / TILES, strips = ((table.num_row + 255) / 256 + 7) / 8;  // strips of an XCD
    const uint32_t xcd = blockIdx.x % 8, side = min(parts, 8u);
    uint32_t turn = blockIdx.x / 8, strip = 0, tile0 = 0;
    const auto find = [&] {  // the square of this turn or of the next that has one
        for (; turn < parts * strips; turn += gridDim.x / 8) {
            const uint32_t column = turn / (side * strips), width = min(side, parts - column * side);
            const uint32_t inside = turn - column * side * strips, row_group = inside / (width * 8), height = min(8u, strips - row_group * 8);
            const uint32_t rest = inside - row_group * width * 8;
            strip = xcd * strips + row_group * 8 + rest % height, tile0 = (column * side + rest / height) * TILES;
            if ((uint64_t)strip * 256 < table.num_row) return true;
        }
        return false;
    };
    if (!find()) return;  // the whole workgroup
    // the wave's first candidate; of a table of 64 or more the last wave's are moved back to end with it
    const auto begin = [&] { return WHOLE ? min(strip * 256 + wave * 64, table.num_row - 64) : strip * 256 + wave * 64; };
    std::conditional_t<WHOLE, whole_rows, table_rows> rows(table, begin());
    uint4 raw[4][2];
    uint32_t exponent[4];
    const auto stage = [&](uint4 *into, int block) {
        const uint32_t at = lane_here() * 8;
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const uint32_t tile = min(tile0 + i, tiles - 1);  // tiles behind the last one: computed, never stored
            const __bf16 *from = fragments + ((size_t)block * tiles + tile) * 4 * kFragment + wave * kFragment + at;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                             (__attribute__((address_space(3))) void *)&into[i * 256 + wave * 64], 16, 0, 0);
        }
    };
    bool more = true;
    const auto step = [&](const uint4 *staged, uint4 *other, int block, f32x4 (&acc)[TILES][4]) {
        meet();  // this wave's loads into LDS had landed, and now everyone's: this block is there, and the one before is done with
        const bool last = block + 1 == table.blocks;
        if (last) {
            turn += gridDim.x / 8;
            more = find();
            rows.move(table, begin());  // where there is no more: the same again, loaded for nothing
        }
        const int after = last ? 0 : block + 1;
        if (more) stage(other, after);
        uint32_t next_exponent[4];
        const auto place = rows.at_block(after);
        // a fragment is asked for RING fragments before it is used: LDS answers meanwhile
        constexpr int RING = 2;
        bf16x8 ring[RING];
        const uint4 *const mine = staged + lane_here();
        const auto fragment = [&](int t) {  // t = (step, tile)
            return __builtin_bit_cast(bf16x8, mine[((t % TILES) * 4 + t / TILES) * 64]);
        };
#pragma unroll
        for (int t = 0; t < RING && t < 4 * TILES; t++) ring[t] = fragment(t);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            bf16x8 a[4][2];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (j == 0) change_places(raw[i][0], raw[i][1]);
                widen(raw[i][j], __uint_as_float(exponent[i] << 23), a[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                raw[i][j] = rows.load(place, i, after, j);
                if (j == 0) next_exponent[i] = rows.exponent_byte(place, i, after);
            }
            __builtin_amdgcn_sched_barrier(0);  // left alone, they are asked for at the block's end and waited for at once
#pragma unroll
            for (int t = 2 * j * TILES; t < 2 * (j + 1) * TILES; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++) acc[t % TILES][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][t / TILES - 2 * j], ring[t % RING], acc[t % TILES][i], 0, 0, 0);
                if (t + RING < 4 * TILES) ring[t % RING] = fragment(t + RING);
                __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);    // four matrix instructions
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one read of LDS
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) exponent[i] = next_exponent[i];
        if (!last) wait_for_loads();
    };
    const auto square = [&](uint4 *staged, uint4 *other) {
        const uint32_t first = begin(), first_tile = tile0;
        const bool empty = strip * 256 + wave * 64 >= table.num_row;
        f32x4 acc[TILES][4] = {};
        for (int block = 0; block + 1 < table.blocks; block += 2) step(staged, other, block, acc), step(other, staged, block + 1, acc);
        if constexpr (ODD) step(staged, other, table.blocks - 1, acc);
        meet();                             // the turns lie over the fragments that everyone is done with
        __builtin_amdgcn_sched_barrier(0);  // no load moves behind the stores
        wave_turn<T> &turned = reinterpret_cast<wave_turn<T> *>(ODD ? staged : other)[wave];
        const auto store = [&](int tile) {
            const uint32_t m0 = (first_tile + tile) * 16;
            store_turned<WHOLE>(turned, logits, logit_stride, WHOLE ? min(m0, num_query - 16) : m0, num_query, first, table.num_row, acc[tile]);
        };
        // The next square's first loads are older than these stores, and loads and stores come back in order: all but the stores having
        // come back means that the loads have, and the stores go on.
        if (WHOLE && !empty && first_tile + TILES <= tiles) {
#pragma unroll
            for (int tile = 0; tile < TILES; tile++) store(tile);
            wait_for_loads_before<TILES * (int)sizeof(T)>();  // a wave's stores of a tile: 16 x 64 logits, sixteen bytes a lane
        } else {
            if (!empty) {
#pragma unroll
                for (int tile = 0; tile < TILES; tile++)
                    if (first_tile + tile < tiles) store(tile);
            }
            wait_for_loads();
        }
        __builtin_amdgcn_sched_barrier(0);
        return more;
    };
    stage(even, 0);
    const auto place = rows.at_block(0);
#pragma unroll
    for (int i = 0; i < 4; i++) raw[i][0] = rows.load(place, i, 0, 0), raw[i][1] = rows.load(place, i, 0, 1), exponent[i] = rows.exponent_byte(place, i, 0);
    wait_for_loads();
    if constexpr (ODD) {
        while (square(even, odd) && square(odd, even)) {}
    } else {
        while (square(even, odd)) {}
    }
}

bool aligned(const void *p, int64_t stride_bytes, size_t to) { return (uintptr_t)p % to == 0 && stride_bytes % (int64_t)to == 0; }

int check_rows(const char *who, int dtype, int64_t num_row, int dim, int64_t stride) {
    if (dtype != GVK_F32 && dtype != GVK_BF16 && dtype != GVK_F16) return gvk_fail(GVK_EINVAL, "%s: unknown type %d", who, dtype);
    if (num_row < 0 || num_row > GVK_MAX_BLOCK_ROWS) return gvk_fail(GVK_EINVAL, "%s: %lld rows", who, (long long)num_row);
    if (dim < 1 || dim > GVK_MAX_BLOCK_DIM) return gvk_fail(GVK_EDIM, "%s: dim must be 1 to %d, not %d", who, GVK_MAX_BLOCK_DIM, dim);
    if (stride < dim) return gvk_fail(GVK_EINVAL, "%s: a row of %d columns with a stride of %lld", who, dim, (long long)stride);
    return GVK_OK;
}

int check_table(const char *who, const void *values, int64_t value_stride, const void *exponents, int dim) {
    if (!values || !exponents) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    if (value_stride < (dim + 15) / 16 * 16) return gvk_fail(GVK_EINVAL, "%s: %d columns need a value stride of %d, not %lld", who, dim, (dim + 15) / 16 * 16, (long long)value_stride);
    if (value_stride > GVK_MAX_BLOCK_STRIDE) return gvk_fail(GVK_EINVAL, "%s: a value stride of %lld", who, (long long)value_stride);
    if (!aligned(values, value_stride, 16)) return gvk_fail(GVK_EINVAL, "%s: values and their stride must be multiples of 16 bytes", who);
    return GVK_OK;
}

dim3 item_grid(uint64_t items) {  // one half wave per item, eight to a workgroup; more items than this take turns
    const uint64_t groups = (items + 7) / 8;
    return dim3((unsigned)(groups < (1u << 20) ? groups : (1u << 20)));
}

int launched(const char *who) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? GVK_OK : gvk_fail(GVK_EHIP, "%s: %s", who, hipGetErrorString(err));
}

template<class Q, class T>
int launch_logits(hipStream_t stream, const Q *query, int64_t query_stride, uint32_t num_query, int dim, const table_view &table, T *logits,
                  int64_t logit_stride, void *workspace) {
    const bool query_wide = aligned(query, query_stride * (int64_t)sizeof(Q), 4 * sizeof(Q));
    if (num_query <= 16 && table.blocks <= kFewBlocks) {
        const uint32_t groups = (table.num_row + 255) / 256;
        hipLaunchKernelGGL((few_queries_kernel<Q, T>), dim3(groups < 2048 ? groups : 2048), dim3(256), 0, stream, query, query_stride, query_wide,
                           num_query, dim, table, logits, logit_stride);
        return launched("gvk_block_logits");
    }
    const uint32_t tiles = (num_query + 15) / 16;
    __bf16 *fragments = reinterpret_cast<__bf16 *>(workspace);
    const bool whole = num_query > 16 && table.num_row >= 64, narrow = whole && table.blocks == 1 && table.num_row >= 256;
    const auto lay_out = [&] {
        hipLaunchKernelGGL((fragment_kernel<Q>), dim3((tiles * 16 * table.blocks + 7) / 8), dim3(256), 0, stream, query, query_stride, query_wide,
                           num_query, tiles, dim, table.blocks, whole, fragments);
    };
    const uint64_t strips = ((uint64_t)table.num_row + 255) / 256;
    if (narrow) {
        // The chip holds 1024 workgroups: as many parts as make the longest row of them on one place shortest, the table's rows counting as
        // four tiles (777 x 99991: 391 strips x 5 parts of ten tiles, two in a row; 4 parts of thirteen: two in a row as well)
        uint32_t parts = 1;
        uint64_t least = ~0ull;
        for (uint32_t p = 1; p <= tiles && p <= 64; p++) {
            const uint64_t cost = ((strips + 7) / 8 * 8 * p + 1023) / 1024 * ((tiles + p - 1) / p + 4);
            if (cost < least) least = cost, parts = p;
        }
        const uint64_t grid = (strips + 7) / 8 * 8 * parts;
        if (grid > 0xffffffull) return gvk_fail(GVK_EINVAL, "gvk_block_logits: too many logits for one call");
        // Few tiles to a workgroup (50 x 10312: one): laying them out where they are used takes 1 us a tile, a launch before this one 2.5
        // (7.5 us against 10; at eight tiles, 256 x 100000, 22 against 19).
        if ((tiles + parts - 1) / parts <= 2) {
            hipLaunchKernelGGL((narrow_kernel<true, Q, T>), dim3((unsigned)grid), dim3(256), 0, stream, query, query_stride, query_wide, dim, nullptr, tiles, num_query, parts,
                               table, logits, logit_stride);
            return launched("gvk_block_logits");
        }
        lay_out();
        hipLaunchKernelGGL((narrow_kernel<false, __bf16, T>), dim3((unsigned)grid), dim3(256), 0, stream, nullptr, 0, false, dim, fragments, tiles, num_query, parts, table, logits,
                           logit_stride);
        return launched("gvk_block_logits");
    }
    lay_out();
#define GVK_LOGITS(TILES, WHOLE)                                                                                                            \
    {                                                                                                                                       \
        const uint64_t squares = (strips + 7) / 8 * 8 * ((tiles + TILES - 1) / TILES), chip = 256 * staying_groups<TILES>();               \
        if (squares > 0xffffffffull) return gvk_fail(GVK_EINVAL, "gvk_block_logits: too many logits for one call");                       \
        const dim3 grid((unsigned)(squares < chip ? squares : chip));                                                                      \
        if (table.blocks % 2)                                                                                                               \
            hipLaunchKernelGGL((logits_kernel<TILES, T, WHOLE, true>), grid, dim3(256), 0, stream, fragments, tiles, num_query, table, logits, logit_stride); \
        else                                                                                                                                \
            hipLaunchKernelGGL((logits_kernel<TILES, T, WHOLE, false>), grid, dim3(256), 0, stream, fragments, tiles, num_query, table, logits, logit_stride); \
    }
    // What is not there is computed all the same, so few tiles take few; what is there is read once for all the tiles of a square.  bf16 logits of 1M
    // candidates, d256, with two / four / eight tiles to a square: 32 queries 65 / 69 / 77 us, 64 queries 99 / 83 / 87, 128 queries 184 / 129 / 113
    // (65: 132 / 104 / 89).  A small table is too few squares of eight for the chip: 128 x 10312 x d512 12.4 / 12.7 / 15.1.
    if (!whole) GVK_LOGITS(1, false)
    else if (tiles <= 2) GVK_LOGITS(2, true)
    else if (tiles <= 4) GVK_LOGITS(4, true)
    else GVK_LOGITS(8, true)
#undef GVK_LOGITS
    return launched("gvk_block_logits");
}

template<class Q>
int launch_logits_to(hipStream_t stream, const Q *query, int64_t query_stride, uint32_t num_query, int dim, const table_view &table, int out, void *logits,
                     int64_t logit_stride, void *workspace) {
    switch (out) {
        case GVK_F32: return launch_logits(stream, query, query_stride, num_query, dim, table, (float *)logits, logit_stride, workspace);
        case GVK_BF16: return launch_logits(stream, query, query_stride, num_query, dim, table, (__bf16 *)logits, logit_stride, workspace);
        default: return launch_logits(stream, query, query_stride, num_query, dim, table, (_Float16 *)logits, logit_stride, workspace);
    }
}

}  // namespace

extern "C" int gvk_block_quantize(void *stream, int dtype, const void *rows, int64_t num_row, int dim, int64_t row_stride, uint8_t *values,
                                  int64_t value_stride, uint8_t *exponents) {
    const char *who = "gvk_block_quantize";
    int rc = check_rows(who, dtype, num_row, dim, row_stride);
    if (rc != GVK_OK) return rc;
    if (num_row == 0) return GVK_OK;
    if (!rows) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    if ((rc = check_table(who, values, value_stride, exponents, dim)) != GVK_OK) return rc;
    const int blocks = (dim + kBlockColumns - 1) / kBlockColumns, padded = (dim + 15) / 16 * 16;
    const dim3 grid = item_grid((uint64_t)num_row * blocks);
#define GVK_QUANTIZE(T)                                                                                                                    \
    hipLaunchKernelGGL((quantize_kernel<T>), grid, dim3(256), 0, (hipStream_t)stream, (const T *)rows, row_stride,                           \
                       aligned(rows, row_stride * (int64_t)sizeof(T), 4 * sizeof(T)), (uint32_t)num_row, dim, blocks, padded, values, value_stride, exponents)
    if (dtype == GVK_F32) GVK_QUANTIZE(float);
    else if (dtype == GVK_BF16) GVK_QUANTIZE(__bf16);
    else GVK_QUANTIZE(_Float16);
#undef GVK_QUANTIZE
    return launched(who);
}

extern "C" int gvk_block_dequantize(void *stream, const uint8_t *values, int64_t value_stride, const uint8_t *exponents, int64_t num_row, int dim,
                                    int dtype, void *rows, int64_t row_stride) {
    const char *who = "gvk_block_dequantize";
    int rc = check_rows(who, dtype, num_row, dim, row_stride);
    if (rc != GVK_OK) return rc;
    if (num_row == 0) return GVK_OK;
    if (!rows) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    if ((rc = check_table(who, values, value_stride, exponents, dim)) != GVK_OK) return rc;
    const int blocks = (dim + kBlockColumns - 1) / kBlockColumns;
    const dim3 grid = item_grid((uint64_t)num_row * blocks);
#define GVK_DEQUANTIZE(T)                                                                                                                 \
    hipLaunchKernelGGL((dequantize_kernel<T>), grid, dim3(256), 0, (hipStream_t)stream, values, value_stride, exponents, (uint32_t)num_row, dim, blocks, \
                       (T *)rows, row_stride, aligned(rows, row_stride * (int64_t)sizeof(T), 4 * sizeof(T)))
    if (dtype == GVK_F32) GVK_DEQUANTIZE(float);
    else if (dtype == GVK_BF16) GVK_DEQUANTIZE(__bf16);
    else GVK_DEQUANTIZE(_Float16);
#undef GVK_DEQUANTIZE
    return launched(who);
}

extern "C" size_t gvk_block_logits_workspace(int64_t num_query, int dim) {
    const int64_t blocks = (dim + kBlockColumns - 1) / kBlockColumns;
    if (num_query < 1 || dim < 1 || (num_query <= 16 && blocks <= kFewBlocks)) return 0;
    return (size_t)((num_query + 15) / 16 * blocks) * 4 * kFragment * sizeof(__bf16);
}

extern "C" int gvk_block_logits(void *stream, int query_dtype, const void *query, int64_t num_query, int64_t query_stride, const uint8_t *values,
                                int64_t value_stride, const uint8_t *exponents, int64_t num_row, int dim, int logit_dtype, void *logits,
                                int64_t logit_stride, void *workspace, size_t workspace_bytes) {
    const char *who = "gvk_block_logits";
    int rc = check_rows(who, query_dtype, num_query, dim, query_stride);
    if (rc != GVK_OK) return rc;
    if (num_query > GVK_MAX_BLOCK_QUERIES) return gvk_fail(GVK_EINVAL, "%s: %lld queries; a call takes %d", who, (long long)num_query, GVK_MAX_BLOCK_QUERIES);
    if (logit_dtype != GVK_F32 && logit_dtype != GVK_BF16 && logit_dtype != GVK_F16) return gvk_fail(GVK_EINVAL, "%s: unknown type %d", who, logit_dtype);
    if (num_row < 0 || num_row > GVK_MAX_BLOCK_ROWS) return gvk_fail(GVK_EINVAL, "%s: %lld rows", who, (long long)num_row);
    if (logit_stride < num_row) return gvk_fail(GVK_EINVAL, "%s: rows of %lld logits with a stride of %lld", who, (long long)num_row, (long long)logit_stride);
    if (num_query == 0 || num_row == 0) return GVK_OK;
    if (!query || !logits) return gvk_fail(GVK_EINVAL, "%s: null pointer", who);
    if ((rc = check_table(who, values, value_stride, exponents, dim)) != GVK_OK) return rc;
    const size_t need = gvk_block_logits_workspace(num_query, dim);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return gvk_fail(GVK_EINVAL, "%s: needs a workspace of %zu bytes on a multiple of 16, %zu given", who, need, workspace ? workspace_bytes : (size_t)0);
    const table_view table = {values, exponents, value_stride, (uint32_t)num_row, (dim + kBlockColumns - 1) / kBlockColumns, (dim + 15) / 16 * 16};
    void *const space = need ? workspace : nullptr;
    switch (query_dtype) {
        case GVK_F32: return launch_logits_to((hipStream_t)stream, (const float *)query, query_stride, (uint32_t)num_query, dim, table, logit_dtype, logits, logit_stride, space);
        case GVK_BF16: return launch_logits_to((hipStream_t)stream, (const __bf16 *)query, query_stride, (uint32_t)num_query, dim, table, logit_dtype, logits, logit_stride, space);
        default: return launch_logits_to((hipStream_t)stream, (const _Float16 *)query, query_stride, (uint32_t)num_query, dim, table, logit_dtype, logits, logit_stride, space);
    }
}
