// What the kernels that run a quantised layer share: element conversions and
// the tiled layouts of their operands.
//
// Operands of the products are stored in tiles of 16 rows x 1024 bytes, in the
// order in which a wave's lanes hold a matrix instruction's operand: lane
// l = 16 g + r holds 16 consecutive bytes of row r.  A tile is one contiguous
// 1 KB load for a wave, and lands in LDS free of bank conflicts.  Per tile:
//   INT8   64 columns;  byte j of lane (g, r) is column 16 g + j
//   INT4  128 columns;  low nibble of byte j: column 16 g + j, high nibble:
//         column 64 + 16 g + j, so both halves of a word unpack to operands in
//         order with a shift and a mask
//   E2M1  128 columns;  columns 32 g .. 32 g + 31, even column in the low
//         nibble; the lane's one E8M0 scale is byte t % 4 of the 32-bit word
//         [row tile][t / 4][lane] for column tile t
// Rows are padded to 16 and columns to 128 (scales: 512) with zeros.
#pragma once

#include "common.hpp"

namespace icq {

constexpr int64_t kActPad = 128;        // columns of 8-bit activations are padded to this many
constexpr int64_t kMaxRows = 1048560;   // a grid's second axis ends at 65535 tiles of 16 rows

template <int DT>
__device__ __forceinline__ float half_word(uint32_t w, int hi) {
    if (DT == IC_DTYPE_BF16) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
    return f16_bits_to_f32((uint16_t)(hi ? w >> 16 : w & 0xffffu));
}

typedef float lb_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 lb_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 lb_f16x2 __attribute__((ext_vector_type(2)));

// Two fp32 values as a word of two 16-bit ones, nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack_half_words(float a, float b) {
    const lb_f32x2 v = {a, b};
    if (DT == IC_DTYPE_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, lb_bf16x2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, lb_f16x2));
}

__device__ __forceinline__ void store_from_f32(void* p, int dtype, int64_t i, float v) {
    if (dtype == IC_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == IC_DTYPE_BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)pack_half_words<IC_DTYPE_BF16>(v, 0.0f);
    else static_cast<uint16_t*>(p)[i] = f32_to_f16_bits(v);
}

typedef float lb_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int lb_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int lb_u32x2 __attribute__((ext_vector_type(2)));

// Vectors of 16 bytes at the alignment of their elements: gfx950 loads and
// stores them whole at any such address.
typedef float lb_f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int lb_u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// 16 consecutive elements of a row as fp32, zeros behind the last column.
template <int DT>
__device__ __forceinline__ void load16(const void* p, int64_t base, int64_t c0, int64_t cols, float (&v)[16]) {
    if (c0 + 16 <= cols) {
        if (DT == IC_DTYPE_F32) {
            const lb_f32x4_any* q = reinterpret_cast<const lb_f32x4_any*>(static_cast<const float*>(p) + base + c0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const lb_f32x4 t = q[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[4 * i + k] = t[k];
            }
        } else {
            const lb_u32x4_any* q = reinterpret_cast<const lb_u32x4_any*>(static_cast<const uint16_t*>(p) + base + c0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const lb_u32x4 t = q[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[8 * i + 2 * k] = half_word<DT>(t[k], 0);
                    v[8 * i + 2 * k + 1] = half_word<DT>(t[k], 1);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = c0 + i < cols ? load_as_f32(p, DT, base + c0 + i) : 0.0f;
    }
}

// N (8 or 16) consecutive elements of a row, those before the last column.
template <int DT, int N>
__device__ __forceinline__ void store_cols(void* p, int64_t base, int64_t c0, int64_t cols, const float (&v)[N]) {
    if (c0 + N <= cols) {
        if (DT == IC_DTYPE_F32) {
            lb_f32x4_any* q = reinterpret_cast<lb_f32x4_any*>(static_cast<float*>(p) + base + c0);
#pragma unroll
            for (int i = 0; i < N / 4; ++i) q[i] = lb_f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        } else {
            lb_u32x4_any* q = reinterpret_cast<lb_u32x4_any*>(static_cast<uint16_t*>(p) + base + c0);
#pragma unroll
            for (int i = 0; i < N / 8; ++i) {
                lb_u32x4 t;
#pragma unroll
                for (int k = 0; k < 4; ++k) t[k] = pack_half_words<DT>(v[8 * i + 2 * k], v[8 * i + 2 * k + 1]);
                q[i] = t;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c0 + i < cols) store_from_f32(p, DT, base + c0 + i, v[i]);
    }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace icq
