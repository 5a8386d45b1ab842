// Low-rank adapters beside a quantised product: y[m, n] += sum_r t[m, r] B_a[n, r],
// t = scale_a A_a x, with an adapter a for each row m.
#pragma once

#include "lowbit.hpp"

namespace icq {

constexpr int kMaxRank = 128;
__host__ __device__ inline int padded_rank(int rank) { return (rank + 15) / 16 * 16; }

struct Adapted {
    const int32_t* ids;      // [M], outside [0, adapters): no adapter
    float* t;                // [M, rank], of rows with an adapter
    const uint16_t* up;      // [adapters, N, rank], zeros behind an adapter's own rank
    int f16;                 // up is fp16, else bf16
    int rank;                // padded to 16
    int adapters;
};

// t for every row that has an adapter.
int launch_shrink(const Adapted& ad, const int8_t* a, int64_t ld_a, const float* sa, int64_t M, int64_t K, const void* down, int rank,
                  const float* scaling, const int32_t* offsets, const int32_t* order, hipStream_t st);

typedef float lb_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 lb_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lb_f16x8 __attribute__((ext_vector_type(8)));

// The adapter's part of four consecutive outputs of row m from column n: a dot
// product in fp32, for few rows, which seldom share an adapter.
__device__ __forceinline__ lb_f32x4 adapter_dot4(const Adapted& ad, int64_t N, int64_t m, int64_t n0) {
    lb_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    const int id = ad.ids[m];
    if (id < 0 || id >= ad.adapters) return s;
    const lb_f32x4* t = reinterpret_cast<const lb_f32x4*>(ad.t + m * ad.rank);
    const lb_u32x4* b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        b[i] = reinterpret_cast<const lb_u32x4*>(ad.up + (id * N + (n0 + i < N ? n0 + i : N - 1)) * ad.rank);
    for (int c = 0; c < ad.rank / 8; ++c) {
        const lb_f32x4 t0 = t[2 * c], t1 = t[2 * c + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const lb_u32x4 w = b[i][c];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float lo = ad.f16 ? half_word<IC_DTYPE_F16>(w[k], 0) : half_word<IC_DTYPE_BF16>(w[k], 0);
                const float hi = ad.f16 ? half_word<IC_DTYPE_F16>(w[k], 1) : half_word<IC_DTYPE_BF16>(w[k], 1);
                s[i] = __builtin_fmaf(k < 2 ? t0[2 * k] : t1[2 * k - 4], lo, s[i]);
                s[i] = __builtin_fmaf(k < 2 ? t0[2 * k + 1] : t1[2 * k - 3], hi, s[i]);
            }
        }
    }
    return s;
}

// The adapters' part of a block of 32 columns x 32 rows of y on the matrix
// cores, added to v: lane (h, r) has row `m` (row r of the block) and, as the
// operand of B, column n; v is laid out like the product's own result.  t is
// split into two 16-bit values, t = hi + lo to 2^-16 of it at least (bf16: hi by
// truncation, which cannot overflow; fp16: 22 bits, of the row brought to a
// magnitude of 1 by a power of two, since t may lie outside fp16's range).  Rows
// of one block may have different adapters: each adapter's products are formed
// with all 32 rows and added to its own.
__device__ __forceinline__ void add_adapters(const Adapted& ad, int64_t N, int m, int64_t n, int h, lb_f32x16& v) {
    int id = ad.ids[m];
    if (id >= ad.adapters) id = -1;
    const lb_f32x4* t = reinterpret_cast<const lb_f32x4*>(ad.t + (int64_t)m * ad.rank) + h * 2;
    const int64_t column = (n < N ? n : N - 1) * ad.rank + h * 8;
    unsigned long long left = __ballot(id >= 0);
    float down = 1.0f, up = 1.0f;
    if (ad.f16 && left) {
        unsigned top = 0;
        if (id >= 0) {
#pragma unroll 1
            for (int c = 0; c < ad.rank / 16; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const unsigned u = __float_as_uint(t[4 * c + (k >> 2)][k & 3]) & 0x7fffffffu;
                    top = top > u ? top : u;
                }
        }
        const unsigned other = (unsigned)__shfl_xor((int)top, 32, 64);
        top = top > other ? top : other;
        const int e = (int)(top >> 23);
        if (e >= 1 && e <= 253) {          // (else 0, subnormal, past fp32's range or not a number: as it is)
            down = __uint_as_float((unsigned)(254 - e) << 23);
            up = __uint_as_float((unsigned)e << 23);
        }
    }
    while (left) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const bool mine = id == a;
        left &= ~__ballot(mine);
        const uint16_t* b = ad.up + a * N * ad.rank + column;
        lb_f32x16 part = {};
#pragma unroll 1
        for (int c = 0; c < ad.rank / 16; ++c) {
            const lb_f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
            const lb_f32x4 t0 = mine ? t[4 * c] : zero, t1 = mine ? t[4 * c + 1] : zero;
            const lb_u32x4 w = *reinterpret_cast<const lb_u32x4*>(b + c * 16);
            lb_u32x4 hi, lo;
            if (ad.f16) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float u0 = (k < 2 ? t0[2 * k & 3] : t1[2 * k & 3]) * down, u1 = (k < 2 ? t0[(2 * k + 1) & 3] : t1[(2 * k + 1) & 3]) * down;
                    hi[k] = pack_half_words<IC_DTYPE_F16>(u0, u1);
                    lo[k] = pack_half_words<IC_DTYPE_F16>(u0 - half_word<IC_DTYPE_F16>(hi[k], 0), u1 - half_word<IC_DTYPE_F16>(hi[k], 1));
                }
                part = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lb_f16x8, w), __builtin_bit_cast(lb_f16x8, hi), part, 0, 0, 0);
                part = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lb_f16x8, w), __builtin_bit_cast(lb_f16x8, lo), part, 0, 0, 0);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float u0 = k < 2 ? t0[2 * k & 3] : t1[2 * k & 3], u1 = k < 2 ? t0[(2 * k + 1) & 3] : t1[(2 * k + 1) & 3];
                    hi[k] = __builtin_amdgcn_perm(__float_as_uint(u1), __float_as_uint(u0), 0x07060302);
                    lo[k] = pack_half_words<IC_DTYPE_BF16>(u0 - half_word<IC_DTYPE_BF16>(hi[k], 0), u1 - half_word<IC_DTYPE_BF16>(hi[k], 1));
                }
                part = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lb_bf16x8, w), __builtin_bit_cast(lb_bf16x8, hi), part, 0, 0, 0);
                part = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lb_bf16x8, w), __builtin_bit_cast(lb_bf16x8, lo), part, 0, 0, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = mine ? v[k] + part[k] * up : v[k];
    }
}

}  // namespace icq
