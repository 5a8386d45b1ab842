// Low-rank adapters beside a quantised product: y[m, n] += sum_r t[m, r] B_a[n, r],
// t = scale_a A_a x, with an adapter a for each row m.
#pragma once

#include "lowbit.hpp"

namespace icq {

constexpr int kMaxRank = 128;
constexpr int kRankPart = 32;           // ranks are padded to parts of 32 with zeros
__host__ __device__ inline int rank_parts(int rank) { return (rank + kRankPart - 1) / kRankPart; }

// t is kept as two bf16 values, hi + lo (hi by truncation, which cannot overflow):
// within 2^-16 of it.  A row has 128 bytes a part, 32 values of hi and then of lo;
// behind the last row there is one of zeros.
//
// B is kept in tiles of 16 columns x 32 ranks, 1 KB, in the order of weight tiles
// (lowbit.hpp): 16 bytes a column are 8 ranks, those of 16 columns follow one
// another.  [adapter][column tile][part][plane]: a bf16 value has one plane; an
// fp16 value has three, itself for dot products and two bf16 values (exact: 11
// bits in 8 + 3) for the matrix cores, whose sums are with t in bf16's range.
__host__ __device__ inline int up_planes(int f16) { return f16 ? 3 : 1; }

struct Adapted {
    const int32_t* ids;      // [M], outside [0, adapters): no adapter
    uint16_t* t;             // [M + 1, parts, 64]
    const uint8_t* up;
    int f16, parts, adapters;
    int eights;              // of ranks that are not all padding
};

// t for every row that has an adapter.
int launch_shrink(const Adapted& ad, const int8_t* a, int64_t ld_a, const float* sa, int64_t M, int64_t K, const void* down, int rank,
                  const float* scaling, const int32_t* offsets, const int32_t* order, hipStream_t st);

typedef float lb_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 lb_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lb_f16x8 __attribute__((ext_vector_type(8)));

// The adapter's part of four consecutive outputs of row m from column n (a
// multiple of 4), share k of n of its ranks: a dot product in fp32, for few rows,
// which seldom share an adapter.  64 rows with 48 adapters of rank 16, INT4 12288
// x 4096: 16.0 to 16.8 us traced, 11.8 without adapters; 19 MB of B are most of
// the difference.
__device__ __forceinline__ lb_f32x4 adapter_dot4(const Adapted& ad, int64_t N, int64_t m, int64_t n, int share, int shares) {
    lb_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    const int id = ad.ids[m];
    if (id < 0 || id >= ad.adapters) return s;
    const int planes = up_planes(ad.f16);
    const lb_u32x4* t = reinterpret_cast<const lb_u32x4*>(ad.t + m * ad.parts * 64);
    const lb_u32x4* b = reinterpret_cast<const lb_u32x4*>(ad.up + (id * cdiv(N, 16) + n / 16) * (ad.parts * planes) * 1024) + n % 16;
    const int c1 = ad.eights * (share + 1) / shares;
#pragma unroll 2
    for (int c = ad.eights * share / shares; c < c1; ++c) {
        const lb_u32x4 hi = t[(c >> 2) * 8 + (c & 3)], lo = t[(c >> 2) * 8 + (c & 3) + 4];
        const lb_u32x4* w = b + (c >> 2) * planes * 64 + (c & 3) * 16;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = half_word<IC_DTYPE_BF16>(hi[k >> 1], k & 1) + half_word<IC_DTYPE_BF16>(lo[k >> 1], k & 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const lb_u32x4 u = w[i];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                s[i] = __builtin_fmaf(v[k], ad.f16 ? half_word<IC_DTYPE_F16>(u[k >> 1], k & 1) : half_word<IC_DTYPE_BF16>(u[k >> 1], k & 1), s[i]);
        }
    }
    return s;
}

}  // namespace icq
