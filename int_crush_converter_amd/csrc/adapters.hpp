// Low-rank adapters beside a quantised product: y[m, n] += sum_r t[m, r] B_a[n, r],
// t = scale_a A_a x, with an adapter a for each row m.
#pragma once

#include "lowbit.hpp"

namespace icq {

constexpr int kMaxRank = 128;
constexpr int kRankPart = 32;           // ranks are padded to parts of 32 with zeros
__host__ __device__ inline int rank_parts(int rank) { return (rank + kRankPart - 1) / kRankPart; }

// How t is kept goes by the result.  A 16-bit result has 8 or 11 bits: t as two
// bf16 values, each the nearest to what is left (the first by truncation where the
// nearest is infinite), within 2^-18 of it, is what the matrix cores take as it
// lies.  An fp32 result has t whole: in
// fp32 for the forms for few rows, which split it in registers, and for the tiled
// ones, whose stages go straight to LDS, as three bf16 values of 8 bits each.
// They are exact where the last is one (|t| >= 2^-110).
//
//   kTwo     128 bytes a row and part, 32 values of hi and then of lo
//   kWhole   128 bytes, 32 fp32 values
//   kThree   256 bytes, 32 values of each and 32 zeros (an INT4 stage is 128 bytes)
//
// Behind the last row there is one of zeros.
//
// B is kept in tiles of 16 columns x 32 ranks, 1 KB, in the order of weight tiles
// (lowbit.hpp): 16 bytes a column are 8 ranks, those of 16 columns follow one
// another.  [adapter][column tile][part][plane]: a bf16 value has one plane; an
// fp16 value has three, itself for dot products and two bf16 values (exact: 11
// bits in 8 + 3) for the matrix cores, whose sums are with t in bf16's range.
__host__ __device__ inline int up_planes(int f16) { return f16 ? 3 : 1; }

enum RankForm { kTwo, kWhole, kThree };

struct Adapted {
    const int32_t* ids;      // [M], outside [0, adapters): no adapter
    uint16_t* t;             // [M + 1, parts, 64 (kThree: 128)]
    const uint8_t* up;
    int f16, parts, adapters;
    int eights;              // of ranks that are not all padding
};

// t for every row that has an adapter.
int launch_shrink(const Adapted& ad, RankForm form, const int8_t* a, int64_t ld_a, const float* sa, int64_t M, int64_t K, const void* down, int rank,
                  const float* scaling, const int32_t* offsets, const int32_t* order, hipStream_t st);

typedef float lb_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 lb_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lb_f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ lb_f32x4 mma_ranks(lb_u32x4 w, lb_u32x4 x, lb_f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lb_bf16x8, w), __builtin_bit_cast(lb_bf16x8, x), acc, 0, 0, 0);
}

// Adapter id's part of four consecutive outputs of row m from column n (a multiple
// of 4), share k of n of its ranks: a dot product in fp32, for rows that seldom share
// an adapter (t: kTwo or, where WHOLE, kWhole).  64 rows with 48 adapters of rank 16, INT4 12288 x 4096: 16.6 to 17.3 us
// traced, 11.8 without adapters; 19 MB of B are most of the difference.
template <bool WHOLE>
__device__ __forceinline__ lb_f32x4 adapter_dot4(const Adapted& ad, int64_t N, int64_t m, int id, int64_t n, int share, int shares) {
    lb_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    const int planes = up_planes(ad.f16);
    const lb_u32x4* t = reinterpret_cast<const lb_u32x4*>(ad.t + m * ad.parts * 64);
    const lb_u32x4* b = reinterpret_cast<const lb_u32x4*>(ad.up + (id * cdiv(N, 16) + n / 16) * (ad.parts * planes) * 1024) + n % 16;
    const int c1 = ad.eights * (share + 1) / shares;
#pragma unroll 2
    for (int c = ad.eights * share / shares; c < c1; ++c) {
        const lb_u32x4 first = t[WHOLE ? c * 2 : (c >> 2) * 8 + (c & 3)], second = t[WHOLE ? c * 2 + 1 : (c >> 2) * 8 + (c & 3) + 4];
        const lb_u32x4* w = b + (c >> 2) * planes * 64 + (c & 3) * 16;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            v[k] = WHOLE ? __uint_as_float((k < 4 ? first : second)[k & 3])
                         : half_word<IC_DTYPE_BF16>(first[k >> 1], k & 1) + half_word<IC_DTYPE_BF16>(second[k >> 1], k & 1);
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

// The upper 16 bits of 8 fp32 values as an operand, and what is left of them.
__device__ __forceinline__ lb_u32x4 take_upper(float (&v)[8]) {
    lb_u32x4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t a = __float_as_uint(v[2 * k]) & 0xffff0000u, b = __float_as_uint(v[2 * k + 1]) & 0xffff0000u;
        o[k] = a >> 16 | b;
        v[2 * k] -= __uint_as_float(a);
        v[2 * k + 1] -= __uint_as_float(b);
    }
    return o;
}

// The adapters' part of 16 rows x 16 columns, this lane's four outputs as above:
// row m of `rows`, with adapter `id` (-1: none, or no row), columns nt * 16 + g * 4.
// Where the rows share adapters, one adapter after another on the matrix cores,
// rows of others with t of zeros; the loads for four tiles of B wait together.
// Where few do, dot products: the matrix cores read a tile of B for each adapter
// of the rows, a dot product its own row's part, and they meet at two or four
// such tiles for 8 ranks (dots / matrix cores, 12288 x 4096 INT4 but for the
// last, us; of the adapters, 64 rows drew at random):
//   rank 16, bf16, 48: 23.5 / 26.5        rank 64, bf16, 12: 33.6 / 26.5, 48: 37.7 / 33.7
//   rank 32, bf16, 48: 28.5 / 27.6, 8: 24.9 / 22.3        rank 64, fp16, 12: 33.5 / 33.9, 48: 37.4 / 44.4
//   rank 128, 8, fp16: 48.5 / 44.5; bf16, 200 rows of 2816 x 4096: 46.3 / 31.2, 25 rows one after another 40.6 / 22.9
template <bool WHOLE>
__device__ __forceinline__ lb_f32x4 adapter_tile(const Adapted& ad, int64_t N, int rows, int m, int id, int nt, int share, int shares) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n_tiles = (int)cdiv(N, 16);
    lb_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (nt >= n_tiles) return s;
    if (id >= ad.adapters) id = -1;
    unsigned left = (unsigned)__ballot(id >= 0) & 0xffffu;
    int now = -1;
    auto pick = [&]() {                                    // the next adapter, in the order of its first row
        now = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
        left &= ~(unsigned)__ballot(id == now);
    };
    const unsigned all = left;
    const int planes = up_planes(ad.f16), per = ad.parts * (ad.f16 ? 2 : 1), most = (ad.eights < 4 ? 2 : 4) * ad.eights;
    int tiles = 0;
    while (left && tiles <= most) {
        pick();
        tiles += per;
    }
    if (tiles > most) return id >= 0 && nt * 16 + g * 4 < N ? adapter_dot4<WHOLE>(ad, N, m, id, nt * 16 + g * 4, share, shares) : s;
    const int first = tiles * share / shares, last = tiles * (share + 1) / shares;
    int at = first;                                        // the adapter's tile: part and plane
    left = all;
    if (left) pick();
    for (; at >= per && left; at -= per) pick();
    for (int p = first; p < last; p += 4) {
        lb_u32x4 b[4], hi[4], lo[4];                       // (WHOLE: the lane's first four values of t and the others)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (p + k >= last) break;
            const int part = ad.f16 ? at >> 1 : at;
            const lb_u32x4* u = reinterpret_cast<const lb_u32x4*>(ad.up) + (((int64_t)now * n_tiles + nt) * ad.parts + part) * planes * 64 + lane;
            const lb_u32x4* t = reinterpret_cast<const lb_u32x4*>(ad.t) + ((int64_t)(id == now ? m : rows) * ad.parts + part) * 8 + (WHOLE ? g * 2 : g);
            b[k] = u[ad.f16 ? 64 + (at & 1) * 64 : 0];
            hi[k] = t[0];
            lo[k] = t[WHOLE ? 1 : 4];
            if (++at == per && left) {
                at = 0;
                pick();
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (p + k >= last) break;
            if (WHOLE) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float((i < 4 ? hi[k] : lo[k])[i & 3]);
                const lb_u32x4 first = take_upper(v), second = take_upper(v);
                s = mma_ranks(b[k], take_upper(v), mma_ranks(b[k], second, mma_ranks(b[k], first, s)));
            } else {
                s = mma_ranks(b[k], lo[k], mma_ranks(b[k], hi[k], s));
            }
        }
    }
    return s;
}

}  // namespace icq
