// Low-rank adapters of many requests beside one quantised weight: their
// factors laid out once, and t = scale_a A_a x for every row's own adapter.
#include "adapters.hpp"
#include "groups.hpp"
#include "prof.hpp"

namespace icq {
namespace {

// A [adapters, rank, K] -> tiles of 16 ranks x 64 columns, [adapter][rank / 16][K / 64]: two words of 16 bytes a lane,
// lane 16 g + r holding columns 16 g .. 16 g + 7 and + 8 .. + 15 of rank r, as a lane holds 16 consecutive codes of
// a row.  Zeros behind the last rank and column.
__global__ __launch_bounds__(256) void pack_down_kernel(const uint16_t* __restrict__ src, int64_t adapters, int rank, int64_t K,
                                                        lb_u32x4* __restrict__ dst, int64_t tiles) {
    const int lane = threadIdx.x & 63, r = lane & 15;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);     // [adapter][rank tile][column tile]
    const int rt = padded_rank(rank) / 16;
    if (at >= adapters * rt * tiles) return;
    const int64_t a = at / (rt * tiles);
    const int row = (int)(at / tiles % rt) * 16 + r;
    const int64_t k0 = at % tiles * 64 + (lane >> 4) * 16;
    lb_u32x4 w[2] = {};
    if (row < rank) {
        const uint16_t* s = src + (a * rank + row) * K;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (k0 + i < K) w[i >> 3][i >> 1 & 3] |= (unsigned)s[k0 + i] << (16 * (i & 1));
    }
    dst[at * 128 + lane] = w[0];
    dst[at * 128 + 64 + lane] = w[1];
}

// B [adapters, N, rank] -> rows padded with zeros to whole 16 ranks.
__global__ __launch_bounds__(256) void pack_up_kernel(const uint16_t* __restrict__ src, int64_t rows, int rank, uint16_t* __restrict__ dst) {
    const int padded = padded_rank(rank);
    const int64_t total = rows * padded, stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const int64_t row = i / padded;
        const int c = (int)(i - row * padded);
        dst[i] = c < rank ? src[row * rank + c] : (uint16_t)0;
    }
}

// 8 codes of a lane as the 16-bit values of an operand (exact: |q| <= 128).
template <int DT>
__device__ __forceinline__ lb_u32x4 code_values(uint32_t a, uint32_t b) {
    lb_u32x4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t w = k < 2 ? a : b;
        const int s = 16 * (k & 1);
        o[k] = pack_half_words<DT>((float)(int8_t)(w >> s), (float)(int8_t)(w >> (s + 8)));
    }
    return o;
}

template <int DT>
__device__ __forceinline__ lb_f32x4 mma16(lb_u32x4 w, lb_u32x4 x, lb_f32x4 acc) {
    if constexpr (DT == IC_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lb_f16x8, w), __builtin_bit_cast(lb_f16x8, x), acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lb_bf16x8, w), __builtin_bit_cast(lb_bf16x8, x), acc, 0, 0, 0);
}

// A work-group of 8 waves takes 16 ranks and 16 rows of one adapter, its waves
// a share of K each; the sums are joined in LDS in a fixed order.
template <int DT>
__global__ __launch_bounds__(512) void shrink_kernel(const int8_t* __restrict__ a, int64_t ld_a, const float* __restrict__ sa, int M,
                                                     const lb_u32x4* __restrict__ down, int64_t tiles, int rank, int adapters,
                                                     const float* __restrict__ scaling, const int32_t* __restrict__ offsets,
                                                     const int32_t* __restrict__ order, float* __restrict__ t) {
    constexpr int WAVES = 8;
    __shared__ lb_f32x4 part[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int padded = padded_rank(rank), rts = padded / 16, rt = blockIdx.x % rts;
    const GroupTile tile = find_tile(offsets, adapters, M, 16, blockIdx.x / rts);
    if (tile.group < 0) return;
    const int at = tile.first + r < tile.end ? tile.first + r : tile.end - 1;
    int m = order[at];
    m = m < 0 ? 0 : m < M ? m : M - 1;
    const lb_u32x4* x = reinterpret_cast<const lb_u32x4*>(a + m * ld_a) + g;
    const lb_u32x4* w = down + ((int64_t)tile.group * rts + rt) * tiles * 128 + lane;
    lb_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t t0 = tiles * wave / WAVES, t1 = tiles * (wave + 1) / WAVES;
    for (int64_t k = t0; k < t1; ++k) {
        const lb_u32x4 q = x[k * 4];
        acc = mma16<DT>(w[k * 128], code_values<DT>(q[0], q[1]), acc);
        acc = mma16<DT>(w[k * 128 + 64], code_values<DT>(q[2], q[3]), acc);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    lb_f32x4 s = part[0][lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) s += part[k][lane];
    const float f = sa[m] * scaling[tile.group];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = rt * 16 + g * 4 + i < rank ? s[i] * f : 0.0f;
    if (tile.first + r < tile.end) *reinterpret_cast<lb_f32x4*>(t + (int64_t)m * padded + rt * 16 + g * 4) = s;
}

}  // namespace

int launch_shrink(const Adapted& ad, const int8_t* a, int64_t ld_a, const float* sa, int64_t M, int64_t K, const void* down, int rank,
                  const float* scaling, const int32_t* offsets, const int32_t* order, hipStream_t st) {
    const dim3 grid((unsigned)(most_tiles(M, ad.adapters, 16) * (ad.rank / 16)));
    const lb_u32x4* d = static_cast<const lb_u32x4*>(down);
    const int64_t tiles = cdiv(K, kActPad) * 2;
    if (ad.f16) hipLaunchKernelGGL(shrink_kernel<IC_DTYPE_F16>, grid, dim3(512), 0, st, a, ld_a, sa, (int)M, d, tiles, rank, ad.adapters, scaling, offsets, order, ad.t);
    else hipLaunchKernelGGL(shrink_kernel<IC_DTYPE_BF16>, grid, dim3(512), 0, st, a, ld_a, sa, (int)M, d, tiles, rank, ad.adapters, scaling, offsets, order, ad.t);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

}  // namespace icq

using namespace icq;

extern "C" int64_t ic_adapter_down_bytes(int64_t adapters, int rank, int64_t K) {
    if (adapters < 0 || rank < 1 || rank > kMaxRank || K < 0) return 0;
    return adapters * padded_rank(rank) * cdiv(K, kActPad) * kActPad * 2;
}

extern "C" int64_t ic_adapter_up_bytes(int64_t adapters, int64_t N, int rank) {
    if (adapters < 0 || rank < 1 || rank > kMaxRank || N < 0) return 0;
    return adapters * N * padded_rank(rank) * 2;
}

extern "C" int64_t ic_adapted_linear_workspace_bytes(int64_t M, int rank) {
    if (M < 0 || rank < 1 || rank > kMaxRank) return 0;
    return M * padded_rank(rank) * 4;
}

extern "C" int ic_adapter_pack(const void* a, const void* b, int64_t adapters, int rank, int64_t N, int64_t K, void* down, void* up,
                               void* stream) {
    IC_REQUIRE(adapters >= 1 && rank >= 1 && N >= 1 && K >= 1, "ic_adapter_pack: sizes must be >= 1");
    if (adapters > kMaxGroups || rank > kMaxRank || K > 65536 || N > kMaxRows)
        return fail(IC_ERR_RANGE, "ic_adapter_pack: at most 1024 adapters, rank 128, 65536 for K, 1048560 for N");
    IC_REQUIRE(a && b && down && up && aligned16(down) && aligned16(up), "ic_adapter_pack: null pointer, or results not 16-byte aligned");
    const int64_t tiles = cdiv(K, kActPad) * 2, n = adapters * (padded_rank(rank) / 16) * tiles;
    hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(pack_down_kernel, dim3((unsigned)cdiv(n, 4)), dim3(256), 0, st, static_cast<const uint16_t*>(a), adapters, rank, K,
                       static_cast<lb_u32x4*>(down), tiles);
    const int64_t blocks = cdiv(adapters * N * padded_rank(rank), 256);
    hipLaunchKernelGGL(pack_up_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, static_cast<const uint16_t*>(b),
                       adapters * N, rank, static_cast<uint16_t*>(up));
    IC_CHECK_LAUNCH();
    return IC_OK;
}
