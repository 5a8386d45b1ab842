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

// A work-group of 8 waves takes 16 RT ranks and 16 MT rows of one adapter, its
// waves a share of K each; the sums are joined in LDS in a fixed order.
template <int DT, int MT, int RT>
__global__ __launch_bounds__(512) void shrink_kernel(const int8_t* __restrict__ a, int64_t ld_a, const float* __restrict__ sa, int M,
                                                     const lb_u32x4* __restrict__ down, int64_t tiles, int rank, int adapters,
                                                     const float* __restrict__ scaling, const int32_t* __restrict__ offsets,
                                                     const int32_t* __restrict__ order, float* __restrict__ t) {
    constexpr int WAVES = 8;
    __shared__ lb_f32x4 part[WAVES][MT * RT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int padded = padded_rank(rank), rts = padded / 16, groups = (rts + RT - 1) / RT, rt0 = blockIdx.x % groups * RT;
    const GroupTile tile = find_tile(offsets, adapters, M, 16 * MT, blockIdx.x / groups);
    if (tile.group < 0) return;
    auto row_of = [&](int i) {             // (rows past the last repeat the last)
        const int at = tile.first + i * 16 + r < tile.end ? tile.first + i * 16 + r : tile.end - 1, m = order[at];
        return m < 0 ? 0 : m < M ? m : M - 1;
    };
    const lb_u32x4* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = reinterpret_cast<const lb_u32x4*>(a + row_of(i) * ld_a) + g;
    const lb_u32x4* w[RT];
#pragma unroll
    for (int k = 0; k < RT; ++k) w[k] = down + ((int64_t)tile.group * rts + (rt0 + k < rts ? rt0 + k : rts - 1)) * tiles * 128 + lane;
    lb_f32x4 acc[MT][RT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < RT; ++k) acc[i][k] = lb_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int t0 = (int)(tiles * wave / WAVES), t1 = (int)(tiles * (wave + 1) / WAVES);
    for (int c = t0; c < t1; ++c) {
        lb_u32x4 q[MT], lo[RT], hi[RT];
#pragma unroll
        for (int i = 0; i < MT; ++i) q[i] = x[i][c * 4];
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            lo[k] = w[k][c * 128];
            hi[k] = w[k][c * 128 + 64];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const lb_u32x4 u = code_values<DT>(q[i][0], q[i][1]), v = code_values<DT>(q[i][2], q[i][3]);
#pragma unroll
            for (int k = 0; k < RT; ++k) acc[i][k] = mma16<DT>(hi[k], v, mma16<DT>(lo[k], u, acc[i][k]));
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < RT; ++k) part[wave][i * RT + k][lane] = acc[i][k];
    __syncthreads();
    for (int u = wave; u < MT * RT; u += WAVES) {
        const int i = u / RT, rt = rt0 + u % RT;
        if (tile.first + i * 16 + r >= tile.end || rt >= rts) continue;
        lb_f32x4 s = part[0][u][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) s += part[k][u][lane];
        const int m = row_of(i);
        const float f = sa[m] * scaling[tile.group];
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = rt * 16 + g * 4 + k < rank ? s[k] * f : 0.0f;
        *reinterpret_cast<lb_f32x4*>(t + (int64_t)m * padded + rt * 16 + g * 4) = s;
    }
}

}  // namespace

int launch_shrink(const Adapted& ad, const int8_t* a, int64_t ld_a, const float* sa, int64_t M, int64_t K, const void* down, int rank,
                  const float* scaling, const int32_t* offsets, const int32_t* order, hipStream_t st) {
    const lb_u32x4* d = static_cast<const lb_u32x4*>(down);
    const int64_t tiles = cdiv(K, kActPad) * 2;
    auto go = [&](auto dt, auto mt, auto rt) {
        constexpr int MT = decltype(mt)::value, RT = decltype(rt)::value;
        const dim3 grid((unsigned)(most_tiles(M, ad.adapters, 16 * MT) * cdiv(ad.rank / 16, RT)));
        hipLaunchKernelGGL((shrink_kernel<decltype(dt)::value, MT, RT>), grid, dim3(512), 0, st, a, ld_a, sa, (int)M, d, tiles, rank, ad.adapters,
                           scaling, offsets, order, ad.t);
    };
    auto shape = [&](auto dt) {
        typedef std::integral_constant<int, 1> one;
        if (M <= 1024) go(dt, one{}, one{});
        else if (ad.rank <= 16) go(dt, std::integral_constant<int, 2>{}, one{});
        else if (ad.rank <= 32) go(dt, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
        else go(dt, std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
    };
    if (ad.f16) shape(std::integral_constant<int, IC_DTYPE_F16>{});
    else shape(std::integral_constant<int, IC_DTYPE_BF16>{});
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
