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
__host__ __device__ inline int down_tiles(int rank) { return (rank + 15) / 16; }

__global__ __launch_bounds__(256) void pack_down_kernel(const uint16_t* __restrict__ src, int64_t adapters, int rank, int64_t K,
                                                        lb_u32x4* __restrict__ dst, int64_t tiles) {
    const int lane = threadIdx.x & 63, r = lane & 15;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);     // [adapter][rank tile][column tile]
    const int rt = down_tiles(rank);
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

// B [adapters, N, rank] -> tiles (adapters.hpp), a lane one column's 8 ranks.
__global__ __launch_bounds__(256) void pack_up_kernel(const uint16_t* __restrict__ src, int64_t adapters, int64_t N, int rank, int f16,
                                                      lb_u32x4* __restrict__ dst) {
    const int lane = threadIdx.x & 63, parts = rank_parts(rank), planes = up_planes(f16);
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), n_tiles = cdiv(N, 16);     // [adapter][column tile][part][plane]
    if (at >= adapters * n_tiles * parts * planes) return;
    const int64_t n = at / (parts * planes) % n_tiles * 16 + (lane & 15), a = at / (parts * planes) / n_tiles;
    const int rank0 = (int)(at / planes % parts) * kRankPart + (lane >> 4) * 8, plane = (int)(at % planes);
    lb_u32x4 w = {0, 0, 0, 0};
    if (n < N) {
        const uint16_t* s = src + (a * N + n) * rank;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (rank0 + k >= rank) continue;
            unsigned v = s[rank0 + k];
            if (plane) {
                const float x = f16_bits_to_f32((uint16_t)v), hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
                v = __float_as_uint(plane == 2 ? x - hi : hi) >> 16;
            }
            w[k >> 1] |= v << (16 * (k & 1));
        }
    }
    dst[at * 64 + lane] = w;
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

// t = scale_a sa A_a q for 16 RT ranks and 16 MT rows of one adapter: the codes
// are exact in 16 bits, the products are summed in fp32.  A work-group's waves
// take a share of K each; the sums are joined in LDS in a fixed order.
//
// Few rows: 48 adapters of 64 rows, rank 16, K = 4096 5.3 to 5.5 us traced, the
// launch and three loads that wait for one another (6.3 MB of A).  Many: 8192 x
// 12288, rank 64 38 to 40 us traced (codes from HBM: 20 us), 8192 x 4096 15 us.
// There a CU's work bounds it: 28 us of it with no loads at all, 2.5 operations a code for
// its value and as many matrix instructions; a round of CUs is what counts, so
// the rows of a work-group are 32 or 48, whichever needs fewer rounds for its
// height (32 rows left 6 of 262 work-groups for a second round: 56 us).  16 waves,
// or two steps' loads in flight, made no difference.
template <int DT, int MT, int RT, int WAVES, RankForm FORM>
__global__ __launch_bounds__(64 * WAVES) void shrink_kernel(const int8_t* __restrict__ a, int64_t ld_a, const float* __restrict__ sa, int M,
                                                     const lb_u32x4* __restrict__ down, int64_t tiles, int rank, int adapters,
                                                     const float* __restrict__ scaling, const int32_t* __restrict__ offsets,
                                                     const int32_t* __restrict__ order, uint16_t* __restrict__ t) {
    __shared__ lb_f32x4 part[WAVES][MT * RT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int parts = rank_parts(rank), rts = down_tiles(rank), groups = (rts + RT - 1) / RT;
    // work-groups are dealt to the 8 XCDs in turn: each gets one run of rows, whose adapter its L2 keeps
    const int per = gridDim.x >> 3, extra = gridDim.x & 7, xcd = blockIdx.x & 7;
    const int at_run = xcd * per + (xcd < extra ? xcd : extra) + (blockIdx.x >> 3), rt0 = at_run % groups * RT;
    constexpr int PITCH = FORM == kThree ? 128 : 64;   // of a row's part
    if (blockIdx.x == 0 && threadIdx.x < parts * PITCH) t[(int64_t)M * parts * PITCH + threadIdx.x] = 0;       // the row of zeros
    const GroupTile tile = find_tile(offsets, adapters, M, 16 * MT, at_run / groups);
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
        const bool rest = rt == rts - 1 && rts % 2;    // of the last part: zeros
        uint16_t* const row = t + ((int64_t)m * parts + rt / 2) * PITCH;
        const int at = rt % 2 * 16 + g * 4;
        lb_f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = rt * 16 + g * 4 + k < rank ? s[k] * f : 0.0f;
        if constexpr (FORM == kWhole) {
            lb_f32x4* to = reinterpret_cast<lb_f32x4*>(reinterpret_cast<float*>(row) + at);
            to[0] = v;
            if (rest) to[4] = lb_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        } else {
            uint32_t value[4][2] = {};                 // hi, lo (kThree: the middle and the last 8 bits, zeros)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t hi = __float_as_uint(v[k]) & 0xffff0000u;
                if (FORM == kTwo) {                    // the nearest, if it is finite: half the rest, with a sign, for lo
                    const uint32_t near = pack_half_words<IC_DTYPE_BF16>(0.0f, v[k]) & 0xffff0000u;
                    hi = (near & 0x7fffffffu) == 0x7f800000u ? hi : near;
                }
                const float low = v[k] - __uint_as_float(hi);
                const uint32_t mid = __float_as_uint(low) & 0xffff0000u, last = __float_as_uint(low - __uint_as_float(mid));
                value[0][k >> 1] |= hi >> (16 * (1 - (k & 1)));
                value[1][k >> 1] |= (FORM == kThree ? mid >> 16 : pack_half_words<IC_DTYPE_BF16>(low, 0.0f)) << (16 * (k & 1));
                value[2][k >> 1] |= last >> 16 << (16 * (k & 1));
            }
#pragma unroll
            for (int k = 0; k < PITCH / kRankPart; ++k) {
                lb_u32x2* to = reinterpret_cast<lb_u32x2*>(row + k * kRankPart + at);
                to[0] = lb_u32x2{value[k][0], value[k][1]};
                if (rest) to[4] = lb_u32x2{0, 0};
            }
        }
    }
}

}  // namespace

int launch_shrink(const Adapted& ad, RankForm form, const int8_t* a, int64_t ld_a, const float* sa, int64_t M, int64_t K, const void* down, int rank,
                  const float* scaling, const int32_t* offsets, const int32_t* order, hipStream_t st) {
    const lb_u32x4* d = static_cast<const lb_u32x4*>(down);
    const int64_t tiles = cdiv(K, kActPad) * 2;
    auto launch = [&](auto dt, auto mt, auto rt, auto waves, auto kept) {
        constexpr int MT = decltype(mt)::value, RT = decltype(rt)::value, WAVES = decltype(waves)::value;
        const dim3 grid((unsigned)(most_tiles(M, ad.adapters, 16 * MT) * cdiv(down_tiles(rank), RT)));
        hipLaunchKernelGGL((shrink_kernel<decltype(dt)::value, MT, RT, WAVES, decltype(kept)::value>), grid, dim3(64 * WAVES), 0, st, a, ld_a, sa, (int)M, d, tiles, rank,
                           ad.adapters, scaling, offsets, order, ad.t);
    };
    auto go = [&](auto dt, auto mt, auto rt, auto waves) {
        if (form == kTwo) launch(dt, mt, rt, waves, std::integral_constant<RankForm, kTwo>{});
        else if (form == kWhole) launch(dt, mt, rt, waves, std::integral_constant<RankForm, kWhole>{});
        else launch(dt, mt, rt, waves, std::integral_constant<RankForm, kThree>{});
    };
    auto shape = [&](auto dt) {
        typedef std::integral_constant<int, 1> c1;
        typedef std::integral_constant<int, 2> c2;
        typedef std::integral_constant<int, 3> c3;
        typedef std::integral_constant<int, 4> c4;
        typedef std::integral_constant<int, 8> c8;
        if (M <= 1024) return go(dt, c1{}, c1{}, std::integral_constant<int, 16>{});
        // 32 or 48 rows: what takes fewer rounds of the CUs for its height
        auto cost = [&](int mt) { return mt * cdiv(most_tiles(M, ad.adapters, 16 * mt) * cdiv(rank, 64), 256); };
        const bool high = cost(3) < cost(2);
        if (rank <= 16) high ? go(dt, c3{}, c1{}, c8{}) : go(dt, c2{}, c1{}, c8{});
        else if (rank <= 32) high ? go(dt, c3{}, c2{}, c8{}) : go(dt, c2{}, c2{}, c8{});
        else high ? go(dt, c3{}, c4{}, c8{}) : go(dt, c2{}, c4{}, c8{});
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
    return adapters * down_tiles(rank) * 16 * cdiv(K, kActPad) * kActPad * 2;
}

extern "C" int64_t ic_adapter_up_bytes(int64_t adapters, int64_t N, int rank, int dtype) {
    if (adapters < 0 || rank < 1 || rank > kMaxRank || N < 0 || (dtype != IC_DTYPE_BF16 && dtype != IC_DTYPE_F16)) return 0;
    return adapters * cdiv(N, 16) * rank_parts(rank) * up_planes(dtype == IC_DTYPE_F16) * 1024;
}

extern "C" int64_t ic_adapted_linear_workspace_bytes(int64_t M, int rank) {
    if (M < 0 || rank < 1 || rank > kMaxRank) return 0;
    return (M + 1) * rank_parts(rank) * (M <= 64 ? 128 : 256);       // (tiles, which may ask for kThree, have more than 64 rows)
}

extern "C" int ic_adapter_pack(const void* a, const void* b, int dtype, int64_t adapters, int rank, int64_t N, int64_t K, void* down, void* up,
                               void* stream) {
    IC_REQUIRE(adapters >= 1 && rank >= 1 && N >= 1 && K >= 1, "ic_adapter_pack: sizes must be >= 1");
    IC_REQUIRE(dtype == IC_DTYPE_BF16 || dtype == IC_DTYPE_F16, "ic_adapter_pack: adapters are bf16 or fp16");
    if (adapters > kMaxGroups || rank > kMaxRank || K > 65536 || N > kMaxRows)
        return fail(IC_ERR_RANGE, "ic_adapter_pack: at most 1024 adapters, rank 128, 65536 for K, 1048560 for N");
    IC_REQUIRE(a && b && down && up && aligned16(down) && aligned16(up), "ic_adapter_pack: null pointer, or results not 16-byte aligned");
    const int64_t tiles = cdiv(K, kActPad) * 2, n = adapters * down_tiles(rank) * tiles;
    const int64_t u = adapters * cdiv(N, 16) * rank_parts(rank) * up_planes(dtype == IC_DTYPE_F16);
    if (u > 1 << 25) return fail(IC_ERR_RANGE, "ic_adapter_pack: b takes more than 2^25 KB");
    hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(pack_down_kernel, dim3((unsigned)cdiv(n, 4)), dim3(256), 0, st, static_cast<const uint16_t*>(a), adapters, rank, K,
                       static_cast<lb_u32x4*>(down), tiles);
    hipLaunchKernelGGL(pack_up_kernel, dim3((unsigned)cdiv(u, 4)), dim3(256), 0, st, static_cast<const uint16_t*>(b), adapters, N, rank,
                       dtype == IC_DTYPE_F16, static_cast<lb_u32x4*>(up));
    IC_CHECK_LAUNCH();
    return IC_OK;
}
