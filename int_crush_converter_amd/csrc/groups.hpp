// Rows ordered by group (expert, adapter), as the kernels that work on them see them.
#pragma once

#include "common.hpp"

namespace icq {

constexpr int kMaxGroups = 1024;

// v of another lane by DPP, `none` where there is no such lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or(int none, int v) {
    return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}
constexpr int kShr1 = 0x111, kShr2 = 0x112, kShr4 = 0x114, kShr8 = 0x118;     // within 16 lanes
constexpr int kLast15 = 0x142, kLast31 = 0x143;     // the last lane of 16 to the next 16, of 32 to the upper 32

// Inclusive sum over the 64 lanes: within 16 lanes, then across them.
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp_or<kShr1, 0xf>(0, v);
    v += dpp_or<kShr2, 0xf>(0, v);
    v += dpp_or<kShr4, 0xf>(0, v);
    v += dpp_or<kShr8, 0xf>(0, v);
    v += dpp_or<kLast15, 0xa>(0, v);
    v += dpp_or<kLast31, 0xc>(0, v);
    return v;
}

// The largest of the 64 lanes, the same scalar for all.  One instruction a
// step, which the compiler makes three of (a lane without a partner keeps its
// value; a DPP operand needs two wait states behind its own writing).
__device__ __forceinline__ unsigned wave_top(unsigned v) {
    asm("s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t"
        "s_nop 1"                          // (and readlane one)
        : "+v"(v));
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// a in the lanes of the mask, else b.
__device__ __forceinline__ unsigned lanes_of(unsigned long long mask, unsigned a, unsigned b) {
    unsigned d;
    asm("v_cndmask_b32_e64 %0, %1, %2, %3" : "=v"(d) : "v"(b), "v"(a), "s"(mask));
    return d;
}

// The sum of the 64 lanes in one order, the same scalar for all.
__device__ __forceinline__ float wave_total(float v) {
    auto part = [](float x, auto ctrl, auto rows) {
        return __int_as_float(dpp_or<decltype(ctrl)::value, decltype(rows)::value>(0, __float_as_int(x)));
    };
    typedef std::integral_constant<int, 0xf> all;
    v += part(v, std::integral_constant<int, kShr1>{}, all{});
    v += part(v, std::integral_constant<int, kShr2>{}, all{});
    v += part(v, std::integral_constant<int, kShr4>{}, all{});
    v += part(v, std::integral_constant<int, kShr8>{}, all{});
    v += part(v, std::integral_constant<int, kLast15>{}, std::integral_constant<int, 0xa>{});
    v += part(v, std::integral_constant<int, kLast31>{}, std::integral_constant<int, 0xc>{});
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Rows [first, end) of group g; ends past `rows` count as `rows`.
__device__ __forceinline__ int group_edge(const int32_t* offsets, int g, int rows) {
    const int o = offsets[g];
    return o < 0 ? 0 : o < rows ? o : rows;
}

struct GroupTile {
    int group, first, end;      // rows [first, end) of the group, of which the tile has the first `height`
};

// Tile number `index` of the groups' rows cut into tiles of `height` rows
// (a group's last one may be shorter; empty groups have none).  Every lane of
// the wave gets the same answer; group -1 behind the last tile.  Two steps of
// a sum over lanes: runs of groups, then the groups of one run.
__device__ __forceinline__ GroupTile find_tile(const int32_t* offsets, int groups, int rows, int height, int index) {
    const int lane = threadIdx.x & 63, run = (groups + 63) >> 6;
    int tiles = 0;
    int edge = lane * run < groups ? group_edge(offsets, lane * run, rows) : 0;
    const int first_edge = edge;
    for (int i = 0; i < run; ++i) {
        const int g = lane * run + i;
        if (g < groups) {
            const int next = group_edge(offsets, g + 1, rows);
            if (next > edge) tiles += (next - edge + height - 1) / height;
            edge = next;
        }
    }
    const int sum = wave_scan(tiles);
    const unsigned long long past = __ballot(sum > index);
    if (!past) return GroupTile{-1, 0, 0};
    const int l = __builtin_ctzll(past);
    int rest = index - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
    if (run == 1) return GroupTile{l, __builtin_amdgcn_readlane(first_edge, l) + rest * height, __builtin_amdgcn_readlane(edge, l)};
    const int g = l * run + lane;
    const bool mine = lane < run && g < groups;
    const int lo = mine ? group_edge(offsets, g, rows) : 0, hi = mine ? group_edge(offsets, g + 1, rows) : 0;
    const int own = hi > lo ? (hi - lo + height - 1) / height : 0, upto = wave_scan(own);
    const int k = __builtin_ctzll(__ballot(upto > rest));
    rest -= __builtin_amdgcn_readlane(upto, k) - __builtin_amdgcn_readlane(own, k);
    return GroupTile{l * run + k, __builtin_amdgcn_readlane(lo, k) + rest * height, __builtin_amdgcn_readlane(hi, k)};
}

// starts[g] = tiles of `height` rows of the groups before g, for g <= groups
// (LDS; one wave).  Fewer than 2^16 for a height of 32 and more: 2^20 rows.
// (Edges that are not in order could have more: what is past 2^16 is left out.)
__device__ __forceinline__ void group_starts(const int32_t* offsets, int groups, int rows, int height, uint16_t* starts) {
    const int lane = threadIdx.x & 63;
    auto held = [](int n) { return (uint16_t)(n < 0xffff ? n : 0xffff); };
    int before = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) {
        const int g = g0 + lane;
        const int lo = g < groups ? group_edge(offsets, g, rows) : 0, hi = g < groups ? group_edge(offsets, g + 1, rows) : 0;
        const int own = hi > lo ? (hi - lo + height - 1) / height : 0, upto = wave_scan(own);
        if (g < groups) starts[g] = held(before + upto - own);
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (lane == 0) starts[groups] = held(before);
}

// At most so many tiles of `height` rows, wherever the groups' edges lie.
inline int64_t most_tiles(int64_t rows, int64_t groups, int64_t height) {
    return rows / height + (rows < groups ? rows : groups);
}

}  // namespace icq
