// Rows of activations and the groups they belong to: the router's choice of
// experts for a token, the order of (row, choice) pairs by group, and the
// weighted sum that brings the ordered rows back.
//
//   chosen:  the k largest of x[t, :], of equals the lowest; -inf is never chosen
//   weight:  exp(x_e - m) / sum exp(x - m), m = max x, over the chosen or over all
//   order:   pair t k + j is at offsets[g] + #{earlier pairs of group g}
//   back:    y[t] = r[t] + sum_j w[t, j] y[position[t, j]]
//
// The order is that of a counting sort whose counts are integers, so it does
// not depend on which work-group comes first.
#include "common.hpp"
#include "groups.hpp"
#include "lowbit.hpp"
#include "prof.hpp"

namespace icq {
namespace {

constexpr int kThreads = 1024;          // of a work-group that counts or places
constexpr int kMaxTop = 64;

// Keys order like the values, a NaN above all of them and the two zeros equal;
// 0 is what a mask (-inf) took out, or what has been chosen already.
__device__ __forceinline__ unsigned logit_key(float x) {
    if (x != x) return 0xffffffffu;
    return x == -INFINITY ? 0u : float_key(x + 0.0f);
}
__device__ __forceinline__ float key_logit(unsigned k) { return k == 0xffffffffu ? __uint_as_float(0x7fc00000u) : key_float(k); }

// The choice of one token by one wave.  A lane has SLOTS consecutive experts and
// sorts them, largest first and of equals the lowest, so that a choice is a
// maximum over the lanes' first ones, and of lanes with that maximum the lowest.
template <int SLOTS>
__device__ __forceinline__ void choose(const float (&logit)[SLOTS], int top, int renormalize, int& id, float& weight) {
    const int lane = threadIdx.x & 63;
    unsigned key[SLOTS];
    int expert[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        expert[i] = lane * SLOTS + i;
        key[i] = logit_key(logit[i]);
    }
#pragma unroll
    for (int n = SLOTS - 1; n > 0; --n)
#pragma unroll
        for (int i = 0; i < n; ++i) {          // neighbours change places only if the second is larger: equals keep their order
            const bool swap = key[i + 1] > key[i];
            const unsigned k = key[i];
            const int e = expert[i];
            key[i] = swap ? key[i + 1] : k;
            expert[i] = swap ? expert[i + 1] : e;
            key[i + 1] = swap ? k : key[i + 1];
            expert[i + 1] = swap ? e : expert[i + 1];
        }
    unsigned best = wave_top(key[0]);
    const float peak = key_logit(best);
    float total = 0.0f;
    if (!renormalize) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) total += key[i] ? expf(key_logit(key[i]) - peak) : 0.0f;
        total = wave_total(total);
    }
    id = -1;
    unsigned own = 0;                          // lane j: the value of choice j
    for (int j = 0; j < top && best; ++j) {
        const unsigned long long at_best = __ballot(key[0] == best), taken = at_best & (0 - at_best);
        const unsigned long long mine = 1ull << j;
        id = (int)lanes_of(mine, (unsigned)__builtin_amdgcn_readlane(expert[0], __builtin_ctzll(at_best)), (unsigned)id);
        own = lanes_of(mine, best, own);
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            key[i] = lanes_of(taken, i + 1 < SLOTS ? key[i + 1 < SLOTS ? i + 1 : i] : 0u, key[i]);
            if (i + 1 < SLOTS) expert[i] = (int)lanes_of(taken, (unsigned)expert[i + 1 < SLOTS ? i + 1 : i], (unsigned)expert[i]);
        }
        best = wave_top(key[0]);
    }
    const float e = id < 0 ? 0.0f : expf(key_logit(own) - peak);
    if (renormalize) total = wave_total(e);
    weight = id < 0 ? 0.0f : e / total;
}

// What a unit of consecutive pairs adds to each group, for the units behind it.
struct Units {
    int64_t pairs;       // of all units
    int per_unit, units, groups;
    uint16_t* counts;    // [units, pitch]: a unit has fewer than 2^16 pairs
    __host__ __device__ int pitch() const { return (groups + 7) / 8 * 8; }
};

// Places this unit's pairs: groups' ids from `ids` (-1: none, ordered behind
// all groups), edges and earlier units' shares from the counts.
struct PlaceLds {
    int total[kMaxGroups + 1], before[kMaxGroups], base[kMaxGroups + 1], waves[2][kThreads / 64];
    uint16_t share[kThreads / 64][kMaxGroups + 1];       // of a wave's 64 pairs, then of the waves before it
};
__device__ __forceinline__ void write_counts(const Units& u, int unit, const int* count) {
    for (int g = threadIdx.x; g < u.pitch(); g += kThreads) u.counts[(int64_t)unit * u.pitch() + g] = (uint16_t)(g < u.groups ? count[g] : 0);
}
__device__ __forceinline__ void place_unit(const Units& u, int unit, const int32_t* ids, PlaceLds& s, int32_t* offsets,
                                           int32_t* order, int32_t* position) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t first = (int64_t)unit * u.per_unit, last = first + u.per_unit < u.pairs ? first + u.per_unit : u.pairs;
    int next = first + tid < last ? ids[first + tid] : -1;
    s.total[tid] = 0;
    s.before[tid] = 0;
    __syncthreads();
    // rows of `width` threads, 8 groups a thread; each row sums every so manieth unit (at most 32 rows meet in LDS)
    const int eights = u.pitch() / 8, width = eights <= 8 ? 8 : eights <= 16 ? 16 : eights <= 32 ? 32 : eights <= 64 ? 64 : 128;
    const int col = tid & (width - 1), row = tid / width, rows = kThreads / width < 32 ? kThreads / width : 32;
    if (col < eights && row < rows) {
        int total[8] = {}, before[8] = {};
#pragma unroll 8
        for (int k = row; k < u.units; k += rows) {
            const lb_u32x4 c = *reinterpret_cast<const lb_u32x4*>(u.counts + (int64_t)k * u.pitch() + col * 8);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int n = (int)(i & 1 ? c[i >> 1] >> 16 : c[i >> 1] & 0xffffu);
                total[i] += n;
                before[i] += k < unit ? n : 0;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {        // (group col * 8 + i at i * 128 + col: lanes on different banks)
            atomicAdd(&s.total[i * 128 + col], total[i]);        // integers: any order gives the same sum
            atomicAdd(&s.before[i * 128 + col], before[i]);
        }
    }
    __syncthreads();
    const int at_lds = (tid & 7) * 128 + (tid >> 3), total = s.total[at_lds], before = s.before[at_lds];      // (zeros behind the last group)
    const int upto = wave_scan(total), earlier = wave_scan(before);
    if (lane == 63) {
        s.waves[0][wave] = upto;
        s.waves[1][wave] = earlier;
    }
    __syncthreads();
    int start = upto - total, all = 0, mine = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
        start += w < wave ? s.waves[0][w] : 0;
        all += s.waves[0][w];
        mine += s.waves[1][w];
    }
    if (tid < u.groups) s.base[tid] = start + before;
    if (tid == 0) s.base[u.groups] = all + (int)(first - mine);          // pairs of no group
    if (unit == 0) {
        if (tid < u.groups) offsets[tid] = start;
        if (tid == 0) offsets[u.groups] = all;
    }
    __syncthreads();
    // 1024 pairs at a time: each wave ranks its 64, and the groups' shares of the 16 waves are summed in order
    for (int64_t p1 = first;; p1 += kThreads) {
        const int64_t p = p1 + tid;
        const bool have = p < last;
        const int id = next, key = id < 0 ? u.groups : id;
        next = p + kThreads < last ? ids[p + kThreads] : -1;
        for (int g = lane; g <= u.groups; g += 64) s.share[wave][g] = 0;
        unsigned long long same = __ballot(have);
        for (int b = 0; (u.groups >> b) != 0; ++b) {
            const unsigned long long m = __ballot((key >> b) & 1);
            same &= (key >> b) & 1 ? m : ~m;
        }
        const int rank = (int)__builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
        lds_wave_fence();
        if (have && rank == 0) s.share[wave][key] = (uint16_t)__builtin_popcountll(same);
        __syncthreads();
        for (int g = tid; g <= u.groups; g += kThreads) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < kThreads / 64; ++w) {
                const int own = s.share[w][g];
                s.share[w][g] = (uint16_t)sum;
                sum += own;
            }
            s.total[g] = sum;
        }
        __syncthreads();
        if (have) {
            const int at = s.base[key] + s.share[wave][key] + rank;
            order[at] = id < 0 ? -1 : (int32_t)p;
            position[p] = id < 0 ? -1 : at;
        }
        if (p1 + kThreads >= last) break;
        __syncthreads();
        for (int g = tid; g <= u.groups; g += kThreads) s.base[g] += s.total[g];
    }
}

// Tokens of a unit, a wave each in turn; with one unit the pairs are placed at once.
// 8191 x 256 fp32, top 8, in a graph 17.0 us with the placing, traced 9.8 to 10.6
// and 7.4 to 7.6 us (two kernels that do next to nothing take 9 in a graph; 9.4
// MB).  A token takes a wave some 390 vector instructions, 5 us of the first.  One
// token of 64 experts: 4.8 us traced, all of it latency.
template <int DT, int SLOTS>
__global__ __launch_bounds__(kThreads) void route_kernel(const void* __restrict__ logits, int64_t tokens, int64_t ld, int top,
                                                         int renormalize, int tokens_per_unit, Units u,
                                                         int32_t* __restrict__ ids, float* __restrict__ weights,
                                                         int32_t* offsets, int32_t* order, int32_t* position) {
    __shared__ PlaceLds s;
    const int tid = threadIdx.x, lane = tid & 63, unit = blockIdx.x;
    int* count = s.total;
    count[tid] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)unit * tokens_per_unit, t1 = t0 + tokens_per_unit < tokens ? t0 + tokens_per_unit : tokens;
    float next[SLOTS];                       // of the wave's next token
    auto load = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) next[i] = t < t1 && lane * SLOTS + i < u.groups ? load_as_f32(logits, DT, t * ld + lane * SLOTS + i) : -INFINITY;
    };
    load(t0 + (tid >> 6));
    for (int64_t t = t0 + (tid >> 6); t < t1; t += kThreads / 64) {
        float logit[SLOTS];
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) logit[i] = next[i];
        load(t + kThreads / 64);
        int id;
        float w;
        choose<SLOTS>(logit, top, renormalize, id, w);
        if (lane < top) {
            ids[t * top + lane] = id;
            weights[t * top + lane] = w;
            if (id >= 0) atomicAdd(&count[id], 1);
        }
    }
    __syncthreads();
    write_counts(u, unit, count);
    if (u.units == 1) {
        __syncthreads();
        place_unit(u, 0, ids, s, offsets, order, position);
    }
}

// Ids from elsewhere: those outside [0, groups) become -1.
template <typename ID>
__global__ __launch_bounds__(kThreads) void count_kernel(const ID* __restrict__ given, Units u, int32_t* __restrict__ ids,
                                                         int32_t* offsets, int32_t* order, int32_t* position) {
    __shared__ PlaceLds s;
    const int tid = threadIdx.x, unit = blockIdx.x;
    int* count = s.total;
    count[tid] = 0;
    __syncthreads();
    const int64_t first = (int64_t)unit * u.per_unit, last = first + u.per_unit < u.pairs ? first + u.per_unit : u.pairs;
    for (int64_t p = first + tid; p < last; p += kThreads) {
        const ID id = given[p];
        const bool is = id >= 0 && id < u.groups;
        ids[p] = is ? (int32_t)id : -1;
        if (is) atomicAdd(&count[(int)id], 1);
    }
    __syncthreads();
    write_counts(u, unit, count);
    if (u.units == 1) {
        __syncthreads();
        place_unit(u, 0, ids, s, offsets, order, position);
    }
}

__global__ __launch_bounds__(kThreads) void place_kernel(Units u, const int32_t* __restrict__ ids, int32_t* offsets,
                                                         int32_t* order, int32_t* position) {
    __shared__ PlaceLds s;
    place_unit(u, blockIdx.x, ids, s, offsets, order, position);
}

// Units of whole rows (a row has `per_row` pairs): at least 16 rows, one a wave
// of the work-group, and at most 256 units.
int rows_per_unit(int64_t rows) {
    const int64_t n = cdiv(rows, 256);
    return (int)(n < 16 ? 16 : n);
}

// Rows back to their tokens: a lane has 8 columns, and four rows' loads in flight.
// HBM bounds it: 8192 x 4096 bf16, top 4, with residual 76 us, 5.3 TB/s.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t base, int c0, int cols, float (&v)[8]) {
    if (c0 + 8 <= cols) {
        if (DT == IC_DTYPE_F32) {
            const lb_f32x4_any* q = reinterpret_cast<const lb_f32x4_any*>(static_cast<const float*>(p) + base + c0);
            const lb_f32x4 a = q[0], b = q[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
        } else {
            const lb_u32x4 t = *reinterpret_cast<const lb_u32x4_any*>(static_cast<const uint16_t*>(p) + base + c0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = half_word<DT>(t[i], 0);
                v[2 * i + 1] = half_word<DT>(t[i], 1);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? load_as_f32(p, DT, base + c0 + i) : 0.0f;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void combine_kernel(const void* __restrict__ y, int64_t pairs, int cols, int64_t ld_y,
                                                      const int32_t* __restrict__ position, const float* __restrict__ weights,
                                                      int top, const void* residual, int64_t ld_r, void* out, int64_t ld_out,
                                                      int64_t tokens, int chunks) {
    const int64_t piece = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, t = piece / chunks;
    const int c0 = ((int)(piece - t * chunks) * 256 + threadIdx.x) * 8;
    if (t >= tokens || c0 >= cols) return;
    float sum[8];
    if (residual) load8<DT>(residual, t * ld_r, c0, cols, sum);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
    }
    for (int j0 = 0; j0 < top; j0 += 4) {
        float v[4][8];
        int at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            at[j] = j0 + j < top ? position[t * top + j0 + j] : -1;
            if (at[j] >= pairs) at[j] = -1;
            if (at[j] >= 0) load8<DT>(y, at[j] * ld_y, c0, cols, v[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (at[j] < 0) continue;
            const float w = weights[t * top + j0 + j];
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = __builtin_fmaf(w, v[j][i], sum[i]);
        }
    }
    store_cols<DT, 8>(out, t * ld_out, c0, cols, sum);
}

int check_groups(const char* who, int64_t rows, int64_t per_row, int64_t groups) {
    const std::string w(who);
    if (rows < 0 || per_row < 1 || groups < 1) return fail(IC_ERR_ARG, w + ": rows must be >= 0, groups and choices >= 1");
    if (groups > kMaxGroups || per_row > kMaxTop || rows > kMaxRows || rows * per_row > kMaxRows)
        return fail(IC_ERR_RANGE, w + ": at most 1024 groups, 64 choices a row and 1048560 pairs");
    return IC_OK;
}

template <int DT>
void launch_route(const void* logits, int64_t tokens, int64_t ld, int top, int renormalize, int per, const Units& u, int32_t* ids,
                  float* weights, int32_t* offsets, int32_t* order, int32_t* position, hipStream_t st) {
    auto go = [&](auto slots) {
        hipLaunchKernelGGL((route_kernel<DT, decltype(slots)::value>), dim3(u.units), dim3(kThreads), 0, st, logits, tokens, ld, top,
                           renormalize, per, u, ids, weights, offsets, order, position);
    };
    if (u.groups <= 64) go(std::integral_constant<int, 1>{});
    else if (u.groups <= 128) go(std::integral_constant<int, 2>{});
    else if (u.groups <= 256) go(std::integral_constant<int, 4>{});
    else if (u.groups <= 512) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
}

}  // namespace
}  // namespace icq

using namespace icq;

extern "C" int64_t ic_group_workspace_bytes(int64_t rows, int64_t groups) {
    if (rows < 0 || groups < 1 || groups > kMaxGroups || rows > kMaxRows) return 0;
    return cdiv(rows, rows_per_unit(rows)) * cdiv(groups, 8) * 16;
}

extern "C" int ic_route_tokens(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t ld, int top, int renormalize,
                               int32_t* ids, float* weights, int32_t* offsets, int32_t* order, int32_t* position,
                               void* workspace, void* stream) {
    if (const int rc = check_groups("ic_route_tokens", tokens, top, experts)) return rc;
    IC_REQUIRE(dtype >= 0 && dtype <= 2, "ic_route_tokens: unknown dtype");
    IC_REQUIRE(top <= experts, "ic_route_tokens: more choices than experts");
    IC_REQUIRE(offsets && (tokens == 0 || (logits && ids && weights && order && position && workspace)),
               "ic_route_tokens: null pointer");
    IC_REQUIRE(aligned16(workspace), "ic_route_tokens: workspace not 16-byte aligned");
    IC_REQUIRE(tokens <= 1 || ld >= experts, "ic_route_tokens: leading dimension below the number of experts");
    hipStream_t st = as_stream(stream);
    const int per = rows_per_unit(tokens);
    const int units = tokens ? (int)cdiv(tokens, per) : 1;
    ProfScope prof(st, PT_OTHER, 0.0, (double)tokens * experts * (dtype == IC_DTYPE_F32 ? 4 : 2) + 16.0 * tokens * top);
    const Units u{tokens * top, per * top, units, (int)experts, static_cast<uint16_t*>(workspace)};
    if (tokens == 0) {
        hipLaunchKernelGGL(place_kernel, dim3(1), dim3(kThreads), 0, st, Units{0, 1, 0, (int)experts, nullptr}, ids, offsets, order, position);
        IC_CHECK_LAUNCH();
        return IC_OK;
    }
    if (dtype == IC_DTYPE_F32) launch_route<IC_DTYPE_F32>(logits, tokens, ld, top, renormalize, per, u, ids, weights, offsets, order, position, st);
    else if (dtype == IC_DTYPE_BF16) launch_route<IC_DTYPE_BF16>(logits, tokens, ld, top, renormalize, per, u, ids, weights, offsets, order, position, st);
    else launch_route<IC_DTYPE_F16>(logits, tokens, ld, top, renormalize, per, u, ids, weights, offsets, order, position, st);
    if (units > 1) hipLaunchKernelGGL(place_kernel, dim3(units), dim3(kThreads), 0, st, u, ids, offsets, order, position);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

extern "C" int ic_group_rows(const void* given, int wide, int64_t rows, int64_t per_row, int64_t groups, int32_t* ids, int32_t* offsets,
                             int32_t* order, int32_t* position, void* workspace, void* stream) {
    if (const int rc = check_groups("ic_group_rows", rows, per_row, groups)) return rc;
    IC_REQUIRE(offsets && (rows == 0 || (given && ids && order && position && workspace)), "ic_group_rows: null pointer");
    IC_REQUIRE(aligned16(workspace), "ic_group_rows: workspace not 16-byte aligned");
    hipStream_t st = as_stream(stream);
    // up to 2048 pairs need no second launch (64 rows 5.2 us in a graph, 7.2 with two; a router's tokens do: a wave takes
    // some microseconds for each, 64 tokens 9.5 us with two launches and 15.9 with one)
    const int per = rows * per_row <= 2048 ? (int)(rows ? rows : 1) : rows_per_unit(rows);
    const int units = rows ? (int)cdiv(rows, per) : 1;
    ProfScope prof(st, PT_OTHER, 0.0, (wide ? 20.0 : 16.0) * rows * per_row);
    const Units u{rows * per_row, (int)(per * per_row), units, (int)groups, static_cast<uint16_t*>(workspace)};
    if (rows == 0) {
        hipLaunchKernelGGL(place_kernel, dim3(1), dim3(kThreads), 0, st, Units{0, 1, 0, (int)groups, nullptr}, ids, offsets, order, position);
        IC_CHECK_LAUNCH();
        return IC_OK;
    }
    if (wide) hipLaunchKernelGGL(count_kernel<int64_t>, dim3(units), dim3(kThreads), 0, st, static_cast<const int64_t*>(given), u, ids, offsets, order, position);
    else hipLaunchKernelGGL(count_kernel<int32_t>, dim3(units), dim3(kThreads), 0, st, static_cast<const int32_t*>(given), u, ids, offsets, order, position);
    if (units > 1) hipLaunchKernelGGL(place_kernel, dim3(units), dim3(kThreads), 0, st, u, ids, offsets, order, position);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

extern "C" int ic_combine_rows(const void* y, int dtype, int64_t tokens, int64_t top, int64_t cols, int64_t ld_y, const int32_t* position,
                               const float* weights, const void* residual, int64_t ld_r, void* out, int64_t ld_out, void* stream) {
    IC_REQUIRE(tokens >= 0 && top >= 1 && cols >= 1, "ic_combine_rows: tokens must be >= 0, top and cols >= 1");
    IC_REQUIRE(dtype >= 0 && dtype <= 2, "ic_combine_rows: unknown dtype");
    if (tokens > kMaxRows || top > kMaxTop || tokens * top > kMaxRows || cols > kMaxRows)
        return fail(IC_ERR_RANGE, "ic_combine_rows: at most 64 choices a token, 1048560 pairs and as many columns");
    if (tokens == 0) return IC_OK;
    IC_REQUIRE(y && position && weights && out, "ic_combine_rows: null pointer");
    IC_REQUIRE(ld_y >= cols && ld_out >= cols && (!residual || ld_r >= cols), "ic_combine_rows: leading dimension below cols");
    const int chunks = (int)cdiv(cols, 2048);
    // along one axis a launch has fewer than 2^32 threads: pieces in runs of 2^20
    const int64_t pieces = tokens * chunks, run = pieces < (1 << 20) ? pieces : 1 << 20;
    hipStream_t st = as_stream(stream);
    const int es = dtype == IC_DTYPE_F32 ? 4 : 2;
    ProfScope prof(st, PT_OTHER, 2.0 * tokens * top * cols, (double)es * tokens * cols * (top + (residual ? 2 : 1)));
    auto go = [&](auto dt) {
        hipLaunchKernelGGL(combine_kernel<decltype(dt)::value>, dim3((unsigned)run, (unsigned)cdiv(pieces, run)), dim3(256), 0, st, y,
                           tokens * top, (int)cols, ld_y, position, weights, (int)top, residual, ld_r, out, ld_out, tokens, chunks);
    };
    if (dtype == IC_DTYPE_F32) go(std::integral_constant<int, IC_DTYPE_F32>{});
    else if (dtype == IC_DTYPE_BF16) go(std::integral_constant<int, IC_DTYPE_BF16>{});
    else go(std::integral_constant<int, IC_DTYPE_F16>{});
    IC_CHECK_LAUNCH();
    return IC_OK;
}
