// Products with quantised weights, y = x W^T + b:
//   INT8 / INT4 weights [N, K] with a scale (and zero-point) a row, 8-bit
//   activations [M, K] with a scale a row:
//     y[m, n] = sa[m] sw[n] (sum_k a q - zp[n] sum_k a) + b[n],
//   the sums exact in 32-bit integers; and both operands in microscaled
//   4-bit floating point, accumulated in fp32.
// The weights are the matrix instructions' first operand, so a lane ends
// with four consecutive outputs of one row of y.
//
// Two further modes of the integer kinds:
//   grouped   rows of y are ordered by group, each group has a weight of its
//             own, and row i of y may come from another row of x;
//   adapted   y[m, n] += sum_r t[m, r] B_a[n, r], a the adapter of row m and
//             t = scale_a A_a x (adapters.hip).
#include "common.hpp"
#include "prof.hpp"
#include "lowbit.hpp"
#include "adapters.hpp"
#include "groups.hpp"

namespace icq {
namespace {

enum Kind { kInt8 = 0, kInt4 = 1, kMx = 2 };
enum Mode { kPlain, kGrouped, kAdapted, kAdaptedWhole };       // (kAdaptedWhole: t to its last bit, for fp32 results)
constexpr bool adapted(int mode) { return mode == kAdapted || mode == kAdaptedWhole; }

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Operands {
    const uint8_t* a;        // activations: int8 rows (pitch ld_a), or E2M1 tiles
    const uint32_t* a_scale; // E8M0 words of the activations (kMx)
    int64_t ld_a;
    const float* sa;         // [M] (integer kinds)
    const int32_t* sums;     // [M] (integer kinds with zero-points)
    const uint8_t* w;        // weight tiles
    const uint32_t* w_scale; // E8M0 words of the weights (kMx)
    const void* sw;          // [N] fp16 or fp32 (integer kinds)
    int sw_f32;
    const int8_t* zp;        // [N] or null
    const void* bias;        // [N] or null
    int bias_dtype;
    int64_t M, N, K;
    void* out;
    int out_dtype;
    int64_t ld_out;
    int wide;                // rows of out are 16-byte aligned and whole groups of 8 values
    // kGrouped: w, sw, zp and bias are those of all groups, one after another
    const int32_t* offsets;  // [groups + 1]
    const int32_t* order;    // [M], where top > 0: row i of y is of row order[i] / top of the activations
    int groups, top;
    int a_rows;              // rows of the activations
    int64_t w_group;         // bytes of a group's tiles
    Adapted ad;              // kAdapted
};

// The row of activations that row m of y comes from (the last, where the order
// names none of them: -1 / 1 is past the last as an unsigned number too).
template <int MODE>
__device__ __forceinline__ int source_row(const Operands& p, int m) {
    if (MODE != kGrouped || !p.top) return m;
    const unsigned s = (unsigned)p.order[m] / (unsigned)p.top;
    return s < (unsigned)p.a_rows ? (int)s : p.a_rows - 1;
}

template <int KIND> struct Acc { typedef i32x4 T; };
template <> struct Acc<kMx> { typedef lb_f32x4 T; };

// What the outputs of four consecutive columns from n0 need (columns past the
// last repeat the last).
template <int KIND>
struct Columns {
    float sw[4], bias[4];
    int zp[4];
    __device__ __forceinline__ void load(const Operands& p, int64_t n0, int64_t first = 0) {    // (first: a group's columns)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = first + (n0 + i < p.N ? n0 + i : p.N - 1);
            if (KIND != kMx) {
                sw[i] = p.sw_f32 ? static_cast<const float*>(p.sw)[n] : f16_bits_to_f32(static_cast<const uint16_t*>(p.sw)[n]);
                zp[i] = p.zp ? p.zp[n] : 0;
            }
            bias[i] = p.bias ? load_as_f32(p.bias, p.bias_dtype, n) : 0.0f;
        }
    }
    // y from the accumulated sums of a row with scale sa and code sum `sum`
    __device__ __forceinline__ lb_f32x4 finish(typename Acc<KIND>::T acc, float sa, int sum) const {
        lb_f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (KIND == kMx) {
                v[i] = acc[i] + bias[i];
            } else {
                // INT4 operands are held as 16 q; the shift is exact.  |sum_k a (q - zp)| < 2^31 for K <= 65536, so
                // the difference is right even where a term has wrapped
                const int d = (int)((unsigned)(KIND == kInt4 ? acc[i] >> 4 : acc[i]) - (unsigned)zp[i] * (unsigned)sum);
                v[i] = (float)d * (sa * sw[i]) + bias[i];
            }
        }
        return v;
    }
};

// Four consecutive outputs of row m from column n.
__device__ __forceinline__ void store4(const Operands& p, lb_f32x4 v, int64_t m, int64_t n, int64_t end) {
    if (m >= end || n >= p.N) return;
    const int64_t at = m * p.ld_out + n;
    if (p.wide && n + 4 <= p.N) {
        if (p.out_dtype == IC_DTYPE_F32)
            *reinterpret_cast<lb_f32x4*>(static_cast<float*>(p.out) + at) = v;
        else if (p.out_dtype == IC_DTYPE_BF16)
            *reinterpret_cast<lb_u32x2*>(static_cast<uint16_t*>(p.out) + at) =
                lb_u32x2{pack_half_words<IC_DTYPE_BF16>(v[0], v[1]), pack_half_words<IC_DTYPE_BF16>(v[2], v[3])};
        else
            *reinterpret_cast<lb_u32x2*>(static_cast<uint16_t*>(p.out) + at) =
                lb_u32x2{pack_half_words<IC_DTYPE_F16>(v[0], v[1]), pack_half_words<IC_DTYPE_F16>(v[2], v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) store_from_f32(p.out, p.out_dtype, at + i, v[i]);
    }
}

// acc += W tile (16 n x 128 k) * X tile (128 k x 16 m).
__device__ __forceinline__ i32x4 mma_i8(lb_u32x4 w, lb_u32x4 x, i32x4 acc) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), acc, 0, 0, 0);
}
__device__ __forceinline__ lb_f32x4 mma_mx(lb_u32x4 w, lb_u32x4 x, lb_f32x4 acc, int sw, int sx) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, sw, 0, sx);
}
// The same products of 32 rows and 32 columns, with twice the operations an
// instruction (a wave alone on its SIMD reaches 4.7 POP/s and 8.9 PFLOP/s with
// these over the card, 2.9 and 5.1 with the smaller ones).
template <typename T>
__device__ __forceinline__ T mma32_ranks(lb_u32x4 w, lb_u32x4 x, T acc) {      // (acc: fp32 values)
    return __builtin_bit_cast(T, __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lb_bf16x8, w), __builtin_bit_cast(lb_bf16x8, x),
                                                                                     __builtin_bit_cast(lb_f32x16, acc), 0, 0, 0));
}
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <int KIND> struct Acc32 { typedef i32x16 T; };
template <> struct Acc32<kMx> { typedef f32x16 T; };
__device__ __forceinline__ i32x16 mma32_i8(lb_u32x4 w, lb_u32x4 x, i32x16 acc) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), acc, 0, 0, 0);
}
// (byte B of each scale word)
template <int B>
__device__ __forceinline__ f32x16 mma32_mx(lb_u32x4 w, lb_u32x4 x, f32x16 acc, int sw, int sx) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 4, 4, B, sw, B, sx);
}
// 32 INT4 values of a lane as two operands of 16 bytes, each value times 16.
__device__ __forceinline__ lb_u32x4 low_nibbles(lb_u32x4 p) { return (p << 4) & 0xf0f0f0f0u; }
__device__ __forceinline__ lb_u32x4 high_nibbles(lb_u32x4 p) { return p & 0xf0f0f0f0u; }

// The 16 bytes that lane `from` holds.  Activations are loaded with four lanes
// on 64 consecutive bytes of a row (an operand's own order, 16 rows in 16
// consecutive lanes, makes 64 requests of a load instead of 16) and then
// exchanged into an operand's order.
__device__ __forceinline__ lb_u32x4 to_operand(lb_u32x4 v, int from) {
    lb_u32x4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (uint32_t)__builtin_amdgcn_ds_bpermute(from * 4, (int)v[k]);
    return o;
}

// Few rows: a work-group of 8 waves takes 16 columns of y and 16 MT rows,
// its waves a share of K each; the sums are joined in LDS in a fixed order.
// One row is bound by the weights' bytes (25 MB) and the launch: INT4 1 x 12288 x
// 4096 6.4 us traced alone, 5.3 us a call in a graph with its weights in cache
// (4.8 TB/s), 8.3 us from HBM (3.0 TB/s, many weights in turn); MXFP4 8 x 4096 x
// 12288 6.1, 5.6 and 11.4 us.  More rows are bound by their activations, which
// every work-group reads and exchanges again: INT8 333 x 1000 x 2901 10.8 us.
template <int KIND, int MT>
__global__ __launch_bounds__(512) void linear_direct_kernel(Operands p) {
    typedef typename Acc<KIND>::T acc_t;
    constexpr int WAVES = 8;
    __shared__ acc_t part[WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int64_t nt = blockIdx.x, mt0 = (int64_t)blockIdx.y * MT;
    const int64_t tiles = cdiv(p.K, 128), words = cdiv(p.K, 512);
    const int64_t t0 = tiles * wave / WAVES, t1 = tiles * (wave + 1) / WAVES;
    const lb_u32x4* wt = reinterpret_cast<const lb_u32x4*>(p.w) + nt * tiles * (KIND == kInt8 ? 128 : 64) + lane;
    const int64_t m_tiles = cdiv(p.M, 16);
    acc_t acc[MT];
    const uint8_t* row[MT];            // rows past the last are read from the last, and dropped at the end
    const lb_u32x4* xt[MT];
    const uint32_t* xs[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        acc[i] = acc_t{0, 0, 0, 0};
        if (KIND == kMx) {
            const int64_t mt = mt0 + i < m_tiles ? mt0 + i : m_tiles - 1;
            xt[i] = reinterpret_cast<const lb_u32x4*>(p.a) + mt * tiles * 64 + lane;
            xs[i] = p.a_scale + mt * words * 64 + lane;
        } else {
            const int64_t m = (mt0 + i) * 16 + (lane >> 2) < p.M ? (mt0 + i) * 16 + (lane >> 2) : p.M - 1;
            row[i] = p.a + m * p.ld_a + (lane & 3) * 16;
        }
    }
    const uint32_t* ws = KIND == kMx ? p.w_scale + nt * words * 64 + lane : nullptr;
    for (int64_t t = t0; t < t1; ++t) {
        if constexpr (KIND == kMx) {
            const lb_u32x4 w = wt[t * 64];
            const int sw = (int)(ws[(t >> 2) * 64] >> (8 * (t & 3)));
#pragma unroll
            for (int i = 0; i < MT; ++i)
                acc[i] = mma_mx(w, xt[i][t * 64], acc[i], sw & 255, (int)(xs[i][(t >> 2) * 64] >> (8 * (t & 3))) & 255);
        } else {
            lb_u32x4 w0, w1;
            if (KIND == kInt8) {
                w0 = wt[t * 128];
                w1 = wt[t * 128 + 64];
            } else {
                const lb_u32x4 q = wt[t * 64];
                w0 = low_nibbles(q);
                w1 = high_nibbles(q);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const lb_u32x4* x = reinterpret_cast<const lb_u32x4*>(row[i] + t * 128);
                const lb_u32x4 x0 = x[0], x1 = x[4];
                acc[i] = mma_i8(w0, to_operand(x0, r * 4 + g), acc[i]);
                acc[i] = mma_i8(w1, to_operand(x1, r * 4 + g), acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    Columns<KIND> cols;
    cols.load(p, nt * 16 + g * 4);
    for (int i = wave; i < MT; i += WAVES) {
        acc_t s = part[0][i][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) s += part[k][i][lane];
        const int64_t m = (mt0 + i) * 16 + r < p.M ? (mt0 + i) * 16 + r : p.M - 1;
        store4(p, cols.finish(s, KIND == kMx ? 1.0f : p.sa[m], KIND != kMx && p.zp ? p.sums[m] : 0), (mt0 + i) * 16 + r,
               nt * 16 + g * 4, p.M);
    }
}

// The same for grouped and adapted products: a work-group of 8 waves takes 16 NT
// columns and 16 MT rows, its waves a share of K each, so that activations that
// have been loaded and exchanged serve NT tiles of weights.  The next step's
// loads are on their way during a step's products.  Sums are integers: waves
// add theirs in LDS in any order.
//
// One token's four experts of 64, INT4 2816 x 4096: traced 7.1 to 7.7 us, 9.0 to
// 9.6 a launch in a graph with weights from HBM (23 MB: 2.5 TB/s); 8 experts 10.9
// us (4.2 TB/s).  Latency bounds it: the launch, the tile's place, then 4 steps of
// a wave.  With two or four steps' loads in flight it was slower (12 and 22 %
// with 64 groups of 4 rows), as fewer waves fit.
template <int KIND, int MT, int NT, int MODE>
__global__ __launch_bounds__(512) void linear_wide_kernel(Operands p) {
    constexpr int WAVES = 8, W = KIND == kInt8 ? 2 : 1;
    static_assert(KIND != kMx && MODE != kPlain, "integer kinds");
    __shared__ int sum[MT * NT][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int n_tiles = (int)cdiv(p.N, 16), nt0 = (int)blockIdx.x * NT;
    int m0 = (int)blockIdx.y * 16 * MT, m_end = (int)p.M;
    int64_t column0 = 0;
    const uint8_t* weight = p.w;
    if constexpr (MODE == kGrouped) {
        const GroupTile tile = find_tile(p.offsets, p.groups, (int)p.M, 16 * MT, blockIdx.y);
        if (tile.group < 0) return;
        m0 = tile.first;
        m_end = tile.end;
        column0 = tile.group * p.N;
        weight += tile.group * p.w_group;
    }
    const int tiles = (int)cdiv(p.K, 128), t0 = tiles * wave / WAVES, t1 = tiles * (wave + 1) / WAVES;
    const lb_u32x4* wt[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)       // (tiles past the last repeat the last; their outputs are dropped)
        wt[j] = reinterpret_cast<const lb_u32x4*>(weight) + (int64_t)(nt0 + j < n_tiles ? nt0 + j : n_tiles - 1) * tiles * (64 * W) + lane;
    const lb_u32x4* row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = m0 + i * 16 + (lane >> 2) < m_end ? m0 + i * 16 + (lane >> 2) : m_end - 1;
        row[i] = reinterpret_cast<const lb_u32x4*>(p.a + source_row<MODE>(p, m) * p.ld_a) + (lane & 3);
    }
    i32x4 acc[MT][NT];
    lb_u32x4 w[NT][W], x[MT][2];
    auto load = [&](int t) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < W; ++k) w[j][k] = wt[j][(t * W + k) * 64];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            x[i][0] = row[i][t * 8];
            x[i][1] = row[i][t * 8 + 4];
        }
    };
    // the adapters' part of the wave's outputs, whose loads wait together with the first of the product
    // (with fewer tiles than waves a tile's ranks are shared among waves)
    constexpr int OWN = (MT * NT + WAVES - 1) / WAVES, SHARES = MT * NT < WAVES ? WAVES / (MT * NT) : 1;
    __shared__ lb_f32x4 shared[adapted(MODE) && SHARES > 1 ? WAVES : 1][64];
    lb_f32x4 added[OWN];
    const int own_wave = __builtin_amdgcn_readfirstlane(wave), u0 = own_wave % (MT * NT < WAVES ? MT * NT : WAVES);
    int id[OWN];
    if constexpr (adapted(MODE)) {
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int u = u0 + k * WAVES, m = m0 + u / NT * 16 + r;
            id[k] = u < MT * NT && m < m_end ? p.ad.ids[m] : -1;
        }
    }
    if (t0 < t1) load(t0);
    if constexpr (adapted(MODE)) {
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int u = u0 + k * WAVES;
            added[k] = adapter_tile<MODE == kAdaptedWhole>(p.ad, p.N, m_end, m0 + u / NT * 16 + r, id[k], nt0 + u % NT, SHARES > 1 ? own_wave / (MT * NT) : 0, SHARES);
        }
        if (SHARES > 1) shared[wave][lane] = added[0];
    }
    for (int k = threadIdx.x; k < MT * NT * 256; k += 64 * WAVES) (&sum[0][0][0])[k] = 0;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        lb_u32x4 now[NT][W], to[MT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < W; ++k) now[j][k] = w[j][k];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            to[i][0] = x[i][0];
            to[i][1] = x[i][1];
        }
        if (t + 1 < t1) load(t + 1);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const lb_u32x4 x0 = to_operand(to[i][0], r * 4 + g), x1 = to_operand(to[i][1], r * 4 + g);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                acc[i][j] = mma_i8(KIND == kInt8 ? now[j][0] : low_nibbles(now[j][0]), x0, acc[i][j]);
                acc[i][j] = mma_i8(KIND == kInt8 ? now[j][W - 1] : high_nibbles(now[j][0]), x1, acc[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) atomicAdd(&sum[i * NT + j][k][lane], acc[i][j][k]);
    __syncthreads();
#pragma unroll
    for (int own = 0; own < OWN; ++own) {
        const int u = wave + own * WAVES;
        if (u >= MT * NT) break;
        const int i = u / NT, j = u % NT, m = m0 + i * 16 + r, n = (nt0 + j) * 16 + g * 4;
        if (m >= m_end || n >= p.N) continue;
        Columns<KIND> cols;
        cols.load(p, n, column0);
        const int from = source_row<MODE>(p, m);
        const i32x4 s = {sum[u][0][lane], sum[u][1][lane], sum[u][2][lane], sum[u][3][lane]};
        lb_f32x4 y = cols.finish(s, p.sa[from], p.zp ? p.sums[from] : 0);
        if constexpr (adapted(MODE) && SHARES == 1) y += added[own];
        else if constexpr (adapted(MODE)) {
            lb_f32x4 a = shared[u][lane];
#pragma unroll
            for (int k = 1; k < SHARES; ++k) a += shared[u + k * MT * NT][lane];
            y += a;
        }
        store4(p, y, m, n, m_end);
    }
}

// Waits until at most N of this wave's global loads (copies to LDS among
// them) are outstanding and all its LDS reads are done, then meets the other
// waves of the work-group.  (A fence before a plain barrier would wait for
// every copy in flight.)
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Many rows.  A work-group of WM x WN waves takes tiles of y of 32 WM FM rows
// and 32 WN FN columns one after another, a wave FM x FN blocks of 32 x 32 of
// each.  K advances in stages (128 columns of 4-bit weights, 64 of INT8)
// through BUF buffers in LDS that are filled straight from global memory,
// BUF - 1 stages ahead of the products; a tile's first stages are on their way
// while the outputs of the tile before are stored.  Operands go from LDS to
// registers one set (32 bytes of each row) ahead of their products, between
// matrix instructions, so a wave waits neither for LDS nor long at the one
// barrier that a stage has: when it gets there, what is left of the stage is
// in registers, and its buffer is filled again.
//
// Measured, one call after another: INT4 8192 x 4096 x 12288 326 us, 2.5 POP/s
// (341 to 345 on another card; traced alone 325 to 376); MXFP4 8192 x 12288 x
// 4096 226 us, 3.7 PFLOP/s (traced 216 to 256).  What bounds the first is power:
// the chip clocks at 1.7 GHz under it, its matrix units are busy for 63 % of the
// cycles, and the same instructions with the same reads from LDS and nothing
// else reach 2.7 POP/s on random operands, 305 us (5.4 PFLOP/s for E2M1, 153 us
// for the second; 3.5 and 6.5 from registers alone).  The second's matrix units
// are busy for 47 %: nobody multiplies at the ends of its 32-stage tiles.  4
// waves of 128 x 128 read less LDS but took 383 and 301 us, a wave alone on its
// SIMD standing still at copies, barriers and outputs.  For INT4 an earlier
// kernel with 16 x 16 instructions, a work-group a tile, was faster: 318 to 323
// us where this one took 341 to 345 in turn on the same card.
//
// The 256 x 256 forms of INT4 and INT8 spill 16 and 4 registers (adapted 81 to
// 93; the grouped ones of 128 x 256 20 and 3), at a tile's start and end, none
// in the K loop.  Spills are vector-memory operations like those that meet()
// counts.  It lets the newest N stay outstanding; with spills among these it
// waits for more copies than it needs, never for fewer.
//
// Grouped: tiles are numbered group by group, whatever their number of rows; a
// work-group finds its tile's group by bisection in LDS.  8192 tokens x 4 of 32
// experts 2816 x 4096 INT4 370 to 383 us a call (traced, medians on three cards
// 403 to 421, least 378), 2.0 POP/s (K = 4096 gives 2.2 in whole tiles; a group's
// last tile is half empty on average): 128 x 256 by two work-groups of 4 waves a
// CU, one at its products while the other is at a tile's end.  64 x 256
// took 409, 256 x 256 414.  Running only the blocks of 32 rows that a last tile
// has took as long (425 against 424, 256 x 256): rows that repeat cost little of
// the power that bounds the rest.  512 tokens x 4 of 64 experts, 32 rows each, 64 x
// 256 tiles: 83 to 87 us, 4.3 to 4.5 TB/s of weights (a large copy: 4.7 to 5.1).
//
// Adapted: 8192 x 4096 x 12288 INT4 with rank 64 traced 358 to 372 us (medians on
// three cards, least 347) where the plain product takes 343 to 349, 8192 x 4096 x
// 4096 149 and 124.  That is with one adapter or two a tile: each that its rows
// have costs the stages of its ranks over the whole tile.  8192 x 4096 x 4096, rank
// 64, a call: 172 us with 64 adapters' rows one after another, 480 with each row
// one of them at random.  Adding the adapters' products block by block behind the
// K loop, each waiting for its operands from L2, took 437 us.
template <int KIND, int WM, int WN, int FM, int FN, int BUF, int MODE = kPlain>
__global__ __launch_bounds__(64 * WM * WN, adapted(MODE) || FM == 4 ? 2 : 1) void linear_tiled_kernel(Operands p, int grid_m, int grid_n) {
    typedef typename Acc32<KIND>::T acc_t;
    constexpr int WAVES = WM * WN, BM = 32 * WM * FM, BN = 32 * WN * FN;
    constexpr int X_KB = BM / 16 * (KIND == kInt4 ? 2 : 1), W_KB = BN / 16;      // a stage's KB
    constexpr int X_LOADS = X_KB / WAVES, W_LOADS = W_KB / WAVES, LOADS = X_LOADS + W_LOADS;   // a wave's copies of 1 KB a stage
    constexpr int STAGE = (X_KB + W_KB) * 64;                                     // in 16-byte words
    constexpr int S_TILES = KIND == kMx ? (BM + BN) / 16 : 0, S_LOADS = S_TILES / (4 * WAVES), S_WORDS = S_TILES * 16;
    static_assert(X_KB % WAVES == 0 && W_KB % WAVES == 0 && S_TILES % (4 * WAVES) == 0, "each wave copies the same share");
    static_assert(FN == 2 && W_KB + X_KB >= WAVES * 4, "the epilogue stores 64 columns a wave, through one buffer");
    static_assert(BM <= 64 * WAVES && BN <= 64 * WAVES, "a thread holds one row's and one column's scale");
    constexpr int STORES = FM * 4;                                                // a lane's stores of a whole 16-bit tile
    // one array for all of it: the compiler guards reads of a second one with waits for every copy in flight.
    // BUF stages; two sets of scale words; a column's bias, scale and zero-point; a row's scale and code sum
    // (and a group's first row of tiles)
    constexpr int SCALES = BUF * STAGE, COLS = SCALES + 2 * S_WORDS, ROWS = COLS + BN * 3 / 4, GROUPS = ROWS + (KIND == kMx ? 0 : BM / 2);
    // (kAdapted: each row's adapter, and which of the adapters the rows have, a bit each, for two tiles in turn)
    __shared__ lb_u32x4 lds[GROUPS + (MODE == kGrouped ? kMaxGroups / 8 + 1 : adapted(MODE) ? BM / 4 + kMaxGroups / 64 : 0)];
    int* const row_id = reinterpret_cast<int*>(lds + GROUPS);
    unsigned* const present = reinterpret_cast<unsigned*>(lds + GROUPS + BM / 4);
    float* const col = reinterpret_cast<float*>(lds + COLS);
    float* const row = reinterpret_cast<float*>(lds + ROWS);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, r = lane & 31;
    const int wm = wave / WN, wn = wave % WN;
    const int lane16 = lane * 16;

    uint16_t* const starts = reinterpret_cast<uint16_t*>(lds + GROUPS);
    if constexpr (MODE == kGrouped) {
        if (wave == 0) group_starts(p.offsets, p.groups, (int)p.M, BM, starts);
        __syncthreads();
        grid_m = __builtin_amdgcn_readfirstlane((int)starts[p.groups]);
    }

    // work-groups are dealt to the 8 XCDs in turn: each XCD gets one run of tiles, walked in bands of 8 tile rows so
    // that what its L2 holds is used again
    const int total = grid_m * grid_n, xcd = blockIdx.x & 7, per = total >> 3, extra = total & 7;
    const int first = xcd * per + (xcd < extra ? xcd : extra), last = first + per + (xcd < extra ? 1 : 0);
    int tile = first + (blockIdx.x >> 3);
    if (tile >= last) return;

    const int k_tiles = (int)cdiv(p.K, 128), words = (int)cdiv(p.K, 512);
    const int n_tiles = (int)cdiv(p.N, 16), m_tiles = (int)cdiv(p.M, 16);
    const int k_stages = KIND == kInt8 ? (int)cdiv(p.K, 64) : k_tiles;
    int stages = k_stages;                                 // (kAdapted: and those of the adapters of the tile's rows)
    constexpr int W_STEP = 1024, X_STEP = KIND == kMx ? 1024 : KIND == kInt4 ? 128 : 64;
    const int w_pitch = k_tiles * (KIND == kInt8 ? 2048 : 1024);                  // bytes of a row of tiles

    // ---- copies.  Rows and tiles past the last repeat the last; their outputs are dropped.
    int bm = 0, bn = 0;
    int group = 0, row0 = 0, row_end = (int)p.M;           // the tile's first row, and the end of the rows it may have
    __amdgpu_buffer_rsrc_t x_buf, w_buf, xs_buf, ws_buf;
    int x_row[KIND == kMx ? X_LOADS : 1], w_row[W_LOADS], x_off[KIND == kMx ? 1 : X_LOADS], s_off[S_LOADS + 1];
    auto buffer = [](const void* base, int bytes = 0x7fffffff) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
    };
    auto aim = [&]() {
        int at = tile, rows_of = grid_m;                   // the tile's place among those of its group
        if constexpr (MODE == kGrouped) {
            // the last group that starts at or before the tile's row of tiles (empty groups start where the next one does)
            const int tile_row = tile / grid_n;
            int past = p.groups;
            group = 0;
            while (past - group > 1) {
                const int mid = (group + past) >> 1;
                if ((int)starts[mid] <= tile_row) group = mid;
                else past = mid;
            }
            group = __builtin_amdgcn_readfirstlane(group);
            const int s0 = __builtin_amdgcn_readfirstlane((int)starts[group]);
            rows_of = __builtin_amdgcn_readfirstlane((int)starts[group + 1]) - s0;
            at -= s0 * grid_n;
        }
        const int band = at / (8 * grid_n), rows_in = rows_of - band * 8 < 8 ? rows_of - band * 8 : 8;
        const int in_band = at - band * 8 * grid_n;
        bm = band * 8 + in_band % rows_in;
        bn = in_band / rows_in;
        if constexpr (MODE == kGrouped) {
            row0 = group_edge(p.offsets, group, (int)p.M) + bm * BM;
            row_end = group_edge(p.offsets, group + 1, (int)p.M);
        } else {
            row0 = bm * BM;
        }
        const int nt = bn * (BN / 16), nl = n_tiles - 1 - nt;
        w_buf = buffer(p.w + (MODE == kGrouped ? group * p.w_group : 0) + (int64_t)nt * w_pitch);
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i) w_row[i] = (i * WAVES + wave < nl ? i * WAVES + wave : nl) * w_pitch;
        if constexpr (KIND == kMx) {
            const int mt = bm * (BM / 16), ml = m_tiles - 1 - mt;
            x_buf = buffer(p.a + (int64_t)mt * w_pitch);
#pragma unroll
            for (int i = 0; i < X_LOADS; ++i) x_row[i] = (i * WAVES + wave < ml ? i * WAVES + wave : ml) * w_pitch;
            // 16 lanes copy the 256 bytes of a tile's word of scales; a copy takes four tiles of one operand
            xs_buf = buffer(p.a_scale + (int64_t)mt * words * 64);
            ws_buf = buffer(p.w_scale + (int64_t)nt * words * 64);
#pragma unroll
            for (int i = 0; i < S_LOADS; ++i) {
                const int t = (i * WAVES + wave) * 4, u = (t < BM / 16 ? t : t - BM / 16) + (lane >> 4), l = t < BM / 16 ? ml : nl;
                s_off[i] = (u < l ? u : l) * words * 256 + (lane & 15) * 16;
            }
        } else {
            // INT4: 8 rows of 128 bytes a copy, chunk c of row r in slot c ^ (r >> 1 & 7); INT8: 16 rows of 64 bytes, chunk
            // c in slot c ^ (r >> 2 & 3).  16 lanes that read one chunk of 16 rows then touch all 64 banks once.
            const int lane_row = KIND == kInt4 ? lane >> 3 : lane >> 2;
            const int chunk = KIND == kInt4 ? (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4)) : (lane & 3) ^ (lane >> 4);
            static_assert(WAVES % 2 == 0, "a wave's copies begin at rows of one parity of 8");
            const int ml = row_end - 1 - row0;
            // (gathered rows lie anywhere in the activations, which have less than 2^32 bytes then)
            if (MODE == kGrouped && p.top) x_buf = buffer(p.a, -1);
            else x_buf = buffer(p.a + (int64_t)row0 * p.ld_a);
#pragma unroll
            for (int i = 0; i < X_LOADS; ++i) {
                int row = (i * WAVES + wave) * (KIND == kInt4 ? 8 : 16) + lane_row;
                row = row < ml ? row : ml;
                if (MODE == kGrouped && p.top) row = source_row<MODE>(p, row0 + row);
                x_off[i] = (int)((unsigned)row * (unsigned)p.ld_a) + chunk * 16;
            }
        }
    };
    auto copy = [&](__amdgpu_buffer_rsrc_t from, int lane_off, int off, lb_u32x4* to) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, lane_off, off, 0, 0);
    };
    // kAdapted.  Behind the stages of K come those of each adapter that the tile's rows have: an operand of t lies like one
    // of the activations (INT4: 32 ranks of two of t's values in a stage, INT8: of one of them), one of B like one of the
    // weights.  Rows with another adapter or none take the row of zeros.  Fetched one after another: adapter `ad_now`,
    // its stage `ad_stage`.
    constexpr int T_BYTES = MODE == kAdaptedWhole ? 256 : 128;                    // of a row's part of t (kThree or kTwo), and its stages
    constexpr int T_STAGES = KIND == kInt8 ? (MODE == kAdaptedWhole ? 3 : 2) : T_BYTES / 128;
    const int ad_planes = p.ad.f16 ? 2 : 1, ad_stages = p.ad.parts * ad_planes * T_STAGES;
    int ad_now = -1, ad_stage = 0, ad_set = 0;
    auto next_adapter = [&]() {                            // the lowest in the set above ad_now (there is one)
        const unsigned* set = present + ad_set * (kMaxGroups / 32);
        const int at = ad_now + 1, l = lane & 31;
        unsigned w = set[l];
        w &= l < at >> 5 ? 0u : l == at >> 5 ? ~0u << (at & 31) : ~0u;
        const int first = __builtin_ctzll(__ballot(w != 0));
        ad_now = first * 32 + __builtin_ctz((unsigned)__builtin_amdgcn_readlane((int)w, first));
    };
    auto fetch_adapter = [&](int buf) {
        if constexpr (adapted(MODE)) {
            if (ad_stage == 0) next_adapter();
            lb_u32x4* to = lds + buf * STAGE + wave * 64;
            const int tile_of = ad_stage / T_STAGES;       // (part and plane)
            const int pitch = p.ad.parts * T_BYTES, part = tile_of / ad_planes;
            const int from = part * T_BYTES + (ad_stage - tile_of * T_STAGES) * (KIND == kInt8 ? 64 : 128);
            const int lane_row = KIND == kInt4 ? lane >> 3 : lane >> 2;
            const int chunk = KIND == kInt4 ? (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4)) : (lane & 3) ^ (lane >> 4);
            const __amdgpu_buffer_rsrc_t t_buf = buffer(p.ad.t);
#pragma unroll
            for (int i = 0; i < X_LOADS; ++i) {
                const int at = (i * WAVES + wave) * (KIND == kInt4 ? 8 : 16) + lane_row;
                copy(t_buf, (row_id[at] == ad_now ? row0 + at : (int)p.M) * pitch + chunk * 16, from, to + i * WAVES * 64);
            }
            const int nt = bn * (BN / 16), nl = n_tiles - 1 - nt, up_pitch = p.ad.parts * up_planes(p.ad.f16) * 1024;
            const __amdgpu_buffer_rsrc_t up_buf = buffer(p.ad.up + ((int64_t)ad_now * n_tiles + nt) * up_pitch);
#pragma unroll
            for (int i = 0; i < W_LOADS; ++i) {
                const int at = i * WAVES + wave < nl ? i * WAVES + wave : nl;
                copy(up_buf, lane16, at * up_pitch + (p.ad.f16 ? part * 3 + 1 + tile_of % 2 : part) * 1024, to + (X_LOADS + i) * WAVES * 64);
            }
            ad_stage = ad_stage + 1 == ad_stages ? 0 : ad_stage + 1;
        }
    };
    auto fetch = [&](int t, int buf) {
        if (adapted(MODE) && t >= k_stages) {
            fetch_adapter(buf);
            return;
        }
        lb_u32x4* to = lds + buf * STAGE + wave * 64;
        if constexpr (KIND == kMx) {
            if ((t & 3) == 0) {
                lb_u32x4* set = lds + SCALES + (t >> 2 & 1) * S_WORDS + wave * 64;
#pragma unroll
                for (int i = 0; i < S_LOADS; ++i) {
                    if ((i * WAVES + wave) * 4 < BM / 16) copy(xs_buf, s_off[i], (t >> 2) * 256, set + i * WAVES * 64);
                    else copy(ws_buf, s_off[i], (t >> 2) * 256, set + i * WAVES * 64);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < X_LOADS; ++i) {
            if constexpr (KIND == kMx) copy(x_buf, lane16, x_row[i] + t * X_STEP, to + i * WAVES * 64);
            else copy(x_buf, x_off[i], t * X_STEP, to + i * WAVES * 64);
        }
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i) copy(w_buf, lane16, w_row[i] + t * W_STEP, to + (X_LOADS + i) * WAVES * 64);
    };

    // ---- operands in registers: of a block of 32 rows, chunk 2 c + h of row r for set c.  Row r of a column block is
    // column (r / 16) 16 + (r / 4 & 1) 8 + (r / 8 & 1) 4 + r % 4 of the block's outputs, so that a lane ends with groups
    // of 8 consecutive outputs.
    lb_u32x4 xv[2][FM], wv[2][FN];
    int xs[KIND == kMx ? FM : 1][2], ws[KIND == kMx ? FN : 1][2];
    const int w_lane = (r >> 4) * 64 + h * 16 + (r >> 2 & 1) * 8 + (r >> 3 & 1) * 4 + (r & 3);
    auto read_x = [&](const lb_u32x4* s, lb_u32x4 (&to)[FM], int c) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int block = wm * FM + i;
            if (KIND == kMx) to[i] = s[block * 128 + (r >> 4) * 64 + (c * 2 + h) * 16 + (r & 15)];
            else if (KIND == kInt8) to[i] = s[(block * 32 + r) * 4 + ((c * 2 + h) ^ (r >> 2 & 3))];
            else to[i] = s[(block * 32 + r) * 8 + ((c * 2 + h) ^ (r >> 1 & 7))];
        }
    };
    auto read_w = [&](const lb_u32x4* s, lb_u32x4 (&to)[FN], int c) {
#pragma unroll
        for (int j = 0; j < FN; ++j) to[j] = s[X_KB * 64 + (wn * FN + j) * 128 + c * 32 + w_lane];
    };
    auto read_scales = [&](int t, int c) {
        if constexpr (KIND == kMx) {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(lds + SCALES + (t >> 2 & 1) * S_WORDS);
#pragma unroll
            for (int i = 0; i < FM; ++i) xs[i][c] = (int)q[(wm * FM + i) * 128 + (r >> 4) * 64 + (c * 2 + h) * 16 + (r & 15)];
#pragma unroll
            for (int j = 0; j < FN; ++j) ws[j][c] = (int)q[BM * 4 + (wn * FN + j) * 128 + c * 32 + w_lane];
        }
    };

    acc_t acc[FM][FN];
    int buf = 0;
    float c_scale = 1.0f, c_bias = 0.0f, r_scale = 1.0f;   // of the thread's column and row
    int c_zero = 0, r_sum = 0;
    auto start = [&]() {                                   // a tile's first copies
        aim();
        const int tid = threadIdx.x;
        int64_t n = bn * BN + tid < p.N ? bn * BN + tid : p.N - 1, m = row0 + tid < row_end ? row0 + tid : row_end - 1;
        if constexpr (MODE == kGrouped) {
            n += group * p.N;
            m = source_row<MODE>(p, (int)m);
        }
        if (KIND != kMx) {
            c_scale = p.sw_f32 ? static_cast<const float*>(p.sw)[n] : f16_bits_to_f32(static_cast<const uint16_t*>(p.sw)[n]);
            r_scale = p.sa[m];
            if (p.zp) {
                c_zero = p.zp[n];
                r_sum = p.sums[m];
            }
        }
        if (p.bias) c_bias = load_as_f32(p.bias, p.bias_dtype, n);
        if constexpr (adapted(MODE)) {                  // (K has BUF - 1 stages at least; the set is read behind the next barrier)
            int id = tid < BM && row0 + tid < row_end ? p.ad.ids[row0 + tid] : -1;
            if (id >= p.ad.adapters) id = -1;
            if (tid < BM) row_id[tid] = id;
            ad_set ^= 1;
            if (id >= 0) atomicOr(&present[ad_set * (kMaxGroups / 32) + (id >> 5)], 1u << (id & 31));
        }
#pragma unroll
        for (int b = 0; b < BUF - 1; ++b)
            if (b < k_stages) fetch(b, b);
    };
    // in stage t, when this wave has read the last of it: stage t + 1 has landed, and all waves are done with stage t's
    // buffer.  Behind the last stage whatever the next buffer holds is read, and not used: no branch parts the reads
    // from the products.
    auto advance = [&](int t) {
        if (t + 2 < BUF) meet<63>();                       // the first BUF - 1 had landed at the tile's start
        else if (t + BUF <= stages) meet<(BUF - 2) * LOADS>();
        else meet<0>();
        if (t + BUF < stages) fetch(t + BUF, buf);
        buf = buf + 1 == BUF ? 0 : buf + 1;
        return lds + buf * STAGE;
    };
    // a read from LDS, then its share of the matrix instructions
    auto interleave = [](auto reads_) {
        constexpr int READS = decltype(reads_)::value;
        auto one = [](auto i_) {
            constexpr int i = decltype(i_)::value, share = FM * FN * (i + 1) / READS - FM * FN * i / READS;
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, share, 0);
        };
        static_for<0, READS>(one);
    };

    // y from the accumulated sum: INT4 operands are held as 16 q, and the shift is exact.  |zp| <= 2^7 and
    // |sum| <= 2^23 for K <= 65536, so the 24-bit product is exact, and |sum_k a (q - zp)| < 2^31, so the
    // difference is right even where a term has wrapped.
    auto value = [&](auto s, float sw, float zero, float bias, float sa, float sum) {
        if constexpr (KIND == kMx) return s + bias;
        else {
            const unsigned d = (unsigned)(KIND == kInt4 ? s >> 4 : s) - (unsigned)__mul24(__float_as_int(zero), __float_as_int(sum));
            return (float)(int)d * (sa * sw) + bias;
        }
    };
    // kAdapted: whole values in place of the sums, before the adapters' stages.  (Each matrix instruction that follows
    // rounds the value: four for 32 ranks, six or eight with t whole, twice as many with fp16 factors.  A sum of the
    // adapters' part alone would take as many registers again as the sums have, and at 256 x 256 they have all.)
    auto whole_values = [&]() {
        // (two addresses, made here: the compiler would keep 80 of them over the K loop, spilled)
        const float* my_col = col + wn * FN * 32 + h * 8;
        const float* my_row = row + wm * FM * 32 + r;
        int at_col = (int)(my_col - reinterpret_cast<const float*>(lds)), at_row = (int)(my_row - reinterpret_cast<const float*>(lds));
        asm volatile("" : "+v"(at_col), "+v"(at_row));
        my_col = reinterpret_cast<const float*>(lds) + at_col;
        my_row = reinterpret_cast<const float*>(lds) + at_row;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const float sa = my_row[i * 32], sum = my_row[BM + i * 32];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                f32x16 v;
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float* c = my_col + j * 32 + (k >> 3) * 16 + (k & 7);
                    const lb_f32x4 bias = *reinterpret_cast<const lb_f32x4*>(c), sw = *reinterpret_cast<const lb_f32x4*>(c + BN);
                    const lb_f32x4 zero = *reinterpret_cast<const lb_f32x4*>(c + 2 * BN);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[k + e] = value(acc[i][j][k + e], sw[e], zero[e], bias[e], sa, sum);
                }
                acc[i][j] = __builtin_bit_cast(acc_t, v);
            }
        }
    };

    if constexpr (adapted(MODE)) {
        if (threadIdx.x < kMaxGroups / 16) present[threadIdx.x] = 0;
        lds_barrier();
    }
    start();
    meet<0>();
    for (;;) {
        if constexpr (adapted(MODE)) {
            const int own = lane < 32 ? __builtin_popcount(present[ad_set * (kMaxGroups / 32) + lane]) : 0;
            stages = k_stages + __builtin_amdgcn_readlane(wave_scan(own), 63) * ad_stages;
            ad_now = -1;
            ad_stage = 0;
            if (threadIdx.x < kMaxGroups / 32) present[(ad_set ^ 1) * (kMaxGroups / 32) + threadIdx.x] = 0;      // for the next tile
        }
        if (threadIdx.x < BN) {
            col[threadIdx.x] = c_bias;
            if (KIND != kMx) {
                col[BN + threadIdx.x] = c_scale;
                col[2 * BN + threadIdx.x] = __int_as_float(c_zero);
            }
        }
        if (KIND != kMx && threadIdx.x < BM) {
            row[threadIdx.x] = r_scale;
            row[BM + threadIdx.x] = __int_as_float(r_sum);
        }
        if (BUF <= stages) fetch(BUF - 1, BUF - 1);
        read_x(lds, xv[0], 0);
        read_w(lds, wv[0], 0);
        read_scales(0, 0);
        buf = 0;
        if constexpr (KIND == kInt4) {
            // four sets a stage: the low nibbles of both words of weights, then the high ones
            auto stage = [&](int t, auto first_, auto of_k) {
                constexpr bool FIRST = decltype(first_)::value, OF_K = decltype(of_k)::value;
                auto products = [&](int word, bool high, const lb_u32x4 (&x)[FM], bool fresh) {
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        if constexpr (OF_K) {
                            const lb_u32x4 w = high ? high_nibbles(wv[word][j]) : low_nibbles(wv[word][j]);
#pragma unroll
                            for (int i = 0; i < FM; ++i) acc[i][j] = mma32_i8(w, x[i], fresh ? acc_t{} : acc[i][j]);
                        } else {
#pragma unroll
                            for (int i = 0; i < FM; ++i) acc[i][j] = mma32_ranks(wv[word][j], x[i], acc[i][j]);
                        }
                    }
                };
                const lb_u32x4* here = lds + buf * STAGE;
                read_x(here, xv[1], 1);
                read_w(here, wv[1], 1);
                products(0, false, xv[0], FIRST);
                interleave(std::integral_constant<int, FM + FN>{});
                __builtin_amdgcn_sched_barrier(0);
                read_x(here, xv[0], 2);
                products(1, false, xv[1], false);
                interleave(std::integral_constant<int, FM>{});
                __builtin_amdgcn_sched_barrier(0);
                read_x(here, xv[1], 3);
                products(0, true, xv[0], false);
                interleave(std::integral_constant<int, FM>{});
                const lb_u32x4* s = advance(t);
                read_x(s, xv[0], 0);
                read_w(s, wv[0], 0);
                products(1, true, xv[1], false);
                interleave(std::integral_constant<int, FM + FN>{});
            };
            stage(0, std::true_type{}, std::true_type{});
#pragma unroll 1
            for (int t = 1; t < k_stages; ++t) stage(t, std::false_type{}, std::true_type{});
            if constexpr (adapted(MODE)) {
                whole_values();
#pragma unroll 1
                for (int t = k_stages; t < stages; ++t) stage(t, std::false_type{}, std::false_type{});
            }
        } else {
            // (stage t with t % 4 = B: the byte of its scales)
            auto stage = [&](int t, auto byte, auto first_, auto of_k) {
                constexpr int B = decltype(byte)::value;
                constexpr bool FIRST = decltype(first_)::value, OF_K = decltype(of_k)::value;
                auto products = [&](auto set, bool fresh) {
                    constexpr int C = decltype(set)::value;
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int i = 0; i < FM; ++i) {
                            const acc_t a = fresh ? acc_t{} : acc[i][j];
                            if constexpr (KIND == kMx) acc[i][j] = mma32_mx<B>(wv[C][j], xv[C][i], a, ws[j][C], xs[i][C]);
                            else if constexpr (!OF_K) acc[i][j] = mma32_ranks(wv[C][j], xv[C][i], acc[i][j]);
                            else acc[i][j] = mma32_i8(wv[C][j], xv[C][i], a);
                        }
                };
                const lb_u32x4* here = lds + buf * STAGE;
                read_x(here, xv[1], 1);
                read_w(here, wv[1], 1);
                if (B == 0) read_scales(t, 1);
                products(std::integral_constant<int, 0>{}, FIRST);
                interleave(std::integral_constant<int, FM + FN>{});
                const lb_u32x4* s = advance(t);
                read_x(s, xv[0], 0);
                read_w(s, wv[0], 0);
                if (B == 3) read_scales(t + 1, 0);
                products(std::integral_constant<int, 1>{}, false);
                interleave(std::integral_constant<int, FM + FN>{});
            };
            stage(0, std::integral_constant<int, 0>{}, std::true_type{}, std::true_type{});
            if constexpr (KIND == kMx) {
#pragma unroll 1
                for (int t = 1; t < stages; t += 4) {
                    stage(t, std::integral_constant<int, 1>{}, std::false_type{}, std::true_type{});
                    if (t + 1 < stages) stage(t + 1, std::integral_constant<int, 2>{}, std::false_type{}, std::true_type{});
                    if (t + 2 < stages) stage(t + 2, std::integral_constant<int, 3>{}, std::false_type{}, std::true_type{});
                    if (t + 3 < stages) stage(t + 3, std::integral_constant<int, 0>{}, std::false_type{}, std::true_type{});
                }
            } else {
                // Where the loop's branches land among the 32 bytes that are fetched at a time counts for 4 % of the INT8 128 x
                // 128 tiles.  Here the loop begins on such a line (a nop, and 28 bytes that the compiler puts behind it):
                // 256 x 4096 x 4096 23.8 us, 1024 x 4096 x 12288 65.4; 8, 16 and 24 bytes behind one 24.0, 24.1 and 24.8, and
                // 65.3, 65.6 and 66.7.
                if constexpr (KIND == kInt8 && FM == 2 && MODE == kPlain) asm volatile(".p2align 5\n\ts_nop 0");
#pragma unroll 1
                for (int t = 1; t < k_stages; ++t) stage(t, std::integral_constant<int, 1>{}, std::false_type{}, std::true_type{});
                if constexpr (adapted(MODE)) {
                    whole_values();
#pragma unroll 1
                    for (int t = k_stages; t < stages; ++t) stage(t, std::integral_constant<int, 1>{}, std::false_type{}, std::false_type{});
                }
            }
        }

        // ---- outputs, after the next tile's first copies
        const int m0 = row0 + wm * FM * 32, n0 = bn * BN + wn * FN * 32, m_end = row_end;
        const bool whole = p.wide && p.out_dtype != IC_DTYPE_F32 && row0 + BM <= m_end && (bn + 1) * BN <= p.N;
        tile += gridDim.x >> 3;
        const bool more = tile < last;                     // (all waves are done with the buffers)
        if (p.wide) {
            if (more) start();
            // 32 rows of 128 bytes at a time through the wave's part of the last buffer, so that 8 lanes store a line;
            // chunk c of row r lies in slot c ^ (r >> 1 & 7)
            lb_u32x4* area = lds + (BUF - 1) * STAGE + wave * 256;
            const int chunk = (lane & 7) ^ (lane >> 4), m1 = m0 + (lane >> 3);     // (of rows k 8 + lane / 8, k even)
            auto flush = [&](int i, int n0, int width) {
                lds_wave_fence();
                lb_u32x4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = area[k * 64 + lane];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int m = m1 + i * 32 + k * 8, n = n0 + (chunk ^ (k & 1) * 4) * width;
                    if (m >= m_end || n >= p.N) continue;
                    if (p.out_dtype == IC_DTYPE_F32) *reinterpret_cast<lb_u32x4*>(static_cast<float*>(p.out) + m * p.ld_out + n) = v[k];
                    else *reinterpret_cast<lb_u32x4*>(static_cast<uint16_t*>(p.out) + m * p.ld_out + n) = v[k];
                }
                lds_wave_fence();
            };
            const int cw = wn * FN * 32, rw = wm * FM * 32;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const float sa = KIND == kMx ? 0.0f : row[rw + i * 32 + r], sum = KIND == kMx ? 0.0f : row[BM + rw + i * 32 + r];
#pragma unroll
                for (int j = 0; j < FN; ++j) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        lb_f32x4 v[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int c = cw + j * 32 + q * 16 + h * 8 + k * 4;
                            const lb_f32x4 bias = *reinterpret_cast<const lb_f32x4*>(col + c);
                            lb_f32x4 sw = {}, zero = {};
                            if (KIND != kMx && !adapted(MODE)) {
                                sw = *reinterpret_cast<const lb_f32x4*>(col + BN + c);
                                zero = *reinterpret_cast<const lb_f32x4*>(col + 2 * BN + c);
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (adapted(MODE)) v[k][e] = __int_as_float(acc[i][j][8 * q + 4 * k + e]);
                                else v[k][e] = value(acc[i][j][8 * q + 4 * k + e], sw[e], zero[e], bias[e], sa, sum);
                            }
                        }
                        if (p.out_dtype == IC_DTYPE_F32) {
                            area[r * 8 + ((q * 4 + h * 2) ^ (r >> 1 & 7))] = __builtin_bit_cast(lb_u32x4, v[0]);
                            area[r * 8 + ((q * 4 + h * 2 + 1) ^ (r >> 1 & 7))] = __builtin_bit_cast(lb_u32x4, v[1]);
                        } else {
                            lb_u32x4 w;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                w[e] = p.out_dtype == IC_DTYPE_BF16 ? pack_half_words<IC_DTYPE_BF16>(v[e >> 1][2 * (e & 1)], v[e >> 1][2 * (e & 1) + 1])
                                                                    : pack_half_words<IC_DTYPE_F16>(v[e >> 1][2 * (e & 1)], v[e >> 1][2 * (e & 1) + 1]);
                            area[r * 8 + ((j * 4 + q * 2 + h) ^ (r >> 1 & 7))] = w;
                        }
                    }
                    if (p.out_dtype == IC_DTYPE_F32) flush(i, n0 + j * 32, 4);
                }
                if (p.out_dtype != IC_DTYPE_F32) flush(i, n0, 8);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!more) break;
            if (whole) meet<STORES>();                     // the copies were issued before the stores
            else meet<0>();
        } else {
            // rows of y at any alignment: 32 rows at a time through LDS, then value by value
            constexpr int PITCH = FN * 32 + 4;
            static_assert(WAVES * 32 * PITCH * 4 <= SCALES * 16, "the waves' areas lie in the buffers");
            typedef std::conditional_t<KIND == kMx, float, int> sum_t;
            typedef sum_t sum4_t __attribute__((ext_vector_type(4)));
            sum_t* area = reinterpret_cast<sum_t*>(lds) + wave * 32 * PITCH;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
#pragma unroll
                for (int j = 0; j < FN; ++j) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<sum4_t*>(area + r * PITCH + j * 32 + (k >> 1) * 16 + h * 8 + (k & 1) * 4) =
                            sum4_t{acc[i][j][4 * k], acc[i][j][4 * k + 1], acc[i][j][4 * k + 2], acc[i][j][4 * k + 3]};
                }
                lds_wave_fence();
                const int rows = m_end - (m0 + i * 32) < 32 ? m_end - (m0 + i * 32) : 32;
#pragma unroll 4
                for (int e = lane; e < rows * FN * 32; e += 64) {
                    const int m = e / (FN * 32), n = e % (FN * 32);
                    if (n0 + n >= p.N) continue;
                    const sum_t s = area[m * PITCH + n];
                    const int c = wn * FN * 32 + n, o = wm * FM * 32 + i * 32 + m;
                    const float v = adapted(MODE) ? __builtin_bit_cast(float, s)
                                    : KIND == kMx    ? value(s, 0.0f, 0.0f, col[c], 0.0f, 0.0f)
                                                     : value(s, col[BN + c], col[2 * BN + c], col[c], row[o], row[BM + o]);
                    store_from_f32(p.out, p.out_dtype, (m0 + i * 32 + m) * p.ld_out + n0 + n, v);
                }
                lds_wave_fence();
            }
            if (!more) break;
            meet<0>();
            start();
            meet<0>();
        }
    }
}

// Weights as the converter stores them -> tiles.
template <int BITS>
__global__ __launch_bounds__(256) void pack_weight_kernel(const uint8_t* __restrict__ src, int64_t N, int64_t K,
                                                          int64_t ld, lb_u32x4* __restrict__ dst, int64_t tiles) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), n = (int64_t)blockIdx.y * 16 + (lane & 15);
    if (t >= tiles) return;
    const int64_t k0 = t * (BITS == 4 ? 128 : 64) + (lane >> 4) * 16;
    lb_u32x4 w = {0, 0, 0, 0};
    if (n < N) {
        const uint8_t* row = src + n * ld;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            unsigned v;
            if (BITS == 8) {
                v = k0 + i < K ? row[k0 + i] : 0u;
            } else {
                const int64_t lo = k0 + i, hi = k0 + 64 + i;
                v = lo < K ? (row[lo >> 1] >> (4 * (lo & 1))) & 15u : 0u;
                v |= hi < K ? ((row[hi >> 1] >> (4 * (hi & 1))) & 15u) << 4 : 0u;
            }
            w[i >> 2] |= v << (8 * (i & 3));
        }
    }
    dst[((int64_t)blockIdx.y * tiles + t) * 64 + lane] = w;
}

template <int KIND, int MT>
void launch_direct(const Operands& p, hipStream_t st) {
    const dim3 grid((unsigned)cdiv(p.N, 16), (unsigned)cdiv(p.M, 16 * MT));
    hipLaunchKernelGGL((linear_direct_kernel<KIND, MT>), grid, dim3(512), 0, st, p);
}

template <int KIND, int MT, int NT, int MODE>
void launch_wide(const Operands& p, hipStream_t st) {
    const int64_t rows = MODE == kGrouped ? most_tiles(p.M, p.groups, 16 * MT) : cdiv(p.M, 16 * MT);
    hipLaunchKernelGGL((linear_wide_kernel<KIND, MT, NT, MODE>), dim3((unsigned)cdiv(p.N, 16 * NT), (unsigned)rows), dim3(512), 0, st, p);
}

// As many work-groups as run at once (one a CU with tiles of 256 x 256, whose
// buffers take most of its LDS, two with 128 x 128, 128 x 256 and 64 x 256, three
// or four with 32 x 128), each of which walks its XCD's tiles.
template <int KIND, int WM, int WN, int FM, int FN, int BUF, int MODE>
void launch_tiled(const Operands& p, hipStream_t st) {
    const int gm = (int)(MODE == kGrouped ? most_tiles(p.M, p.groups, 32 * WM * FM) : cdiv(p.M, 32 * WM * FM)), gn = (int)cdiv(p.N, 32 * WN * FN);
    const int64_t tiles = (int64_t)gm * gn;
    constexpr int64_t at_once = WM * WN == 8 ? 256 : WM * WN == 4 ? 512 : 1024;
    const unsigned grid = (unsigned)(tiles < at_once ? cdiv(tiles, 8) * 8 : at_once);
    hipLaunchKernelGGL((linear_tiled_kernel<KIND, WM, WN, FM, FN, BUF, MODE>), dim3(grid), dim3(64 * WM * WN), 0, st, p, gm, gn);
}

// Which form.  The direct one while it has few work-groups (of 64 rows x 16
// columns each): a tile of 128 x 128 takes its K steps one after another and
// leaves CUs idle when there are few.  Its line is where the two meet at K =
// 4096 (a longer K has it lower, a shorter one higher).  Measured (calls one
// after another, operands in cache; us), direct against 128 x 128, K = 1024 /
// 4096 / 12288, 128 x 128 being 10/23/57, 10/22/53 and 7.8/15/33 in each line:
//   groups (y)             INT8         INT4         MXFP4
//    693 ( 701 x 1000)    7.7/20/55    8.0/15/34    6.8/9.3/24
//   1008 ( 192 x 5376)    9.5/25/68    8.5/18/43    6.9/12/26
//   1152 ( 256 x 4608)     11/28/81    8.7/20/54    6.7/14/41
//   1280 ( 320 x 4096)     12/30/83    8.8/20/59    6.9/15/44
//   1344 ( 192 x 7168)     11/32/98    9.9/23/60    7.3/17/44
// Then tiles of 256 x 256, one a CU, where they fill more than half of a first
// round over the 256 CUs (up to there 128 x 128 tiles need one round too), or of
// two and more rounds three quarters, with INT4 two thirds (between these two the
// forms are within 4 %); else of 128 x 128.
// 128 x 128 against 256 x 256, y of 4096 columns, K = 1024 / 4096 / 12288:
//   rows (256-tiles)            INT8                        INT4                         MXFP4
//   2048 (1/2 round)     17/44/115 - 23/55/139      16/41/101 - 24/52/127      12/25/59  - 16/34/82
//   2304 (0.56)          24/62/160 - 25/59/143      22/53/136 - 24/53/128      16/34/86  - 16/34/84
//   4096 (1 round)       31/82/225 - 28/69/178      29/76/196 - 27/65/166      25/46/111 - 22/41/99
//   5120 (0.63 of two)  36/101/279 - 44/117/305    36/91/236 - 44/109/286      32/57/143 - 28/66/171
//   5632 (0.69 of two)  42/115/328 - 45/118/309    40/106/283 - 44/110/286     34/63/155 - 28/67/171
//   6144 (0.75 of two)  43/120/336 - 46/121/319    41/111/291 - 45/113/291     35/65/163 - 29/68/174
//   8192 (2 rounds)     55/157/446 - 53/133/348    52/145/385 - 51/127/327     37/85/216 - 48/77/191
int linear_form(int kind, int64_t M, int64_t N) {      // 0, 128 or 256
    const int64_t groups = cdiv(N, 16) * cdiv(M, 64), tiles = cdiv(M, 256) * cdiv(N, 256), rounds = cdiv(tiles, 256);
    if (M <= 64 || groups < (kind == kInt8 ? 1000 : kind == kInt4 ? 1300 : 1150)) return 0;
    if (rounds == 1) return tiles > 128 ? 256 : 128;
    return tiles * 12 >= rounds * 256 * (kind == kInt4 ? 8 : 9) ? 256 : 128;
}

template <int KIND> constexpr int kBuffers = KIND == kInt4 ? 3 : 4;

// The same for adapted products.  The end of a tile takes longer, which two
// work-groups a CU hide: 256 x 256 from K = 4096 on, and where they fill three
// quarters of their rounds.  128 against 256, INT4 / INT8, rank 16 where not said,
// us: 8192 x 4096 x 1024 68 to 77 / 75 to 87; 2304 x 4096 x 2048 43 to 51 / 47 to
// 58; 4096 x 4096 x 4096 90 to 89 / 100 to 99; 8192 x 4096 x 4096 rank 64 173 to
// 165 / 189 to 184; 8192 x 4100 x 4096 (0.71) 192 to 242.  The rule sees neither
// the number of adapters nor the rank, nor which rows share one: 512 x 4096 x 4096
// INT4 takes 22 us plain, 39 with 48 adapters of rank 16 in order and 58 mixed,
// 126 with 512 adapters, 245 with 512 of rank 64.
int adapted_form(int kind, int64_t M, int64_t N, int64_t K) {
    // (a tile's adapters are known when all but one of the buffers have been asked for)
    if (cdiv(K, kind == kInt8 ? 64 : 128) < (kind == kInt8 ? kBuffers<kInt8> : kBuffers<kInt4>) - 1) return 0;
    const int form = linear_form(kind, M, N);
    const int64_t tiles = cdiv(M, 256) * cdiv(N, 256);
    return form == 256 && (K < 4096 || (tiles > 256 && tiles * 12 < cdiv(tiles, 256) * 256 * 9)) ? 128 : form;
}

template <int KIND, int MODE = kPlain>
int launch_linear(const Operands& p, hipStream_t st) {
    constexpr int BUF = kBuffers<KIND>;
    const int form = adapted(MODE) ? adapted_form(KIND, p.M, p.N, p.K) : linear_form(KIND, p.M, p.N);
    if (form == 256) launch_tiled<KIND, 2, 4, 4, 2, BUF, MODE>(p, st);
    else if (form == 128) launch_tiled<KIND, 2, 2, 2, 2, BUF, MODE>(p, st);
    else if constexpr (MODE == kPlain) {
        if (p.M <= 16) launch_direct<KIND, 1>(p, st);
        else if (p.M <= 32) launch_direct<KIND, 2>(p, st);
        else launch_direct<KIND, 4>(p, st);
    } else {
        // More than 32 rows: one work-group of 4 x 3 or 4 x 4 runs a CU, so the fewer rounds count, and 2 x 2 where they
        // would leave a quarter of the CUs idle.  2 x 2 / 4 x 3 / 4 x 4, K = 4096, rank 16, INT4, us: 64 x 8192 17.8 / 19.6 /
        // 22.1; 64 x 10240 23.9 / 20.0 / 22.5; 64 x 12288 25.3 / 20.9 / 24.6; 64 x 14336 24.8 / 33.0 / 22.9; 64 x 24576 38.3
        // / 35.1 / 38.3; 128 x 4096 16.8 / 20.8 / 21.0; 192 x 4096 23.3 / 32.6 / 21.6; INT8 64 x 12288 28.5 / 24.8 / 29.9.
        const int64_t high = cdiv(p.M, 64), threes = high * cdiv(p.N, 48), fours = high * cdiv(p.N, 64);
        if (p.M <= 16 && cdiv(p.N, 32) < 256) launch_wide<KIND, 1, 1, MODE>(p, st);
        else if (p.M <= 16) launch_wide<KIND, 1, 2, MODE>(p, st);
        else if (p.M > 32 && threes >= 200 && cdiv(threes, 256) <= cdiv(fours, 256)) launch_wide<KIND, 4, 3, MODE>(p, st);
        else if (p.M > 32 && threes >= 200) launch_wide<KIND, 4, 4, MODE>(p, st);
        else launch_wide<KIND, 2, 2, MODE>(p, st);
    }
    IC_CHECK_LAUNCH();
    return IC_OK;
}

// Which form a grouped product takes.  The groups' sizes are on the GPU, so it
// goes by their average, and by whether a row of 64 x 256 tiles of every group
// that can have rows fills the CUs (`many`).  Measured, weights from HBM, rows
// at random over 8 (few) and 64 groups (many), us:
//                  2816 x 4096                               4096 x 1408
//   rows a group   wide 16  wide 32  32x128  64x256  128x256  wide 16  wide 32  32x128  64x256  128x256
//   INT4,  8,   1    10.9     11.8    17.6    25.3              8.7     11.2    11.1    14.8
//               8    14.2     17.8    17.9    25.0              9.4     12.8    11.3    15.0
//              16    14.6     18.3    17.9    25.4             11.6     13.0    11.4    15.1
//              32    18.7     19.2    18.3    25.4             16.2     17.4    13.5    15.1
//              64    28.5     30.0    22.3    25.7             25.1     25.8    14.3    16.1
//             128                     36.2    27.0    39.9                      23.9    19.8
//             512                             60.0    62.4                              45.2    48.0
//            1024                              111     101                              71.8    74.5
//            2048                              216     191                               136     129
//   INT4, 64,   1    47.7     61.6    56.2    50.0             31.5     56.8    30.7    33.8
//               2    63.8     87.4    64.9    80.8             43.7     77.0    40.9    43.2
//               4    73.8     96.9    71.3    78.8             51.4     90.7    51.7    45.7
//              16    98.7    102.4    75.8    79.5             68.1     94.1    54.7    50.7
//              64     197      207     136    97.4     115      162      198     103    67.9
//             256                              252     240                               163     158
//            1024                              887     801                               568     528
//                  wide 16  wide 32  128x128  128x256          wide 16  wide 32  128x128  128x256
//   INT8,  8,   8    21.1     25.5    29.0                      13.4     15.6    16.4
//              16    25.6     26.4    28.8                      15.3     15.9    17.1
//              32    29.9     28.8    29.2     42.9             20.4     20.5    16.7
//              64    41.0     37.6    30.8                      32.0     29.6    17.6
//             128                     36.5     49.3                               22.4     23.5
//             256                     56.4     49.6                               31.6     30.9
//            1024                      135      109                               83.0     78.0
//   INT8, 64,   1    85.7     86.9    96.0                      49.1     65.0    56.2
//               4     124      133     137                      90.9      113    85.9
//              16     147      148     145                       116      122    89.7
//              32                      152      140                               94.0     93.0
//             128                      237      216                                145      123
//            1024                     1175      897                                683      570
// 256 x 256 tiles, one work-group a CU, took 117 us (INT8 125) where the table
// has 101 (109), and 836 (847) where it has 801 (897): they lead by 13 % at best,
// INT8 with 8 groups of 512 rows, and lose by up to 30 %.
// Where 32 x 128 tiles would leave a third of the CUs idle, the wide form with
// 32 rows, and for INT8, whose next are 128 x 128, up to 250 of them: 10 groups of
// 70 rows, 1000 x 2901 (240), 16.7 against 21.7; 2 of 90, 4096 x 1024 (192), 10.8
// and 13.2; 4 of 90, 2000 x 2000 (192), 17.7 and 17.6; 6 of 70, 2000 x 4096 (288),
// 33.0 and 28.7; 2 of 128, 4096 x 1024 (256), 14.6 and 13.2.  INT4: one group of
// 64 rows, 4096 x 4096, 8.1 against 16.8, 4096 x 12288 12.3 against 35.5; 32 x 128
// tiles where there are up to 128 of 64 x 256: 13 groups of 78 rows, 823 x 3662
// (104), 22.9 against 29.6; 8 of 128, 2816 x 4096 (176), 36.2 and 27.0.  A K below 1024 has fewer steps than the wide
// form has waves: 16 groups of one row, 9668 x 120, 16.6 against 10.5 (64 x 256).
int expert_form(int kind, int64_t rows, int64_t groups, int64_t N, int64_t K) {      // 1, 2 (wide), 32, 64, 128 or 256 (128 x 256)
    const int64_t met = rows < groups ? rows : groups, each = met ? cdiv(rows, met) : 0;
    const bool many = met * cdiv(N, 256) >= 256;
    if (each <= (!many ? 16 : K >= 1024 ? 2 : 0)) return 1;
    if (met * cdiv(each, 32) * cdiv(N, 128) < (kind == kInt8 ? 250 : 170)) return 2;
    if (kind == kInt4 && met * cdiv(each, 64) * cdiv(N, 256) <= 128) return 32;
    const int64_t tiles = met * cdiv(each, 128) * cdiv(N, 256);
    if (kind == kInt4 ? each >= 256 && tiles >= 512 : tiles >= (each >= 128 ? 170 : 512)) return 256;
    return kind == kInt8 ? 128 : 64;
}

template <int KIND>
int launch_experts(const Operands& p, hipStream_t st) {
    const int form = expert_form(KIND, p.M, p.groups, p.N, p.K);
    constexpr int BUF = kBuffers<KIND>;
    if (form == 256) launch_tiled<KIND, 1, 4, 4, 2, BUF - 1, kGrouped>(p, st);
    else if (form >= 32) {
        if constexpr (KIND == kInt8) launch_tiled<KIND, 2, 2, 2, 2, BUF, kGrouped>(p, st);
        else if (form == 32) launch_tiled<KIND, 1, 2, 1, 2, BUF, kGrouped>(p, st);
        else launch_tiled<KIND, 1, 4, 2, 2, BUF, kGrouped>(p, st);
    } else if (form == 2) launch_wide<KIND, 2, 2, kGrouped>(p, st);
    // four column tiles for INT4 where work-groups abound: 64 groups of 4096 x 1408, 1 row each, 35.4 against 40.3 us
    // (INT8 50.7 against 53.0, but 2816 x 4096 95 against 83); few: 8 groups of 4 rows, 2816 x 4096, 16.2 against 14.6
    else if (KIND == kInt4 && (p.M < p.groups ? p.M : p.groups) * cdiv(p.N, 256) >= 256) launch_wide<KIND, 1, 4, kGrouped>(p, st);
    else launch_wide<KIND, 1, 2, kGrouped>(p, st);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

int check_product(const char* who, const Operands& p) {
    const std::string w(who);
    if (p.M < 0 || p.N < 1 || p.K < 1) return fail(IC_ERR_ARG, w + ": M must be >= 0, N and K >= 1");
    if (p.out_dtype < 0 || p.out_dtype > 2 || (p.bias && (p.bias_dtype < 0 || p.bias_dtype > 2)))
        return fail(IC_ERR_ARG, w + ": unknown dtype");
    if (p.K > 65536 || p.M > kMaxRows || p.N > kMaxRows)
        return fail(IC_ERR_RANGE, w + ": at most 65536 for K, 1048560 for M and N");
    return IC_OK;
}

}  // namespace
}  // namespace icq

using namespace icq;

extern "C" int ic_linear_form(int kind, int64_t M, int64_t N) {
    IC_REQUIRE(kind >= kInt8 && kind <= kMx && M >= 0 && N >= 1, "ic_linear_form: kind must be 0, 1 or 2, M >= 0, N >= 1");
    return linear_form(kind, M, N);
}

extern "C" int64_t ic_linear_weight_bytes(int64_t N, int64_t K, int bits) {
    if (N < 0 || K < 0 || (bits != 4 && bits != 8)) return 0;
    return cdiv(N, 16) * cdiv(K, 128) * (bits == 8 ? 2048 : 1024);
}

extern "C" int ic_linear_pack_weight(const void* stored, int bits, int64_t N, int64_t K, int64_t ld, void* tiles,
                                     void* stream) {
    IC_REQUIRE(bits == 4 || bits == 8, "ic_linear_pack_weight: bits must be 4 or 8");
    IC_REQUIRE(N >= 1 && K >= 1 && ld >= (bits == 4 ? cdiv(K, 2) : K), "ic_linear_pack_weight: bad sizes");
    IC_REQUIRE(stored && tiles && aligned16(tiles), "ic_linear_pack_weight: null pointer, or tiles not 16-byte aligned");
    if (K > 65536 || N > kMaxRows) return fail(IC_ERR_RANGE, "ic_linear_pack_weight: at most 65536 for K, 1048560 for N");
    const int64_t t = cdiv(K, 128) * (bits == 8 ? 2 : 1);
    const dim3 grid((unsigned)cdiv(t, 4), (unsigned)cdiv(N, 16));
    const uint8_t* s = static_cast<const uint8_t*>(stored);
    lb_u32x4* d = static_cast<lb_u32x4*>(tiles);
    if (bits == 8) hipLaunchKernelGGL(pack_weight_kernel<8>, grid, dim3(256), 0, as_stream(stream), s, N, K, ld, d, t);
    else hipLaunchKernelGGL(pack_weight_kernel<4>, grid, dim3(256), 0, as_stream(stream), s, N, K, ld, d, t);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

namespace icq {
namespace {

// The operands of the integer kinds, checked.  Rows of y and of the activations differ where groups gather.
int integer_product(const char* who, Operands& p, const int8_t* a, int64_t ld_a, const float* sa, const int32_t* sums, int64_t M,
                    const void* tiles, int bits, const void* sw, int sw_kind, const int8_t* zp, const void* bias, int bias_dtype,
                    int64_t N, int64_t K, void* out, int out_dtype, int64_t ld_out) {
    const std::string w(who);
    p.a = reinterpret_cast<const uint8_t*>(a); p.ld_a = ld_a; p.sa = sa; p.sums = sums;
    p.w = static_cast<const uint8_t*>(tiles); p.sw = sw; p.sw_f32 = sw_kind; p.zp = zp;
    p.bias = bias; p.bias_dtype = bias_dtype; p.M = M; p.N = N; p.K = K;
    p.out = out; p.out_dtype = out_dtype; p.ld_out = ld_out;
    if (const int rc = check_product(who, p)) return rc;
    IC_REQUIRE(bits == 4 || bits == 8, w + ": bits must be 4 or 8");
    IC_REQUIRE(sw_kind == 0 || sw_kind == 1, w + ": sw_kind must be 0 (fp16) or 1 (fp32)");
    if (M == 0) return IC_OK;
    IC_REQUIRE(a && sa && tiles && sw && out && (!zp || sums), w + ": null pointer");
    IC_REQUIRE(ld_a >= cdiv(K, kActPad) * kActPad && ld_a % 16 == 0 && aligned16(a) && aligned16(tiles),
               w + ": activations need rows of ic_activation_pitch codes, 16-byte aligned");
    IC_REQUIRE(ld_out >= N, w + ": ld_out below N");
    if (ld_a > (1 << 20)) return fail(IC_ERR_RANGE, w + ": at most 2^20 for ld_a");   // (a lane's 32-bit offset in 256 rows)
    p.wide = aligned16(out) && ld_out % (out_dtype == IC_DTYPE_F32 ? 4 : 8) == 0 && N % 8 == 0;
    return IC_OK;
}

}  // namespace
}  // namespace icq

extern "C" int ic_quantized_linear(const int8_t* a, int64_t ld_a, const float* sa, const int32_t* sums, int64_t M,
                                   const void* tiles, int bits, const void* sw, int sw_kind, const int8_t* zp,
                                   const void* bias, int bias_dtype, int64_t N, int64_t K, void* out, int out_dtype,
                                   int64_t ld_out, void* stream) {
    Operands p{};
    if (const int rc = integer_product("ic_quantized_linear", p, a, ld_a, sa, sums, M, tiles, bits, sw, sw_kind, zp, bias, bias_dtype, N,
                                       K, out, out_dtype, ld_out)) return rc;
    if (M == 0) return IC_OK;
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 2.0 * M * N * K, (double)M * K + (double)N * K * bits / 8);
    return bits == 8 ? launch_linear<kInt8>(p, st) : launch_linear<kInt4>(p, st);
}

extern "C" int ic_expert_form(int bits, int64_t rows, int64_t groups, int64_t N, int64_t K) {
    IC_REQUIRE((bits == 4 || bits == 8) && rows >= 0 && groups >= 1 && N >= 1 && K >= 1,
               "ic_expert_form: bits must be 4 or 8, rows >= 0, groups, N and K >= 1");
    return expert_form(bits == 8 ? kInt8 : kInt4, rows, groups, N, K);
}

extern "C" int ic_expert_linear(const int8_t* a, int64_t ld_a, const float* sa, const int32_t* sums, int64_t a_rows,
                                const int32_t* offsets, const int32_t* order, int top, int64_t groups, int64_t rows,
                                const void* tiles, int bits, const void* sw, int sw_kind, const int8_t* zp, const void* bias,
                                int bias_dtype, int64_t N, int64_t K, void* out, int out_dtype, int64_t ld_out, void* stream) {
    Operands p{};
    if (const int rc = integer_product("ic_expert_linear", p, a, ld_a, sa, sums, rows, tiles, bits, sw, sw_kind, zp, bias, bias_dtype, N,
                                       K, out, out_dtype, ld_out)) return rc;
    IC_REQUIRE(groups >= 1 && groups <= kMaxGroups, "ic_expert_linear: 1 to 1024 groups");
    if (rows == 0) return IC_OK;
    IC_REQUIRE(top >= 0 && offsets && (top == 0 || order), "ic_expert_linear: gathered rows need their order");
    IC_REQUIRE(top > 0 ? a_rows >= 1 && a_rows <= kMaxRows : a_rows == rows,
               "ic_expert_linear: rows of activations and of the result differ, and none are gathered");
    if (top > 0 && a_rows * ld_a > 0xffffffffll) return fail(IC_ERR_RANGE, "ic_expert_linear: gathered activations have less than 2^32 bytes");
    p.offsets = offsets; p.order = order; p.top = top; p.groups = (int)groups; p.a_rows = (int)a_rows;
    p.w_group = ic_linear_weight_bytes(N, K, bits);
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 2.0 * rows * N * K, (double)a_rows * K + (double)groups * N * K * bits / 8);
    return bits == 8 ? launch_experts<kInt8>(p, st) : launch_experts<kInt4>(p, st);
}

extern "C" int ic_adapted_linear(const int8_t* a, int64_t ld_a, const float* sa, const int32_t* sums, int64_t M,
                                 const void* tiles, int bits, const void* sw, int sw_kind, const int8_t* zp, const void* bias,
                                 int bias_dtype, int64_t N, int64_t K, const void* down, const void* up, int adapter_dtype,
                                 int64_t adapters, int rank, const float* scaling, const int32_t* ids, const int32_t* offsets,
                                 const int32_t* order, void* workspace, void* out, int out_dtype, int64_t ld_out, void* stream) {
    Operands p{};
    if (const int rc = integer_product("ic_adapted_linear", p, a, ld_a, sa, sums, M, tiles, bits, sw, sw_kind, zp, bias, bias_dtype, N, K,
                                       out, out_dtype, ld_out)) return rc;
    IC_REQUIRE(adapter_dtype == IC_DTYPE_BF16 || adapter_dtype == IC_DTYPE_F16, "ic_adapted_linear: adapters are bf16 or fp16");
    IC_REQUIRE(adapters >= 1 && adapters <= kMaxGroups && rank >= 1 && rank <= kMaxRank, "ic_adapted_linear: 1 to 1024 adapters of rank 1 to 128");
    if (M == 0) return IC_OK;
    IC_REQUIRE(down && up && scaling && ids && offsets && order && workspace, "ic_adapted_linear: null pointer");
    IC_REQUIRE(aligned16(down) && aligned16(up) && aligned16(workspace), "ic_adapted_linear: adapters and workspace need 16-byte alignment");
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 2.0 * M * N * K + 2.0 * M * rank * (N + K), (double)M * K + (double)N * K * bits / 8);
    p.ad = Adapted{ids, static_cast<uint16_t*>(workspace), static_cast<const uint8_t*>(up), adapter_dtype == IC_DTYPE_F16, rank_parts(rank), (int)adapters,
                   (rank + 7) / 8};
    const bool whole = out_dtype == IC_DTYPE_F32;
    const RankForm kept = !whole ? kTwo : adapted_form(bits == 8 ? kInt8 : kInt4, M, N, K) ? kThree : kWhole;
    if (const int rc = launch_shrink(p.ad, kept, a, ld_a, sa, M, K, down, rank, scaling, offsets, order, st)) return rc;
    if (bits == 8) return whole ? launch_linear<kInt8, kAdaptedWhole>(p, st) : launch_linear<kInt8, kAdapted>(p, st);
    return whole ? launch_linear<kInt4, kAdaptedWhole>(p, st) : launch_linear<kInt4, kAdapted>(p, st);
}

extern "C" int ic_mxfp4_linear(const void* a, const void* a_scales, int64_t M, const void* w, const void* w_scales,
                               const void* bias, int bias_dtype, int64_t N, int64_t K, void* out, int out_dtype,
                               int64_t ld_out, void* stream) {
    Operands p{};
    p.a = static_cast<const uint8_t*>(a); p.a_scale = static_cast<const uint32_t*>(a_scales);
    p.w = static_cast<const uint8_t*>(w); p.w_scale = static_cast<const uint32_t*>(w_scales);
    p.bias = bias; p.bias_dtype = bias_dtype; p.M = M; p.N = N; p.K = K;
    p.out = out; p.out_dtype = out_dtype; p.ld_out = ld_out;
    if (const int rc = check_product("ic_mxfp4_linear", p)) return rc;
    if (M == 0) return IC_OK;
    IC_REQUIRE(a && a_scales && w && w_scales && out, "ic_mxfp4_linear: null pointer");
    IC_REQUIRE(aligned16(a) && aligned16(w) && aligned16(a_scales) && aligned16(w_scales) && ld_out >= N,
               "ic_mxfp4_linear: operands need 16-byte alignment and ld_out at least N");
    p.wide = aligned16(out) && ld_out % (out_dtype == IC_DTYPE_F32 ? 4 : 8) == 0 && N % 8 == 0;
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 2.0 * M * N * K, ((double)M * K + (double)N * K) * 17 / 32);
    return launch_linear<kMx>(p, st);
}
