// Products with quantised weights, y = x W^T + b:
//   INT8 / INT4 weights [N, K] with a scale (and zero-point) a row, 8-bit
//   activations [M, K] with a scale a row:
//     y[m, n] = sa[m] sw[n] (sum_k a q - zp[n] sum_k a) + b[n],
//   the sums exact in 32-bit integers; and both operands in microscaled
//   4-bit floating point, accumulated in fp32.
// The weights are the matrix instructions' first operand, so a lane ends
// with four consecutive outputs of one row of y.
#include "common.hpp"
#include "prof.hpp"
#include "lowbit.hpp"

namespace icq {
namespace {

enum Kind { kInt8 = 0, kInt4 = 1, kMx = 2 };

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
};

template <int KIND> struct Acc { typedef i32x4 T; };
template <> struct Acc<kMx> { typedef lb_f32x4 T; };

// What the outputs of four consecutive columns from n0 need (columns past the
// last repeat the last).
template <int KIND>
struct Columns {
    float sw[4], bias[4];
    int zp[4];
    __device__ __forceinline__ void load(const Operands& p, int64_t n0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = n0 + i < p.N ? n0 + i : p.N - 1;
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
__device__ __forceinline__ void store4(const Operands& p, lb_f32x4 v, int64_t m, int64_t n) {
    if (m >= p.M || n >= p.N) return;
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
               nt * 16 + g * 4);
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
// The 256 x 256 forms of INT4 and INT8 spill 22 and 8 registers, at a tile's
// start and end, none in the K loop.  Spills are vector-memory operations like
// those that meet() counts.  It lets the newest N stay outstanding; with spills
// among these it waits for more copies than it needs, never for fewer.
template <int KIND, int WM, int WN, int FM, int FN, int BUF>
__global__ __launch_bounds__(64 * WM * WN) void linear_tiled_kernel(Operands p, int grid_m, int grid_n) {
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
    constexpr int SCALES = BUF * STAGE, COLS = SCALES + 2 * S_WORDS, ROWS = COLS + BN * 3 / 4;
    __shared__ lb_u32x4 lds[ROWS + (KIND == kMx ? 0 : BM / 2)];
    float* const col = reinterpret_cast<float*>(lds + COLS);
    float* const row = reinterpret_cast<float*>(lds + ROWS);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, r = lane & 31;
    const int wm = wave / WN, wn = wave % WN;
    const int lane16 = lane * 16;

    // work-groups are dealt to the 8 XCDs in turn: each XCD gets one run of tiles, walked in bands of 8 tile rows so
    // that what its L2 holds is used again
    const int total = grid_m * grid_n, xcd = blockIdx.x & 7, per = total >> 3, extra = total & 7;
    const int first = xcd * per + (xcd < extra ? xcd : extra), last = first + per + (xcd < extra ? 1 : 0);
    int tile = first + (blockIdx.x >> 3);
    if (tile >= last) return;

    const int k_tiles = (int)cdiv(p.K, 128), words = (int)cdiv(p.K, 512);
    const int n_tiles = (int)cdiv(p.N, 16), m_tiles = (int)cdiv(p.M, 16);
    const int stages = KIND == kInt8 ? (int)cdiv(p.K, 64) : k_tiles;
    constexpr int W_STEP = 1024, X_STEP = KIND == kMx ? 1024 : KIND == kInt4 ? 128 : 64;
    const int w_pitch = k_tiles * (KIND == kInt8 ? 2048 : 1024);                  // bytes of a row of tiles

    // ---- copies.  Rows and tiles past the last repeat the last; their outputs are dropped.
    int bm = 0, bn = 0;
    __amdgpu_buffer_rsrc_t x_buf, w_buf, xs_buf, ws_buf;
    int x_row[KIND == kMx ? X_LOADS : 1], w_row[W_LOADS], x_off[KIND == kMx ? 1 : X_LOADS], s_off[S_LOADS + 1];
    auto buffer = [](const void* base) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
    };
    auto aim = [&]() {
        const int band = tile / (8 * grid_n), rows_in = grid_m - band * 8 < 8 ? grid_m - band * 8 : 8;
        const int in_band = tile - band * 8 * grid_n;
        bm = band * 8 + in_band % rows_in;
        bn = in_band / rows_in;
        const int nt = bn * (BN / 16), nl = n_tiles - 1 - nt;
        w_buf = buffer(p.w + (int64_t)nt * w_pitch);
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
            const int row0 = KIND == kInt4 ? lane >> 3 : lane >> 2;
            const int chunk = KIND == kInt4 ? (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4)) : (lane & 3) ^ (lane >> 4);
            static_assert(WAVES % 2 == 0, "a wave's copies begin at rows of one parity of 8");
            const int ml = (int)p.M - 1 - bm * BM;
            x_buf = buffer(p.a + (int64_t)bm * BM * p.ld_a);
#pragma unroll
            for (int i = 0; i < X_LOADS; ++i) {
                const int row = (i * WAVES + wave) * (KIND == kInt4 ? 8 : 16) + row0;
                x_off[i] = (row < ml ? row : ml) * (int)p.ld_a + chunk * 16;
            }
        }
    };
    auto copy = [&](__amdgpu_buffer_rsrc_t from, int lane_off, int off, lb_u32x4* to) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, lane_off, off, 0, 0);
    };
    auto fetch = [&](int t, int buf) {
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
        const int64_t n = bn * BN + tid < p.N ? bn * BN + tid : p.N - 1, m = bm * BM + tid < p.M ? bm * BM + tid : p.M - 1;
        if (KIND != kMx) {
            c_scale = p.sw_f32 ? static_cast<const float*>(p.sw)[n] : f16_bits_to_f32(static_cast<const uint16_t*>(p.sw)[n]);
            r_scale = p.sa[m];
            if (p.zp) {
                c_zero = p.zp[n];
                r_sum = p.sums[m];
            }
        }
        if (p.bias) c_bias = load_as_f32(p.bias, p.bias_dtype, n);
#pragma unroll
        for (int b = 0; b < BUF - 1; ++b)
            if (b < stages) fetch(b, b);
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

    start();
    meet<0>();
    for (;;) {
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
            auto stage = [&](int t, auto first_) {
                constexpr bool FIRST = decltype(first_)::value;
                auto products = [&](int word, bool high, const lb_u32x4 (&x)[FM], bool fresh) {
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        const lb_u32x4 w = high ? high_nibbles(wv[word][j]) : low_nibbles(wv[word][j]);
#pragma unroll
                        for (int i = 0; i < FM; ++i) acc[i][j] = mma32_i8(w, x[i], fresh ? acc_t{} : acc[i][j]);
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
            stage(0, std::true_type{});
#pragma unroll 1
            for (int t = 1; t < stages; ++t) stage(t, std::false_type{});
        } else {
            // (stage t with t % 4 = B: the byte of its scales)
            auto stage = [&](int t, auto byte, auto first_) {
                constexpr int B = decltype(byte)::value;
                constexpr bool FIRST = decltype(first_)::value;
                auto products = [&](auto set, bool fresh) {
                    constexpr int C = decltype(set)::value;
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int i = 0; i < FM; ++i) {
                            const acc_t a = fresh ? acc_t{} : acc[i][j];
                            if constexpr (KIND == kMx) acc[i][j] = mma32_mx<B>(wv[C][j], xv[C][i], a, ws[j][C], xs[i][C]);
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
            stage(0, std::integral_constant<int, 0>{}, std::true_type{});
            if constexpr (KIND == kMx) {
#pragma unroll 1
                for (int t = 1; t < stages; t += 4) {
                    stage(t, std::integral_constant<int, 1>{}, std::false_type{});
                    if (t + 1 < stages) stage(t + 1, std::integral_constant<int, 2>{}, std::false_type{});
                    if (t + 2 < stages) stage(t + 2, std::integral_constant<int, 3>{}, std::false_type{});
                    if (t + 3 < stages) stage(t + 3, std::integral_constant<int, 0>{}, std::false_type{});
                }
            } else {
#pragma unroll 1
                for (int t = 1; t < stages; ++t) stage(t, std::integral_constant<int, 1>{}, std::false_type{});
            }
        }

        // ---- outputs, after the next tile's first copies
        const int m0 = bm * BM + wm * FM * 32, n0 = bn * BN + wn * FN * 32;
        const bool whole = p.wide && p.out_dtype != IC_DTYPE_F32 && (bm + 1) * BM <= p.M && (bn + 1) * BN <= p.N;
        tile += gridDim.x >> 3;
        const bool more = tile < last;                     // (all waves are done with the buffers)
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
                    if (m >= p.M || n >= p.N) continue;
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
                            if (KIND != kMx) {
                                sw = *reinterpret_cast<const lb_f32x4*>(col + BN + c);
                                zero = *reinterpret_cast<const lb_f32x4*>(col + 2 * BN + c);
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[k][e] = value(acc[i][j][8 * q + 4 * k + e], sw[e], zero[e], bias[e], sa, sum);
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
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<sum4_t*>(area + r * PITCH + j * 32 + (k >> 1) * 16 + h * 8 + (k & 1) * 4) =
                            sum4_t{acc[i][j][4 * k], acc[i][j][4 * k + 1], acc[i][j][4 * k + 2], acc[i][j][4 * k + 3]};
                lds_wave_fence();
                const int rows = (int)p.M - (m0 + i * 32) < 32 ? (int)p.M - (m0 + i * 32) : 32;
#pragma unroll 4
                for (int e = lane; e < rows * FN * 32; e += 64) {
                    const int m = e / (FN * 32), n = e % (FN * 32);
                    if (n0 + n >= p.N) continue;
                    const sum_t s = area[m * PITCH + n];
                    const int c = wn * FN * 32 + n, o = wm * FM * 32 + i * 32 + m;
                    const float v = KIND == kMx ? value(s, 0.0f, 0.0f, col[c], 0.0f, 0.0f)
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

// As many work-groups as run at once (one a CU with tiles of 256 x 256, whose
// buffers take most of its LDS, two with 128 x 128), each of which walks its
// XCD's tiles.  (INT4's 128 x 128 takes 260 registers, four too many for two a
// CU: its second half starts as the first ends.)
template <int KIND, int WM, int WN, int FM, int FN, int BUF>
void launch_tiled(const Operands& p, hipStream_t st) {
    const int gm = (int)cdiv(p.M, 32 * WM * FM), gn = (int)cdiv(p.N, 32 * WN * FN);
    const int64_t tiles = (int64_t)gm * gn;
    constexpr int64_t at_once = WM * WN == 4 ? 512 : 256;
    const unsigned grid = (unsigned)(tiles < at_once ? cdiv(tiles, 8) * 8 : at_once);
    hipLaunchKernelGGL((linear_tiled_kernel<KIND, WM, WN, FM, FN, BUF>), dim3(grid), dim3(64 * WM * WN), 0, st, p, gm, gn);
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
// two and more rounds three quarters, with INT4 two thirds; else of 128 x 128.
// 128 x 128 against 256 x 256, y of 4096 columns, K = 1024 / 4096 / 12288:
//   rows (256-tiles)            INT8                        INT4                         MXFP4
//   2048 (1/2 round)     17/44/115 - 23/55/139      22/49/119 - 25/56/137      12/25/59  - 16/34/82
//   2304 (0.56)          24/62/160 - 25/59/143      30/69/168 - 26/57/135      16/34/86  - 16/34/84
//   4096 (1 round)       31/82/225 - 28/69/178      40/94/237 - 29/66/164      25/46/111 - 22/41/99
//   5120 (0.63 of two)  36/101/279 - 44/117/305    49/114/288 - 47/112/285     32/57/143 - 28/66/171
//   5632 (0.69 of two)  42/115/328 - 45/118/309    57/135/343 - 48/115/285     34/63/155 - 28/67/171
//   6144 (0.75 of two)  43/120/336 - 46/121/319    58/138/345 - 50/118/288     35/65/163 - 29/68/174
//   8192 (2 rounds)     55/157/446 - 53/133/348    77/188/479 - 54/126/320     37/85/216 - 48/77/191
int linear_form(int kind, int64_t M, int64_t N) {      // 0, 128 or 256
    const int64_t groups = cdiv(N, 16) * cdiv(M, 64), tiles = cdiv(M, 256) * cdiv(N, 256), rounds = cdiv(tiles, 256);
    if (M <= 64 || groups < (kind == kInt8 ? 1000 : kind == kInt4 ? 1300 : 1150)) return 0;
    if (rounds == 1) return tiles > 128 ? 256 : 128;
    return tiles * 12 >= rounds * 256 * (kind == kInt4 ? 8 : 9) ? 256 : 128;
}

template <int KIND>
int launch_linear(const Operands& p, hipStream_t st) {
    const int form = linear_form(KIND, p.M, p.N);
    if (form == 256) launch_tiled<KIND, 2, 4, 4, 2, KIND == kInt4 ? 3 : 4>(p, st);
    else if (form == 128) launch_tiled<KIND, 2, 2, 2, 2, KIND == kInt4 ? 3 : 4>(p, st);
    else if (p.M <= 16) launch_direct<KIND, 1>(p, st);
    else if (p.M <= 32) launch_direct<KIND, 2>(p, st);
    else launch_direct<KIND, 4>(p, st);
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

extern "C" int ic_quantized_linear(const int8_t* a, int64_t ld_a, const float* sa, const int32_t* sums, int64_t M,
                                   const void* tiles, int bits, const void* sw, int sw_kind, const int8_t* zp,
                                   const void* bias, int bias_dtype, int64_t N, int64_t K, void* out, int out_dtype,
                                   int64_t ld_out, void* stream) {
    Operands p{};
    p.a = reinterpret_cast<const uint8_t*>(a); p.ld_a = ld_a; p.sa = sa; p.sums = sums;
    p.w = static_cast<const uint8_t*>(tiles); p.sw = sw; p.sw_f32 = sw_kind; p.zp = zp;
    p.bias = bias; p.bias_dtype = bias_dtype; p.M = M; p.N = N; p.K = K;
    p.out = out; p.out_dtype = out_dtype; p.ld_out = ld_out;
    if (const int rc = check_product("ic_quantized_linear", p)) return rc;
    IC_REQUIRE(bits == 4 || bits == 8, "ic_quantized_linear: bits must be 4 or 8");
    IC_REQUIRE(sw_kind == 0 || sw_kind == 1, "ic_quantized_linear: sw_kind must be 0 (fp16) or 1 (fp32)");
    if (M == 0) return IC_OK;
    IC_REQUIRE(a && sa && tiles && sw && out && (!zp || sums), "ic_quantized_linear: null pointer");
    IC_REQUIRE(ld_a >= cdiv(K, kActPad) * kActPad && ld_a % 16 == 0 && aligned16(a) && aligned16(tiles),
               "ic_quantized_linear: activations need rows of ic_activation_pitch codes, 16-byte aligned");
    IC_REQUIRE(ld_out >= N, "ic_quantized_linear: ld_out below N");
    if (ld_a > (1 << 20)) return fail(IC_ERR_RANGE, "ic_quantized_linear: at most 2^20 for ld_a");   // (a lane's 32-bit offset in 256 rows)
    p.wide = aligned16(out) && ld_out % (out_dtype == IC_DTYPE_F32 ? 4 : 8) == 0 && N % 8 == 0;
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 2.0 * M * N * K, (double)M * K + (double)N * K * bits / 8);
    return bits == 8 ? launch_linear<kInt8>(p, st) : launch_linear<kInt4>(p, st);
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
