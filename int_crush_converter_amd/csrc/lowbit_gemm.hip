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
    int wide;                // four outputs may be stored at once
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

// A wave's 16 rows x 64 (16 COLS) columns of y from its area of LDS: a lane
// writes 4 COLS consecutive columns of one row, so that 4 lanes write whole
// lines.  Rows of `area` hold 16 COLS + 4 values: 16-byte reads and writes
// then spread over the banks.
template <int COLS>
__device__ __forceinline__ void store_rows(const Operands& p, const float* area, int lane, int64_t m0, int64_t n0) {
    const int64_t m = m0 + (lane >> 2);
    const float* row = area + (lane >> 2) * (16 * COLS + 4) + (lane & 3) * 4 * COLS;
    const int64_t c0 = n0 + (lane & 3) * 4 * COLS;
    if (m >= p.M || c0 >= p.N) return;
    float v[4 * COLS];
#pragma unroll
    for (int i = 0; i < COLS; ++i) *reinterpret_cast<lb_f32x4*>(v + 4 * i) = *reinterpret_cast<const lb_f32x4*>(row + 4 * i);
    const int64_t at = m * p.ld_out + c0;
    if (p.wide && c0 + 4 * COLS <= p.N) {
        if (p.out_dtype == IC_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < COLS; ++i)
                *reinterpret_cast<lb_f32x4*>(static_cast<float*>(p.out) + at + 4 * i) = lb_f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        } else {
            uint32_t w[2 * COLS];
            if (p.out_dtype == IC_DTYPE_BF16) {
#pragma unroll
                for (int i = 0; i < 2 * COLS; ++i) w[i] = pack_half_words<IC_DTYPE_BF16>(v[2 * i], v[2 * i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < 2 * COLS; ++i) w[i] = pack_half_words<IC_DTYPE_F16>(v[2 * i], v[2 * i + 1]);
            }
            uint16_t* q = static_cast<uint16_t*>(p.out) + at;
            if constexpr (COLS % 2 == 0) {
#pragma unroll
                for (int i = 0; i < COLS / 2; ++i)
                    *reinterpret_cast<lb_u32x4*>(q + 8 * i) = lb_u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
            } else {
#pragma unroll
                for (int i = 0; i < COLS; ++i) *reinterpret_cast<lb_u32x2*>(q + 4 * i) = lb_u32x2{w[2 * i], w[2 * i + 1]};
            }
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 4 * COLS && c0 + i < p.N; ++i) store_from_f32(p.out, p.out_dtype, at + i, row[i]);
    }
}

// acc += W tile (16 n x 128 k) * X tile (128 k x 16 m).
__device__ __forceinline__ i32x4 mma_i8(lb_u32x4 w, lb_u32x4 x, i32x4 acc) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), acc, 0, 0, 0);
}
// (byte B of each scale word)
template <int B>
__device__ __forceinline__ lb_f32x4 mma_mx(lb_u32x4 w, lb_u32x4 x, lb_f32x4 acc, int sw, int sx) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, B, sw, B, sx);
}
// 32 INT4 values of a lane as two operands of 16 bytes, each value times 16.
__device__ __forceinline__ lb_u32x4 low_nibbles(lb_u32x4 p) { return (p << 4) & 0xf0f0f0f0u; }
__device__ __forceinline__ lb_u32x4 high_nibbles(lb_u32x4 p) { return p & 0xf0f0f0f0u; }

// Few rows: a work-group of WAVES waves takes 16 columns of y and 16 MT rows,
// its waves a share of K each; the sums are joined in LDS in a fixed order.
template <int KIND, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear_direct_kernel(Operands p) {
    typedef typename Acc<KIND>::T acc_t;
    __shared__ acc_t part[WAVES][MT][64];
    __shared__ float rows[MT][16 * 20];
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
            const int64_t m = (mt0 + i) * 16 + r < p.M ? (mt0 + i) * 16 + r : p.M - 1;
            row[i] = p.a + m * p.ld_a + g * 16;
        }
    }
    const uint32_t* ws = KIND == kMx ? p.w_scale + nt * words * 64 + lane : nullptr;
    for (int64_t t = t0; t < t1; ++t) {
        if constexpr (KIND == kMx) {
            const lb_u32x4 w = wt[t * 64];
            const int sw = (int)(ws[(t >> 2) * 64] >> (8 * (t & 3)));
#pragma unroll
            for (int i = 0; i < MT; ++i)
                acc[i] = mma_mx<0>(w, xt[i][t * 64], acc[i], sw & 255, (int)(xs[i][(t >> 2) * 64] >> (8 * (t & 3))) & 255);
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
                acc[i] = mma_i8(w0, x[0], acc[i]);
                acc[i] = mma_i8(w1, x[4], acc[i]);
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
        const lb_f32x4 v = cols.finish(s, KIND == kMx ? 1.0f : p.sa[m], KIND != kMx && p.zp ? p.sums[m] : 0);
        float* area = rows[i];
        *reinterpret_cast<lb_f32x4*>(area + r * 20 + g * 4) = v;
        lds_wave_fence();
        store_rows<1>(p, area, lane, (mt0 + i) * 16, nt * 16);
    }
}

// Copies 16 bytes a lane from global memory straight to LDS: lane i's bytes
// land at dst + 16 i.
__device__ __forceinline__ void load_to_lds(const void* src, void* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// Waits until at most N of this wave's global loads (copies to LDS among
// them) are outstanding and all its LDS reads are done, then meets the other
// waves of the work-group.  (A fence before a plain barrier would wait for
// every copy in flight.)
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Many rows: a work-group of WM x WN waves takes WM FM 16 rows of y and
// WN FN 16 columns, each wave FM x FN instruction tiles.  K advances by 128
// columns a step through BUF buffers in LDS, filled straight from global
// memory BUF - 1 steps ahead.
template <int KIND, int WM, int WN, int FM, int FN, int BUF>
__global__ __launch_bounds__(64 * WM * WN) void linear_tiled_kernel(Operands p, int grid_m, int grid_n) {
    typedef typename Acc<KIND>::T acc_t;
    constexpr int WAVES = WM * WN, BM = WM * FM * 16, BN = WN * FN * 16;
    constexpr int X_KB = BM / 16 * (KIND == kMx ? 1 : 2), W_KB = BN / 16 * (KIND == kInt8 ? 2 : 1);   // a stage's KB
    constexpr int LOADS = (X_KB + W_KB) / WAVES;
    static_assert((X_KB + W_KB) % WAVES == 0 && X_KB % WAVES == 0, "each wave copies the same number of KB");
    __shared__ lb_u32x4 lds[BUF][(X_KB + W_KB) * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int wm = wave / WN, wn = wave % WN;

    // work-groups are dealt to the 8 XCDs in turn: give each XCD one run of tiles, and walk a run in blocks of
    // 8 tile rows so that what its L2 holds is used again
    const int total = grid_m * grid_n, per = total / 8, extra = total % 8, xcd = blockIdx.x % 8;
    const int id = xcd * per + (xcd < extra ? xcd : extra) + blockIdx.x / 8;
    const int band = id / (8 * grid_n), rows_in = grid_m - band * 8 < 8 ? grid_m - band * 8 : 8;
    const int in_band = id - band * 8 * grid_n;
    const int bm = band * 8 + in_band % rows_in, bn = in_band / rows_in;

    const int64_t tiles = cdiv(p.K, 128), words = cdiv(p.K, 512);
    const int64_t n_tiles = cdiv(p.N, 16), m_tiles = cdiv(p.M, 16);

    // where this wave's copies come from; rows and tiles past the last repeat the last, and are dropped at the end
    const uint8_t* src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int kb = i * WAVES + wave;
        if (kb < X_KB) {
            if (KIND == kMx) {
                const int64_t mt = (int64_t)bm * (BM / 16) + kb;
                src[i] = p.a + (mt < m_tiles ? mt : m_tiles - 1) * tiles * 1024 + lane * 16;
            } else {
                // 8 rows of 128 bytes; 16-byte chunk c of row r lies in slot c ^ (r & 7), so that 8 lanes reading
                // one chunk of 8 rows touch 8 different groups of banks
                const int64_t m = (int64_t)bm * BM + kb * 8 + (lane >> 3);
                src[i] = p.a + (m < p.M ? m : p.M - 1) * p.ld_a + ((lane & 7) ^ (lane >> 3)) * 16;
            }
        } else {
            const int64_t nt = (int64_t)bn * (BN / 16) + (KIND == kInt8 ? (kb - X_KB) / 2 : kb - X_KB);
            src[i] = p.w + ((nt < n_tiles ? nt : n_tiles - 1) * tiles * (KIND == kInt8 ? 2 : 1) +
                            (KIND == kInt8 ? (kb - X_KB) % 2 : 0)) * 1024 + lane * 16;
        }
    }
    auto fetch = [&](int buf) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            load_to_lds(src[i], &lds[buf][(i * WAVES + wave) * 64]);
            src[i] += i * WAVES < X_KB ? (KIND == kMx ? 1024 : 128) : (KIND == kInt8 ? 2048 : 1024);
        }
    };

    acc_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = acc_t{0, 0, 0, 0};

    // the scale words of four steps, BM / 16 + BN / 16 tiles of 256 bytes: 16 lanes copy a tile's
    constexpr int S_TILES = (BM + BN) / 16, S_WAVES = S_TILES / 4;
    static_assert(KIND != kMx || (BM % 64 == 0 && BN % 64 == 0 && S_WAVES <= WAVES), "a wave copies the scales of four tiles");
    __shared__ uint32_t lds_s[KIND == kMx ? 2 : 1][KIND == kMx ? S_TILES * 64 : 1];
    const uint32_t* s_src = nullptr;
    if (KIND == kMx && wave < S_WAVES) {
        const int tile = wave * 4 + (lane >> 4);
        if (tile < BM / 16) {
            const int64_t mt = (int64_t)bm * (BM / 16) + tile;
            s_src = p.a_scale + (mt < m_tiles ? mt : m_tiles - 1) * words * 64 + (lane & 15) * 4;
        } else {
            const int64_t nt = (int64_t)bn * (BN / 16) + tile - BM / 16;
            s_src = p.w_scale + (nt < n_tiles ? nt : n_tiles - 1) * words * 64 + (lane & 15) * 4;
        }
    }
    auto fetch_scales = [&](int half) {
        if (KIND == kMx && wave < S_WAVES) {
            load_to_lds(s_src, &lds_s[half][wave * 256]);
            s_src += 64;
        }
    };
    int xs[KIND == kMx ? FM : 1], ws[KIND == kMx ? FN : 1];
    auto read_scales = [&](int half) {
        if constexpr (KIND == kMx) {
#pragma unroll
            for (int i = 0; i < FM; ++i) xs[i] = (int)lds_s[half][(wm * FM + i) * 64 + lane];
#pragma unroll
            for (int j = 0; j < FN; ++j) ws[j] = (int)lds_s[half][(BM / 16 + wn * FN + j) * 64 + lane];
        }
    };

    auto step = [&](const lb_u32x4* s, auto byte) {
        constexpr int B = decltype(byte)::value;
        const lb_u32x4* x = s + wm * FM * (KIND == kMx ? 64 : 128);
        const lb_u32x4* w = s + X_KB * 64 + wn * FN * (KIND == kInt8 ? 128 : 64) + lane;
        if constexpr (KIND == kMx) {
            lb_u32x4 wv[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) wv[j] = w[j * 64];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const lb_u32x4 xv = x[i * 64 + lane];
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma_mx<B>(wv[j], xv, acc[i][j], ws[j], xs[i]);
            }
        } else {
            lb_u32x4 wv[2][FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if (KIND == kInt4) {
                    const lb_u32x4 q = w[j * 64];
                    wv[0][j] = low_nibbles(q);
                    wv[1][j] = high_nibbles(q);
                } else {
                    wv[0][j] = w[j * 128];
                    wv[1][j] = w[j * 128 + 64];
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const lb_u32x4 xv = x[(i * 16 + r) * 8 + ((h * 4 + g) ^ (r & 7))];
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mma_i8(wv[h][j], xv, acc[i][j]);
                }
        }
    };

    // one step: wait for this wave's own copies of it, meet the others (whose copies have then landed too, and who
    // are done with the buffer of the step before), fill that buffer, multiply.  The scales of four steps are copied
    // just before the first of them, into the half that the last four did not use.
    const int steps = (int)tiles;
    auto turn = [&](int t, int buf, int half, auto byte) {
        constexpr int B = decltype(byte)::value;
        if (t + BUF - 2 < steps) meet<LOADS * (BUF - 2)>();
        else meet<0>();
        if (t + BUF - 1 < steps) {
            if (KIND == kMx && B == 1) fetch_scales(half ^ 1);         // (of step t + 3, the first of its word)
            fetch((buf + BUF - 1) % BUF);
        }
        if (KIND == kMx && B == 0) read_scales(half);
        step(lds[buf], byte);
    };
    if (KIND == kMx) fetch_scales(0);
#pragma unroll
    for (int b = 0; b < BUF - 1; ++b)
        if (b < steps) fetch(b);
    if constexpr (KIND == kMx) {
        static_assert(KIND != kMx || BUF == 4, "a word of scales holds four steps");
        for (int t = 0, half = 0; t < steps; t += 4, half ^= 1) {
            turn(t, 0, half, std::integral_constant<int, 0>{});
            if (t + 1 < steps) turn(t + 1, 1, half, std::integral_constant<int, 1>{});
            if (t + 2 < steps) turn(t + 2, 2, half, std::integral_constant<int, 2>{});
            if (t + 3 < steps) turn(t + 3, 3, half, std::integral_constant<int, 3>{});
        }
    } else {
        for (int t = 0; t < steps; t += BUF) {
#pragma unroll
            for (int b = 0; b < BUF; ++b)
                if (t + b < steps) turn(t + b, b, 0, std::integral_constant<int, 0>{});
        }
    }
    static_assert(FN == 2 || FN == 4, "store_rows takes 32 or 64 columns");
    static_assert(sizeof(lds) >= WAVES * 16 * (16 * FN + 4) * 4, "the areas of the epilogue lie in the buffers");
    Columns<KIND> cols[FN];
    const int64_t m0 = (int64_t)bm * BM + wm * FM * 16, n0 = (int64_t)bn * BN + wn * FN * 16;
#pragma unroll
    for (int j = 0; j < FN; ++j) cols[j].load(p, n0 + j * 16 + g * 4);
    meet<0>();                                               // the buffers are free
    float* area = reinterpret_cast<float*>(&lds[0][0]) + wave * 16 * (16 * FN + 4);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t m = m0 + i * 16 + r < p.M ? m0 + i * 16 + r : p.M - 1;
        const float sa = KIND == kMx ? 1.0f : p.sa[m];
        const int sum = KIND != kMx && p.zp ? p.sums[m] : 0;
#pragma unroll
        for (int j = 0; j < FN; ++j)
            *reinterpret_cast<lb_f32x4*>(area + r * (16 * FN + 4) + j * 16 + g * 4) = cols[j].finish(acc[i][j], sa, sum);
        lds_wave_fence();
        store_rows<FN>(p, area, lane, m0 + i * 16, n0);
        lds_wave_fence();
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

template <int KIND, int MT, int WAVES>
void launch_direct(const Operands& p, hipStream_t st) {
    const dim3 grid((unsigned)cdiv(p.N, 16), (unsigned)cdiv(p.M, 16 * MT));
    hipLaunchKernelGGL((linear_direct_kernel<KIND, MT, WAVES>), grid, dim3(64 * WAVES), 0, st, p);
}

template <int KIND, int WM, int WN, int FM, int FN, int BUF>
void launch_tiled(const Operands& p, hipStream_t st) {
    const int gm = (int)cdiv(p.M, WM * FM * 16), gn = (int)cdiv(p.N, WN * FN * 16);
    hipLaunchKernelGGL((linear_tiled_kernel<KIND, WM, WN, FM, FN, BUF>), dim3((unsigned)gm * gn), dim3(64 * WM * WN), 0, st, p, gm, gn);
}

template <int KIND>
int launch_linear(const Operands& p, hipStream_t st) {
    if (p.M <= 16) launch_direct<KIND, 1, 8>(p, st);
    else if (p.M <= 32) launch_direct<KIND, 2, 8>(p, st);
    else if (p.M <= 64) launch_direct<KIND, 4, 8>(p, st);
    else launch_tiled<KIND, 2, 4, 8, 4, KIND == kMx ? 4 : KIND == kInt4 ? 3 : 2>(p, st);
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
    p.wide = aligned16(out) && ld_out % 4 == 0;
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
    p.wide = aligned16(out) && ld_out % 4 == 0;
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 2.0 * M * N * K, ((double)M * K + (double)N * K) * 17 / 32);
    return launch_linear<kMx>(p, st);
}
