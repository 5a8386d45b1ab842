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

// y for four consecutive n from n0 of row m, from the accumulated sums.
template <int KIND>
__device__ __forceinline__ void finish4(const Operands& p, typename Acc<KIND>::T acc, int64_t m, int64_t n0) {
    if (m >= p.M || n0 >= p.N) return;
    float v[4];
    float sa = 1.0f;
    int sum = 0;
    if (KIND != kMx) {
        sa = p.sa[m];
        if (p.zp) sum = p.sums[m];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t n = n0 + i < p.N ? n0 + i : p.N - 1;
        if constexpr (KIND == kMx) {
            v[i] = acc[i];
        } else {
            // INT4 operands are held as 16 q; the shift is exact.  |sum_k a (q - zp)| < 2^31 for K <= 65536, so the
            // difference is right even where a term has wrapped
            int d = KIND == kInt4 ? acc[i] >> 4 : acc[i];
            if (p.zp) d = (int)((unsigned)d - (unsigned)((int)p.zp[n] * sum));
            const float sw = p.sw_f32 ? static_cast<const float*>(p.sw)[n]
                                      : f16_bits_to_f32(static_cast<const uint16_t*>(p.sw)[n]);
            v[i] = (float)d * (sa * sw);
        }
        if (p.bias) v[i] += load_as_f32(p.bias, p.bias_dtype, n);
    }
    const int64_t at = m * p.ld_out + n0;
    if (p.wide && n0 + 4 <= p.N) {
        if (p.out_dtype == IC_DTYPE_F32) {
            *reinterpret_cast<lb_f32x4*>(static_cast<float*>(p.out) + at) = lb_f32x4{v[0], v[1], v[2], v[3]};
        } else {
            lb_u32x2 w;
            if (p.out_dtype == IC_DTYPE_BF16)
                w = lb_u32x2{pack_half_words<IC_DTYPE_BF16>(v[0], v[1]), pack_half_words<IC_DTYPE_BF16>(v[2], v[3])};
            else
                w = lb_u32x2{pack_half_words<IC_DTYPE_F16>(v[0], v[1]), pack_half_words<IC_DTYPE_F16>(v[2], v[3])};
            *reinterpret_cast<lb_u32x2*>(static_cast<uint16_t*>(p.out) + at) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < p.N) store_from_f32(p.out, p.out_dtype, at + i, v[i]);
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
// 32 INT4 values of a lane as two operands of 16 bytes, each value times 16.
__device__ __forceinline__ lb_u32x4 low_nibbles(lb_u32x4 p) { return (p << 4) & 0xf0f0f0f0u; }
__device__ __forceinline__ lb_u32x4 high_nibbles(lb_u32x4 p) { return p & 0xf0f0f0f0u; }

// Few rows: a work-group of WAVES waves takes 16 columns of y and 16 MT rows,
// its waves a share of K each; the sums are joined in LDS in a fixed order.
template <int KIND, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear_direct_kernel(Operands p) {
    typedef typename Acc<KIND>::T acc_t;
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
                acc[i] = mma_i8(w0, x[0], acc[i]);
                acc[i] = mma_i8(w1, x[4], acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < MT; i += WAVES) {
        acc_t s = part[0][i][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) s += part[k][i][lane];
        finish4<KIND>(p, s, (mt0 + i) * 16 + r, nt * 16 + g * 4);
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

template <int KIND>
int launch_linear(const Operands& p, hipStream_t st) {
    if (p.M <= 16) launch_direct<KIND, 1, 8>(p, st);
    else if (p.M <= 32) launch_direct<KIND, 2, 8>(p, st);
    else launch_direct<KIND, 4, 8>(p, st);
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
