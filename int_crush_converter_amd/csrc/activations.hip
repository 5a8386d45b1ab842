// 8-bit activations for a quantised layer: residual addition, root-mean-square
// norm, group-wise Hadamard rotation and quantisation of a row in one pass.
//
//   h = x + r,  y = h rsqrt(mean(h^2) + eps) g,  z = R pad(y),
//   s = max(|z|_max, 1e-30) / 127,  q = clamp(rhaz(z / s), -127, 127)
//
// A row stays in registers from its load to its codes, so HBM sees each
// input and each output once.
#include "common.hpp"
#include "prof.hpp"
#include "lowbit.hpp"

namespace icq {
namespace {

// Work-groups in runs of 2^20 along the grid's second axis: along one axis a
// launch has fewer than 2^32 threads, which 2^22 rows of 16 waves fill.
inline dim3 group_grid(int64_t groups) {
    const int64_t run = 1 << 20;
    return dim3((unsigned)(groups < run ? groups : run), (unsigned)cdiv(groups, run));
}
__device__ __forceinline__ int64_t group_index() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

constexpr float kTinyMax = 1e-30f;   // the smallest row maximum that a scale stands for
constexpr float kTopScale = 0x1.020406p+121f;   // the largest whose 127-fold is finite (fp32's largest value / 127 rounds up)

__device__ __forceinline__ void bfly4(float& a, float& b, float& c, float& d) {
    const float s = (a + b) + (c + d);
    const float na = __builtin_fmaf(s, 0.5f, -d), nb = __builtin_fmaf(s, 0.5f, -c);
    const float nc = __builtin_fmaf(s, 0.5f, -b), nd = __builtin_fmaf(s, 0.5f, -a);
    a = na; b = nb; c = nc; d = nd;
}

template <int CTRL>
__device__ __forceinline__ float dppf(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E;                   // quad permutations
constexpr int kRor4 = 0x124, kRor8 = 0x128;                 // rotations within 16 lanes

// One base-4 digit across lanes, twice its value: with the digits' values
// x_0 .. x_3 in four lanes, 2 y_d = (x_d + x_(d^1)) + (x_(d^2) - x_(d^3)), a
// sum, a difference and one exchange of the difference.  Across a quad:
__device__ __forceinline__ float digit_quad(float v) {
    const float p = v + dppf<kXor1>(v), q = v - dppf<kXor1>(v);
    return p + dppf<kXor2>(q);
}
// and across lane bits 2 and 3 of a row of 16 (d ^ 2: 8 lanes on).  A rotation
// by 4 brings lane i the difference of lane i - 4: that of d ^ 1 where bit 2 is
// set, else that 8 lanes from it, which is its negative.
__device__ __forceinline__ float digit_row16(float v, float sign) {
    const float p = v + dppf<kRor8>(v), q = v - dppf<kRor8>(v);
    return __builtin_fmaf(dppf<kRor4>(q), sign, p);
}

// R of order rot in {4, 16, 64, 256} on chunks of 16 consecutive columns, 16
// consecutive lanes holding 256 columns; for 64 and 256 the result is 2 and 4
// times the rotation's.
__device__ __forceinline__ void rotate16(float (&v)[16], int rot, float sign) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) bfly4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    if (rot >= 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) bfly4(v[i], v[i + 4], v[i + 8], v[i + 12]);
    }
    if (rot >= 64) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = digit_quad(v[i]);
    }
    if (rot >= 256) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = digit_row16(v[i], sign);
    }
}

// op over the 64 lanes: within rows of 16 by DPP, between them by two exchanges.
// The rotations give the four quads of a row their sums in different orders, so
// one lane's result is taken for all: a row has one norm and one scale.
template <int CTRL, typename T>
__device__ __forceinline__ T dpp_any(T v) {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int WAVES, typename T, typename F>
__device__ __forceinline__ T row_reduce(T v, T* lds, F op) {
    v = op(v, dpp_any<kXor1>(v));
    v = op(v, dpp_any<kXor2>(v));
    v = op(v, dpp_any<kRor4>(v));
    v = op(v, dpp_any<kRor8>(v));
    v = op(v, __shfl_xor(v, 16, 64));
    v = op(v, __shfl_xor(v, 32, 64));
    if (WAVES > 1) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[w] = v;
        lds_barrier();                       // (each reduction has LDS of its own)
        v = lds[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = op(v, lds[i]);
        return v;
    }
    return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// WAVES waves hold one row, NC chunks of 16 columns a lane; for WAVES = 1 a
// work-group of 4 waves holds 4 rows.  HBM bounds it.  Traced alone (median of
// 30): 8192 x 4096 bf16 with residual and rotation 43.8 us, 5.4 TB/s; 8192 x
// 12288 without rotation 61.5 us (least 56.4), 4.9 TB/s; one call after another
// 41.8 and 53.7 us (a large copy: 5.1 TB/s).  Four waves a row with one chunk a
// lane, as one wave with four of them took a fifth longer for the first (62
// against 51 us, with the loads of that time): three reductions meet at
// barriers, but four times the waves cover the loads' latency.  16 waves of
// four chunks spill 16 registers of the row.
template <int DT, int WAVES, int NC>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void quantize_rows_kernel(
    const void* __restrict__ x, int64_t rows, int64_t cols, int64_t ld_x, const void* residual, int64_t ld_r,
    const void* __restrict__ weight, int weight_f32, float eps, int rot, int8_t* __restrict__ codes,
    int64_t ld_q, float* __restrict__ scales, int32_t* __restrict__ sums, void* residual_out,
    int64_t ld_ro) {
    __shared__ float red_f[WAVES], red_f2[WAVES];
    __shared__ unsigned red_u[WAVES], red_u2[WAVES];
    __shared__ int red_i[WAVES];
    const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = WAVES == 1 ? group_index() * 4 + (threadIdx.x >> 6) : group_index();
    if (row >= rows) return;
    constexpr int SPAN = 64 * WAVES * 16;

    float v[NC][16];
#pragma unroll
    for (int c = 0; c < NC; ++c) load16<DT>(x, row * ld_x, c * SPAN + lane * 16, cols, v[c]);
    if (residual) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float r[16];
            load16<DT>(residual, row * ld_r, c * SPAN + lane * 16, cols, r);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[c][i] += r[i];
            store_cols<DT, 16>(residual_out, row * ld_ro, c * SPAN + lane * 16, cols, v[c]);
        }
    }
    if (weight) {
        // the weight is on its way while the squares are summed, unless it and the row fill the registers (128 a lane
        // with 1024 threads, where 89 were spilled: 2048 x 65536 bf16 153 us, 166 with the early load and 16 spilled;
        // 1024 x 65536 fp32 107 against 97, with residual and rotation 226 against 227)
        constexpr bool EARLY = WAVES * NC < 64;
        float g[EARLY ? NC : 1][16];
        auto load_weight = [&](int c, float (&to)[16]) {
            if (weight_f32) load16<IC_DTYPE_F32>(weight, 0, c * SPAN + lane * 16, cols, to);
            else load16<DT>(weight, 0, c * SPAN + lane * 16, cols, to);
        };
        if (EARLY) {
#pragma unroll
            for (int c = 0; c < NC; ++c) load_weight(c, g[c]);
        }
        auto squares = [&]() {
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(v[c][i], v[c][i], ss);
            return ss;
        };
        const auto add = [](float a, float b) { return a + b; };
        const auto larger = [](unsigned a, unsigned b) { return max(a, b); };
        float ms = row_reduce<WAVES>(squares(), red_f, add) / (float)cols + eps;
        if (!(ms >= 0x1p-100f && ms < INFINITY)) {
            // Squares past fp32's range, or all below it (the whole row takes this branch): again with the row, and
            // eps, brought to a magnitude of 1 by a power of two.  Rows with Inf or NaN end as NaN here as well.
            unsigned top = __float_as_uint(sqrtf(eps));
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[c][i]) & 0x7fffffffu);
            top = row_reduce<WAVES>(top, red_u2, larger);
            const int e = min(max((int)(top >> 23), 1), 253);          // (254: the power's own would be subnormal)
            const float f = __uint_as_float((unsigned)(254 - e) << 23);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) v[c][i] *= f;
            ms = row_reduce<WAVES>(squares(), red_f2, add) / (float)cols + eps * f * f;
        }
        const float rs = 1.0f / sqrtf(ms);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (!EARLY) load_weight(c, g[0]);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[c][i] = v[c][i] * rs * g[EARLY ? c : 0][i];
        }
    }
    if (rot > 1) {
#pragma unroll
        for (int c = 0; c < NC; ++c) rotate16(v[c], rot, lane & 4 ? 1.0f : -1.0f);
    }
    // the maximum of the magnitudes' bits: Inf and NaN compare above every finite value
    unsigned top = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[c][i]) & 0x7fffffffu);
    top = row_reduce<WAVES>(top, red_u, [](unsigned a, unsigned b) { return max(a, b); });
    const bool bad = top >= 0x7f800000u;
    // z is `unit` times the values held; |z| / s <= 127 (1 + 2^-22), whose halves round to 127 at most.  The factor
    // 127 / peak is held as two fp32 values: with the first alone, whose rounding may lie below, a half (z = peak / 2
    // gives 63.5) would now and then round towards zero.
    const float unit = rot >= 256 ? 0.25f : rot >= 64 ? 0.5f : 1.0f;
    const float peak = bad ? 1.0f : fmaxf(__uint_as_float(top) * unit, kTinyMax);
    const float ratio = 127.0f / peak;
    const float inv = bad ? 0.0f : ratio * unit, rest = bad ? 0.0f : __builtin_fmaf(-ratio, peak, 127.0f) / peak * unit;
    int sum = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int64_t c0 = c * SPAN + lane * 16;
        lb_u32x4 word;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            int q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = v[c][4 * w + k];
                q[k] = bad ? 0 : (int)__builtin_fmaf(z, inv, __builtin_fmaf(z, rest, __builtin_copysignf(0.5f, z)));    // truncates
            }
            const unsigned lo = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(q[3], q[2], 0x04000c0c);
            word[w] = lo | hi;
            sum = __builtin_amdgcn_sdot4(word[w], 0x01010101, sum, false);
        }
        if (c0 < ld_q) *reinterpret_cast<lb_u32x4*>(codes + row * ld_q + c0) = word;
    }
    sum = row_reduce<WAVES>(sum, red_i, [](int a, int b) { return a + b; });
    if (lane == 0) {
        scales[row] = bad ? __uint_as_float(0x7fc00000u) : fminf(peak / 127.0f, kTopScale);
        sums[row] = sum;
    }
}

// q * s back as values: one lane per 16 codes.  HBM-bound: 8192 x 12288 to bf16
// 48.2 us traced alone, 6.3 TB/s (behind the quantisation, whose codes are partly
// in cache).
template <int DT>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const int8_t* __restrict__ codes, int64_t rows,
                                                              int64_t cols, int64_t ld_q,
                                                              const float* __restrict__ scales, void* __restrict__ out,
                                                              int64_t ld_out) {
    const int64_t upr = cdiv(cols, 16), total = rows * upr, stride = (int64_t)gridDim.x * 256;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += stride) {
        const int64_t r = u / upr, c0 = (u - r * upr) * 16;
        const lb_u32x4 w = *reinterpret_cast<const lb_u32x4*>(codes + r * ld_q + c0);
        const float s = scales[r];
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * s;
        store_cols<DT, 16>(out, r * ld_out, c0, cols, v);
    }
}

// Row sums of 8-bit codes: one wave a row.
__global__ __launch_bounds__(256) void row_sums_kernel(const int8_t* __restrict__ codes, int64_t rows, int64_t cols,
                                                       int64_t ld_q, int32_t* __restrict__ sums) {
    const int64_t row = group_index() * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    int sum = 0;
    for (int64_t c = threadIdx.x & 63; c < cols; c += 64) sum += codes[row * ld_q + c];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[row] = sum;
}

struct RowArgs {
    const void* x; int64_t rows, cols, ld_x; const void* residual; int64_t ld_r; const void* weight;
    int weight_f32; float eps; int rot; int8_t* codes; int64_t ld_q; float* scales; int32_t* sums; void* residual_out;
    int64_t ld_ro; hipStream_t st;
};

template <int DT, int WAVES, int NC>
void launch_rows(const RowArgs& a) {
    const dim3 grid = group_grid(WAVES == 1 ? cdiv(a.rows, 4) : a.rows), block(WAVES == 1 ? 256 : 64 * WAVES);
    hipLaunchKernelGGL((quantize_rows_kernel<DT, WAVES, NC>), grid, block, 0, a.st, a.x, a.rows, a.cols, a.ld_x,
                       a.residual, a.ld_r, a.weight, a.weight_f32, a.eps, a.rot, a.codes, a.ld_q, a.scales, a.sums,
                       a.residual_out, a.ld_ro);
}

// One wave a row up to 1024 columns, four up to 16384, else sixteen.
template <int DT>
void launch_waves(const RowArgs& a) {
    if (a.ld_q <= 1024) return launch_rows<DT, 1, 1>(a);
    if (a.ld_q <= 4096) return launch_rows<DT, 4, 1>(a);
    if (a.ld_q <= 8192) return launch_rows<DT, 4, 2>(a);
    if (a.ld_q <= 12288) return launch_rows<DT, 4, 3>(a);
    if (a.ld_q <= 16384) return launch_rows<DT, 4, 4>(a);
    if (a.ld_q <= 32768) return launch_rows<DT, 16, 2>(a);
    if (a.ld_q <= 49152) return launch_rows<DT, 16, 3>(a);
    launch_rows<DT, 16, 4>(a);
}

}  // namespace
}  // namespace icq

using namespace icq;

extern "C" int64_t ic_activation_pitch(int64_t cols) { return cols < 0 ? 0 : cdiv(cols, kActPad) * kActPad; }

extern "C" int ic_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld_x,
                                const void* residual, int64_t ld_r, const void* weight, int weight_dtype,
                                float eps, int rot, int8_t* codes, int64_t ld_q, float* scales, int32_t* sums, void* residual_out,
                                int64_t ld_ro, void* stream) {
    IC_REQUIRE(rows >= 0 && cols >= 1, "ic_quantize_rows: rows must be >= 0 and cols >= 1");
    IC_REQUIRE(dtype >= 0 && dtype <= 2, "ic_quantize_rows: unknown dtype");
    IC_REQUIRE(!weight || weight_dtype == dtype || weight_dtype == IC_DTYPE_F32,
               "ic_quantize_rows: the norm's weight is of x's dtype or fp32");
    IC_REQUIRE(rot == 1 || rot == 4 || rot == 16 || rot == 64 || rot == 256,
               "ic_quantize_rows: rot must be 1, 4, 16, 64 or 256");
    if (rows == 0) return IC_OK;
    IC_REQUIRE(x && codes && scales && sums, "ic_quantize_rows: null pointer");
    IC_REQUIRE(!residual == !residual_out, "ic_quantize_rows: residual and residual_out go together");
    const int64_t cols_pad = cdiv(cols, rot) * rot;
    if (cols_pad > 65536 || rows > 0x7fffffff) return fail(IC_ERR_RANGE, "ic_quantize_rows: at most 65536 columns and 2^31 - 1 rows");
    IC_REQUIRE(ld_x >= cols && (!residual || (ld_r >= cols && ld_ro >= cols)), "ic_quantize_rows: leading dimension below cols");
    IC_REQUIRE(ld_q == ic_activation_pitch(cols_pad) && aligned16(codes),
               "ic_quantize_rows: codes need ic_activation_pitch columns and 16-byte alignment");
    const int64_t es = dtype == IC_DTYPE_F32 ? 4 : 2;
    RowArgs a{x, rows, cols, ld_x, residual, ld_r, weight, weight && weight_dtype == IC_DTYPE_F32, eps, rot, codes, ld_q, scales, sums,
              residual_out, ld_ro, as_stream(stream)};
    ProfScope prof(a.st, PT_OTHER, 0.0, (double)rows * cols * (es * (residual ? 3 : 1) + 1));
    if (dtype == IC_DTYPE_F32) launch_waves<IC_DTYPE_F32>(a);
    else if (dtype == IC_DTYPE_BF16) launch_waves<IC_DTYPE_BF16>(a);
    else launch_waves<IC_DTYPE_F16>(a);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

extern "C" int ic_dequantize_rows(const int8_t* codes, int64_t rows, int64_t cols, int64_t ld_q, const float* scales,
                                  void* out, int dtype, int64_t ld_out, void* stream) {
    IC_REQUIRE(rows >= 0 && cols >= 1, "ic_dequantize_rows: rows must be >= 0 and cols >= 1");
    IC_REQUIRE(dtype >= 0 && dtype <= 2, "ic_dequantize_rows: unknown dtype");
    if (rows == 0) return IC_OK;
    IC_REQUIRE(codes && scales && out, "ic_dequantize_rows: null pointer");
    IC_REQUIRE(ld_q >= cdiv(cols, 16) * 16 && ld_q % 16 == 0 && aligned16(codes) && ld_out >= cols,
               "ic_dequantize_rows: rows of codes need a pitch of whole 16-byte words");
    const int64_t es = dtype == IC_DTYPE_F32 ? 4 : 2;
    const int64_t grid = cdiv(rows * cdiv(cols, 16), 256);
    const dim3 g((unsigned)(grid < 65536 ? grid : 65536)), b(256);
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 0.0, (double)rows * cols * (es + 1));
    if (dtype == IC_DTYPE_F32)
        hipLaunchKernelGGL(dequantize_rows_kernel<IC_DTYPE_F32>, g, b, 0, st, codes, rows, cols, ld_q, scales, out, ld_out);
    else if (dtype == IC_DTYPE_BF16)
        hipLaunchKernelGGL(dequantize_rows_kernel<IC_DTYPE_BF16>, g, b, 0, st, codes, rows, cols, ld_q, scales, out, ld_out);
    else
        hipLaunchKernelGGL(dequantize_rows_kernel<IC_DTYPE_F16>, g, b, 0, st, codes, rows, cols, ld_q, scales, out, ld_out);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

extern "C" int ic_row_sums_i8(const int8_t* codes, int64_t rows, int64_t cols, int64_t ld_q, int32_t* sums,
                              void* stream) {
    IC_REQUIRE(rows >= 0 && cols >= 1 && ld_q >= cols, "ic_row_sums_i8: bad sizes");
    if (rows == 0) return IC_OK;
    IC_REQUIRE(codes && sums, "ic_row_sums_i8: null pointer");
    if (cols > 65536 || rows > 0x7fffffff) return fail(IC_ERR_RANGE, "ic_row_sums_i8: at most 65536 columns and 2^31 - 1 rows");
    hipLaunchKernelGGL(row_sums_kernel, group_grid(cdiv(rows, 4)), dim3(256), 0, as_stream(stream), codes, rows,
                       cols, ld_q, sums);
    IC_CHECK_LAUNCH();
    return IC_OK;
}
