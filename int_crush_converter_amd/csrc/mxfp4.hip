// Microscaled 4-bit floating point (OCP MX: E2M1 elements, one E8M0 scale for
// 32 consecutive columns): quantisation, its inverse, and the change between
// the row-major and the tiled layout of lowbit.hpp.
//
//   e = floor(log2(max|x|)) - 2 (clamped to [-127, 125]),
//   element = nearest E2M1 value of x / 2^e, ties to even, at most 6
//
// A block that holds Inf or NaN gets the scale NaN (byte 255) and codes 0.
#include "common.hpp"
#include "prof.hpp"
#include "lowbit.hpp"

namespace icq {
namespace {

// 32 values as one block: 16 bytes of codes and the scale's byte.
__device__ __forceinline__ lb_u32x4 quantize_block(float (&a)[16], float (&b)[16], unsigned& scale) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
    const bool bad = top >= 0x7f800000u;
    const int e8 = max((int)(top >> 23) - 2, 0);
    scale = bad ? 255u : (unsigned)e8;
    // the conversion divides by a normal power of two; 2^-127 is none, so such blocks (all magnitudes below 2^-124)
    // are doubled first, which is exact
    const bool low = e8 == 0;
    if (__builtin_amdgcn_ballot_w64(low) != 0) {
        const float f = low ? 2.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { a[i] *= f; b[i] *= f; }
    }
    const float s = __uint_as_float((unsigned)max(e8, 1) << 23);
    lb_u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float* v = k < 2 ? a + 8 * k : b + 8 * (k - 2);
        unsigned u = 0;
        u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0], v[1], s, 0);
        u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], s, 1);
        u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], s, 2);
        u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], s, 3);
        w[k] = bad ? 0u : u;
    }
    return w;
}

// One wave per tile of 16 rows x 128 columns; the four waves of a work-group
// take the four tiles that share a word of scales.  HBM-bound: 8192 x 12288 bf16
// 57.1 us (least 52.4), 4.5 TB/s; 5000 x 2900 fp16, rows at no alignment, 9.7 us,
// 3.8 TB/s (traced alone, medians of 30).
template <int DT>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const void* __restrict__ x, int64_t rows, int64_t cols,
                                                             int64_t ld, lb_u32x4* __restrict__ codes,
                                                             uint8_t* __restrict__ scales, int64_t tiles) {
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.y * 16 + (lane & 15), t = (int64_t)blockIdx.x * 4 + j;
    const int64_t c0 = t * 128 + (lane >> 4) * 32;
    float a[16], b[16];
    const int64_t n = row < rows ? cols : 0;
    load16<DT>(x, row * ld, c0, n, a);
    load16<DT>(x, row * ld, c0 + 16, n, b);
    unsigned s;
    const lb_u32x4 w = quantize_block(a, b, s);
    if (t < tiles) codes[((int64_t)blockIdx.y * tiles + t) * 64 + lane] = w;
    scales[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 64 + lane) * 4 + j] = (uint8_t)s;
}

// One wave per tile again, but a lane takes 8 columns of one row at a time, so
// that 16 lanes write 128 consecutive values: 8192 x 12288 to bf16 37.6 us traced
// alone, 6.8 TB/s (behind the quantisation, whose codes are in cache); 32 columns
// a lane (64 bytes of 64 rows a store) took half as long again.
template <int DT>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, int64_t rows,
                                                               int64_t cols, void* __restrict__ out, int64_t ld,
                                                               int64_t tiles) {
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6, part = lane & 15, g = part >> 2;
    const int64_t t = (int64_t)blockIdx.x * 4 + j, c0 = t * 128 + part * 8;
    if (c0 >= cols) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = k * 4 + (lane >> 4);
        const int64_t row = (int64_t)blockIdx.y * 16 + r;
        if (row >= rows) return;
        const uint32_t w = codes[(((int64_t)blockIdx.y * tiles + t) * 64 + g * 16 + r) * 4 + (part & 3)];
        const unsigned e = scales[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 64 + g * 16 + r) * 4 + j];
        // (2^-127 is no normal number: such a block is taken at 2^-126 and halved, which is exact)
        const float s = __uint_as_float((e ? e : 1u) << 23);
        float v[8];
        const lb_f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
        const lb_f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
        const float unit = e == 255 ? __uint_as_float(0x7fc00000u) : e ? 1.0f : 0.5f;
        v[0] = p0[0] * unit; v[1] = p0[1] * unit; v[2] = p1[0] * unit; v[3] = p1[1] * unit;
        v[4] = p2[0] * unit; v[5] = p2[1] * unit; v[6] = p3[0] * unit; v[7] = p3[1] * unit;
        store_cols<DT, 8>(out, row * ld, c0, cols, v);
    }
}

// Row-major bytes (blocks of 16, scales one a block) to tiles, or back.
template <bool PACK>
__global__ __launch_bounds__(256) void mxfp4_layout_kernel(uint8_t* __restrict__ flat, int64_t ld_c,
                                                           uint8_t* __restrict__ flat_s, int64_t ld_s, int64_t rows,
                                                           int64_t cols, lb_u32x4* __restrict__ codes,
                                                           uint8_t* __restrict__ scales, int64_t tiles) {
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.y * 16 + (lane & 15), t = (int64_t)blockIdx.x * 4 + j;
    const int64_t b = t * 4 + (lane >> 4), c0 = b * 32;
    const int64_t at = ((int64_t)blockIdx.y * tiles + t) * 64 + lane;
    const int64_t at_s = (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 64 + lane) * 4 + j;
    const bool in = row < rows && c0 < cols;
    const int left = in ? (int)(cols - c0 < 32 ? cols - c0 : 32) : 0, bytes = (left + 1) / 2;   // of this block
    if (PACK) {
        lb_u32x4 w = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            unsigned v = i < bytes ? flat[row * ld_c + c0 / 2 + i] : 0;
            if (2 * i + 1 >= left) v &= 15;                 // a column past the last is 0
            w[i >> 2] |= v << (8 * (i & 3));
        }
        if (t < tiles) codes[at] = w;
        scales[at_s] = in ? flat_s[row * ld_s + b] : 0;
    } else if (in) {
        const lb_u32x4 w = codes[at];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < bytes) flat[row * ld_c + c0 / 2 + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        flat_s[row * ld_s + b] = scales[at_s];
    }
}

int check_sizes(const char* who, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1) return fail(IC_ERR_ARG, std::string(who) + ": rows must be >= 0 and cols >= 1");
    if (rows > kMaxRows || cols > (1 << 20))
        return fail(IC_ERR_RANGE, std::string(who) + ": at most 1048560 rows and 2^20 columns");
    return IC_OK;
}

}  // namespace
}  // namespace icq

using namespace icq;

extern "C" int64_t ic_mxfp4_code_bytes(int64_t rows, int64_t cols) {
    return rows < 0 || cols < 0 ? 0 : cdiv(rows, 16) * cdiv(cols, 128) * 1024;
}
extern "C" int64_t ic_mxfp4_scale_bytes(int64_t rows, int64_t cols) {
    return rows < 0 || cols < 0 ? 0 : cdiv(rows, 16) * cdiv(cols, 512) * 256;
}

extern "C" int ic_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld_x, void* codes,
                                 void* scales, void* stream) {
    if (const int rc = check_sizes("ic_mxfp4_quantize", rows, cols)) return rc;
    IC_REQUIRE(dtype >= 0 && dtype <= 2, "ic_mxfp4_quantize: unknown dtype");
    if (rows == 0) return IC_OK;
    IC_REQUIRE(x && codes && scales, "ic_mxfp4_quantize: null pointer");
    IC_REQUIRE(ld_x >= cols && aligned16(codes), "ic_mxfp4_quantize: leading dimension below cols, or codes not 16-byte aligned");
    const int64_t es = dtype == IC_DTYPE_F32 ? 4 : 2;
    const dim3 g((unsigned)cdiv(cols, 512), (unsigned)cdiv(rows, 16)), b(256);
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 0.0, (double)rows * cols * (es + 17.0 / 32));
    lb_u32x4* c = static_cast<lb_u32x4*>(codes);
    uint8_t* s = static_cast<uint8_t*>(scales);
    const int64_t tiles = cdiv(cols, 128);
    if (dtype == IC_DTYPE_F32)
        hipLaunchKernelGGL(mxfp4_quantize_kernel<IC_DTYPE_F32>, g, b, 0, st, x, rows, cols, ld_x, c, s, tiles);
    else if (dtype == IC_DTYPE_BF16)
        hipLaunchKernelGGL(mxfp4_quantize_kernel<IC_DTYPE_BF16>, g, b, 0, st, x, rows, cols, ld_x, c, s, tiles);
    else
        hipLaunchKernelGGL(mxfp4_quantize_kernel<IC_DTYPE_F16>, g, b, 0, st, x, rows, cols, ld_x, c, s, tiles);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

extern "C" int ic_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out,
                                   int dtype, int64_t ld_out, void* stream) {
    if (const int rc = check_sizes("ic_mxfp4_dequantize", rows, cols)) return rc;
    IC_REQUIRE(dtype >= 0 && dtype <= 2, "ic_mxfp4_dequantize: unknown dtype");
    if (rows == 0) return IC_OK;
    IC_REQUIRE(codes && scales && out, "ic_mxfp4_dequantize: null pointer");
    IC_REQUIRE(ld_out >= cols && aligned16(codes), "ic_mxfp4_dequantize: leading dimension below cols, or codes not 16-byte aligned");
    const int64_t es = dtype == IC_DTYPE_F32 ? 4 : 2;
    const dim3 g((unsigned)cdiv(cols, 512), (unsigned)cdiv(rows, 16)), b(256);
    hipStream_t st = as_stream(stream);
    ProfScope prof(st, PT_OTHER, 0.0, (double)rows * cols * (es + 17.0 / 32));
    const uint32_t* c = static_cast<const uint32_t*>(codes);
    const uint8_t* s = static_cast<const uint8_t*>(scales);
    const int64_t tiles = cdiv(cols, 128);
    if (dtype == IC_DTYPE_F32)
        hipLaunchKernelGGL(mxfp4_dequantize_kernel<IC_DTYPE_F32>, g, b, 0, st, c, s, rows, cols, out, ld_out, tiles);
    else if (dtype == IC_DTYPE_BF16)
        hipLaunchKernelGGL(mxfp4_dequantize_kernel<IC_DTYPE_BF16>, g, b, 0, st, c, s, rows, cols, out, ld_out, tiles);
    else
        hipLaunchKernelGGL(mxfp4_dequantize_kernel<IC_DTYPE_F16>, g, b, 0, st, c, s, rows, cols, out, ld_out, tiles);
    IC_CHECK_LAUNCH();
    return IC_OK;
}

extern "C" int ic_mxfp4_relayout(void* flat_codes, int64_t ld_codes, void* flat_scales, int64_t ld_scales, int64_t rows,
                                 int64_t cols, void* codes, void* scales, int to_tiles, void* stream) {
    if (const int rc = check_sizes("ic_mxfp4_relayout", rows, cols)) return rc;
    if (rows == 0) return IC_OK;
    IC_REQUIRE(flat_codes && flat_scales && codes && scales, "ic_mxfp4_relayout: null pointer");
    IC_REQUIRE(ld_codes >= cdiv(cols, 2) && ld_scales >= cdiv(cols, 32) && aligned16(codes),
               "ic_mxfp4_relayout: a leading dimension is too small, or the tiles are not 16-byte aligned");
    const dim3 g((unsigned)cdiv(cols, 512), (unsigned)cdiv(rows, 16)), b(256);
    uint8_t *f = static_cast<uint8_t*>(flat_codes), *fs = static_cast<uint8_t*>(flat_scales);
    lb_u32x4* c = static_cast<lb_u32x4*>(codes);
    uint8_t* s = static_cast<uint8_t*>(scales);
    hipStream_t st = as_stream(stream);
    if (to_tiles)
        hipLaunchKernelGGL(mxfp4_layout_kernel<true>, g, b, 0, st, f, ld_codes, fs, ld_scales, rows, cols, c, s, cdiv(cols, 128));
    else
        hipLaunchKernelGGL(mxfp4_layout_kernel<false>, g, b, 0, st, f, ld_codes, fs, ld_scales, rows, cols, c, s, cdiv(cols, 128));
    IC_CHECK_LAUNCH();
    return IC_OK;
}
