// Packed 4-bit matrices (MXFP4): packing, reading back and the product.
#include "b200_mx4.h"

namespace b200 {
namespace mx4 {
namespace {

__host__ __device__ inline uint64_t scale_offset(uint64_t r, uint64_t b, uint64_t tiles) {
    return 512 * ((r / 128) * tiles + b / 4) + 16 * (r % 32) + 4 * (r % 128 / 32) + b % 4;
}

__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i) {
    switch (dtype) {
        case SNN_B200_F32: return ((const float *)p)[i];
        case SNN_B200_F16: return to_float(((const __half *)p)[i]);
        case SNN_B200_BF16: return to_float(((const __nv_bfloat16 *)p)[i]);
        default: return to_float(((const Spike *)p)[i]);
    }
}
__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float v) {
    switch (dtype) {
        case SNN_B200_F32: ((float *)p)[i] = v; break;
        case SNN_B200_F16: ((__half *)p)[i] = from_float<__half>(v); break;
        default: ((__nv_bfloat16 *)p)[i] = from_float<__nv_bfloat16>(v); break;
    }
}

// The scale byte of a block from its largest magnitude (bits of a
// non-negative float): exponent - 2, at least 2^-127, 255 when not finite.
// Scale byte s stands for 2^(s - 127) and the float's exponent field f for
// 2^(f - 127), so the byte is f - 2.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const uint32_t f = amax_bits >> 23;
    return f == 255u ? 255u : f > 2u ? f - 2u : 0u;
}
// 2^(127 - s) for s of 0..252.
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127), the smallest one subnormal.
__device__ __forceinline__ float scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fffffffu) : s ? __uint_as_float(s << 23) : __uint_as_float(0x00400000u);
}
// e2m1 code of v, ties to the even code, saturating.
__device__ __forceinline__ uint32_t encode(float v) {
    const float m = fabsf(v);
    uint32_t c = (m > 0.25f) + (m >= 0.75f) + (m > 1.25f) + (m >= 1.75f) + (m > 2.5f) + (m >= 3.5f) + (m > 5.0f);
    return c | (__float_as_uint(v) >> 31 << 3);
}
__device__ __forceinline__ float decode(uint32_t c) {
    const uint32_t m = c & 7u;
    const float v = m < 4u ? 0.5f * (float)m : m < 6u ? (float)(m - 2u) : (m == 6u ? 4.0f : 6.0f);
    return c & 8u ? -v : v;
}

// One thread a (padded) block.
__global__ void mx4_quantize_kernel(const void *src, int dtype, uint64_t rows, uint64_t cols, int64_t rs, int64_t cs,
                                    uint4 *codes, uint8_t *scales) {
    const uint64_t nb = blocks_of(cols), tiles = scale_tiles(cols);
    const uint64_t padded_rows = (rows + 127) / 128 * 128, padded_blocks = tiles * 4;
    const uint64_t step = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < padded_rows * padded_blocks; i += step) {
        const uint64_t r = i / padded_blocks, b = i % padded_blocks;
        uint32_t s = 0;
        if (r < rows && b < nb) {
            float v[kBlock];
            uint32_t top = 0;
            for (uint32_t k = 0; k < kBlock; ++k) {
                const uint64_t c = b * kBlock + k;
                v[k] = c < cols ? load_any(src, dtype, (int64_t)r * rs + (int64_t)c * cs) : 0.0f;
                top = max(top, __float_as_uint(fabsf(v[k])));
            }
            s = scale_byte(top);
            uint32_t w[4] = {};
            if (s != 255u) {
                const float inv = inverse_scale(s);
                for (uint32_t k = 0; k < kBlock; ++k) w[k / 8] |= encode(__fmul_rn(v[k], inv)) << (4 * (k % 8));
            }
            codes[r * nb + b] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        scales[scale_offset(r, b, tiles)] = (uint8_t)s;
    }
}

__global__ void mx4_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, uint64_t rows, uint64_t cols,
                                      void *dst, int dtype, int64_t rs) {
    const uint64_t nb = blocks_of(cols), tiles = scale_tiles(cols);
    const uint64_t step = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * cols; i += step) {
        const uint64_t r = i / cols, c = i % cols;
        const uint32_t code = codes[r * nb * 16 + c / 2] >> (4 * (c & 1)) & 15u;
        store_any(dst, dtype, (int64_t)r * rs + (int64_t)c,
                  __fmul_rn(decode(code), scale_value(scales[scale_offset(r, c / kBlock, tiles)])));
    }
}

// A product over no columns: the bias, or zero.
__global__ void mx4_no_columns_kernel(uint64_t m, uint64_t n, const float *bias, void *out, int dtype, int64_t rs) {
    const uint64_t step = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m * n; i += step)
        store_any(out, dtype, (int64_t)(i / n) * rs + (int64_t)(i % n), bias ? bias[i % n] : 0.0f);
}

int grid_for(int device, uint64_t threads, uint32_t block) {
    const uint64_t want = (threads + block - 1) / block, most = (uint64_t)sm_count(device) * 16;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

snn_status_t check_source(const void *src, int dtype, snn_size_t rows, snn_size_t cols, int64_t rs, int64_t cs) {
    if (!is_dtype(dtype) || !offset_fits(rows, rs) || !offset_fits(cols, cs)) return SNN_ERR_INVALID_ARGUMENT;
    if (rows && cols && (src == nullptr || !aligned_to(src, dtype_bytes(dtype)))) return SNN_ERR_INVALID_ARGUMENT;
    return SNN_OK;
}

snn_status_t check_packed(const void *codes, const void *scales, snn_size_t rows, snn_size_t cols) {
    if (rows == 0 || cols == 0) return SNN_OK;
    return codes && scales && aligned_to(codes, 16) && aligned_to(scales, 16) ? SNN_OK : SNN_ERR_INVALID_ARGUMENT;
}

snn_status_t check_rows(const void *out, int dtype, snn_size_t rows, snn_size_t cols, int64_t rs) {
    if (!is_float_dtype(dtype) || !offset_fits(rows, rs) || !disjoint_runs(rows, rs, 1, 0, cols))
        return SNN_ERR_INVALID_ARGUMENT;
    if (rows && cols && (out == nullptr || !aligned_to(out, dtype_bytes(dtype)))) return SNN_ERR_INVALID_ARGUMENT;
    return SNN_OK;
}

void enqueue_quantize(int device, cudaStream_t s, const void *src, int dtype, uint64_t rows, uint64_t cols, int64_t rs,
                      int64_t cs, void *codes, void *scales) {
    const uint64_t padded = (rows + 127) / 128 * 128 * scale_tiles(cols) * 4;
    mx4_quantize_kernel<<<grid_for(device, padded, 128), 128, 0, s>>>(src, dtype, rows, cols, rs, cs, (uint4 *)codes,
                                                                      (uint8_t *)scales);
}

cudaError_t enqueue_matmul(int device, cudaStream_t s, const Packed &x, const Packed &w, uint64_t k, const float *bias,
                           void *out, int dtype, int64_t rs) {
    if (k) return matmul(device, s, x, w, k, bias, out, dtype, rs);
    mx4_no_columns_kernel<<<grid_for(device, x.rows * w.rows, 256), 256, 0, s>>>(x.rows, w.rows, bias, out, dtype, rs);
    return cudaGetLastError();
}

}  // namespace
}  // namespace mx4
}  // namespace b200

using namespace b200;
using namespace b200::mx4;

extern "C" {

snn_status_t snn_b200_mx4_sizes(snn_size_t rows, snn_size_t cols, snn_size_t *out_code_bytes,
                                snn_size_t *out_scale_bytes) {
    if (out_code_bytes == nullptr || out_scale_bytes == nullptr) return SNN_ERR_INVALID_ARGUMENT;
    *out_code_bytes = *out_scale_bytes = 0;
    if (rows > kMaxCount || cols > kMaxCount) return SNN_ERR_OVERFLOW;
    *out_code_bytes = code_bytes(rows, cols);
    *out_scale_bytes = scale_bytes(rows, cols);
    return SNN_OK;
}

snn_status_t snn_b200_mx4_quantize_async(int device, void *stream, const void *src, int src_dtype, snn_size_t rows,
                                         snn_size_t cols, int64_t row_stride, int64_t col_stride, void *codes,
                                         void *scales) {
    if (rows > kMaxCount || cols > kMaxCount) return SNN_ERR_OVERFLOW;
    snn_status_t st = check_source(src, src_dtype, rows, cols, row_stride, col_stride);
    if (st == SNN_OK) st = check_packed(codes, scales, rows, cols);
    if (st != SNN_OK || device < 0) return st != SNN_OK ? st : SNN_ERR_INVALID_ARGUMENT;
    if (rows == 0 || cols == 0) return SNN_OK;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    enqueue_quantize(device, (cudaStream_t)stream, src, src_dtype, rows, cols, row_stride, col_stride, codes, scales);
    return op_status(cudaGetLastError(), __func__);
}

snn_status_t snn_b200_mx4_dequantize_async(int device, void *stream, const void *codes, const void *scales,
                                           snn_size_t rows, snn_size_t cols, void *dst, int dst_dtype,
                                           int64_t row_stride) {
    if (rows > kMaxCount || cols > kMaxCount) return SNN_ERR_OVERFLOW;
    snn_status_t st = check_packed(codes, scales, rows, cols);
    if (st == SNN_OK) st = check_rows(dst, dst_dtype, rows, cols, row_stride);
    if (st != SNN_OK || device < 0) return st != SNN_OK ? st : SNN_ERR_INVALID_ARGUMENT;
    if (rows == 0 || cols == 0) return SNN_OK;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    mx4_dequantize_kernel<<<grid_for(device, rows * cols, 256), 256, 0, (cudaStream_t)stream>>>(
        (const uint8_t *)codes, (const uint8_t *)scales, rows, cols, dst, dst_dtype, row_stride);
    return op_status(cudaGetLastError(), __func__);
}

snn_status_t snn_b200_mx4_matmul_async(int device, void *stream, const void *x_codes, const void *x_scales,
                                       snn_size_t m, const void *w_codes, const void *w_scales, snn_size_t n,
                                       snn_size_t k, const float *bias, void *out, int out_dtype,
                                       int64_t out_row_stride) {
    if (m > kMaxCount || n > kMaxCount || k > kMaxCount) return SNN_ERR_OVERFLOW;
    snn_status_t st = check_packed(x_codes, x_scales, m, k);
    if (st == SNN_OK) st = check_packed(w_codes, w_scales, n, k);
    if (st == SNN_OK) st = check_rows(out, out_dtype, m, n, out_row_stride);
    if (st != SNN_OK || device < 0 || !aligned_to(bias, 4)) return st != SNN_OK ? st : SNN_ERR_INVALID_ARGUMENT;
    if (m == 0 || n == 0) return SNN_OK;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    const Packed x = {(const uint8_t *)x_codes, (const uint8_t *)x_scales, m};
    const Packed w = {(const uint8_t *)w_codes, (const uint8_t *)w_scales, n};
    return op_status(enqueue_matmul(device, (cudaStream_t)stream, x, w, k, bias, out, out_dtype, out_row_stride),
                     __func__);
}

snn_size_t snn_b200_mx4_linear_workspace(snn_size_t m, snn_size_t k) {
    if (m > kMaxCount || k > kMaxCount) return 0;
    return code_bytes(m, k) + scale_bytes(m, k);
}

snn_status_t snn_b200_mx4_linear_async(int device, void *stream, const void *x, int x_dtype, snn_size_t m,
                                       snn_size_t k, int64_t x_row_stride, int64_t x_col_stride, const void *w_codes,
                                       const void *w_scales, snn_size_t n, const float *bias, void *out,
                                       int out_dtype, int64_t out_row_stride, void *workspace,
                                       snn_size_t workspace_bytes) {
    if (m > kMaxCount || n > kMaxCount || k > kMaxCount) return SNN_ERR_OVERFLOW;
    snn_status_t st = check_source(x, x_dtype, m, k, x_row_stride, x_col_stride);
    if (st == SNN_OK) st = check_packed(w_codes, w_scales, n, k);
    if (st == SNN_OK) st = check_rows(out, out_dtype, m, n, out_row_stride);
    if (st != SNN_OK || device < 0 || !aligned_to(bias, 4)) return st != SNN_OK ? st : SNN_ERR_INVALID_ARGUMENT;
    const uint64_t need = snn_b200_mx4_linear_workspace(m, k);
    if (need && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (m == 0 || n == 0) return SNN_OK;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    uint8_t *codes = (uint8_t *)workspace, *scales = codes + code_bytes(m, k);
    if (k) enqueue_quantize(device, (cudaStream_t)stream, x, x_dtype, m, k, x_row_stride, x_col_stride, codes, scales);
    cudaError_t e = cudaGetLastError();
    const Packed xq = {codes, scales, m}, w = {(const uint8_t *)w_codes, (const uint8_t *)w_scales, n};
    if (e == cudaSuccess)
        e = enqueue_matmul(device, (cudaStream_t)stream, xq, w, k, bias, out, out_dtype, out_row_stride);
    return op_status(e, __func__);
}

}  // extern "C"
