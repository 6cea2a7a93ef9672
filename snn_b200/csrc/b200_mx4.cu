// Packed 4-bit matrices (MXFP4): packing, reading back, and the calls (the
// product itself: b200_mx4_mma.cu).
#include "b200_mx4.cuh"

namespace b200 {
namespace mx4 {
namespace {

__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float v) {
    switch (dtype) {
        case SNN_B200_F32: ((float *)p)[i] = v; break;
        case SNN_B200_F16: ((__half *)p)[i] = from_float<__half>(v); break;
        default: ((__nv_bfloat16 *)p)[i] = from_float<__nv_bfloat16>(v); break;
    }
}

// 128 rows x 4 blocks: the unit of the packers' CTAs, and one tile of scales.
constexpr uint32_t kTileRows = 128, kTileCols = 128;

// Rows of neighbouring elements. Lanes lie across a row, each with 16 bytes of
// it, and find their block's largest magnitude by shuffles, so loads and
// stores are whole runs; a CTA takes one tile of scales, which leaves whole.
// 16384 x 8192 bf16: 62 us, 5.4 TB/s (cold 3.9 TB/s with 70% of the issue slots
// taken: the arithmetic is close behind the bytes). Rows that do not start on 16
// bytes are read element by element, out of lines that the lanes share in L1
// (34654 x 3873 bf16: 117 us, against 62 at 3872 columns and 210 in the form below).
template <typename T, bool Aligned>
__global__ void __launch_bounds__(256) mx4_quantize_rows_kernel(const T *src, uint32_t rows, uint32_t cols, int64_t rs,
                                                                uint8_t *codes, uint8_t *scales, uint32_t tiles) {
    constexpr uint32_t kOwn = 16 / sizeof(T), kAcross = kTileCols / kOwn;  // elements of a lane, lanes on a row
    constexpr uint32_t kRowsAtOnce = 256 / kAcross, kPasses = kTileRows / kRowsAtOnce, kLanes = kBlock / kOwn;
    constexpr uint32_t kHeld = kPasses < 8 ? kPasses : 8;  // loads under way
    __shared__ __align__(16) uint8_t s_scales[512];
    const uint32_t tile = blockIdx.x, r0 = blockIdx.y * kTileRows;
    const uint32_t part = threadIdx.x % kAcross, first = threadIdx.x / kAcross, c = tile * kTileCols + part * kOwn;
    const uint64_t pitch = blocks_of(cols) * 16;
    after_previous();
#pragma unroll 1
    for (uint32_t pass = 0; pass < kPasses; pass += kHeld) {
        Piece<T> v[kHeld];
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) {
            const uint32_t r = r0 + (pass + i) * kRowsAtOnce + first;
            if (r < rows && c < cols) v[i] = load_piece<Aligned>(src + (int64_t)r * rs + c, cols - c);
            else v[i] = Piece<T>{};
        }
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) {
            const uint32_t at = (pass + i) * kRowsAtOnce + first, r = r0 + at;
            uint32_t top = v[i].largest();
#pragma unroll
            for (uint32_t d = 1; d < kLanes; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
            const uint32_t s = scale_byte(top);
            v[i].store(codes + r * pitch + c / 2, s, r < rows && c / kBlock < (cols + kBlock - 1) / kBlock);
            if (part % kLanes == 0) s_scales[scale_slot(at, part / kLanes)] = (uint8_t)s;
        }
    }
    __syncthreads();
    if (threadIdx.x < 32)
        reinterpret_cast<uint4 *>(scales + ((uint64_t)blockIdx.y * tiles + tile) * 512)[threadIdx.x] =
            reinterpret_cast<const uint4 *>(s_scales)[threadIdx.x];
}

// Other strides: a thread a block, lanes along the rows, so a transposed source
// is read in whole runs; all of a block's elements are on their way before the
// first is looked at (3873 x 34654 transposed: f32 109 us, bf16 110 us, 250 us with
// the magnitude taken on the way; the two rows of a word in a thread took 327).
template <typename T>
__global__ void __launch_bounds__(512) mx4_quantize_any_kernel(const T *src, uint32_t rows, uint32_t cols, int64_t rs,
                                                               int64_t cs, uint8_t *codes, uint8_t *scales,
                                                               uint32_t tiles) {
    __shared__ __align__(16) uint8_t s_scales[512];
    const uint32_t tile = blockIdx.x, at = threadIdx.x % kTileRows, b = threadIdx.x / kTileRows;
    const uint64_t r = (uint64_t)blockIdx.y * kTileRows + at, c = (uint64_t)tile * kTileCols + b * kBlock;
    const uint32_t n = r < rows && c < cols ? min(kBlock, (uint32_t)(cols - c)) : 0;
    const T *p = src + (int64_t)r * rs + (int64_t)c * cs;
    T e[kBlock];
    after_previous();
#pragma unroll
    for (uint32_t k = 0; k < kBlock; ++k) e[k] = k < n ? p[(int64_t)k * cs] : T{};
    uint32_t top = 0, w[4];
#pragma unroll
    for (uint32_t k = 0; k < kBlock; ++k) top = max(top, __float_as_uint(fabsf(to_float(e[k]))));
    const uint32_t s = scale_byte(top);
    const float inv = inverse_scale(s);
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
        float v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) v[k] = to_float(e[8 * q + k]);
        w[q] = s == 255u ? 0u : encode8(v, inv);
    }
    if (n) reinterpret_cast<uint4 *>(codes)[r * blocks_of(cols) + c / kBlock] = make_uint4(w[0], w[1], w[2], w[3]);
    s_scales[scale_slot(at, b)] = (uint8_t)s;
    __syncthreads();
    if (threadIdx.x < 32)
        reinterpret_cast<uint4 *>(scales + ((uint64_t)blockIdx.y * tiles + tile) * 512)[threadIdx.x] =
            reinterpret_cast<const uint4 *>(s_scales)[threadIdx.x];
}

// A CTA 16 rows of 512 elements at a time, a thread 8 elements (4 bytes of
// codes) of four rows. Whole: they are written in 16-byte pieces; else they go
// through shared memory and leave element by element, lanes side by side, so
// that rows that do not start on 16 bytes are written in whole runs too
// (34654 x 3873 -> bf16: 87 us, against 53 at 3872 columns).
template <typename T, bool Whole>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, uint32_t rows,
                                                             uint32_t cols, uint32_t tiles, T *dst, int64_t rs) {
    __shared__ __align__(16) T s_row[Whole ? 1 : 16][Whole ? 8 : 512];
    const uint64_t pitch = blocks_of(cols) * 16;
    const uint32_t first = blockIdx.x * 512, lane = threadIdx.x % 64, c = first + lane * 8, b = c / kBlock;
    after_previous();
    for (uint64_t base = (uint64_t)blockIdx.y * 16; base < rows; base += (uint64_t)gridDim.y * 16) {
        const uint64_t r0 = base + threadIdx.x / 64;
        uint32_t w[4] = {}, s[4] = {};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint64_t r = r0 + 4 * i;
            if (r >= rows || c >= cols) continue;
            w[i] = *reinterpret_cast<const uint32_t *>(codes + r * pitch + c / 2);
            s[i] = scales[512 * ((r / kTileRows) * tiles + b / 4) + scale_slot((uint32_t)(r % kTileRows), b % 4)];
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint64_t r = r0 + 4 * i;
            float v[8];
            decode8(w[i], scale_value(s[i]), v);
            Eight<T> o;
#pragma unroll
            for (int q = 0; q < 8; ++q) o.v[q] = from_float<T>(v[q]);
            T *to = Whole ? dst + (int64_t)r * rs + c : &s_row[threadIdx.x / 64 + 4 * i][lane * 8];
            if (Whole && (r >= rows || c >= cols)) continue;
            if (!Whole || c + 8 <= cols) {
#pragma unroll
                for (uint32_t q = 0; q < sizeof(T) / 2; ++q)
                    reinterpret_cast<uint4 *>(to)[q] = reinterpret_cast<const uint4 *>(&o)[q];
            } else {
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q)
                    if (c + q < cols) to[q] = o.v[q];
            }
        }
        if constexpr (!Whole) {
            __syncthreads();
            for (uint32_t i = 0; i < 4; ++i) {
                const uint64_t r = r0 + 4 * i;
                if (r >= rows) break;
                T *to = dst + (int64_t)r * rs + first;
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q)
                    if (first + q * 64 + lane < cols) to[q * 64 + lane] = s_row[threadIdx.x / 64 + 4 * i][q * 64 + lane];
            }
            __syncthreads();
        }
    }
}

// A product over no columns: the bias, or zero.
__global__ void mx4_no_columns_kernel(uint64_t m, uint64_t n, const float *bias, void *out, int dtype, int64_t rs) {
    after_previous();
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

template <typename T>
cudaError_t quantize_as(cudaStream_t s, const void *src, uint64_t rows, uint64_t cols, int64_t rs, int64_t cs,
                        uint8_t *codes, uint8_t *scales) {
    const uint32_t tiles = (uint32_t)scale_tiles(cols);
    cudaError_t e = cudaSuccess;
    // Tiles of rows beyond a grid's height go in several launches.
    for (uint64_t r0 = 0; e == cudaSuccess && r0 < rows; r0 += 65535ull * kTileRows) {
        const uint64_t n = rows - r0 < 65535ull * kTileRows ? rows - r0 : 65535ull * kTileRows;
        const dim3 grid(tiles, (uint32_t)((n + kTileRows - 1) / kTileRows));
        const T *from = (const T *)src + (int64_t)r0 * rs;
        uint8_t *c = codes + code_bytes(r0, cols), *x = scales + scale_bytes(r0, cols);
        if (cs == 1 && aligned_to(src, 16) && rs * (int64_t)sizeof(T) % 16 == 0)
            e = launch_early(mx4_quantize_rows_kernel<T, true>, grid, 256, 0, s, 1, from, n, cols, rs, c, x, tiles);
        else if (cs == 1)
            e = launch_early(mx4_quantize_rows_kernel<T, false>, grid, 256, 0, s, 1, from, n, cols, rs, c, x, tiles);
        else
            e = launch_early(mx4_quantize_any_kernel<T>, grid, 512, 0, s, 1, from, n, cols, rs, cs, c, x, tiles);
    }
    return e;
}
cudaError_t enqueue_quantize(cudaStream_t s, const void *src, int dtype, uint64_t rows, uint64_t cols, int64_t rs,
                             int64_t cs, void *codes, void *scales) {
    uint8_t *c = (uint8_t *)codes, *x = (uint8_t *)scales;
    switch (dtype) {
        case SNN_B200_F32: return quantize_as<float>(s, src, rows, cols, rs, cs, c, x);
        case SNN_B200_F16: return quantize_as<__half>(s, src, rows, cols, rs, cs, c, x);
        case SNN_B200_BF16: return quantize_as<__nv_bfloat16>(s, src, rows, cols, rs, cs, c, x);
        default: return quantize_as<Spike>(s, src, rows, cols, rs, cs, c, x);
    }
}
template <typename T>
cudaError_t dequantize_as(cudaStream_t s, const void *codes, const void *scales, uint64_t rows, uint64_t cols, void *dst,
                          int64_t rs) {
    const uint64_t high = (rows + 15) / 16;
    const dim3 grid((uint32_t)((cols + 511) / 512), (uint32_t)(high < 65535 ? high : 65535));
    const bool whole = aligned_to(dst, 16) && rs * (int64_t)sizeof(T) % 16 == 0;
    return launch_early(whole ? mx4_dequantize_kernel<T, true> : mx4_dequantize_kernel<T, false>, grid, 256, 0, s, 1,
                        (const uint8_t *)codes, (const uint8_t *)scales, rows, cols, scale_tiles(cols), (T *)dst, rs);
}

cudaError_t enqueue_matmul(int device, cudaStream_t s, const Packed &x, const Packed &w, uint64_t k, const float *bias,
                           void *out, int dtype, int64_t rs) {
    if (k) return matmul(device, s, x, w, k, bias, out, dtype, rs);
    return launch_early(mx4_no_columns_kernel, grid_for(device, x.rows * w.rows, 256), 256, 0, s, 1, x.rows, w.rows, bias,
                        out, dtype, rs);
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
    return op_status(
        enqueue_quantize((cudaStream_t)stream, src, src_dtype, rows, cols, row_stride, col_stride, codes, scales), __func__);
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
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = dst_dtype == SNN_B200_F32   ? dequantize_as<float>(s, codes, scales, rows, cols, dst, row_stride)
                          : dst_dtype == SNN_B200_F16 ? dequantize_as<__half>(s, codes, scales, rows, cols, dst, row_stride)
                                                      : dequantize_as<__nv_bfloat16>(s, codes, scales, rows, cols, dst,
                                                                                     row_stride);
    return op_status(e, __func__);
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

snn_size_t snn_b200_mx4_linear_workspace(const void *x, int x_dtype, snn_size_t m, snn_size_t k, int64_t x_row_stride,
                                         int64_t x_col_stride) {
    if (m > kMaxCount || k > kMaxCount || packs_on_the_way(x, x_dtype, m, x_row_stride, x_col_stride)) return 0;
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
    const uint64_t need = snn_b200_mx4_linear_workspace(x, x_dtype, m, k, x_row_stride, x_col_stride);
    if (need && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (m == 0 || n == 0) return SNN_OK;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    const cudaStream_t s = (cudaStream_t)stream;
    const Packed w = {(const uint8_t *)w_codes, (const uint8_t *)w_scales, n};
    if (k && packs_on_the_way(x, x_dtype, m, x_row_stride, x_col_stride))
        return op_status(linear(device, s, x, x_dtype, m, x_row_stride, w, k, bias, out, out_dtype, out_row_stride),
                         __func__);
    uint8_t *codes = (uint8_t *)workspace, *scales = codes + code_bytes(m, k);
    cudaError_t e = k ? enqueue_quantize(s, x, x_dtype, m, k, x_row_stride, x_col_stride, codes, scales) : cudaSuccess;
    const Packed xq = {codes, scales, m};
    if (e == cudaSuccess) e = enqueue_matmul(device, s, xq, w, k, bias, out, out_dtype, out_row_stride);
    return op_status(e, __func__);
}

}  // extern "C"
