// Packed 4-bit matrices: layout and the launchers shared by b200_mx4.cu (the
// calls) and b200_mx4_mma.cu (the product).
#pragma once

#include "b200_ops.h"

namespace b200 {
namespace mx4 {

constexpr uint32_t kBlock = 32;  // elements that share a scale

__host__ __device__ inline uint64_t blocks_of(uint64_t cols) { return (cols + kBlock - 1) / kBlock; }
__host__ __device__ inline uint64_t scale_tiles(uint64_t cols) { return (blocks_of(cols) + 3) / 4; }
inline uint64_t code_bytes(uint64_t rows, uint64_t cols) { return rows * blocks_of(cols) * 16; }
inline uint64_t scale_bytes(uint64_t rows, uint64_t cols) { return (rows + 127) / 128 * scale_tiles(cols) * 512; }

struct Packed {
    const uint8_t *codes, *scales;
    uint64_t rows;
};

// out[i, j] = x row i . w row j + bias[j]; k >= 1, m >= 1, n >= 1.
cudaError_t matmul(int device, cudaStream_t s, const Packed &x, const Packed &w, uint64_t k, const float *bias,
                   void *out, int dtype, int64_t row_stride);

// The same with up to 16 rows of plain x, packed by the product's own kernel,
// where packs_on_the_way.
bool packs_on_the_way(const void *x, int x_dtype, uint64_t m, int64_t row_stride, int64_t col_stride);
cudaError_t linear(int device, cudaStream_t s, const void *x, int x_dtype, uint64_t m, int64_t x_stride, const Packed &w,
                   uint64_t k, const float *bias, void *out, int dtype, int64_t row_stride);

}  // namespace mx4
}  // namespace b200
