// The tile layouts that the row projections (rows.h) read and write, for kernels that hand their rows on to them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>

namespace navi_amd {
namespace rows {

// Tile layouts of the packed kernels (the prompt prefill): every operand load of a wave is one
// contiguous 1 KB instead of 16 rows x 64 B. Reads of L2-resident data run about twice as fast that
// way (16 rows x 64 B touch 16 cache lines per instruction, 1 KB touches 8).
// f32 activations [M][K] (K % 32 == 0): element (m, k) of 16-row tile m / 16 and 32-column step
// k / 32 sits where lane (m % 16) + 16 ((k / 8) % 4) of the MFMA A operand loads it, as two 1 KB
// halves (k % 8 < 4, then >= 4) of 64 lanes x 4 floats.
__host__ __device__ inline size_t pk_a(int m, int k, int K) {
    return ((static_cast<size_t>(m >> 4) * (K >> 5) + (k >> 5)) * 2 + ((k >> 2) & 1)) * 256 +
           static_cast<size_t>((m & 15) + 16 * ((k >> 3) & 3)) * 4 + (k & 3);
}
// f16 weights [N][K]: element (n, k) where lane (n % 16) + 16 ((k / 8) % 4) of the MFMA B operand
// loads it, 64 lanes x 8 halves per 16-row tile and 32-column step.
__host__ __device__ inline size_t pk_w(int n, int k, int K) {
    return (static_cast<size_t>(n >> 4) * (K >> 5) + (k >> 5)) * 512 + static_cast<size_t>((n & 15) + 16 * ((k >> 3) & 3)) * 8 +
           (k & 7);
}

} // namespace rows
} // namespace navi_amd
