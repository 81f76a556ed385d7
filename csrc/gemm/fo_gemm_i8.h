// Product of 8-bit integers with a scale for each token and each channel (no counterpart in the reference):
//   C[m, n] = round16(SA[m] * SB[e, n] * sum_k A[m, k] * B[e, n, k]),
// the sums exact in 32-bit integers.  Without offsets there is one matrix B [N, K]; with offsets [experts + 1] rows
// offsets[e] .. offsets[e + 1] - 1 of A are multiplied by B[e], and the rows outside all of these are set to zero.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <string>

namespace fo {

constexpr int kI8BK = 128;            // elements of K in one 128-byte swizzle atom
constexpr int kI8MaxK = 131071;       // 128 * 128 * K stays below 2^31
constexpr int kI8MaxExperts = 1024;
constexpr int kI8MaxRows = INT32_MAX - 1023;  // of A and of a weight matrix: tiles that begin inside end below 2^31

struct GemmI8Params {
  int M, N, K;
  int experts;            // of B; 1 without offsets
  int tiles_n;            // column tiles of the kernel that runs
  int raster_sw;          // wide kernel: strip width in column tiles
  int token_tiles;        // narrow kernel: token tiles that are launched (with offsets an upper bound)
  const int32_t* offsets;  // [experts + 1] or nullptr
  const float* SA;        // [M]
  const float* SB;        // [experts, N]
  uint16_t* C;            // [M, N]
  int32_t* status;
  uint64_t timeout_ns;
};

struct GemmI8Maps {
  CUtensorMap a, b, c;
  CUtensorMap b_half;  // wide kernel: boxes of half of b's rows, for half-width tiles
};

// What runs for a problem: the wide kernel (256 x 256 tiles, CTA pairs), or the narrow one (tiles of `tokens` tokens x 128
// channels, K split over the `split` CTAs of a cluster).
struct GemmI8Plan {
  int tokens;  // 0: wide
  int split;   // narrow; wide: 1, or 2 for tiles of 512 rows
};
GemmI8Plan choose_i8(int M, int N, int K, int experts, bool grouped);

// A [M, K], B [experts * N, K] int8.  Returns an empty string, or why the call cannot be made.
std::string gemm_i8_launch(const GemmI8Plan& plan, GemmI8Params p, const void* A, const void* B, bool bf16,
                           cudaStream_t stream);

}  // namespace fo
