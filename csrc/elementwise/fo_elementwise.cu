#include "fo_elementwise.h"

#include <cstdint>

#include "../common/fo_pack16.cuh"
#include "../common/fo_ptx.cuh"

namespace fo {

namespace {

constexpr int kThreads = 256;

// Bound by memory: 4096 tokens x 9 heads of 128 (19 MB moved) took 284 us as the fourteen eager
// operators of the two rotations (fp32 intermediates, strided pairs) and take 9 us here.
// A thread owns 8 adjacent elements (4 pairs) of one position and walks kHeadsPerThread heads, whose
// loads are all in flight while it computes the four angles they share.
constexpr int kHeadsPerThread = 8;

template <bool BF16>
__global__ void __launch_bounds__(kThreads)
    rope_kernel(uint16_t* __restrict__ qkv, int tokens, int seq, int heads, int head_dim, int row_elems, float theta) {
  const int per_head = head_dim / 8;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t token = idx / per_head;
  if (token >= tokens) return;
  const int d = static_cast<int>(idx - token * per_head) * 8;
  const int h0 = blockIdx.y * kHeadsPerThread;
  const int h1 = min(heads, h0 + kHeadsPerThread);
  uint16_t* row = qkv + token * row_elems + d;
  uint4 x[kHeadsPerThread];
#pragma unroll
  for (int i = 0; i < kHeadsPerThread; ++i) {
    if (h0 + i < h1) x[i] = *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h0 + i) * head_dim);
  }
  const float pos = static_cast<float>(token % seq);
  float c[4], s[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float inv = powf(theta, -static_cast<float>(d + 2 * k) / static_cast<float>(head_dim));
    sincosf(pos * inv, &s[k], &c[k]);
  }
#pragma unroll
  for (int i = 0; i < kHeadsPerThread; ++i) {
    if (h0 + i < h1) {
      uint32_t* u = reinterpret_cast<uint32_t*>(&x[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = unpack2<BF16>(u[k]);
        u[k] = pack2<BF16>(v.x * c[k] - v.y * s[k], v.x * s[k] + v.y * c[k]);
      }
      *reinterpret_cast<uint4*>(row + static_cast<int64_t>(h0 + i) * head_dim) = x[i];
    }
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t silu_mul(uint32_t g, uint32_t u) {
  const float2 a = unpack2<BF16>(g);
  // silu is rounded to the storage type before the product, as two operators in a row round it
  const uint32_t r = pack2<BF16>(silu(a.x), silu(a.y));
  const float2 p = unpack2<BF16>(r), q = unpack2<BF16>(u);
  return pack2<BF16>(p.x * q.x, p.y * q.y);
}

template <bool BF16>
__device__ __forceinline__ uint4 silu_mul8(const uint4& g, const uint4& u) {
  return make_uint4(silu_mul<BF16>(g.x, u.x), silu_mul<BF16>(g.y, u.y), silu_mul<BF16>(g.z, u.z),
                    silu_mul<BF16>(g.w, u.w));
}

// Bound by memory: 4096 x 7168 -> 3584 (88 MB) took 81 us as silu and a product over strided halves
// and takes 20 us here.  One row at a time per CTA (grid-strided), two vectors of each operand in flight per thread.
template <bool BF16>
__global__ void __launch_bounds__(kThreads)
    swiglu_kernel(const uint16_t* __restrict__ gu, uint16_t* __restrict__ y, int rows, int f) {
  const int nvec = f / 8;
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const uint4* g = reinterpret_cast<const uint4*>(gu + static_cast<int64_t>(r) * 2 * f);
    const uint4* u = g + nvec;
    uint4* o = reinterpret_cast<uint4*>(y + static_cast<int64_t>(r) * f);
    for (int j = threadIdx.x; j < nvec; j += 2 * kThreads) {
      const bool two = j + kThreads < nvec;
      const uint4 g0 = __ldcs(g + j), u0 = __ldcs(u + j);
      uint4 g1 = {}, u1 = {};
      if (two) {
        g1 = __ldcs(g + j + kThreads);
        u1 = __ldcs(u + j + kThreads);
      }
      o[j] = silu_mul8<BF16>(g0, u0);
      if (two) o[j + kThreads] = silu_mul8<BF16>(g1, u1);
    }
  }
}

// Bound by memory: 3 bytes an element (8192 x 28672: 107 us, 6.6 TB/s).  A row stays in registers between the maximum and the
// rounding; a CTA takes it, or a warp (WARP: rows of up to 1024 elements), which then needs no barrier and no launch of a CTA for
// each row (16384 x 1024, whole calls on cold inputs: 23 -> 12 us; back to back it takes 7).
constexpr int kQuantizeThreads = 512, kQuantizeWarps = 8;

template <bool BF16, int VPT, bool WARP>
__global__ void __launch_bounds__(kQuantizeThreads)
    quantize_rows_kernel(const uint16_t* __restrict__ X, int8_t* __restrict__ Q, float* __restrict__ S, int rows, int dim) {
  __shared__ uint32_t red[kQuantizeThreads / 32];
  const int nvec = dim / 8, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = WARP ? static_cast<int>(blockIdx.x) * kQuantizeWarps + warp : static_cast<int>(blockIdx.x);
  const int first = WARP ? lane : static_cast<int>(threadIdx.x), step = WARP ? 32 : static_cast<int>(blockDim.x);
  const size_t base = static_cast<size_t>(row) * dim;
  const uint4* x = reinterpret_cast<const uint4*>(X + base);
  uint4 v[VPT];
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  if (WARP && row >= rows) return;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = first + i * step;
    v[i] = j < nvec ? __ldcs(x + j) : make_uint4(0, 0, 0, 0);
  }
  // magnitudes compare like their bits, and those of infinities and NaNs lie above all numbers
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) top = __vmaxu2(top, u[k] & 0x7fff7fffu);
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if (!WARP) {
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < static_cast<int>(blockDim.x >> 5) ? red[lane] : 0u);
  }
  const bool finite = top < (BF16 ? 0x7f80u : 0x7c00u);
  const float amax = fmaxf(unpack2<BF16>(top).x, 0x1p-100f);
  const float inv = __fdiv_rn(127.f, amax);
  if (first == 0) S[row] = finite ? __fdiv_rn(amax, 127.f) : __int_as_float(0x7fc00000);
  uint2* q = reinterpret_cast<uint2*>(Q + base);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = first + i * step;
    if (j < nvec) {
      const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t b[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2<BF16>(u[k]);
        // (at most 127 in magnitude: the quotient's rounding is less than half a step there)
        b[2 * k] = finite ? static_cast<uint32_t>(__float2int_rn(__fmul_rn(f.x, inv))) & 0xffu : 0u;
        b[2 * k + 1] = finite ? static_cast<uint32_t>(__float2int_rn(__fmul_rn(f.y, inv))) & 0xffu : 0u;
      }
      q[j] = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
    }
  }
}

template <bool BF16, int VPT, bool WARP>
cudaError_t launch_quantize(const uint16_t* x, int8_t* q, float* s, int rows, int dim, cudaStream_t stream) {
  const int nvec = dim / 8;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(WARP ? (rows - 1) / kQuantizeWarps + 1 : rows, 1, 1);
  cfg.blockDim = dim3(WARP ? 32 * kQuantizeWarps : ((nvec + VPT - 1) / VPT + 31) / 32 * 32, 1, 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, quantize_rows_kernel<BF16, VPT, WARP>, x, q, s, rows, dim);
  if (e != cudaSuccess) cudaGetLastError();  // reported to the caller, not left for the next one
  return e;
}

template <bool BF16>
cudaError_t quantize(const uint16_t* x, int8_t* q, float* s, int rows, int dim, cudaStream_t stream) {
  const int nvec = dim / 8;
  if (nvec <= 32) return launch_quantize<BF16, 1, true>(x, q, s, rows, dim, stream);
  if (nvec <= 128) return launch_quantize<BF16, 4, true>(x, q, s, rows, dim, stream);
  if (nvec <= kQuantizeThreads / 2) return launch_quantize<BF16, 1, false>(x, q, s, rows, dim, stream);
  if (nvec <= kQuantizeThreads) return launch_quantize<BF16, 2, false>(x, q, s, rows, dim, stream);
  if (nvec <= 2 * kQuantizeThreads) return launch_quantize<BF16, 4, false>(x, q, s, rows, dim, stream);
  return launch_quantize<BF16, 8, false>(x, q, s, rows, dim, stream);
}

}  // namespace

cudaError_t quantize_rows_launch(const void* X, void* Q, float* S, int rows, int dim, bool bf16, cudaStream_t stream) {
  if (dim < 8 || dim % 8 != 0 || dim > kMaxQuantizeDim) return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  const uint16_t* x = static_cast<const uint16_t*>(X);
  int8_t* q = static_cast<int8_t*>(Q);
  return bf16 ? quantize<true>(x, q, S, rows, dim, stream) : quantize<false>(x, q, S, rows, dim, stream);
}

cudaError_t rope_launch(void* QKV, int tokens, int seq, int heads, int head_dim, int row_elems, float theta, bool bf16,
                        cudaStream_t stream) {
  if (head_dim < 8 || head_dim % 8 != 0 || row_elems % 8 != 0 || seq < 1) return cudaErrorInvalidValue;
  if (tokens == 0 || heads == 0) return cudaSuccess;
  const int64_t threads = static_cast<int64_t>(tokens) * (head_dim / 8);
  const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads),
                  static_cast<unsigned>((heads + kHeadsPerThread - 1) / kHeadsPerThread));
  uint16_t* q = static_cast<uint16_t*>(QKV);
  if (bf16) {
    rope_kernel<true><<<grid, kThreads, 0, stream>>>(q, tokens, seq, heads, head_dim, row_elems, theta);
  } else {
    rope_kernel<false><<<grid, kThreads, 0, stream>>>(q, tokens, seq, heads, head_dim, row_elems, theta);
  }
  return cudaGetLastError();
}

cudaError_t swiglu_launch(const void* GU, void* Y, int rows, int f, bool bf16, int sm_count, cudaStream_t stream) {
  if (f % 8 != 0) return cudaErrorInvalidValue;
  if (rows == 0 || f == 0) return cudaSuccess;
  const int grid = rows < sm_count * 32 ? rows : sm_count * 32;
  const uint16_t* g = static_cast<const uint16_t*>(GU);
  uint16_t* y = static_cast<uint16_t*>(Y);
  if (bf16) {
    swiglu_kernel<true><<<grid, kThreads, 0, stream>>>(g, y, rows, f);
  } else {
    swiglu_kernel<false><<<grid, kThreads, 0, stream>>>(g, y, rows, f);
  }
  return cudaGetLastError();
}

}  // namespace fo
