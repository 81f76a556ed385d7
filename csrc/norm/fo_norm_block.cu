// The norms around a block of a decoder layer, in one pass over the rows, and their gradients:
//   u = T r1 PW,  r1 = 1 / sqrt(mean T^2 + eps);   H = alpha X + G u;   Y = H r2 W,  r2 = 1 / sqrt(mean H^2 + eps)
// Everything between the loads and the stores is fp32; H, Y and the gradients are rounded once, when they are stored.
// In particular the second norm takes H as it is, not as it is rounded for the residual stream: Y is then as
// exact as its type allows (rounding H first costs another 2^-9 of it in bf16), and the backward pass, which
// recomputes H from X and T, differentiates exactly what the forward pass computed.
#include "fo_norm_block.h"

#include <algorithm>
#include <cstdint>

#include "../common/fo_pack16.cuh"
#include "../common/fo_ptx.cuh"

namespace fo {

namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxDim = 16384;

struct Vec8 {
  float v[8];
};

template <bool BF16>
__device__ __forceinline__ Vec8 unpack8(const uint4& p) {
  Vec8 r;
  const uint32_t u[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = unpack2<BF16>(u[k]);
    r.v[2 * k] = f.x;
    r.v[2 * k + 1] = f.y;
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const Vec8& r) {
  return make_uint4(pack2<BF16>(r.v[0], r.v[1]), pack2<BF16>(r.v[2], r.v[3]), pack2<BF16>(r.v[4], r.v[5]),
                    pack2<BF16>(r.v[6], r.v[7]));
}

// Sum over the CTA, the same in every thread.  `red` alternates between two buffers, so one barrier per sum is
// enough: a warp writes a buffer again only behind the barrier of the sum in between, which every
// warp reaches after its reads of this one.
__device__ __forceinline__ float block_sum(float v, float (*red)[kMaxThreads / 32], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* r = red[turn];
  turn ^= 1;
  if (lane == 0) r[warp] = v;
  __syncthreads();
  float t = lane < warps ? r[lane] : 0.f;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return __shfl_sync(0xffffffffu, t, 0);
}

__device__ __forceinline__ uint4 ld_vec(const uint16_t* p, int j) { return __ldg(reinterpret_cast<const uint4*>(p) + j); }

// Bound by memory: 8 bytes an element.  A CTA takes a run of rows; a thread owns VPT vectors of a row and requests
// the next row's before it reduces this one's.
template <bool BF16, int VPT>
__global__ void __launch_bounds__(kMaxThreads, VPT <= 2 ? 2 : 1)
    norm_block_kernel(const uint16_t* __restrict__ X, const uint16_t* __restrict__ T, const uint16_t* __restrict__ PW,
                      const uint16_t* __restrict__ W, const uint16_t* __restrict__ G, uint16_t* __restrict__ H,
                      uint16_t* __restrict__ Y, float2* __restrict__ stats, int rows, int dim, int rows_per_line,
                      float alpha, float eps) {
  __shared__ float red[2][kMaxThreads / 32];
  int turn = 0;
  const int nvec = dim / 8;
  const int row_begin = static_cast<int>(static_cast<int64_t>(rows) * blockIdx.x / gridDim.x);
  const int row_end = static_cast<int>(static_cast<int64_t>(rows) * (blockIdx.x + 1) / gridDim.x);
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  uint4 x[VPT], t[VPT];
  auto load_row = [&](int b) {
    const size_t base = static_cast<size_t>(b) * dim;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * blockDim.x;
      if (j < nvec) {
        t[i] = __ldcs(reinterpret_cast<const uint4*>(T + base) + j);
        x[i] = __ldcs(reinterpret_cast<const uint4*>(X + base) + j);
      }
    }
  };
  if (row_begin < row_end) load_row(row_begin);
  for (int b = row_begin; b < row_end; ++b) {
    const size_t base = static_cast<size_t>(b) * dim;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (threadIdx.x + i * blockDim.x < nvec) {
        const Vec8 tv = unpack8<BF16>(t[i]);
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += tv.v[k] * tv.v[k];
      }
    }
    const float r1 = rsqrtf(block_sum(ss, red, turn) / static_cast<float>(dim) + eps);
    const uint16_t* g = G != nullptr ? G + static_cast<size_t>(b / rows_per_line) * dim : nullptr;
    Vec8 h[VPT];
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * blockDim.x;
      if (j < nvec) {
        const Vec8 tv = unpack8<BF16>(t[i]), xv = unpack8<BF16>(x[i]), pw = unpack8<BF16>(ld_vec(PW, j));
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i].v[k] = tv.v[k] * r1 * pw.v[k];
        if (g != nullptr) {
          const Vec8 gv = unpack8<BF16>(ld_vec(g, j));
#pragma unroll
          for (int k = 0; k < 8; ++k) h[i].v[k] *= gv.v[k];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          h[i].v[k] += alpha * xv.v[k];
          ss += h[i].v[k] * h[i].v[k];
        }
      }
    }
    if (b + 1 < row_end) load_row(b + 1);
    const float r2 = rsqrtf(block_sum(ss, red, turn) / static_cast<float>(dim) + eps);
    if (stats != nullptr && threadIdx.x == 0) stats[b] = make_float2(r1, r2);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = threadIdx.x + i * blockDim.x;
      if (j < nvec) {
        __stcs(reinterpret_cast<uint4*>(H + base) + j, pack8<BF16>(h[i]));
        const Vec8 w = unpack8<BF16>(ld_vec(W, j));
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i].v[k] = h[i].v[k] * r2 * w.v[k];
        __stcs(reinterpret_cast<uint4*>(Y + base) + j, pack8<BF16>(h[i]));
      }
    }
  }
}

// Column sums a thread keeps over its rows: in registers, or, for rows that leave none, in shared memory (each
// thread its own words: no barrier).
template <int VPT, bool SHARED>
struct ColumnSum {
  Vec8 r[SHARED ? 1 : VPT];
  float4* s;
  __device__ __forceinline__ void init(float4* smem) {
    s = smem + threadIdx.x;
    clear();
  }
  __device__ __forceinline__ float4* at(int i, int half) const { return s + (2 * i + half) * kMaxThreads; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if constexpr (SHARED) {
        *at(i, 0) = *at(i, 1) = make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) r[i].v[k] = 0.f;
      }
    }
  }
  __device__ __forceinline__ void add(int i, const Vec8& a) {
    if constexpr (SHARED) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float4 w = *at(i, half);
        w.x += a.v[4 * half];
        w.y += a.v[4 * half + 1];
        w.z += a.v[4 * half + 2];
        w.w += a.v[4 * half + 3];
        *at(i, half) = w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) r[i].v[k] += a.v[k];
    }
  }
  __device__ __forceinline__ Vec8 get(int i) const {
    if constexpr (SHARED) {
      const float4 a = *at(i, 0), b = *at(i, 1);
      return Vec8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    } else {
      return r[i];
    }
  }
};

__device__ __forceinline__ void store_sum(float* dst, int j, const Vec8& a) {
  float4* d = reinterpret_cast<float4*>(dst) + 2 * j;
  d[0] = make_float4(a.v[0], a.v[1], a.v[2], a.v[3]);
  d[1] = make_float4(a.v[4], a.v[5], a.v[6], a.v[7]);
}

struct BackwardArgs {
  const uint16_t *X, *T, *PW, *W, *G, *GH, *GY;
  const float2* stats;
  uint16_t *DX, *DT, *DG;  // DG: gradients of whole lines, when chunks == 1
  float *sum_pw, *sum_w;   // [gridDim.x][dim]
  float* sum_g;            // [lines * chunks][dim], when chunks > 1
  int rows, dim, lines, chunks;
  float alpha;
};

// n1 = T r1, n2 = H r2:  dH = GH + r2 (GY W - n2 mean(GY W n2)),  dX = alpha dH,  b = dH G PW,
// dT = r1 (b - n1 mean(b n1)),  dPW = sum dH G n1,  dW = sum GY n2,  dG = sum over the line's rows of dH n1 PW.
// 12 bytes an element; two sums over the row follow one another.  Column sums stay in registers over a CTA's rows and
// are added up over the CTAs by column_sum_kernel, in a fixed order.
template <bool BF16, int VPT, bool GATE>
__global__ void __launch_bounds__(kMaxThreads, 1) norm_block_backward_kernel(const __grid_constant__ BackwardArgs p) {
  constexpr bool kShared = VPT > 2;
  extern __shared__ float4 sums[];
  __shared__ float red[2][kMaxThreads / 32];
  int turn = 0;
  const int dim = p.dim, nvec = dim / 8;
  const float inv_dim = 1.f / static_cast<float>(dim);
  ColumnSum<VPT, kShared> acc_pw, acc_w, acc_g;
  acc_pw.init(sums);
  acc_w.init(sums + 2 * VPT * kMaxThreads);
  if constexpr (GATE) acc_g.init(sums + 4 * VPT * kMaxThreads);
  const int64_t units = static_cast<int64_t>(p.lines) * p.chunks;
  const int unit_begin = static_cast<int>(units * blockIdx.x / gridDim.x);
  const int unit_end = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
  const int rows_per_line = p.rows / p.lines;
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int unit = unit_begin; unit < unit_end; ++unit) {
    const int line = unit / p.chunks, chunk = unit - line * p.chunks;
    const int row_begin = line * rows_per_line + static_cast<int>(static_cast<int64_t>(rows_per_line) * chunk / p.chunks);
    const int row_end = line * rows_per_line + static_cast<int>(static_cast<int64_t>(rows_per_line) * (chunk + 1) / p.chunks);
    [[maybe_unused]] const uint16_t* g = p.G + static_cast<size_t>(line) * dim;
    uint4 x[VPT], t[VPT], gh[VPT], gy[VPT];
    auto load_row = [&](int b) {
      const size_t base = static_cast<size_t>(b) * dim;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = threadIdx.x + i * blockDim.x;
        if (j < nvec) {
          x[i] = __ldcs(reinterpret_cast<const uint4*>(p.X + base) + j);
          t[i] = __ldcs(reinterpret_cast<const uint4*>(p.T + base) + j);
          gy[i] = p.GY != nullptr ? __ldcs(reinterpret_cast<const uint4*>(p.GY + base) + j) : zero;
          gh[i] = p.GH != nullptr ? __ldcs(reinterpret_cast<const uint4*>(p.GH + base) + j) : zero;
        }
      }
    };
    for (int b = row_begin; b < row_end; ++b) {
      load_row(b);
      const float2 st = p.stats[b];
      const float r1 = st.x, r2 = st.y;
      const size_t base = static_cast<size_t>(b) * dim;
      float s = 0.f;
      Vec8 n2[VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = threadIdx.x + i * blockDim.x;
        if (j < nvec) {
          const Vec8 tv = unpack8<BF16>(t[i]), xv = unpack8<BF16>(x[i]), gyv = unpack8<BF16>(gy[i]);
          const Vec8 pw = unpack8<BF16>(ld_vec(p.PW, j)), w = unpack8<BF16>(ld_vec(p.W, j));
          Vec8 u;
#pragma unroll
          for (int k = 0; k < 8; ++k) u.v[k] = tv.v[k] * r1 * pw.v[k];
          if constexpr (GATE) {
            const Vec8 gv = unpack8<BF16>(ld_vec(g, j));
#pragma unroll
            for (int k = 0; k < 8; ++k) u.v[k] *= gv.v[k];
          }
          Vec8 dw;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            n2[i].v[k] = (u.v[k] + p.alpha * xv.v[k]) * r2;
            dw.v[k] = gyv.v[k] * n2[i].v[k];
            s += dw.v[k] * w.v[k];
          }
          acc_w.add(i, dw);
        }
      }
      const float c2 = block_sum(s, red, turn) * inv_dim;
      s = 0.f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = threadIdx.x + i * blockDim.x;
        if (j < nvec) {
          const Vec8 tv = unpack8<BF16>(t[i]), gyv = unpack8<BF16>(gy[i]), ghv = unpack8<BF16>(gh[i]);
          const Vec8 pw = unpack8<BF16>(ld_vec(p.PW, j)), w = unpack8<BF16>(ld_vec(p.W, j));
          Vec8 dh, dx, dpw;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            dh.v[k] = ghv.v[k] + r2 * (gyv.v[k] * w.v[k] - n2[i].v[k] * c2);
            dx.v[k] = p.alpha * dh.v[k];
          }
          __stcs(reinterpret_cast<uint4*>(p.DX + base) + j, pack8<BF16>(dx));
#pragma unroll
          for (int k = 0; k < 8; ++k) dpw.v[k] = dh.v[k] * (tv.v[k] * r1);
          if constexpr (GATE) {
            const Vec8 gv = unpack8<BF16>(ld_vec(g, j));
            Vec8 dg;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              dg.v[k] = dpw.v[k] * pw.v[k];
              dpw.v[k] *= gv.v[k];
              dh.v[k] *= gv.v[k];
            }
            acc_g.add(i, dg);
          }
          acc_pw.add(i, dpw);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            n2[i].v[k] = dh.v[k] * pw.v[k];  // b
            s += dpw.v[k] * pw.v[k];         // b n1
          }
        }
      }
      const float c1 = block_sum(s, red, turn) * inv_dim;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = threadIdx.x + i * blockDim.x;
        if (j < nvec) {
          const Vec8 tv = unpack8<BF16>(t[i]);
          Vec8 dt;
#pragma unroll
          for (int k = 0; k < 8; ++k) dt.v[k] = r1 * (n2[i].v[k] - tv.v[k] * r1 * c1);
          __stcs(reinterpret_cast<uint4*>(p.DT + base) + j, pack8<BF16>(dt));
        }
      }
    }
    if constexpr (GATE) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = threadIdx.x + i * blockDim.x;
        if (j < nvec) {
          if (p.chunks == 1) {
            __stcs(reinterpret_cast<uint4*>(p.DG + static_cast<size_t>(unit) * dim) + j, pack8<BF16>(acc_g.get(i)));
          } else {
            store_sum(p.sum_g + static_cast<size_t>(unit) * dim, j, acc_g.get(i));
          }
        }
      }
      acc_g.clear();
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = threadIdx.x + i * blockDim.x;
    if (j < nvec) {
      store_sum(p.sum_pw + static_cast<size_t>(blockIdx.x) * dim, j, acc_pw.get(i));
      store_sum(p.sum_w + static_cast<size_t>(blockIdx.x) * dim, j, acc_w.get(i));
    }
  }
}

struct ColumnJob {
  const float* src;  // [lines][count][dim]
  uint16_t* dst;     // [lines][dim]
  int lines, count;
};
struct ColumnJobs {
  ColumnJob job[3];
  int dim;
};

// dst[l, j] = round16(sum over c of src[l, c, j]): 128 columns and one line per CTA, eight runs of c added in order.
template <bool BF16>
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ ColumnJobs p) {
  __shared__ float4 part[8][32];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  int line = blockIdx.y, which = 0;
  while (line >= p.job[which].lines) line -= p.job[which++].lines;
  const ColumnJob job = p.job[which];
  const int col = (blockIdx.x * 32 + lane) * 4;
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < p.dim) {
    const float* src = job.src + static_cast<size_t>(line) * job.count * p.dim + col;
#pragma unroll 8
    for (int c = y; c < job.count; c += 8) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src + static_cast<size_t>(c) * p.dim));
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
  }
  part[y][lane] = s;
  __syncthreads();
  if (y == 0 && col < p.dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      const float4 v = part[i][lane];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    *reinterpret_cast<uint2*>(job.dst + static_cast<size_t>(line) * p.dim + col) =
        make_uint2(pack2<BF16>(s.x, s.y), pack2<BF16>(s.z, s.w));
  }
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) cudaGetLastError();  // reported to the caller, not left for the next one
  return e;
}

int threads_for(int nvec, int vpt) { return std::min(kMaxThreads, ((nvec + vpt - 1) / vpt + 31) / 32 * 32); }

template <bool BF16, int VPT>
cudaError_t launch_forward(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream) {
  const int threads = threads_for(p.dim / 8, VPT);
  const int grid = std::min(p.rows, sm_count * 8 * (kMaxThreads / threads));
  return launch(norm_block_kernel<BF16, VPT>, dim3(grid), threads, 0, stream, static_cast<const uint16_t*>(p.X),
                static_cast<const uint16_t*>(p.T), static_cast<const uint16_t*>(p.PW), static_cast<const uint16_t*>(p.W),
                static_cast<const uint16_t*>(p.G), static_cast<uint16_t*>(H), static_cast<uint16_t*>(Y),
                reinterpret_cast<float2*>(stats), p.rows, p.dim, p.rows / p.lines, p.alpha, p.eps);
}

template <bool BF16>
cudaError_t forward(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream) {
  const int nvec = p.dim / 8;
  if (nvec <= kMaxThreads) return launch_forward<BF16, 1>(p, H, Y, stats, sm_count, stream);
  if (nvec <= 2 * kMaxThreads) return launch_forward<BF16, 2>(p, H, Y, stats, sm_count, stream);
  return launch_forward<BF16, 4>(p, H, Y, stats, sm_count, stream);
}

int backward_vpt(int dim) { return dim / 8 <= kMaxThreads / 2 ? 1 : (dim / 8 <= 2 * kMaxThreads ? 2 : 4); }

template <bool BF16, int VPT, bool GATE>
cudaError_t launch_backward(const BackwardArgs& a, int ctas, cudaStream_t stream) {
  auto kernel = norm_block_backward_kernel<BF16, VPT, GATE>;
  const int smem = VPT > 2 ? (GATE ? 6 : 4) * VPT * kMaxThreads * static_cast<int>(sizeof(float4)) : 0;
  if (smem > 0) {
    static bool set[16] = {};  // the same whoever sets it
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 16 || !set[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      if (dev >= 0 && dev < 16) set[dev] = true;
    }
  }
  return launch(kernel, dim3(ctas), threads_for(a.dim / 8, VPT), smem, stream, a);
}

template <bool BF16>
cudaError_t backward(const BackwardArgs& a, bool gate, int ctas, cudaStream_t stream) {
  switch (backward_vpt(a.dim)) {
    case 1: return gate ? launch_backward<BF16, 1, true>(a, ctas, stream) : launch_backward<BF16, 1, false>(a, ctas, stream);
    case 2: return gate ? launch_backward<BF16, 2, true>(a, ctas, stream) : launch_backward<BF16, 2, false>(a, ctas, stream);
    default: return gate ? launch_backward<BF16, 4, true>(a, ctas, stream) : launch_backward<BF16, 4, false>(a, ctas, stream);
  }
}

bool valid(const NormBlock& p) {
  return p.dim >= 8 && p.dim % 8 == 0 && p.dim <= kMaxDim && p.rows >= 1 && p.lines >= 1 && p.rows % p.lines == 0;
}

}  // namespace

cudaError_t norm_block_launch(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream) {
  if (!valid(p)) return cudaErrorInvalidValue;
  return p.bf16 ? forward<true>(p, H, Y, stats, sm_count, stream) : forward<false>(p, H, Y, stats, sm_count, stream);
}

NormBlockPlan norm_block_plan(const NormBlock& p, int sm_count) {
  NormBlockPlan plan;
  const int threads = threads_for(p.dim / 8, backward_vpt(p.dim));
  const int most = sm_count * std::min(8, kMaxThreads / threads);
  if (p.G == nullptr || p.lines == 1) {
    plan.ctas = plan.chunks = std::min(p.rows, most);
  } else {
    // several runs per CTA, so that uneven numbers of them matter little, but of eight rows at least
    plan.chunks = std::max(1, std::min((4 * most + p.lines - 1) / p.lines, p.rows / p.lines / 8));
    plan.ctas = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(p.lines) * plan.chunks, most));
  }
  plan.workspace = static_cast<size_t>(2) * plan.ctas * p.dim;
  if (p.G != nullptr && plan.chunks > 1) plan.workspace += static_cast<size_t>(p.lines) * plan.chunks * p.dim;
  return plan;
}

cudaError_t norm_block_backward_launch(const NormBlock& p, const float* stats, const void* GH, const void* GY, void* DX,
                                       void* DT, void* DPW, void* DW, void* DG, float* workspace,
                                       const NormBlockPlan& plan, cudaStream_t stream) {
  if (!valid(p)) return cudaErrorInvalidValue;
  const bool gate = p.G != nullptr;
  BackwardArgs a;
  a.X = static_cast<const uint16_t*>(p.X);
  a.T = static_cast<const uint16_t*>(p.T);
  a.PW = static_cast<const uint16_t*>(p.PW);
  a.W = static_cast<const uint16_t*>(p.W);
  a.G = static_cast<const uint16_t*>(p.G);
  a.GH = static_cast<const uint16_t*>(GH);
  a.GY = static_cast<const uint16_t*>(GY);
  a.stats = reinterpret_cast<const float2*>(stats);
  a.DX = static_cast<uint16_t*>(DX);
  a.DT = static_cast<uint16_t*>(DT);
  a.DG = static_cast<uint16_t*>(DG);
  a.sum_pw = workspace;
  a.sum_w = a.sum_pw + static_cast<size_t>(plan.ctas) * p.dim;
  a.sum_g = a.sum_w + static_cast<size_t>(plan.ctas) * p.dim;
  a.rows = p.rows;
  a.dim = p.dim;
  a.lines = gate ? p.lines : 1;
  a.chunks = plan.chunks;
  a.alpha = p.alpha;
  cudaError_t e = p.bf16 ? backward<true>(a, gate, plan.ctas, stream) : backward<false>(a, gate, plan.ctas, stream);
  if (e != cudaSuccess) return e;
  ColumnJobs jobs;
  jobs.dim = p.dim;
  jobs.job[0] = {a.sum_pw, static_cast<uint16_t*>(DPW), 1, plan.ctas};
  jobs.job[1] = {a.sum_w, static_cast<uint16_t*>(DW), 1, plan.ctas};
  jobs.job[2] = {a.sum_g, a.DG, gate && plan.chunks > 1 ? p.lines : 0, plan.chunks};
  const dim3 grid((p.dim + 127) / 128, 2 + jobs.job[2].lines);
  return p.bf16 ? launch(column_sum_kernel<true>, grid, 256, 0, stream, jobs)
                : launch(column_sum_kernel<false>, grid, 256, 0, stream, jobs);
}

}  // namespace fo
