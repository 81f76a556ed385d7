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

// Eight elements in fp32, as four pairs, whose products and sums are one instruction each on sm_100 (f32x2): 84 instead of 101 million
// warp instructions for the backward pass of 8192 x 8192 (no less time: it is the latencies that count).
struct Vec8 {
  float2 v[4];
};

__device__ __forceinline__ float2 f2(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 operator*(const float2& a, const float2& b) { return __fmul2_rn(a, b); }
// a * b + c
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) { return __ffma2_rn(a, b, c); }

template <bool BF16>
__device__ __forceinline__ Vec8 unpack8(const uint4& p) {
  if constexpr (BF16) {  // a bf16 is the upper half of an fp32
    const uint32_t u[4] = {p.x, p.y, p.z, p.w};
    Vec8 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r.v[k] = make_float2(__uint_as_float(u[k] << 16), __uint_as_float(u[k] & 0xffff0000u));
    return r;
  } else {
    return Vec8{{unpack2<BF16>(p.x), unpack2<BF16>(p.y), unpack2<BF16>(p.z), unpack2<BF16>(p.w)}};
  }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const Vec8& r) {
  return make_uint4(pack2<BF16>(r.v[0].x, r.v[0].y), pack2<BF16>(r.v[1].x, r.v[1].y), pack2<BF16>(r.v[2].x, r.v[2].y),
                    pack2<BF16>(r.v[3].x, r.v[3].y));
}

// A row of up to kCtaDim elements is one CTA's, a longer one is shared by a cluster of two, the first taking kCtaDim of
// it: the registers and the shared memory of one SM hold no more (16384 elements in one CTA leave the backward pass no room to
// load ahead: 4096 rows took 264 us, in clusters 167).  Sharing shorter rows too loses: 8192 x 8192 forward 94 -> 112 us.
constexpr int kCtaDim = 8192;

// Four sums over a row's threads, the same in all of them and added in a fixed order.  One barrier: `red` alternates between two
// buffers, and a warp writes a buffer again only behind the barrier of the sums in between, which every warp reaches after
// its reads of this one.  In a cluster every warp leaves its part in both CTAs.
template <int CTAS>
__device__ __forceinline__ float4 row_sums(const float4& v, float (*red)[128], int& turn) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // each lane ends up with one of the four, number lane & 3: two exchanges of halves, then sums over the other lanes
  const bool b0 = lane & 1, b1 = lane & 2;
  const float a = (b0 ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, b0 ? v.x : v.y, 1);
  const float b = (b0 ? v.w : v.z) + __shfl_xor_sync(0xffffffffu, b0 ? v.z : v.w, 1);
  float t = (b1 ? b : a) + __shfl_xor_sync(0xffffffffu, b1 ? a : b, 2);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (CTAS > 1 || warps > 1) {
    float* r = red[turn];
    turn ^= 1;
    if constexpr (CTAS == 1) {
      if (lane < 4) r[4 * warp + lane] = t;
      __syncthreads();
    } else {
      const uint32_t at = (static_cast<uint32_t>(ptx::cluster_ctarank()) * 16 + warp) * 4 + (lane & 3);
      if (lane < 4 * CTAS) ptx::st_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(r + at), lane >> 2), __float_as_uint(t));
      __syncwarp();
      ptx::cluster_arrive_release();
      ptx::cluster_wait_acquire();
    }
    t = 0.f;
#pragma unroll
    for (int i = 0; i < (CTAS == 1 ? 2 : 4); ++i) {
      if (CTAS > 1 || lane + 32 * i < 4 * warps) t += r[lane + 32 * i];
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  return make_float4(__shfl_sync(0xffffffffu, t, 0), __shfl_sync(0xffffffffu, t, 1), __shfl_sync(0xffffffffu, t, 2),
                     __shfl_sync(0xffffffffu, t, 3));
}

// Kernels that follow one another closely (ptx::grid_wait) begin before their inputs are written, so no load of an input goes the
// read-only way (ld.global.nc, which __ldg and const __restrict__ pointers are compiled to): it is for data that nobody writes while
// the kernel exists.
__device__ __forceinline__ uint4 ld_vec(const uint16_t* p) { return __ldca(reinterpret_cast<const uint4*>(p)); }

// The rows a thread reads come through a ring in shared memory that it fills with asynchronous copies, STAGES - 1 rows
// ahead.  Every thread copies and reads words of its own only, so the ring needs no barrier, and the loads in
// flight take no registers.
template <int VPT, int ARRAYS, int STAGES>
struct RowRing {
  uint32_t base;  // this thread's first word
  __device__ __forceinline__ explicit RowRing(const uint4* smem) : base(ptx::smem_u32(smem + threadIdx.x)) {}
  __device__ __forceinline__ uint32_t at(int stage, int array, int i) const {
    return base + ((stage * ARRAYS + array) * VPT + i) * blockDim.x * 16;
  }
  __device__ __forceinline__ void fill(int stage, int array, int i, const uint16_t* src) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(stage, array, i)), "l"(src) : "memory");
  }
  __device__ __forceinline__ uint4 get(int stage, int array, int i) const {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at(stage, array, i)) : "memory");
    return v;
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // the oldest of STAGES groups has landed
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
  static constexpr int kStages = STAGES;
  static constexpr int kBytesPerThread = STAGES * ARRAYS * VPT * 16;
};

// Where the gate comes from: a line that lasts kMinLineRows rows or more is read when it begins, shorter ones (a line for
// each row above all) come through the ring like the rows.
enum Gate { kNoGate, kLineGate, kRowGate };
constexpr int kMinLineRows = 8;

template <int VPT, int GATE>
using ForwardRing = RowRing<VPT, GATE == kRowGate ? 3 : 2, 3>;
// three stages, two where the gate takes the third's place
template <int VPT, int GATE>
using BackwardRing = RowRing<VPT, GATE == kRowGate ? 5 : 4, GATE == kRowGate ? 2 : 3>;

// The vectors of a row that a thread owns: number i starts at element first + i * step, and is there if first + i * step < dim.
struct Columns {
  int first, step;
};
template <int CTAS>
__device__ __forceinline__ Columns my_columns() {
  const int cta = CTAS == 1 ? 0 : static_cast<int>(ptx::cluster_ctarank()) * kCtaDim;
  return Columns{cta + static_cast<int>(threadIdx.x) * 8, static_cast<int>(blockDim.x) * 8};
}

// Rows (whole lines of the gate if those are short) are dealt out evenly: CTA or cluster `at` of `of` takes the ones from
// here to the next one's first.
__host__ __device__ __forceinline__ int first_row_of(int at, int of, int rows) {
  return static_cast<int>(static_cast<int64_t>(rows) * at / of);
}
__device__ __forceinline__ int owner_of_row(int row, int of, int rows) {
  return static_cast<int>(((static_cast<int64_t>(row) + 1) * of - 1) / rows);
}

// Bound by memory: 8 bytes an element.  A CTA takes a run of rows; a thread owns VPT vectors of a row, and what it needs of the
// weights and of the gate's line stays in its registers: beside the ring there is little L1, and rows that fetched them again
// from the L2 waited for them (8192 x 4096: 57 -> 48 us; 16384 x 1024, cold: 33 -> 27 us; 16384 x 8192 no difference: 177 us,
// 6.1 TB/s).  Rows of one vector a thread leave registers for two sets of CTAs.
template <bool BF16, int VPT, int CTAS, int GATE>
__global__ void __launch_bounds__(kMaxThreads, 1)
    norm_block_kernel(const uint16_t* __restrict__ X, const uint16_t* __restrict__ T, const uint16_t* __restrict__ PW,
                      const uint16_t* __restrict__ W, const uint16_t* __restrict__ G, uint16_t* __restrict__ H,
                      uint16_t* __restrict__ Y, float2* __restrict__ stats, int rows, int dim, int rows_per_line,
                      float alpha, float eps) {
  extern __shared__ uint4 ring_words[];
  __shared__ float red[2][128];
  using Ring = ForwardRing<VPT, GATE>;
  constexpr int kStages = Ring::kStages;
  const Ring ring(ring_words);
  int turn = 0;
  const Columns c = my_columns<CTAS>();
  const int at = blockIdx.x / CTAS, of = gridDim.x / CTAS;
  const int row_begin = first_row_of(at, of, rows), row_end = first_row_of(at + 1, of, rows);
  const float inv_dim = 1.f / static_cast<float>(dim);
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  auto fill = [&](int stage, int b) {
    if (b < row_end) {
      const size_t row = static_cast<size_t>(b) * dim + c.first;
      [[maybe_unused]] const uint16_t* g =
          GATE == kRowGate ? G + static_cast<size_t>(b / rows_per_line) * dim + c.first : nullptr;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (c.first + i * c.step < dim) {
          ring.fill(stage, 0, i, T + row + i * c.step);
          ring.fill(stage, 1, i, X + row + i * c.step);
          if constexpr (GATE == kRowGate) ring.fill(stage, 2, i, g + i * c.step);
        }
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fill(s, row_begin + s);
  if constexpr (CTAS > 1) {  // the other CTA runs before anything is stored into its shared memory
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait_acquire();
  }
  int stage = 0;
  [[maybe_unused]] int line = row_begin / rows_per_line;
  [[maybe_unused]] int line_left = (line + 1) * rows_per_line - row_begin;  // rows of the gate's line that are left
  Vec8 pg[VPT];
  uint4 w16[VPT], pw16[VPT];
  auto load_line = [&]() {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        pg[i] = unpack8<BF16>(ld_vec(PW + c.first + i * c.step));
        if constexpr (GATE == kLineGate) {
          const Vec8 g = unpack8<BF16>(ld_vec(G + static_cast<size_t>(line) * dim + c.first + i * c.step));
#pragma unroll
          for (int k = 0; k < 4; ++k) pg[i].v[k] = pg[i].v[k] * g.v[k];
        }
      }
    }
  };
  if constexpr (GATE != kRowGate) load_line();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (c.first + i * c.step < dim) {
      w16[i] = ld_vec(W + c.first + i * c.step);
      if constexpr (GATE == kRowGate) pw16[i] = ld_vec(PW + c.first + i * c.step);
    }
  }
  for (int b = row_begin; b < row_end; ++b) {
    const size_t row = static_cast<size_t>(b) * dim + c.first;
    ring.wait();
    // With q = T PW G, H = alpha X + r1 q, and its sum of squares follows from three sums that do not wait for r1: one
    // exchange between the warps a row instead of two.
    auto post_gate = [&](int i) {  // PW G
      if constexpr (GATE == kRowGate) {
        Vec8 v = unpack8<BF16>(pw16[i]);
        const Vec8 g = unpack8<BF16>(ring.get(stage, 2, i));
#pragma unroll
        for (int k = 0; k < 4; ++k) v.v[k] = v.v[k] * g.v[k];
        return v;
      } else {
        return pg[i];
      }
    };
    Vec8 h[VPT];  // q, then H
    float2 tt = f2(0.f), xx = f2(0.f), xq = f2(0.f), qq = f2(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        const Vec8 t = unpack8<BF16>(ring.get(stage, 0, i)), x = unpack8<BF16>(ring.get(stage, 1, i));
        h[i] = post_gate(i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[i].v[k] = h[i].v[k] * t.v[k];
          tt = fma2(t.v[k], t.v[k], tt);
          xx = fma2(x.v[k], x.v[k], xx);
          xq = fma2(x.v[k], h[i].v[k], xq);
          qq = fma2(h[i].v[k], h[i].v[k], qq);
        }
      }
    }
    const float4 sums = row_sums<CTAS>(make_float4(tt.x + tt.y, xx.x + xx.y, xq.x + xq.y, qq.x + qq.y), red, turn);
    const float r1 = rsqrtf(sums.x * inv_dim + eps);
    const float apart = alpha * alpha * sums.y + r1 * r1 * sums.w;
    float hh = apart + 2.f * alpha * r1 * sums.z;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        const Vec8 x = unpack8<BF16>(ring.get(stage, 1, i));
#pragma unroll
        for (int k = 0; k < 4; ++k) h[i].v[k] = fma2(f2(alpha), x.v[k], h[i].v[k] * f2(r1));
      }
    }
    if (!(hh >= 0.25f * apart && apart < __int_as_float(0x7f800000))) {
      // the two parts cancel, or q, which r1 has not scaled yet, is too large to be squared: H in the order of its definition,
      // and a sum of its own
      float2 ss = f2(0.f);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (c.first + i * c.step < dim) {
          const Vec8 t = unpack8<BF16>(ring.get(stage, 0, i)), x = unpack8<BF16>(ring.get(stage, 1, i));
          h[i] = post_gate(i);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            h[i].v[k] = fma2(f2(alpha), x.v[k], t.v[k] * f2(r1) * h[i].v[k]);
            ss = fma2(h[i].v[k], h[i].v[k], ss);
          }
        }
      }
      hh = row_sums<CTAS>(make_float4(ss.x + ss.y, 0.f, 0.f, 0.f), red, turn).x;
    }
    fill(stage, b + kStages);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if constexpr (GATE == kLineGate) {
      if (--line_left == 0) {
        ++line;
        line_left = rows_per_line;
        if (b + 1 < row_end) load_line();
      }
    }
    const float2 r2 = f2(rsqrtf(hh * inv_dim + eps));
    if (stats != nullptr && c.first == 0) stats[b] = make_float2(r1, r2.x);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        __stcs(reinterpret_cast<uint4*>(H + row + i * c.step), pack8<BF16>(h[i]));
        const Vec8 w = unpack8<BF16>(w16[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[i].v[k] = h[i].v[k] * r2 * w.v[k];
        __stcs(reinterpret_cast<uint4*>(Y + row + i * c.step), pack8<BF16>(h[i]));
      }
    }
  }
}

__device__ __forceinline__ void store_sum(float* dst, const Vec8& a) {
  float4* d = reinterpret_cast<float4*>(dst);
  d[0] = make_float4(a.v[0].x, a.v[0].y, a.v[1].x, a.v[1].y);
  d[1] = make_float4(a.v[2].x, a.v[2].y, a.v[3].x, a.v[3].y);
}

struct BackwardArgs {
  const uint16_t *X, *T, *PW, *W, *G, *GH, *GY;
  const float2* stats;
  uint16_t *DX, *DT, *DG;  // DG: gradients of lines that are one CTA's
  float *sum_pw, *sum_w;   // [CTAs or clusters][dim]
  float* sum_g;            // [CTAs or clusters][2][dim]: parts of lines that several of them share, first of the one
                           // that was begun before the CTA's rows or with them, then of the one that begins among them
  int rows, dim, lines;
  float alpha;
};

// n1 = T r1, n2 = H r2:  dH = GH + r2 (GY W - n2 mean(GY W n2)),  dX = alpha dH,  b = dH G PW,
// dT = r1 (b - n1 mean(b n1)),  dW = sum GY n2,  and with m = dH n1 summed over the rows of a line of the gate,
// dG = PW sum m,  dPW = sum over the lines of G sum m: one column sum a row serves both.
// 12 bytes an element: 8192 x 8192 145 us (5.5 TB/s), 16384 x 8192 without a gate 271 us with the sums (5.9 TB/s).  Bound by memory, and by the
// latencies of 16 warps an SM, all that the column sums' registers leave.  Column sums stay in registers over a CTA's rows and are
// added up over the CTAs by the two kernels below, in a fixed order (6 us behind this kernel; 11 us cold, by itself under a profiler).
template <bool BF16, int VPT, int CTAS, int GATE>
__global__ void __launch_bounds__(kMaxThreads, 1) norm_block_backward_kernel(const __grid_constant__ BackwardArgs p) {
  extern __shared__ uint4 ring_words[];
  __shared__ float red[2][128];
  enum { kT, kX, kGY, kGH, kG };
  using Ring = BackwardRing<VPT, GATE>;
  constexpr int kStages = Ring::kStages;
  const Ring ring(ring_words);
  // gate of short lines: this thread's words of the sum for PW, [VPT][2][threads] x 16 bytes behind the ring
  [[maybe_unused]] float4* sum_pw = reinterpret_cast<float4*>(ring_words) + blockDim.x * (Ring::kBytesPerThread / 16) + threadIdx.x;
  int turn = 0;
  const int dim = p.dim;
  const Columns c = my_columns<CTAS>();
  const float inv_dim = 1.f / static_cast<float>(dim);
  Vec8 acc_m[VPT], acc_w[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) acc_m[i].v[k] = acc_w[i].v[k] = f2(0.f);
    if constexpr (GATE == kRowGate) sum_pw[2 * i * blockDim.x] = sum_pw[(2 * i + 1) * blockDim.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int at = blockIdx.x / CTAS, of = gridDim.x / CTAS;
  const int rows_per_line = p.rows / p.lines;
  const int row_begin = GATE == kRowGate ? first_row_of(at, of, p.lines) * rows_per_line : first_row_of(at, of, p.rows);
  const int row_end = GATE == kRowGate ? first_row_of(at + 1, of, p.lines) * rows_per_line : first_row_of(at + 1, of, p.rows);
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  auto fill = [&](int stage, int b) {
    if (b < row_end) {
      const size_t row = static_cast<size_t>(b) * dim + c.first;
      [[maybe_unused]] const uint16_t* g =
          GATE == kRowGate ? p.G + static_cast<size_t>(b / rows_per_line) * dim + c.first : nullptr;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (c.first + i * c.step < dim) {
          if constexpr (GATE == kRowGate) ring.fill(stage, kG, i, g + i * c.step);
          ring.fill(stage, kT, i, p.T + row + i * c.step);
          ring.fill(stage, kX, i, p.X + row + i * c.step);
          if (p.GY != nullptr) ring.fill(stage, kGY, i, p.GY + row + i * c.step);
          if (p.GH != nullptr) ring.fill(stage, kGH, i, p.GH + row + i * c.step);
        }
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fill(s, row_begin + s);
  if constexpr (CTAS > 1) {  // the other CTA runs before anything is stored into its shared memory
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait_acquire();
  }
  const uint4 zero = make_uint4(0, 0, 0, 0);
  int stage = 0;
  [[maybe_unused]] int line = row_begin / rows_per_line;
  [[maybe_unused]] int line_end = min(row_end, (line + 1) * rows_per_line);  // of the rows that are this CTA's
  const uint16_t* g_line = GATE == kLineGate ? p.G + static_cast<size_t>(line) * dim + c.first : nullptr;
  Vec8 pg[VPT];
  uint4 w16[VPT];
  [[maybe_unused]] uint4 pw16[VPT];
  auto load_line = [&]() {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        pg[i] = unpack8<BF16>(ld_vec(p.PW + c.first + i * c.step));
        if constexpr (GATE == kLineGate) {
          const Vec8 g = unpack8<BF16>(ld_vec(g_line + i * c.step));
#pragma unroll
          for (int k = 0; k < 4; ++k) pg[i].v[k] = pg[i].v[k] * g.v[k];
        }
      }
    }
  };
  if constexpr (GATE != kRowGate) load_line();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (c.first + i * c.step < dim) {
      w16[i] = ld_vec(p.W + c.first + i * c.step);
      if constexpr (GATE == kRowGate) pw16[i] = ld_vec(p.PW + c.first + i * c.step);
    }
  }
  float2 next_stats = row_begin < row_end ? __ldca(p.stats + row_begin) : f2(0.f);
  for (int b = row_begin; b < row_end; ++b) {
    const float2 r1 = f2(next_stats.x), r2 = f2(next_stats.y);
    if (b + 1 < row_end) next_stats = __ldca(p.stats + b + 1);
    const size_t row = static_cast<size_t>(b) * dim + c.first;
    ring.wait();
    // s0 = sum GY W n2.  With u = n1 G PW the other mean, sum b n1, is sum GH u + r2 (sum GY W u - s0 / dim sum n2 u): all
    // four sums before any of the means is known, and so one exchange between the warps a row instead of two.
    float2 s0 = f2(0.f), s1 = f2(0.f), s2 = f2(0.f), s3 = f2(0.f);
    Vec8 n2[VPT], v[VPT];  // v: GY W
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        const Vec8 x = unpack8<BF16>(ring.get(stage, kX, i));
        const Vec8 gy = unpack8<BF16>(p.GY != nullptr ? ring.get(stage, kGY, i) : zero);
        const Vec8 gh = unpack8<BF16>(p.GH != nullptr ? ring.get(stage, kGH, i) : zero);
        const Vec8 w = unpack8<BF16>(w16[i]);
        const Vec8 t = unpack8<BF16>(ring.get(stage, kT, i));
        if constexpr (GATE == kRowGate) {
          const Vec8 g = unpack8<BF16>(ring.get(stage, kG, i));
          pg[i] = unpack8<BF16>(pw16[i]);
#pragma unroll
          for (int k = 0; k < 4; ++k) pg[i].v[k] = pg[i].v[k] * g.v[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 u = t.v[k] * r1 * pg[i].v[k];
          n2[i].v[k] = fma2(f2(p.alpha), x.v[k], u) * r2;
          v[i].v[k] = gy.v[k] * w.v[k];
          s0 = fma2(v[i].v[k], n2[i].v[k], s0);
          s1 = fma2(gh.v[k], u, s1);
          s2 = fma2(v[i].v[k], u, s2);
          s3 = fma2(n2[i].v[k], u, s3);
          acc_w[i].v[k] = fma2(gy.v[k], n2[i].v[k], acc_w[i].v[k]);
        }
      }
    }
    const float4 sums = row_sums<CTAS>(make_float4(s0.x + s0.y, s1.x + s1.y, s2.x + s2.y, s3.x + s3.y), red, turn);
    const float c2 = sums.x * inv_dim;
    const float2 minus_c2 = f2(-c2);
    const float2 minus_c1 = f2(-(sums.y + r2.x * (sums.z - c2 * sums.w)) * inv_dim);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (c.first + i * c.step < dim) {
        const Vec8 gh = unpack8<BF16>(p.GH != nullptr ? ring.get(stage, kGH, i) : zero);
        const Vec8 t = unpack8<BF16>(ring.get(stage, kT, i));
        Vec8 dx, dt;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 dh = fma2(r2, fma2(n2[i].v[k], minus_c2, v[i].v[k]), gh.v[k]);
          dx.v[k] = f2(p.alpha) * dh;
          const float2 n1 = t.v[k] * r1;
          acc_m[i].v[k] = fma2(dh, n1, acc_m[i].v[k]);
          dt.v[k] = r1 * fma2(n1, minus_c1, dh * pg[i].v[k]);
        }
        __stcs(reinterpret_cast<uint4*>(p.DX + row + i * c.step), pack8<BF16>(dx));
        __stcs(reinterpret_cast<uint4*>(p.DT + row + i * c.step), pack8<BF16>(dt));
      }
    }
    if constexpr (GATE != kRowGate) fill(stage, b + kStages);  // (the gate is read once more)
    if constexpr (GATE != kNoGate) {
      if (b + 1 == line_end) {
        const bool whole = (line * rows_per_line >= row_begin) && line_end == (line + 1) * rows_per_line;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (c.first + i * c.step < dim) {
            const Vec8 pw = unpack8<BF16>(GATE == kRowGate ? pw16[i] : ld_vec(p.PW + c.first + i * c.step));
            const Vec8 g = unpack8<BF16>(GATE == kRowGate ? ring.get(stage, kG, i) : ld_vec(g_line + i * c.step));
            Vec8 dg;
#pragma unroll
            for (int k = 0; k < 4; ++k) dg.v[k] = acc_m[i].v[k] * pw.v[k];
            if (whole) {
              __stcs(reinterpret_cast<uint4*>(p.DG + static_cast<size_t>(line) * dim + c.first + i * c.step), pack8<BF16>(dg));
            } else {
              const int part = 2 * at + (line * rows_per_line > row_begin ? 1 : 0);
              store_sum(p.sum_g + static_cast<size_t>(part) * dim + c.first + i * c.step, dg);
            }
            float4 *lo, *hi;
            bool begun = true;
            if constexpr (GATE == kRowGate) {
              lo = sum_pw + 2 * i * blockDim.x;
              hi = lo + blockDim.x;
            } else {  // a line's end is rare enough for the CTA's words in global memory
              lo = reinterpret_cast<float4*>(p.sum_pw + static_cast<size_t>(at) * dim + c.first + i * c.step);
              hi = lo + 1;
              begun = line * rows_per_line > row_begin;
            }
            const float4 zero4 = make_float4(0.f, 0.f, 0.f, 0.f);
            const float4 a = begun ? *lo : zero4, d = begun ? *hi : zero4;
            *lo = make_float4(a.x + g.v[0].x * acc_m[i].v[0].x, a.y + g.v[0].y * acc_m[i].v[0].y,
                              a.z + g.v[1].x * acc_m[i].v[1].x, a.w + g.v[1].y * acc_m[i].v[1].y);
            *hi = make_float4(d.x + g.v[2].x * acc_m[i].v[2].x, d.y + g.v[2].y * acc_m[i].v[2].y,
                              d.z + g.v[3].x * acc_m[i].v[3].x, d.w + g.v[3].y * acc_m[i].v[3].y);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) acc_m[i].v[k] = f2(0.f);
        }
        if (b + 1 < row_end) {
          ++line;
          line_end = min(row_end, (line + 1) * rows_per_line);
          if constexpr (GATE == kLineGate) {
            g_line = p.G + static_cast<size_t>(line) * dim + c.first;
            load_line();
          }
        }
      }
    }
    if constexpr (GATE == kRowGate) fill(stage, b + kStages);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (c.first + i * c.step < dim) {
      const size_t to = static_cast<size_t>(at) * dim + c.first + i * c.step;
      if constexpr (GATE == kRowGate) {
        float4* d = reinterpret_cast<float4*>(p.sum_pw + to);
        d[0] = sum_pw[2 * i * blockDim.x];
        d[1] = sum_pw[(2 * i + 1) * blockDim.x];
      } else if constexpr (GATE == kNoGate) {
        store_sum(p.sum_pw + to, acc_m[i]);
      }
      store_sum(p.sum_w + to, acc_w[i]);
    }
  }
}

struct ColumnArgs {
  const float *sum_pw, *sum_w, *sum_g;  // as in BackwardArgs
  uint16_t *DPW, *DW, *DG;
  int dim, of, rows, lines;
};

// The parts of a line's sum in sum_g: rows first, first + more + step, ... of [2 * of][dim]; none if one CTA had the line.
struct LineParts {
  int first, more, count;
};
__device__ __forceinline__ LineParts parts_of_line(const ColumnArgs& p, int line) {
  const int rows_per_line = p.rows / p.lines;
  const int from = owner_of_row(line * rows_per_line, p.of, p.rows);
  const int to = owner_of_row((line + 1) * rows_per_line - 1, p.of, p.rows);
  return LineParts{2 * from, line * rows_per_line > first_row_of(from, p.of, p.rows) ? 1 : 0, to > from ? to - from + 1 : 0};
}

__device__ __forceinline__ void add4(float4& s, const float4& v) {
  s.x += v.x;
  s.y += v.y;
  s.z += v.z;
  s.w += v.w;
}

// Column sums over the CTAs of the kernel above: dPW, dW and, if it has few, the lines of dG.  A CTA takes 32 columns of one result
// (a whole 128-byte piece of every part), adds the parts up in blockDim.x / 8 runs and then the runs, in a fixed
// order.  Bound by latency: many short runs, since few columns leave few CTAs (16384 x 256: 2368 parts).
template <bool BF16>
__global__ void __launch_bounds__(1024) column_sum_kernel(const __grid_constant__ ColumnArgs p) {
  __shared__ float4 part[1024];
  const int lane = threadIdx.x & 7, run = threadIdx.x >> 3, runs = blockDim.x >> 3;
  const int col = (blockIdx.x * 8 + lane) * 4;
  const float* src = blockIdx.y == 0 ? p.sum_pw : p.sum_w;
  uint16_t* dst = blockIdx.y == 0 ? p.DPW : p.DW;
  LineParts l{0, 0, p.of};
  int step = 1;
  if (blockIdx.y >= 2) {
    const int line = static_cast<int>(blockIdx.y) - 2;
    l = parts_of_line(p, line);
    step = 2;
    src = p.sum_g;
    dst = p.DG + static_cast<size_t>(line) * p.dim;
  }
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < p.dim) {
#pragma unroll 8
    for (int c = run; c < l.count; c += runs) {
      const size_t row = static_cast<size_t>(l.first) + static_cast<size_t>(c) * step + (c == 0 ? l.more : 0);
      add4(s, __ldcs(reinterpret_cast<const float4*>(src + row * p.dim + col)));
    }
  }
  part[threadIdx.x] = s;
  for (int half = runs >> 1; half > 0; half >>= 1) {
    __syncthreads();
    if (run < half) {
      add4(s, part[threadIdx.x + 8 * half]);
      part[threadIdx.x] = s;
    }
  }
  if (run == 0 && col < p.dim && l.count > 0) {
    *reinterpret_cast<uint2*>(dst + col) = make_uint2(pack2<BF16>(s.x, s.y), pack2<BF16>(s.z, s.w));
  }
}

// The lines of dG if they are many and each has few parts: a thread adds up four columns of a line.  CTA rows of the grid: the
// lines, or, if those are more than the boundaries between two CTAs' rows, the boundaries (the first one inside a
// line stands for the line).
constexpr int kManyParts = 16;

template <bool BF16>
__global__ void __launch_bounds__(256) line_sum_kernel(const __grid_constant__ ColumnArgs p) {
  int line = blockIdx.y;
  if (p.lines >= p.of) {
    const int rows_per_line = p.rows / p.lines, at = blockIdx.y + 1, row = first_row_of(at, p.of, p.rows);
    line = row / rows_per_line;
    if (row == line * rows_per_line || first_row_of(at - 1, p.of, p.rows) > line * rows_per_line) line = -1;
  }
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  const int col = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (line < 0 || col >= p.dim) return;
  const LineParts l = parts_of_line(p, line);
  if (l.count == 0) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = 0; c < l.count; ++c) {
    const size_t row = static_cast<size_t>(l.first) + 2 * c + (c == 0 ? l.more : 0);
    add4(s, __ldcs(reinterpret_cast<const float4*>(p.sum_g + row * p.dim + col)));
  }
  *reinterpret_cast<uint2*>(p.DG + static_cast<size_t>(line) * p.dim + col) =
      make_uint2(pack2<BF16>(s.x, s.y), pack2<BF16>(s.z, s.w));
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, dim3 grid, int cluster, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) cudaGetLastError();  // reported to the caller, not left for the next one
  return e;
}

int threads_for(int nvec, int vpt) { return std::min(kMaxThreads, ((nvec + vpt - 1) / vpt + 31) / 32 * 32); }

// (per kernel and device, and the same whoever sets it)
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, bool* set) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 16 && set[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024);
  if (e == cudaSuccess && dev >= 0 && dev < 16) set[dev] = true;
  return e;
}

template <bool BF16, int VPT, int CTAS, int GATE>
cudaError_t launch_forward(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream) {
  auto kernel = norm_block_kernel<BF16, VPT, CTAS, GATE>;
  static bool set[16] = {};
  const cudaError_t e = allow_smem(kernel, set);
  if (e != cudaSuccess) return e;
  const int threads = threads_for(p.dim / 8, VPT);
  const int grid = std::min(p.rows, sm_count / CTAS * std::min(16, kMaxThreads / threads * (VPT == 1 ? 2 : 1))) * CTAS;
  return launch(kernel, dim3(grid), CTAS, threads, threads * ForwardRing<VPT, GATE>::kBytesPerThread, stream,
                static_cast<const uint16_t*>(p.X), static_cast<const uint16_t*>(p.T), static_cast<const uint16_t*>(p.PW),
                static_cast<const uint16_t*>(p.W), static_cast<const uint16_t*>(p.G), static_cast<uint16_t*>(H),
                static_cast<uint16_t*>(Y), reinterpret_cast<float2*>(stats), p.rows, p.dim, p.rows / p.lines, p.alpha, p.eps);
}

template <bool BF16, int GATE>
cudaError_t forward(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream) {
  const int nvec = p.dim / 8;
  if (nvec <= kMaxThreads) return launch_forward<BF16, 1, 1, GATE>(p, H, Y, stats, sm_count, stream);
  if (p.dim <= kCtaDim) return launch_forward<BF16, 2, 1, GATE>(p, H, Y, stats, sm_count, stream);
  return launch_forward<BF16, 2, 2, GATE>(p, H, Y, stats, sm_count, stream);
}

// Rows of one warp keep one vector a thread, so that more of them run at once.
int backward_vpt(int dim) { return dim / 8 <= 32 ? 1 : 2; }

template <bool BF16, int VPT, int CTAS, int GATE>
cudaError_t launch_backward(const BackwardArgs& a, int at_once, cudaStream_t stream) {
  auto kernel = norm_block_backward_kernel<BF16, VPT, CTAS, GATE>;
  static bool set[16] = {};
  const cudaError_t e = allow_smem(kernel, set);
  if (e != cudaSuccess) return e;
  const int threads = threads_for(a.dim / 8, VPT);
  return launch(kernel, dim3(at_once * CTAS), CTAS, threads, threads * (BackwardRing<VPT, GATE>::kBytesPerThread + (GATE == kRowGate ? VPT * 32 : 0)),
                stream, a);
}

template <bool BF16, int GATE>
cudaError_t backward(const BackwardArgs& a, int at_once, cudaStream_t stream) {
  if (backward_vpt(a.dim) == 1) return launch_backward<BF16, 1, 1, GATE>(a, at_once, stream);
  if (a.dim <= kCtaDim) return launch_backward<BF16, 2, 1, GATE>(a, at_once, stream);
  return launch_backward<BF16, 2, 2, GATE>(a, at_once, stream);
}

Gate gate_of(const NormBlock& p) {
  return p.G == nullptr ? kNoGate : (p.lines == 1 || p.rows / p.lines >= kMinLineRows ? kLineGate : kRowGate);
}

bool valid(const NormBlock& p) {
  return p.dim >= 8 && p.dim % 8 == 0 && p.dim <= kMaxDim && p.rows >= 1 && p.rows <= kMaxNormBlockRows && p.lines >= 1 && p.rows % p.lines == 0;
}

}  // namespace

cudaError_t norm_block_launch(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream) {
  if (!valid(p)) return cudaErrorInvalidValue;
  switch (gate_of(p)) {
    case kNoGate: return p.bf16 ? forward<true, kNoGate>(p, H, Y, stats, sm_count, stream) : forward<false, kNoGate>(p, H, Y, stats, sm_count, stream);
    case kLineGate: return p.bf16 ? forward<true, kLineGate>(p, H, Y, stats, sm_count, stream) : forward<false, kLineGate>(p, H, Y, stats, sm_count, stream);
    default: return p.bf16 ? forward<true, kRowGate>(p, H, Y, stats, sm_count, stream) : forward<false, kRowGate>(p, H, Y, stats, sm_count, stream);
  }
}

NormBlockPlan norm_block_plan(const NormBlock& p, int sm_count) {
  NormBlockPlan plan;
  const int threads = threads_for(p.dim / 8, backward_vpt(p.dim));
  const int most = p.dim <= kCtaDim ? sm_count * std::min(16, kMaxThreads / threads) : sm_count / 2;
  plan.at_once = std::min(gate_of(p) == kRowGate ? p.lines : p.rows, most);
  plan.workspace = static_cast<size_t>(p.G != nullptr ? 4 : 2) * plan.at_once * p.dim;
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
  a.sum_w = a.sum_pw + static_cast<size_t>(plan.at_once) * p.dim;
  a.sum_g = a.sum_w + static_cast<size_t>(plan.at_once) * p.dim;
  a.rows = p.rows;
  a.dim = p.dim;
  a.lines = gate ? p.lines : 1;
  a.alpha = p.alpha;
  cudaError_t e;
  switch (gate_of(p)) {
    case kNoGate: e = p.bf16 ? backward<true, kNoGate>(a, plan.at_once, stream) : backward<false, kNoGate>(a, plan.at_once, stream); break;
    case kLineGate: e = p.bf16 ? backward<true, kLineGate>(a, plan.at_once, stream) : backward<false, kLineGate>(a, plan.at_once, stream); break;
    default: e = p.bf16 ? backward<true, kRowGate>(a, plan.at_once, stream) : backward<false, kRowGate>(a, plan.at_once, stream); break;
  }
  if (e != cudaSuccess) return e;
  ColumnArgs sums;
  sums.sum_pw = a.sum_pw;
  sums.sum_w = a.sum_w;
  sums.sum_g = a.sum_g;
  sums.DPW = static_cast<uint16_t*>(DPW);
  sums.DW = static_cast<uint16_t*>(DW);
  sums.DG = a.DG;
  sums.dim = p.dim;
  sums.of = plan.at_once;
  sums.rows = p.rows;
  sums.lines = a.lines;
  const bool lines_apart = gate && gate_of(p) == kLineGate && a.lines * kManyParts > plan.at_once;
  const bool lines_too = gate && gate_of(p) == kLineGate && !lines_apart && plan.at_once > 1;
  const dim3 grid((p.dim + 31) / 32, 2 + (lines_too ? a.lines : 0));
  const int threads = plan.at_once > 256 ? 1024 : 512;
  e = p.bf16 ? launch(column_sum_kernel<true>, grid, 1, threads, 0, stream, sums)
             : launch(column_sum_kernel<false>, grid, 1, threads, 0, stream, sums);
  if (e != cudaSuccess || !lines_apart || plan.at_once == 1) return e;
  const dim3 by_line((p.dim + 1023) / 1024, a.lines >= plan.at_once ? plan.at_once - 1 : a.lines);
  return p.bf16 ? launch(line_sum_kernel<true>, by_line, 1, 256, 0, stream, sums)
                : launch(line_sum_kernel<false>, by_line, 1, 256, 0, stream, sums);
}

}  // namespace fo
