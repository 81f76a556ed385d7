// Rows sorted by expert and back.  A router gives every token top_k experts; the products run on each expert's rows
// together, so a token's row is copied to top_k places of a matrix sorted by expert, and afterwards the
// top_k results are summed with the router's weights.  All sums are fp32; there are no atomics on global
// memory, and every result is the same from call to call.
#include "fo_moe.h"

#include <algorithm>

#include "../common/fo_pack16.cuh"
#include "../common/fo_ptx.cuh"

namespace fo {

namespace {

// Kernels that follow one another closely (ptx::grid_wait) begin before their inputs are written, so no load of an input goes the
// read-only way (ld.global.nc, which __ldg and const __restrict__ pointers are compiled to): it is for data that nobody writes while
// the kernel exists.

// ---------------------------------------------------------------------------- the order

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
// Choices up to which one CTA sorts, and eight; sixteen from there on.  1, 8 and 16 CTAs, in us, back to back in a graph: 1024 choices of 64
// experts 3.8, 4.6, 4.9; 2048 of 256 4.8, 5.1, 5.6; 4096 of 64 5.7, 4.8, 5.1; 8192 of 64 9.1, 4.8, 5.1; 12288 of 64 12.4, 5.6, 5.2; 65536
// of 64 56, 10.2, 7.1.
constexpr int kSortOne = 2048, kSortEight = 8192;
constexpr int kSortBatch = 4;

__device__ __forceinline__ uint32_t ld_shared_cluster_u32(uint32_t cluster_addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// A stable counting sort: one CTA, or a cluster of eight or sixteen.  Every warp takes a run of choices and counts them by
// expert in a row of its own in shared memory; the counts of the warps and, through distributed shared memory, of the CTAs in
// front of it give each warp its first row for every expert, and a second walk over the same run hands the rows out, 32
// choices a step: ballots over the expert's bits tell each lane which others have its expert (half the time of match.any, whose
// cost goes with the number of different experts: 16384 x 8 of 256 in 25 against 41 us with eight CTAs).  Bound by latency; back to
// back in a graph, and in brackets cold under a profiler: 16 x 8 choices 2.5 us (6.2), 8192 x 8 of 64 7.0 us (11.8), 16384 x 8 of
// 256 11.5 us (16.1).
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
    moe_sort_kernel(const Id* __restrict__ ids, int64_t n, int experts, int32_t* __restrict__ slot,
                    int32_t* __restrict__ source, int32_t* __restrict__ offsets) {
  extern __shared__ uint32_t smem[];
  uint32_t* total = smem;              // [experts]: this CTA's choices
  uint32_t* base = total + experts;    // [experts]: the first row of these
  uint32_t* count = base + experts;    // [kSortWarps][experts]: each warp's, then its next row behind the first
  __shared__ uint32_t scan[kSortWarps];
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int ctas = static_cast<int>(gridDim.x);  // one cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* mine = count + warp * experts;
  const int64_t per_warp = (n + ctas * kSortThreads - 1) / (ctas * kSortThreads) * 32;
  const int64_t left = n - static_cast<int64_t>(rank) * kSortWarps * per_warp;
  const int warps_used = left <= 0 ? 0 : static_cast<int>(min((left + per_warp - 1) / per_warp, static_cast<int64_t>(kSortWarps)));
  for (int e = threadIdx.x; e < warps_used * experts; e += kSortThreads) count[e] = 0;
  const int64_t begin = min(n, (static_cast<int64_t>(rank) * kSortWarps + warp) * per_warp);
  const int64_t end = min(n, begin + per_warp);
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  __syncthreads();
  // expert of choice i; `experts` for a choice without one and for lanes past the end
  auto expert_at = [&](int64_t i) -> int {
    if (i >= end) return experts;
    const Id v = __ldca(ids + i);
    return v >= 0 && v < static_cast<Id>(experts) ? static_cast<int>(v) : experts;
  };
  // the walks go in batches whose loads are in flight together
  for (int64_t i0 = begin; i0 < end; i0 += 32 * kSortBatch) {
    int ex[kSortBatch];
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) ex[u] = expert_at(i0 + 32 * u + lane);
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) {
      if (ex[u] < experts) atomicAdd(mine + ex[u], 1u);  // a count does not depend on the order
    }
  }
  __syncthreads();
  const int e = threadIdx.x;  // experts <= kSortThreads
  if (e < experts) {
    uint32_t sum = 0;
#pragma unroll 8
    for (int w = 0; w < warps_used; ++w) {
      const uint32_t c = count[w * experts + e];
      count[w * experts + e] = sum;
      sum += c;
    }
    total[e] = sum;
  }
  uint32_t before = 0, all = 0;
  if (ctas > 1) {
    __syncwarp();  // the barrier's aligned forms take whole warps
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
  }
  if (e < experts && ctas == 1) {
    all = total[e];
  } else if (e < experts) {
    for (int c = 0; c < ctas; ++c) {
      const uint32_t v = ld_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(total + e), c));
      if (c < rank) before += v;
      all += v;
    }
  }
  // Nobody reads another CTA's counts from here on.  The release form: a CTA without choices waits at the kernel's end only, and
  // must not leave while a load of its counts is under way.
  __syncwarp();
  if (ctas > 1) ptx::cluster_arrive_release();
  // exclusive sums over the experts
  uint32_t incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  uint32_t warps = scan[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, warps, o);
    if (lane >= o) warps += v;
  }
  const uint32_t rows = __shfl_sync(0xffffffffu, warps, 31);
  const uint32_t in_front = __shfl_sync(0xffffffffu, warps, warp > 0 ? warp - 1 : 0);
  const uint32_t first = incl - all + (warp > 0 ? in_front : 0u);
  if (e < experts) {
    if (rank == 0) offsets[e] = static_cast<int32_t>(first);
    base[e] = first + before;
  }
  if (rank == 0 && threadIdx.x == 0) offsets[experts] = static_cast<int32_t>(rows);
  __syncthreads();
  const int bits = 32 - __clz(experts);
  for (int64_t i0 = begin; i0 < end; i0 += 32 * kSortBatch) {
    int batch[kSortBatch];
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) batch[u] = expert_at(i0 + 32 * u + lane);
#pragma unroll
    for (int u = 0; u < kSortBatch; ++u) {
      if (i0 + 32 * u >= end) break;
      const int ex = batch[u];
      uint32_t same = 0xffffffffu;  // the lanes with this lane's expert
      for (int b = 0; b < bits; ++b) {
        const uint32_t ones = __ballot_sync(0xffffffffu, (ex >> b) & 1);
        same &= (ex >> b) & 1 ? ones : ~ones;
      }
      const int64_t i = i0 + 32 * u + lane;
      int32_t row = -1;
      if (ex < experts) {
        row = static_cast<int32_t>(base[ex] + mine[ex] + __popc(same & ((1u << lane) - 1u)));
        source[row] = static_cast<int32_t>(i);
      }
      __syncwarp();
      if (ex < experts && lane == __ffs(same) - 1) mine[ex] += __popc(same);
      __syncwarp();
      if (i < end) slot[i] = row;
    }
  }
  for (int64_t r = rows + static_cast<int64_t>(rank) * kSortThreads + threadIdx.x; r < n; r += static_cast<int64_t>(ctas) * kSortThreads) {
    source[r] = -1;
  }
  __syncwarp();
  if (ctas > 1) ptx::cluster_wait_acquire();
}

// ---------------------------------------------------------------------------- the rows

constexpr int kRowThreads = 256;

// The row of a choice if it is one of the `rows` there are, else -1: an order made for something else is not followed
// out of the matrix.
__device__ __forceinline__ int row_at(const int32_t* slot, int64_t choice, int64_t rows) {
  const int row = __ldca(slot + choice);
  return static_cast<uint32_t>(row) < static_cast<uint32_t>(rows) ? row : -1;
}

// The rows that belong to experts, as far as the matrix has them.
__device__ __forceinline__ int64_t served_rows(const int32_t* offsets, int experts, int64_t rows) {
  return min(max(static_cast<int64_t>(__ldca(offsets + experts)), static_cast<int64_t>(0)), rows);
}

// Rows [first, last), zeroed by all threads of the grid.
__device__ __forceinline__ void zero_rows(uint4* rows, int64_t first, int64_t last, int nvec) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t end = last * nvec;
  for (int64_t v = first * nvec + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; v < end; v += step) rows[v] = zero;
}

// Rows below `served` that no slot names, zeroed: the row of a choice whose slot was set to -1 in a sorted order.  A thread looks
// after a row, which is named if the choice that back[row] holds names it; so are all rows of a sorted order with its own
// sources.  Where it does not, nobody names the row if `back` is the scratch of moe_inverse_kernel (`exact`), but sources may
// also be of something else: then the CTA goes through all slots.  8192 x 8 rows of 512: 13.0 us sorted (12.8 without any of this),
// 33 with a tenth dropped; with a scratch 14.3 and 14.6, but one launch more, which small calls pay for on the host.  So the scratch is
// made where a call brings no sources, and for more than kNamedScan choices, since the search's cost grows with their square
// (8192 x 8 rows of 4096: 96 us, 106 with a tenth dropped, and 98 with a scratch).
constexpr int64_t kNamedScan = 65536;

struct NamedRows {
  const int32_t* back;
  bool exact;
};

// The row that this thread looks after first.
__device__ __forceinline__ int64_t first_own_row() { return static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; }

// All threads of the grid call this.  `back`: of first_own_row(), fetched ahead (whatever it is where there is no such row).
__device__ __forceinline__ void zero_unnamed_rows(uint4* R, const int32_t* slot, const NamedRows& n, int32_t back, int64_t served,
                                                  int64_t choices, int nvec) {
  __shared__ uint32_t named[kRowThreads / 32];  // a bit for each row of the CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t own = first_own_row(); own - threadIdx.x < served; own += step) {
    if (own >= step) back = own < served ? __ldca(n.back + own) : -1;
    const bool there = own < served;
    const bool is = there && static_cast<uint32_t>(back) < static_cast<uint32_t>(choices) && __ldca(slot + back) == own;
    uint32_t left = __ballot_sync(0xffffffffu, there && !is);
    if (!n.exact && __syncthreads_or(left)) {
      constexpr int kAhead = 8;  // loads in flight
      const int first = static_cast<int>(own - threadIdx.x), last = static_cast<int>(choices);  // kNamedScan at most
      if (lane == 0) named[warp] = 0;
      __syncthreads();
#pragma unroll 1
      for (int c0 = threadIdx.x; c0 < last; c0 += kAhead * blockDim.x) {
        uint32_t r[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int c = c0 + u * static_cast<int>(blockDim.x);
          r[u] = c < last ? static_cast<uint32_t>(__ldca(slot + c)) - first : 0xffffffffu;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (r[u] < blockDim.x) atomicOr(&named[r[u] >> 5], 1u << (r[u] & 31));
        }
      }
      __syncthreads();
      left &= ~named[warp];
      __syncthreads();  // the bits have been read
    }
    for (; left != 0; left &= left - 1) {
      uint4* row = R + (own - lane + __ffs(left) - 1) * nvec;
      for (int j = lane; j < nvec; j += 32) row[j] = make_uint4(0, 0, 0, 0);
    }
  }
}

// inverse[slot[c]] = c.  Rows that no slot names keep what was there, which the look back tells.
__global__ void __launch_bounds__(kRowThreads)
    moe_inverse_kernel(const int32_t* __restrict__ slot, int32_t* __restrict__ inverse, int64_t choices) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  if (c >= choices) return;
  const int row = row_at(slot, c, choices);
  if (row >= 0) inverse[row] = static_cast<int32_t>(c);
}

// Bound by the rows written: every token's row is read once.  A thread copies one vector of a token to its top_k rows.
// 8192 x 8 rows of 4096: 97 us (6.2 TB/s), 16384 x 2 of 8192: 129 us (6.2 TB/s).  32 registers, for eight CTAs an SM: rows that
// are zeros wait for nothing but warps (8192 x 4 rows of 4096, a quarter with a choice, with its sort 59.0 us, at 48 registers 63).
__global__ void __launch_bounds__(kRowThreads, 8)
    moe_dispatch_kernel(const uint4* __restrict__ X, const int32_t* __restrict__ slot,
                        const int32_t* __restrict__ offsets, NamedRows named, uint4* __restrict__ R,
                        int tokens, int top_k, int nvec, int experts) {
  const int64_t v = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  const int64_t token = v / nvec;
  const int64_t rows = static_cast<int64_t>(tokens) * top_k;
  const int64_t served = served_rows(offsets, experts, rows);
  const int32_t back = first_own_row() < rows ? __ldca(named.back + first_own_row()) : -1;
  if (token < tokens) {
    const int j = static_cast<int>(v - token * nvec);
    const uint4 x = __ldcs(X + v);
#pragma unroll 4
    for (int k = 0; k < top_k; ++k) {
      const int row = row_at(slot, token * top_k + k, served);
      if (row >= 0) R[static_cast<int64_t>(row) * nvec + j] = x;
    }
  }
  zero_unnamed_rows(R, slot, named, back, served, rows, nvec);
  zero_rows(R, served, rows, nvec);
}

template <bool BF16>
__device__ __forceinline__ float weight_at(const void* w, bool f32, int64_t i) {
  if (w == nullptr) return 1.f;
  if (f32) return __ldca(static_cast<const float*>(w) + i);
  const uint32_t bits = __ldca(static_cast<const unsigned short*>(w) + i);
  return unpack2<BF16>(bits).x;
}

// The kernels that read a token's rows have a build for each number of rows that a thread requests at once; more choices
// than that are taken in turns.
constexpr int kMostAtOnce = 8;

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& p, float2 (&f)[4]) {
  f[0] = unpack2<BF16>(p.x);
  f[1] = unpack2<BF16>(p.y);
  f[2] = unpack2<BF16>(p.z);
  f[3] = unpack2<BF16>(p.w);
}

// Bound by the rows read.  A thread sums VPT vectors of a token over its top_k rows, in their order; KC rows of them are in flight at
// once, and where a token has few rows more of its vectors are (one vector a thread: 16384 x 2 rows of 8192 in 316 us, now 131;
// 8192 x 8 of 4096: 94 us, 6.4 TB/s).
template <bool BF16, int KC, int VPT>
__global__ void __launch_bounds__(kRowThreads)
    moe_combine_kernel(const uint4* __restrict__ R, const void* __restrict__ w, bool f32,
                       const int32_t* __restrict__ slot, uint4* __restrict__ O, int tokens, int top_k, int nvec) {
  const int groups = (nvec + VPT - 1) / VPT;  // threads of a token: thread j takes vectors j, j + groups, ...
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  const int64_t token = id / groups;
  const int j = static_cast<int>(id - token * groups);
  const int64_t rows = static_cast<int64_t>(tokens) * top_k;
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  if (token >= tokens) return;
  float2 acc[VPT][4];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = make_float2(0.f, 0.f);
  }
  for (int k0 = 0; k0 < top_k; k0 += KC) {
    uint4 r[KC][VPT];
    int row[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) row[k] = k0 + k < top_k ? row_at(slot, token * top_k + k0 + k, rows) : -1;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (row[k] >= 0 && j + i * groups < nvec) r[k][i] = __ldcs(R + static_cast<int64_t>(row[k]) * nvec + j + i * groups);
      }
    }
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      if (row[k] >= 0) {
        const float wk = weight_at<BF16>(w, f32, token * top_k + k0 + k);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (j + i * groups >= nvec) continue;
          float2 f[4];
          unpack8<BF16>(r[k][i], f);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            acc[i][n].x += wk * f[n].x;
            acc[i][n].y += wk * f[n].y;
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (j + i * groups < nvec) {
      __stcs(O + token * nvec + j + i * groups,
             make_uint4(pack2<BF16>(acc[i][0].x, acc[i][0].y), pack2<BF16>(acc[i][1].x, acc[i][1].y),
                        pack2<BF16>(acc[i][2].x, acc[i][2].y), pack2<BF16>(acc[i][3].x, acc[i][3].y)));
    }
  }
}

// Bound by memory: the token's gradient is read once, every row of the experts is read (for its weight's gradient) and its
// gradient written.  A CTA takes a token, three of them an SM; the dots are summed over its threads in a fixed order.  8192 x 8 rows
// of 4096: 182 us (6.3 TB/s; 194 with two an SM), 16384 x 2 of 8192: 212 us (6.3 TB/s).
template <bool BF16, int KC, int VPT, bool ROWS, bool WEIGHTS>
__global__ void __launch_bounds__(kRowThreads, 3)
    moe_combine_backward_kernel(const uint4* __restrict__ GO, const uint4* __restrict__ R, const void* __restrict__ w,
                                bool f32, const int32_t* __restrict__ slot, const int32_t* __restrict__ offsets,
                                NamedRows named, uint4* __restrict__ DR, void* __restrict__ DW, int tokens, int top_k, int nvec,
                                int experts) {
  __shared__ float part[kRowThreads / 32][KC];
  const int64_t token = blockIdx.x;
  const int64_t rows = static_cast<int64_t>(tokens) * top_k;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ptx::grid_launch_dependents();
  ptx::grid_wait();
  [[maybe_unused]] const int64_t served = ROWS ? served_rows(offsets, experts, rows) : 0;
  for (int k0 = 0; k0 < top_k; k0 += KC) {
    int row[KC];
    float wk[KC], dot[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      row[k] = k0 + k < top_k ? row_at(slot, token * top_k + k0 + k, rows) : -1;
      dot[k] = 0.f;
      wk[k] = ROWS && row[k] >= 0 ? weight_at<BF16>(w, f32, token * top_k + k0 + k) : 0.f;
    }
    for (int j0 = threadIdx.x; j0 < nvec; j0 += VPT * blockDim.x) {
      uint4 g[VPT];
      [[maybe_unused]] uint4 r[KC][VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = j0 + i * blockDim.x;
        if (j < nvec) g[i] = __ldca(GO + token * nvec + j);
      }
      if constexpr (WEIGHTS) {
#pragma unroll
        for (int k = 0; k < KC; ++k) {
#pragma unroll
          for (int i = 0; i < VPT; ++i) {
            const int j = j0 + i * blockDim.x;
            if (row[k] >= 0 && j < nvec) r[k][i] = __ldcs(R + static_cast<int64_t>(row[k]) * nvec + j);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = j0 + i * blockDim.x;
        if (j >= nvec) continue;
        float2 gf[4];
        unpack8<BF16>(g[i], gf);
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          if (row[k] < 0) continue;
          if constexpr (WEIGHTS) {
            float2 f[4];
            unpack8<BF16>(r[k][i], f);
#pragma unroll
            for (int n = 0; n < 4; ++n) dot[k] += gf[n].x * f[n].x + gf[n].y * f[n].y;
          }
          if constexpr (ROWS) {
            if (row[k] >= served) continue;
            __stcs(DR + static_cast<int64_t>(row[k]) * nvec + j,
                   make_uint4(pack2<BF16>(wk[k] * gf[0].x, wk[k] * gf[0].y), pack2<BF16>(wk[k] * gf[1].x, wk[k] * gf[1].y),
                              pack2<BF16>(wk[k] * gf[2].x, wk[k] * gf[2].y), pack2<BF16>(wk[k] * gf[3].x, wk[k] * gf[3].y)));
          }
        }
      }
    }
    if constexpr (WEIGHTS) {
#pragma unroll
      for (int k = 0; k < KC; ++k) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
      }
      __syncthreads();  // the previous round's sums have been read
      if (lane == 0) {
#pragma unroll
        for (int k = 0; k < KC; ++k) part[warp][k] = dot[k];
      }
      __syncthreads();
      const int k = threadIdx.x;
      if (k < KC && k0 + k < top_k) {
        float s = 0.f;
        for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s += part[i][k];
        const int64_t at = token * top_k + k0 + k;
        if (f32) {
          static_cast<float*>(DW)[at] = s;
        } else if constexpr (BF16) {
          static_cast<__nv_bfloat16*>(DW)[at] = __float2bfloat16_rn(s);
        } else {
          static_cast<__half*>(DW)[at] = __float2half_rn(s);
        }
      }
    }
  }
  if constexpr (ROWS) {
    const int32_t back = first_own_row() < rows ? __ldca(named.back + first_own_row()) : -1;
    zero_unnamed_rows(DR, slot, named, back, served, rows, nvec);
    zero_rows(DR, served, rows, nvec);
  }
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, int64_t grid, int threads, cudaStream_t stream, Args... args) {
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) cudaGetLastError();  // reported to the caller, not left for the next one
  return e;
}

cudaLaunchConfig_t sort_config(int ctas, int smem, cudaStream_t stream, cudaLaunchAttribute (&attr)[2]) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(kSortThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// The largest cluster of the sort that the current device has a place for, and the kernel's attributes set on the way: sixteen
// CTAs are more than every device or part of one (a partition, a context of fewer SMs) grants.
template <typename Id>
cudaError_t largest_sort(int* ctas) {
  static int cache[16] = {};  // 0: not asked yet; the same whoever sets it
  constexpr int smem = (kSortWarps + 2) * kMaxExperts * static_cast<int>(sizeof(uint32_t));
  auto kernel = moe_sort_kernel<Id>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 16 && cache[dev] != 0) {
    *ctas = cache[dev];
    return cudaSuccess;
  }
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  int most = 1;
  for (int size : {16, 8}) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = sort_config(size, smem, nullptr, attr);
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0) {
      most = size;
      break;
    }
    cudaGetLastError();
  }
  if (dev < 16) cache[dev] = most;
  *ctas = most;
  return cudaSuccess;
}

template <typename Id>
cudaError_t launch_sort(const void* ids, int64_t n, int experts, int most_ctas, int32_t* slot, int32_t* source,
                        int32_t* offsets, cudaStream_t stream) {
  int largest = 1;
  cudaError_t e = largest_sort<Id>(&largest);
  if (e != cudaSuccess) return e;
  const int smem = (kSortWarps + 2) * experts * static_cast<int>(sizeof(uint32_t));
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = sort_config(moe_sort_ctas(n, std::min(most_ctas, largest)), smem, stream, attr);
  e = cudaLaunchKernelEx(&cfg, moe_sort_kernel<Id>, static_cast<const Id*>(ids), n, experts, slot, source, offsets);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}

bool valid(const MoeShape& s) {
  return s.tokens >= 1 && s.top_k >= 1 && s.top_k <= kMaxTopK && s.dim >= 8 && s.dim % 8 == 0 && s.experts >= 1 &&
         s.experts <= kMaxExperts && static_cast<int64_t>(s.tokens) * s.top_k <= INT32_MAX;
}

// How the rows that are named are told, made on the way if it takes the scratch.
cudaError_t named_rows(const MoeShape& s, const int32_t* slot, const MoeSources& from, NamedRows* n, cudaStream_t stream) {
  const int64_t choices = static_cast<int64_t>(s.tokens) * s.top_k;
  *n = NamedRows{from.scratch != nullptr ? from.scratch : from.source, from.scratch != nullptr};
  if (from.scratch == nullptr) return moe_scratch_words(s, from.source != nullptr) == 0 ? cudaSuccess : cudaErrorInvalidValue;
  return launch(moe_inverse_kernel, (choices + kRowThreads - 1) / kRowThreads, kRowThreads, stream, slot, from.scratch, choices);
}

int64_t vec_ctas(const MoeShape& s) { return (static_cast<int64_t>(s.tokens) * (s.dim / 8) + kRowThreads - 1) / kRowThreads; }

// Rows requested at once, and vectors of each, for a number of choices: about eight loads a thread, four where eight take the registers of
// a third CTA an SM (two rows, four vectors each: 16384 x 2 rows of 8192 in 144 us, two vectors: 130).
template <bool BF16, int KC, int VPT>
cudaError_t launch_combine(const MoeShape& s, const uint4* r, MoeWeights w, const int32_t* slot, uint4* o, cudaStream_t stream) {
  const int nvec = s.dim / 8;
  const int64_t threads = static_cast<int64_t>(s.tokens) * ((nvec + VPT - 1) / VPT);
  return launch(moe_combine_kernel<BF16, KC, VPT>, (threads + kRowThreads - 1) / kRowThreads, kRowThreads, stream, r, w.p,
                w.f32, slot, o, s.tokens, s.top_k, nvec);
}

template <bool BF16>
cudaError_t combine(const MoeShape& s, const uint4* r, MoeWeights w, const int32_t* slot, uint4* o, cudaStream_t stream) {
  switch (s.top_k) {
    case 1: return launch_combine<BF16, 1, 4>(s, r, w, slot, o, stream);
    case 2: return launch_combine<BF16, 2, 2>(s, r, w, slot, o, stream);
    case 3: return launch_combine<BF16, 3, 2>(s, r, w, slot, o, stream);
    case 4: return launch_combine<BF16, 4, 2>(s, r, w, slot, o, stream);
    case 5:
    case 6: return launch_combine<BF16, 6, 1>(s, r, w, slot, o, stream);
    default: return launch_combine<BF16, kMostAtOnce, 1>(s, r, w, slot, o, stream);
  }
}

struct BackwardCall {
  MoeShape s;
  const uint4 *go, *r;
  MoeWeights w;
  const int32_t *slot, *offsets;
  NamedRows named;
  uint4* dr;
  void* dw;
};

template <bool BF16, int KC, int VPT>
cudaError_t launch_backward(const BackwardCall& c, cudaStream_t stream) {
  const int nvec = c.s.dim / 8;
  const int threads = std::min(kRowThreads, ((nvec + VPT - 1) / VPT + 31) / 32 * 32);
  auto kernel = c.dr == nullptr   ? moe_combine_backward_kernel<BF16, KC, VPT, false, true>
                : c.dw == nullptr ? moe_combine_backward_kernel<BF16, KC, VPT, true, false>
                                  : moe_combine_backward_kernel<BF16, KC, VPT, true, true>;
  return launch(kernel, c.s.tokens, threads, stream, c.go, c.r, c.w.p, c.w.f32, c.slot, c.offsets, c.named, c.dr, c.dw, c.s.tokens,
                c.s.top_k, nvec, c.s.experts);
}

template <bool BF16>
cudaError_t backward(const BackwardCall& c, cudaStream_t stream) {
  switch (c.s.top_k) {
    case 1: return launch_backward<BF16, 1, 4>(c, stream);
    case 2: return launch_backward<BF16, 2, 4>(c, stream);
    case 3: return launch_backward<BF16, 3, 2>(c, stream);
    case 4: return launch_backward<BF16, 4, 2>(c, stream);
    case 5:
    case 6: return launch_backward<BF16, 6, 1>(c, stream);
    default: return launch_backward<BF16, kMostAtOnce, 1>(c, stream);
  }
}

}  // namespace

int64_t moe_scratch_words(const MoeShape& s, bool sources) {
  const int64_t choices = static_cast<int64_t>(s.tokens) * s.top_k;
  return sources && choices <= kNamedScan ? 0 : choices;
}

int moe_sort_ctas(int64_t choices, int most) {
  const int wanted = choices <= kSortOne ? 1 : (choices <= kSortEight ? 8 : 16);
  return wanted <= most ? wanted : (wanted == 16 && most >= 8 ? 8 : 1);
}

cudaError_t moe_sort_launch(const void* ids, bool ids64, int64_t choices, int experts, int most_ctas, int32_t* slot,
                            int32_t* source, int32_t* offsets, cudaStream_t stream) {
  if (experts < 1 || experts > kMaxExperts || choices < 0 || choices > INT32_MAX || most_ctas < 1) return cudaErrorInvalidValue;
  return ids64 ? launch_sort<int64_t>(ids, choices, experts, most_ctas, slot, source, offsets, stream)
               : launch_sort<int32_t>(ids, choices, experts, most_ctas, slot, source, offsets, stream);
}

cudaError_t moe_dispatch_launch(const MoeShape& s, const void* X, const int32_t* slot, const int32_t* offsets,
                                const MoeSources& from, void* R, cudaStream_t stream) {
  if (!valid(s)) return cudaErrorInvalidValue;
  NamedRows named;
  const cudaError_t e = named_rows(s, slot, from, &named, stream);
  if (e != cudaSuccess) return e;
  return launch(moe_dispatch_kernel, vec_ctas(s), kRowThreads, stream, static_cast<const uint4*>(X), slot, offsets,
                named, static_cast<uint4*>(R), s.tokens, s.top_k, s.dim / 8, s.experts);
}

cudaError_t moe_combine_launch(const MoeShape& s, const void* R, MoeWeights w, const int32_t* slot, void* O,
                               cudaStream_t stream) {
  if (!valid(s)) return cudaErrorInvalidValue;
  const uint4* r = static_cast<const uint4*>(R);
  return s.bf16 ? combine<true>(s, r, w, slot, static_cast<uint4*>(O), stream) : combine<false>(s, r, w, slot, static_cast<uint4*>(O), stream);
}

cudaError_t moe_combine_backward_launch(const MoeShape& s, const void* GO, const void* R, MoeWeights w,
                                        const int32_t* slot, const int32_t* offsets, const MoeSources& from, void* DR,
                                        void* DW, cudaStream_t stream) {
  if (!valid(s) || (DR == nullptr && DW == nullptr)) return cudaErrorInvalidValue;
  NamedRows named{};
  if (DR != nullptr) {
    const cudaError_t e = named_rows(s, slot, from, &named, stream);
    if (e != cudaSuccess) return e;
  }
  const BackwardCall c{s, static_cast<const uint4*>(GO), static_cast<const uint4*>(R), w, slot, offsets, named, static_cast<uint4*>(DR), DW};
  return s.bf16 ? backward<true>(c, stream) : backward<false>(c, stream);
}

}  // namespace fo
