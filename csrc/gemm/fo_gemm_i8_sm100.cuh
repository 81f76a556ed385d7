// tcgen05 kernels for products of 8-bit integers on B200 (sm_100a), see fo_gemm_i8.h.
//
// Wide: CTA pairs on 256 x 256 tiles, persistent, roles and epilogue as in fo_gemm_plain_sm100.cuh.  A stage of the
// operand ring holds the same 128 bytes of every row as there, which are 128 elements of K instead of 64, and one
// tcgen05.mma.kind::i8 takes 32 of them in the time kind::f16 takes 16.  The accumulators are exact 32-bit integers; the
// epilogue converts each once, multiplies by the two scales in fp32 and rounds to 16 bits.  Bound by the tensor pipe (94-96 % of its
// cycles) and, under load, by power: 8192^3 298 to 320 us (3.7 to 3.4 PFLOP/s) by itself, 378 us (2.9) sustained.
//
// Narrow: a batch of few tokens is bound by the weights' way through HBM, so here the weights are the 128 rows of the
// MMA and the tokens its 16 to 128 columns: no tensor-core row is spent on tokens that are not there, and a k-block
// costs the weights' 16 KB and little else (1 x 28672 x 8192: 39 us, 6.0 TB/s, against 55 us wide).  The CTAs of a cluster share
// a tile by splitting K and add their partial sums, exact integers, through distributed shared memory.
//
// Rows by expert.  The wide kernel's units are 256-row tiles that start at each expert's first row; the number
// of units is only known on the device, so every CTA sums up the experts' tiles in its prologue and finds a unit's
// expert by bisection.  A tile's rows past the expert's last one are multiplied (they are the next expert's)
// and not stored.
//
// Kernels that follow one another closely (ptx::grid_wait) begin before their inputs are written, so no load of an input goes the
// read-only way (ld.global.nc, which __ldg and const __restrict__ pointers are compiled to): it is for data that nobody writes while
// the kernel exists.
//
// Every wait is bounded: on expiry the role records a status code, raises a CTA-wide abort flag, the producer drains its
// TMA loads in flight, TMEM is freed and the kernel returns.
#pragma once
#include "../common/fo_pack16.cuh"
#include "../common/fo_ptx.cuh"
#include "fo_gemm_device.cuh"
#include "fo_gemm_i8.h"

namespace fo {

// Rows [0, first) and [last, M) of C, zeroed by `threads` threads of which this is number `at`.
__device__ __forceinline__ void i8_zero_outside(const GemmI8Params& p, int64_t at, int64_t threads) {
  const int first = min(max(__ldca(p.offsets), 0), p.M);
  const int last = min(max(__ldca(p.offsets + p.experts), 0), p.M);
  const int64_t nvec = p.N / 8;
  uint4* c = reinterpret_cast<uint4*>(p.C);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int64_t v = at; v < first * nvec; v += threads) c[v] = zero;
  for (int64_t v = last * nvec + at; v < p.M * nvec; v += threads) c[v] = zero;
}

// Rows of expert e, none where the offsets are out of order or out of range (which `bad` tells).
struct I8Segment {
  int lo, hi;
  bool bad;
};
__device__ __forceinline__ I8Segment i8_segment(const GemmI8Params& p, int e) {
  I8Segment s{__ldca(p.offsets + e), __ldca(p.offsets + e + 1), false};
  if (s.lo < 0 || s.hi < s.lo || s.hi > p.M) {
    s.bad = true;
    s.hi = s.lo = 0;
  }
  return s;
}

// ---------------------------------------------------------------------------- wide

constexpr int kI8Rows = 256, kI8Cols = 256;  // tile of a CTA pair
constexpr int kI8WideThreads = 64 + 256;

// MT = 2: each CTA of a pair owns two 128-row halves that share its B tile (512 x 256 per pair): a quarter fewer operand bytes a
// product, but the two accumulators fill TMEM, so nothing hides a tile's epilogue.
template <bool GROUPED, int MT>
struct I8WideSmem {
  static_assert(MT == 1 || !GROUPED, "experts' rows come in 256-row tiles");
  static constexpr int kStages = MT == 2 ? 4 : (GROUPED ? 5 : 6);  // the experts' tables take a stage's place
  static constexpr int kAHalfBytes = 128 * kI8BK;
  static constexpr int kABytes = MT * kAHalfBytes;
  static constexpr int kBBytes = 128 * kI8BK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kWarpBufBytes = 32 * 128;  // 32 rows x 64 16-bit columns
  static constexpr int kEpiOffset = kStages * kStageBytes;
  static constexpr int kTableOffset = kEpiOffset + 8 * kWarpBufBytes;
  static constexpr int kTableWords = GROUPED ? 2 * (kI8MaxExperts + 1) : 0;  // first unit and first row per expert
  static constexpr int kBarOffset = (kTableOffset + kTableWords * 4 + 7) / 8 * 8;
  static constexpr int kNumBars = 2 * kStages + 4;
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotalBytes = kMiscOffset + 16 + 1024;
};

template <bool BF16, bool GROUPED, int MT>
__global__ void __launch_bounds__(kI8WideThreads, 1)
    fo_gemm_i8_wide_kernel(const __grid_constant__ GemmI8Maps maps, const __grid_constant__ GemmI8Params p) {
  using L = I8WideSmem<GROUPED, MT>;
  constexpr int STAGES = L::kStages;
  constexpr int kRows = MT * kI8Rows;             // of a pair's tile
  constexpr int kAccStages = MT == 2 ? 1 : 2;     // tiles whose accumulators TMEM holds
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full_bar = full_bar + 2 * STAGES;
  uint64_t* tmem_empty_bar = full_bar + 2 * STAGES + 2;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  uint32_t* s_tmem_base = misc;
  volatile int* s_abort = reinterpret_cast<volatile int*>(misc + 1);
  [[maybe_unused]] int* s_first = reinterpret_cast<int*>(smem + L::kTableOffset);  // [experts + 1] first unit
  [[maybe_unused]] int* s_rows = s_first + kI8MaxExperts + 1;                      // [experts + 1] first row

  const int warp_idx = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int num_kb = (p.K + kI8BK - 1) / kI8BK;
  constexpr uint32_t kTmemCols = 2 * kI8Cols;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const bool leader = rank == 0;
  const int unit = static_cast<int>(blockIdx.x >> 1);
  const int num_units = static_cast<int>(gridDim.x >> 1);
  const uint64_t pipe_timeout = 4ull * p.timeout_ns + 1000000000ull;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      ptx::mbar_init(&full_bar[i], 1);
      ptx::mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&tmem_full_bar[i], 1);
      ptx::mbar_init(&tmem_empty_bar[i], 2 * 8);  // one arrival per epilogue warp of both CTAs
    }
    *s_abort = 0;
    ptx::mbar_fence_init();
  }
  if (warp_idx == 0 && lane == 0) {
    ptx::prefetch_tmap(&maps.a);
    ptx::prefetch_tmap(&maps.b);
    ptx::prefetch_tmap(&maps.c);
  }
  if (warp_idx == 1) {
    ptx::tmem_alloc_pair(s_tmem_base, kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncwarp();
  ptx::cluster_arrive_release();  // both CTAs' barriers are initialised before either receives a remote signal
  ptx::cluster_wait_acquire();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *s_tmem_base;
  ptx::grid_launch_dependents();
  ptx::grid_wait();

  int units_m = (p.M + kRows - 1) / kRows;
  if constexpr (GROUPED) {
    for (int e = threadIdx.x; e < p.experts; e += kI8WideThreads) {
      const I8Segment s = i8_segment(p, e);
      if (s.bad && blockIdx.x == 0) ptx::report_status(p.status, kStatusBadArgument, 3, e, __ldca(p.offsets + e));
      s_first[e] = (s.hi - s.lo + kI8Rows - 1) / kI8Rows;
      s_rows[e] = s.lo;
    }
    __syncthreads();
    if (warp_idx == 0) {
      int carry = 0;
      for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int own = e0 + lane < p.experts ? s_first[e0 + lane] : 0;
        int incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        if (e0 + lane < p.experts) s_first[e0 + lane] = carry + incl - own;
        carry += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) s_first[p.experts] = carry;
    }
    __syncthreads();
    units_m = s_first[p.experts];
  }
  // The tiles that are left over after the last full wave are computed as 256 x 128 halves if those fit one wave.
  const int sched_tiles = units_m * p.tiles_n;
  const int left = sched_tiles % num_units;
  const int tail_start = sched_tiles - (MT == 1 && 2 * left <= num_units ? left : 0);
  const int sched_len = 2 * sched_tiles - tail_start;

  struct Work {
    int row, row_end;  // this CTA's first row, and the end of the rows that are stored
    int n0, expert;
    bool narrow;  // 128 columns from n0
  };
  auto work_at = [&](int i) {
    Work w;
    w.narrow = MT == 1 && i >= tail_start;
    const int pos = w.narrow ? tail_start + (i - tail_start) / 2 : i;
    const TileCoord tc = tile_of_position(pos, units_m, p.tiles_n, p.raster_sw);
    w.n0 = tc.n * kI8Cols + (w.narrow ? ((i - tail_start) & 1) * (kI8Cols / 2) : 0);
    if constexpr (GROUPED) {
      int lo = 0, hi = p.experts;  // the last expert whose first unit is not behind tc.m has it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_first[mid] <= tc.m) {
          lo = mid;
        } else {
          hi = mid;
        }
      }
      w.expert = lo;
      w.row = s_rows[lo] + (tc.m - s_first[lo]) * kI8Rows + rank * 128;
      w.row_end = __ldca(p.offsets + lo + 1);
    } else {
      w.expert = 0;
      w.row = tc.m * kRows + rank * MT * 128;
      w.row_end = p.M;
    }
    return w;
  };

  if (warp_idx == 0) {
    // ------------------------------------------------------------------ TMA producer
    const bool elected = ptx::elect_one();
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued = 0;
    bool ok = true;
    for (int pos = unit; ok && pos < sched_len; pos += num_units) {
      const Work work = work_at(pos);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!ptx::mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, s_abort, pipe_timeout)) {
          if (elected) ptx::report_status(p.status, kStatusTimeoutSmemEmpty, pos, kb, stage);
          *s_abort = 1;
          ok = false;
          break;
        }
        if (elected) {
          uint8_t* sa = smem + stage * L::kStageBytes;
          // the leader's barrier collects the bytes of both CTAs
          if (leader) {
            ptx::mbar_arrive_expect_tx(&full_bar[stage], 2 * (work.narrow ? L::kStageBytes - L::kBBytes / 2 : L::kStageBytes));
          }
#pragma unroll
          for (int h = 0; h < MT; ++h) {
            ptx::tma_load_2d_pair(sa + h * L::kAHalfBytes, &maps.a, &full_bar[stage], kb * kI8BK, work.row + h * 128,
                                  ptx::kL2EvictNormal);
          }
          ptx::tma_load_3d_pair(sa + L::kABytes, work.narrow ? &maps.b_half : &maps.b, &full_bar[stage], kb * kI8BK,
                                work.n0 + rank * (work.narrow ? 64 : 128), work.expert, ptx::kL2EvictNormal);
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Drain (the follower's loads are counted on the leader's barriers; it relies on the cluster barrier at the end).
    for (int s = 0; elected && leader && s < STAGES; ++s) {
      if (issued <= static_cast<uint32_t>(s)) continue;
      const uint32_t par = ((issued - 1 - s) / STAGES) & 1u;
      for (uint32_t it = 0; it < ptx::kMbarDrainPolls; ++it) {
        if (ptx::mbar_try_wait(&full_bar[s], par)) break;
      }
    }
  } else if (warp_idx == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader) {
      const bool elected = ptx::elect_one();
      constexpr uint32_t idesc_full = ptx::make_idesc_s8(kI8Rows, kI8Cols);
      constexpr uint32_t idesc_half = ptx::make_idesc_s8(kI8Rows, kI8Cols / 2);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int pos = unit; ok && pos < sched_len; pos += num_units) {
        if (!ptx::mbar_wait_bounded(&tmem_empty_bar[acc], acc_phase ^ 1u, s_abort, pipe_timeout)) {
          if (elected) ptx::report_status(p.status, kStatusTimeoutTmemEmpty, pos, acc, 0);
          *s_abort = 1;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kI8Cols);
        const uint32_t idesc = MT == 1 && pos >= tail_start ? idesc_half : idesc_full;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!ptx::mbar_wait_bounded(&full_bar[stage], phase, s_abort, pipe_timeout)) {
            if (elected) ptx::report_status(p.status, kStatusTimeoutSmemFull, pos, kb, stage);
            *s_abort = 1;
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t sa = ptx::smem_u32(smem + stage * L::kStageBytes);
          const uint64_t da = ptx::make_smem_desc_sw128_kmajor(sa);
          const uint64_t db = ptx::make_smem_desc_sw128_kmajor(sa + L::kABytes);
          if (elected) {
            // advance 32 elements (32 B) along K inside the swizzle atom: +2 in 16-byte units
#pragma unroll
            for (int h = 0; h < MT; ++h) {
#pragma unroll
              for (int k = 0; k < kI8BK / 32; ++k) {
                ptx::umma_s8_ss_pair(tmem_d + static_cast<uint32_t>(h * kI8Cols),
                                     da + static_cast<uint64_t>(h * (L::kAHalfBytes >> 4) + 2 * k),
                                     db + static_cast<uint64_t>(2 * k), idesc, (kb > 0 || k > 0) ? 1u : 0u);
              }
            }
            ptx::umma_commit_pair(&empty_bar[stage], 3);  // slot reusable in both CTAs
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (elected) ptx::umma_commit_pair(&tmem_full_bar[acc], 3);  // accumulators complete in both CTAs
        __syncwarp();
        if (++acc == kAccStages) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp_idx - 2;
    const int wg = ew >> 2;         // every second 64-column chunk, or (MT = 2) all chunks of one half
    const int quad = warp_idx & 3;  // TMEM lane quadrant this warp may read
    uint8_t* buf = smem + L::kEpiOffset + ew * L::kWarpBufBytes;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const uint32_t tmem_empty_addr0 = ptx::mapa_shared(ptx::smem_u32(&tmem_empty_bar[0]), 0u);  // the leader's
    for (int pos = unit; ok && pos < sched_len; pos += num_units) {
      const Work work = work_at(pos);
      const int row0 = work.row + (MT == 2 ? wg * 128 : 0) + quad * 32;
      const bool exists = row0 < work.row_end;
      // whole rows of the warp leave by tensor store (which leaves out what lies beyond the matrix), an expert's last
      // ones by thread, since behind them are the next expert's
      const bool use_tma = !GROUPED || row0 + 32 <= work.row_end;
      const float sa = row0 + lane < work.row_end ? __ldca(p.SA + row0 + lane) : 0.f;
      const float* sb = p.SB + static_cast<size_t>(work.expert) * p.N + work.n0;
      ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(&tmem_full_bar[acc], acc_phase, s_abort, pipe_timeout));
      if (!ok) {
        if (lane == 0) {
          ptx::report_status(p.status, kStatusTimeoutTmemFull, pos, acc, 0);
          *s_abort = 1;
        }
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t t_row =
          tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>((MT == 2 ? wg : acc) * kI8Cols);
      constexpr int kStep = MT == 2 ? 1 : 2;  // chunks a warp steps by
      const bool last_tile = pos + num_units >= sched_len;
      const int chunks = (work.narrow ? kI8Cols / 2 : kI8Cols) / 64;
#pragma unroll 1
      for (int c = MT == 2 ? 0 : wg; c < chunks; c += kStep) {
        uint32_t v0[32], v1[32];
        ptx::tmem_ld_32x32b_x32(t_row + c * 64, v0);
        ptx::tmem_ld_32x32b_x32(t_row + c * 64 + 32, v1);
        ptx::tmem_ld_wait();
        if (c + kStep >= chunks) {
          // accumulator fully read by this warp: hand it back to the leader's MMA warp
          ptx::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster_tmem(tmem_empty_addr0 + static_cast<uint32_t>(acc) * 8u);
        }
        const int cols = p.N - work.n0 - c * 64;  // of the matrix, from the chunk's first on
        if (!exists || cols <= 0) continue;
        // On the CTA's last tile the operand ring is idle: the later chunks go through it instead of waiting for the
        // buffer's previous store.
        static_assert(8 * (kI8Cols / 64) * L::kWarpBufBytes <= L::kEpiOffset, "the ring must hold a tile");
        uint8_t* cbuf = buf;
        if (last_tile && c >= kStep) {
          cbuf = smem + (ew * (kI8Cols / 64) + c) * L::kWarpBufBytes;
        } else {
          if (lane == 0) ptx::bulk_wait_group_read<0>();
          __syncwarp();
        }
        // Row `lane` of the warp's slice, 16-byte pieces swizzled as the tensor store expects.
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t(&v)[32] = j < 4 ? v0 : v1;
          const int b = 8 * (j & 3);
          float s[8] = {};
          if (8 * j < cols) {  // N is a multiple of 8
            const float4 s0 = __ldca(reinterpret_cast<const float4*>(sb + c * 64 + 8 * j));
            const float4 s1 = __ldca(reinterpret_cast<const float4*>(sb + c * 64 + 8 * j + 4));
            s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w;
            s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
          }
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(static_cast<int32_t>(v[b + i])) * sa * s[i];
          *reinterpret_cast<uint4*>(cbuf + lane * 128 + ((j ^ (lane & 7)) * 16)) = make_uint4(
              pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
        }
        if (use_tma) {
          ptx::fence_proxy_async_smem();  // generic-proxy writes before the async-proxy read
          __syncwarp();
          if (lane == 0) {
            ptx::tma_store_2d(&maps.c, cbuf, work.n0 + c * 64, row0);
            ptx::bulk_commit_group();
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int lr = (lane >> 3) + 4 * i;
            const uint4 w = *reinterpret_cast<const uint4*>(cbuf + lr * 128 + (((lane & 7) ^ (lr & 7)) * 16));
            if (row0 + lr < work.row_end && 8 * (lane & 7) < cols) {
              ptx::st_v4(p.C + static_cast<size_t>(row0 + lr) * p.N + work.n0 + c * 64 + 8 * (lane & 7), w);
            }
          }
          __syncwarp();  // everybody has read the buffer before it is written again
        }
      }
      if (++acc == kAccStages) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if constexpr (GROUPED) {
      i8_zero_outside(p, static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x - 64, static_cast<int64_t>(gridDim.x) * 256);
    }
    // No tensor store may still read this CTA's shared memory when the CTA exits.
    if (lane == 0) ptx::bulk_wait_group<0>();
  }

  __syncwarp();  // lanes that drained join theirs: the barriers' aligned forms take whole warps
  ptx::tc_fence_before_sync();
  // Neither CTA may free TMEM or leave while the other can still signal its barriers or its MMAs read this CTA's
  // shared memory.  The release form: the leader waits for nobody's hand-back of its last accumulators, whose signals have
  // to arrive before it leaves.
  ptx::cluster_arrive_release();
  ptx::cluster_wait_acquire();
  if (warp_idx == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------- narrow

constexpr int kI8NarrowThreads = 64 + 128;

template <int TN, int S>
struct I8NarrowSmem {
  static constexpr int kWBytes = 128 * kI8BK;  // weights
  static constexpr int kTBytes = TN * kI8BK;   // tokens
  static constexpr int kStageBytes = kWBytes + kTBytes;
  static constexpr int kOwn = TN / S;  // tokens whose sums a CTA finishes
  static constexpr int kSlotBytes = kOwn * 128 * 4;
  static constexpr int kRecvBytes = (S - 1) * kSlotBytes;  // [senders][own / 4][128 channels] x 16 bytes
  // two CTAs per SM, one where 128 tokens leave no room for that
  static constexpr int kBudget = (TN == 128 ? 220 : 110) * 1024 - kRecvBytes;
  static constexpr int kStages = kBudget / kStageBytes < 8 ? kBudget / kStageBytes : 8;
  static constexpr int kRecvOffset = kStages * kStageBytes;
  static constexpr int kBarOffset = kRecvOffset + kRecvBytes;
  static constexpr int kNumBars = 2 * kStages + 1;
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotalBytes = kMiscOffset + 16 + 1024;
};

template <bool BF16>
__device__ __forceinline__ uint16_t to16(float f) {
  return static_cast<uint16_t>(pack2<BF16>(f, 0.f) & 0xffffu);
}

template <bool BF16, int TN, int S>
__global__ void __launch_bounds__(kI8NarrowThreads)
    fo_gemm_i8_narrow_kernel(const __grid_constant__ GemmI8Maps maps, const __grid_constant__ GemmI8Params p) {
  using L = I8NarrowSmem<TN, S>;
  constexpr int STAGES = L::kStages, kOwn = L::kOwn;
  static_assert(kOwn % 4 == 0 && STAGES >= 3, "sums are exchanged four tokens at a time");
  constexpr uint32_t kTmemCols = TN < 32 ? 32 : TN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full_bar = full_bar + 2 * STAGES;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  uint32_t* s_tmem_base = misc;
  volatile int* s_abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile uint32_t* s_peer_failed = misc + 2;  // set by a CTA of the cluster that sent nothing

  const int warp_idx = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = S > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / S;
  const int u = tile % p.token_tiles;   // token tiles of one weight tile follow one another
  const int n0 = tile / p.token_tiles * 128;
  const int num_kb = (p.K + kI8BK - 1) / kI8BK;
  const int kb_begin = num_kb * rank / S;
  const int kb_end = num_kb * (rank + 1) / S;
  const uint64_t pipe_timeout = 4ull * p.timeout_ns + 1000000000ull;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      ptx::mbar_init(&full_bar[i], 1);
      ptx::mbar_init(&empty_bar[i], 1);
    }
    ptx::mbar_init(tmem_full_bar, 1);
    *s_abort = 0;
    *s_peer_failed = 0;
    ptx::mbar_fence_init();
  }
  if (warp_idx == 0 && lane == 0) {
    ptx::prefetch_tmap(&maps.a);
    ptx::prefetch_tmap(&maps.b);
  }
  if (warp_idx == 1) {
    ptx::tmem_alloc(s_tmem_base, kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  // First phase of the cluster barrier: every CTA runs and has cleared its failure word before anybody stores into its
  // shared memory.  The epilogue waits for it ahead of its sends.
  if constexpr (S > 1) ptx::cluster_arrive_release();
  const uint32_t tmem_base = *s_tmem_base;
  ptx::grid_launch_dependents();
  ptx::grid_wait();

  // The tile's tokens; every warp looks them up by itself.  `work` is the same in all CTAs of the cluster.
  int token0 = u * TN, token_end = p.M, expert = 0;
  bool work = token0 < p.M;
  if (p.offsets != nullptr) {
    work = false;
    int carry = 0;
    // one tile, of the last tokens, looks at all experts: where every tile has found its own, nobody else does
    const bool checks = tile == p.token_tiles - 1;
    for (int e0 = 0; e0 < p.experts && (!work || checks); e0 += 32) {
      I8Segment s{0, 0, false};
      if (e0 + lane < p.experts) s = i8_segment(p, e0 + lane);
      if (s.bad && warp_idx == 0) ptx::report_status(p.status, kStatusBadArgument, 3, e0 + lane, s.lo);
      const int own = (s.hi - s.lo + TN - 1) / TN;
      int incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const int first = carry + incl - own;
      const uint32_t hit = __ballot_sync(0xffffffffu, u >= first && u < first + own);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        work = true;
        expert = e0 + l;
        token0 = __shfl_sync(0xffffffffu, s.lo + (u - first) * TN, l);
        token_end = __shfl_sync(0xffffffffu, s.hi, l);
      }
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  const int quad = warp_idx & 3;  // TMEM lane quadrant this warp may read
  const int row = quad * 32 + lane;
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);

  if (work && warp_idx == 0) {
    // ------------------------------------------------------------------ TMA producer
    const bool elected = ptx::elect_one();
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued = 0;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!ptx::mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, s_abort, pipe_timeout)) {
        if (elected) ptx::report_status(p.status, kStatusTimeoutSmemEmpty, tile, kb, stage);
        *s_abort = 1;
        break;
      }
      if (elected) {
        uint8_t* sw = smem + stage * L::kStageBytes;
        ptx::mbar_arrive_expect_tx(&full_bar[stage], L::kStageBytes);
        ptx::tma_load_3d(sw, &maps.b, &full_bar[stage], kb * kI8BK, n0, expert, ptx::kL2EvictNormal);
        ptx::tma_load_2d(sw + L::kWBytes, &maps.a, &full_bar[stage], kb * kI8BK, token0, ptx::kL2EvictNormal);
      }
      __syncwarp();
      ++issued;
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Drain: no bulk copy may still write this CTA's shared memory when it leaves (bounded).
    for (int s = 0; elected && s < STAGES; ++s) {
      if (issued <= static_cast<uint32_t>(s)) continue;
      const uint32_t par = ((issued - 1 - s) / STAGES) & 1u;
      for (uint32_t it = 0; it < ptx::kMbarDrainPolls; ++it) {
        if (ptx::mbar_try_wait(&full_bar[s], par)) break;
      }
    }
  } else if (work && warp_idx == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const bool elected = ptx::elect_one();
    constexpr uint32_t idesc = ptx::make_idesc_s8(128, TN);
    int stage = 0;
    uint32_t phase = 0;
    bool go = true;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!ptx::mbar_wait_bounded(&full_bar[stage], phase, s_abort, pipe_timeout)) {
        if (elected) ptx::report_status(p.status, kStatusTimeoutSmemFull, tile, kb, stage);
        *s_abort = 1;
        go = false;
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t sw = ptx::smem_u32(smem + stage * L::kStageBytes);
      const uint64_t dw = ptx::make_smem_desc_sw128_kmajor(sw);
      const uint64_t dt = ptx::make_smem_desc_sw128_kmajor(sw + L::kWBytes);
      if (elected) {
#pragma unroll
        for (int k = 0; k < kI8BK / 32; ++k) {
          ptx::umma_s8_ss(tmem_base, dw + static_cast<uint64_t>(2 * k), dt + static_cast<uint64_t>(2 * k), idesc,
                          (kb > kb_begin || k > 0) ? 1u : 0u);
        }
        ptx::umma_commit(&empty_bar[stage]);
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (go && elected) ptx::umma_commit(tmem_full_bar);
  }
  bool ok = work;
  if (work && warp_idx >= 2) {
    // ------------------------------------------------------------------ epilogue, first half
    ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(tmem_full_bar, 0, s_abort, pipe_timeout));
    if (!ok && lane == 0) {
      ptx::report_status(p.status, kStatusTimeoutTmemFull, tile, 0, 0);
      *s_abort = 1;
    }
    __syncwarp();  // the barrier's aligned form takes whole warps
    ptx::tc_fence_after_sync();
  }
  __syncwarp();
  if constexpr (S > 1) {
    ptx::cluster_wait_acquire();
    if (work && warp_idx >= 2) {
      if (ok) {
        // Sums of tokens that other CTAs finish go to their receive buffers.
#pragma unroll
        for (int c = 0; c < TN; c += 16) {
          uint32_t v[16];
          ptx::tmem_ld_32x32b_x16(t_row + c, v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int d = (c + 4 * j) / kOwn;
            if (d == rank) continue;
            const int slot = rank < d ? rank : rank - 1;
            const uint32_t dst = ptx::mapa_shared(ptx::smem_u32(smem + L::kRecvOffset), d) + slot * L::kSlotBytes +
                                 ((c + 4 * j - d * kOwn) / 4 * 128 + row) * 16;
            ptx::st_shared_cluster_v4(dst, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
      } else if (lane < S) {
        ptx::st_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(misc + 2), lane), 1u);
      }
    }
    __syncwarp();
    // Every CTA's partial sums have arrived (release / acquire at cluster scope).
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
    ok = work && *s_peer_failed == 0;  // a CTA that gave up sent nothing: nobody in the cluster stores
  }
  if (ok && warp_idx >= 2) {
    // ------------------------------------------------------------------ epilogue, second half
    const int n = n0 + row;
    const float sb = n < p.N ? __ldca(p.SB + static_cast<size_t>(expert) * p.N + n) : 0.f;
#pragma unroll 4
    for (int c = 0; c < kOwn; c += 4) {
      const int token = token0 + rank * kOwn + c;
      if (token >= token_end) break;
      uint32_t v[4];
      ptx::tmem_ld_32x32b_x4(t_row + rank * kOwn + c, v);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int s = 0; s < S - 1; ++s) {
        const uint4 x = *reinterpret_cast<const uint4*>(smem + L::kRecvOffset + s * L::kSlotBytes + (c / 4 * 128 + row) * 16);
        v[0] += x.x;
        v[1] += x.y;
        v[2] += x.z;
        v[3] += x.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (token + i < token_end && n < p.N) {
          const float f = static_cast<float>(static_cast<int32_t>(v[i])) * __ldca(p.SA + token + i) * sb;
          p.C[static_cast<size_t>(token + i) * p.N + n] = to16<BF16>(f);
        }
      }
    }
  }
  if (p.offsets != nullptr && warp_idx >= 2) {
    i8_zero_outside(p, static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x - 64, static_cast<int64_t>(gridDim.x) * 128);
  }

  // Nobody stores into another CTA's shared memory after the barrier: each leaves by itself.
  __syncwarp();
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp_idx == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace fo
