// Log-probabilities of given tokens from hidden states and the weight of a language model's head, and their gradients, without the logits in
// memory:
//
//   x = h W^T * inv_temp,   logp_r = x_rt - logsumexp_v x_rv,   G_rv = c_r inv_temp (delta_vt - p_rv),   dh = G W,   dW = G^T h
//
// Four products on one persistent CTA-pair kernel (tcgen05, 256 x 256 tiles over two SMs, operands by TMA, two accumulators in tensor memory):
//   stats   h W^T, whose epilogue leaves the largest logit and the sum of exponentials of each row and 128 columns (8 bytes instead of 512)
//           and the target's logit; a join over the vocabulary follows.  Where the whole G is small enough to be held, the epilogue also
//           writes the exponentials in 16 bits, relative to that largest logit, and the gradient is a pass over them;
//   grad    otherwise h W^T again, whose epilogue turns the logits into G in 16 bits: one product more, and G of a bounded number of rows is
//           all that is ever in memory
//   dh, dW  G W and G^T h
// Bound by the tensor cores: 2048 x 2048 x 32000 BF16 at 86 (statistics, exponentials written) and 87 % (dh) of their pipe, 180 us each, 1.49
// PFLOP/s; at 5376 x 4096 x 32000 1.05 ms for each of the three products, 1.33 PFLOP/s (to 1.43 in other runs), under the power cap.  The
// statistics' form spills 40 bytes stored, 56 loaded (168 registers, which ten warps leave it); the others nothing.
// Rows whose target does not count are left out before the first product: the others are brought together in order (their number stays on the
// device and bounds every loop), so that prompts and padding cost no tensor-core time.  A tile is 256 rows: without a gradient, up to that
// many rows stay where they are (with one they would put 0 * h of a row that does not count into dW, and h may hold anything there).
//
// G is rounded to the operands' type, as the tensor cores take it.  FP16 has no room for c p below 2^-24: G is multiplied by the power of two
// that takes the largest |c| to at most 2^15, and the products by its inverse.
#include "common.cuh"
#include "nx_api_objectives.h"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

#include <algorithm>

namespace {
using namespace nx;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBM = 128, kTile = 256, kBK = 64;
constexpr int kThreads = 320;  // warp 0: TMA, warp 1: MMA, warps 2..9: epilogue (two per quarter of the tensor memory's lanes)
constexpr int kOperandBytes = 128 * kBK * 2, kStageBytes = 2 * kOperandBytes, kStages = 5, kSlots = 4;
constexpr int kStoreBytes = 8 * kSlots * 2048;
constexpr int kSmemBytes = kStages * kStageBytes + kStoreBytes + 256;
constexpr int kTmemCols = 512;

enum Mode { kStats = 0, kGrad = 1, kInputGrad = 2, kWeightGrad = 3 };

struct Params {
  int64_t rows;             // of the whole call
  int64_t row0, cap;        // this launch: rows [row0, row0 + cap) of those that count
  const int32_t* count;     // how many count (null: all)
  const int32_t* index;     // where the r-th of them is (null: r)
  const void* targets;
  int64_t ignore;
  int targets_wide;
  int vocab, width;         // columns of the logits; columns of h
  int group;                // stats, grad: row tiles that pass over the vocabulary together
  int part_blocks;          // stats: 64-deep blocks that one accumulator sums
  int keep;                 // stats: write the exponentials
  int slices;               // input gradient: pieces of the vocabulary at most, whose sums have room
  float inv_temp;
  float2* part;             // stats: [2 * column tiles][part_ld]
  int64_t part_ld;
  float* tlogit;
  const float2* stats;      // grad
  const float* coef;
  const float* scale;       // FP16: {2^e, 2^-e}; null: 1
  void* out;                // input gradient: rows of pitch out_ld; weight gradient in FP32
  float* partial;           // input gradient of several slices: [slice][cap][width]
  int64_t out_ld;
  int add;                  // weight gradient: add to the FP32 rows
  int* status;
};

__device__ __forceinline__ int64_t live_rows(const Params& p) {
  const int64_t n = (p.count != nullptr ? static_cast<int64_t>(*p.count) : p.rows) - p.row0;
  return n < 0 ? 0 : (n < p.cap ? n : p.cap);
}
__device__ __forceinline__ int64_t place(const Params& p, int64_t row) { return p.index != nullptr ? p.index[p.row0 + row] : p.row0 + row; }
__device__ __forceinline__ int64_t target_of(const void* targets, int wide, int64_t at) {
  return wide ? reinterpret_cast<const int64_t*>(targets)[at] : static_cast<int64_t>(reinterpret_cast<const int32_t*>(targets)[at]);
}

struct Unit {
  int m0, n0, kb_begin, kb_end, slice;
};
struct Extent {
  int tiles_m, tiles_n, kb, units;
  int slices, per;          // input gradient: pieces of the vocabulary, and blocks of a piece
};
// Pieces of `blocks` 64-deep blocks for each of `tiles` tiles, so that the CTA pairs finish together: rounds times (blocks of a piece and six for
// handing a tile over).  Chosen here, from the number of rows that count: by all rows, 380 of 609 kept 48 of the 74 pairs busy (156 us; now 130
// to 141).
__device__ __forceinline__ void cut(Extent& e, int tiles, int blocks, int most) {
  int best = 0x7fffffff;
  e.slices = 1;
  e.per = blocks;
  for (int s = 1; s <= most; ++s) {
    const int per = (blocks + s - 1) / s;
    const int cost = (tiles * s + kNumSmsB200 / 2 - 1) / (kNumSmsB200 / 2) * (per + 6);
    if (cost < best) {
      best = cost;
      e.per = per;
      e.slices = (blocks + per - 1) / per;
    }
  }
}
template <int MODE>
__device__ __forceinline__ Extent extent(const Params& p, int live) {
  Extent e;
  if (MODE == kStats || MODE == kGrad) {
    e.tiles_m = (live + kTile - 1) / kTile;
    e.tiles_n = (p.vocab + kTile - 1) / kTile;
    e.kb = (p.width + kBK - 1) / kBK;
  } else if (MODE == kInputGrad) {
    e.tiles_m = (live + kTile - 1) / kTile;
    e.tiles_n = (p.width + kTile - 1) / kTile;
    e.kb = (p.vocab + kBK - 1) / kBK;
  } else {
    e.tiles_m = (p.vocab + kTile - 1) / kTile;
    e.tiles_n = (p.width + kTile - 1) / kTile;
    e.kb = (live + kBK - 1) / kBK;
  }
  e.slices = 1;
  e.per = e.kb;
  if (MODE == kInputGrad) cut(e, e.tiles_m * e.tiles_n, e.kb, p.slices);
  e.units = e.tiles_m * e.tiles_n * e.slices;
  return e;
}
template <int MODE>
__device__ __forceinline__ Unit unit_at(const Params& p, const Extent& e, int u) {
  Unit w;
  int tm, tn;
  w.slice = 0;
  w.kb_begin = 0;
  w.kb_end = e.kb;
  if (MODE == kStats || MODE == kGrad) {
    // a group of row tiles stays in L2 while the weight passes by once
    const int per = p.group * e.tiles_n, g = u / per, in = u - g * per;
    const int rows = min(p.group, e.tiles_m - g * p.group);
    tn = in / rows;
    tm = g * p.group + in - tn * rows;
  } else {
    tn = u % e.tiles_n;
    u /= e.tiles_n;
    tm = u % e.tiles_m;
    if (MODE == kInputGrad) {
      w.slice = u / e.tiles_m;
      w.kb_begin = w.slice * e.per;
      w.kb_end = min(e.kb, w.kb_begin + e.per);
    }
  }
  w.m0 = tm * kTile;
  w.n0 = tn * kTile;
  return w;
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) return pack_bf16x2(a, b);
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
// one row of a [32][32] staging tile in the 64-byte swizzle of its tensor map
template <bool BF>
__device__ __forceinline__ void stage_row(uint8_t* buf, int r, const float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 q;
    q.x = pack2<BF>(v[8 * i], v[8 * i + 1]);
    q.y = pack2<BF>(v[8 * i + 2], v[8 * i + 3]);
    q.z = pack2<BF>(v[8 * i + 4], v[8 * i + 5]);
    q.w = pack2<BF>(v[8 * i + 6], v[8 * i + 7]);
    *reinterpret_cast<uint4*>(buf + r * 64 + ((i ^ ((r >> 1) & 3)) << 4)) = q;
  }
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int MODE, bool BF>
__global__ void __launch_bounds__(kThreads, 1)
head_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out,
            const Params p, const uint32_t idesc) {
  constexpr bool kAmn = MODE == kWeightGrad, kBmn = MODE == kInputGrad || MODE == kWeightGrad;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0u) {  // the swizzle needs it; the same in both CTAs
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kStatusBadArgument);
    return;
  }
  uint8_t* const store_base = smem + kStages * kStageBytes;
  uint64_t* const full_bar = reinterpret_cast<uint64_t*>(store_base + kStoreBytes);
  uint64_t* const empty_bar = full_bar + kStages;
  uint64_t* const tfull_bar = empty_bar + kStages;
  uint64_t* const tempty_bar = tfull_bar + 2;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_ctarank();
  const int unit_first = static_cast<int>(blockIdx.x >> 1), unit_step = static_cast<int>(gridDim.x >> 1);
  const int m_off = static_cast<int>(cta_rank) * kBM;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 16);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  cluster_sync_all();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  const int live = static_cast<int>(live_rows(p));
  Extent e = extent<MODE>(p, live);
  if (MODE == kWeightGrad && p.add && live == 0) e.units = 0;  // nothing to add

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = unit_first; u < e.units && ok; u += unit_step) {
        const Unit w = unit_at<MODE>(p, e, u);
        const int m0 = w.m0 + m_off, bn0 = w.n0 + static_cast<int>(cta_rank) * 128;
        for (int kb = w.kb_begin; kb < w.kb_end; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            atomicCAS(p.status, 0, kStatusTimeoutProducer);
            break;
          }
          uint8_t* sa = smem + stage * kStageBytes;
          uint8_t* sb = sa + kOperandBytes;
          const int k0 = kb * kBK;
          // both CTAs' bytes are counted on the even CTA's barrier
          if (cta_rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * kStageBytes);
          const uint32_t bar = mapa_shared(smem_u32(&full_bar[stage]), 0);
          if constexpr (!kAmn) {
            tma_load_3d_pair(sa, &map_a, bar, k0, m0, 0);
          } else {
            tma_load_3d_pair(sa, &map_a, bar, m0, k0, 0);
            tma_load_3d_pair(sa + 64 * kBK * 2, &map_a, bar, m0 + 64, k0, 0);
          }
          if constexpr (!kBmn) {
            tma_load_3d_pair(sb, &map_b, bar, k0, bn0, 0);
          } else {
            tma_load_3d_pair(sb, &map_b, bar, bn0, k0, 0);
            tma_load_3d_pair(sb + 64 * kBK * 2, &map_b, bar, bn0 + 64, k0, 0);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // The even CTA's commits also arrive on this CTA's barriers: every stage filled here has been released before the CTA leaves.
      for (int s = 0; s < kStages && ok; ++s) {
        ok = mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, abort_flag);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (cta_rank == 0) {
      const bool leader = elect_one();
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int u = unit_first; u < e.units && ok; u += unit_step) {
        const Unit w = unit_at<MODE>(p, e, u);
        int kb = w.kb_begin;
        do {
          const int kb_stop = MODE == kStats ? min(w.kb_end, kb + p.part_blocks) : w.kb_end;
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1u, abort_flag))) {
            if (leader) atomicCAS(p.status, 0, kStatusTimeoutMma);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kTile);
          for (const int kb_first = kb; kb < kb_stop; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full_bar[stage], phase, abort_flag))) {
              ok = false;
              if (leader) atomicCAS(p.status, 0, kStatusTimeoutMma);
              break;
            }
            tc_fence_after_sync();
            const uint32_t sa = smem_u32(smem + stage * kStageBytes), sb = sa + kOperandBytes;
            const uint64_t da0 = make_smem_desc_sw128(sa, kAmn ? 64 * kBK * 2 : 16, 1024);
            const uint64_t db0 = make_smem_desc_sw128(sb, kBmn ? 64 * kBK * 2 : 16, 1024);
            if (leader) {
#pragma unroll
              for (int ks = 0; ks < kBK / 16; ++ks)
                umma_f16_ss_pair(tmem_d, da0 + static_cast<uint64_t>(kAmn ? ks * 128 : ks * 2),
                                 db0 + static_cast<uint64_t>(kBmn ? ks * 128 : ks * 2), idesc, (kb > kb_first || ks > 0) ? 1u : 0u);
              umma_commit_pair(&empty_bar[stage], 3);
            }
            __syncwarp();
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          if (leader) umma_commit_pair(&tfull_bar[acc], 3);
          __syncwarp();
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1u;
          }
        } while (kb < w.kb_end);
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint8_t* const st = store_base + (warp - 2) * (kSlots * 2048);
    int acc = 0;
    uint32_t acc_phase = 0;
    const float k2 = p.inv_temp * kLog2e;
    const float up = (MODE == kGrad && p.scale != nullptr) ? p.scale[0] : 1.0f;
    const float down = ((MODE == kInputGrad || MODE == kWeightGrad) && p.scale != nullptr) ? p.scale[1] : 1.0f;
    const int n_end = (MODE == kStats || MODE == kGrad) ? p.vocab : p.width;
    for (int u = unit_first; u < e.units; u += unit_step) {
      const Unit w = unit_at<MODE>(p, e, u);
      const int row0 = w.m0 + m_off + quarter * 32, row = row0 + lane;
      const int c0 = w.n0 + half * 128;  // this warp's columns: four chunks of 32
      // what the rows need, under the tile's MMAs
      int64_t at = 0;
      int tcol = -1;
      float2 mine = make_float2(0.0f, 0.0f);
      float c = 0.0f;
      bool counts = false;
      if (MODE != kWeightGrad && row < live) {
        at = place(p, row);
        if (MODE == kStats || MODE == kGrad) {
          const int64_t tg = target_of(p.targets, p.targets_wide, at);
          counts = tg != p.ignore && tg >= 0 && tg < p.vocab;
          tcol = counts ? static_cast<int>(tg) : -1;
          if (MODE == kGrad && counts) {
            mine = p.stats[p.row0 + row];
            c = p.coef[at] * p.inv_temp * up;
          }
        }
      }
      if constexpr (MODE == kStats) {
        // Accumulators of `part_blocks` blocks are added up here: the tensor cores' own sums truncate at every addition, which over 4096 columns
        // put an error of 1.45e-6 of itself into logp; with accumulators of 1024 columns 3.3e-7, at the same time.
        uint32_t x[4][32];
        const int chunks = c0 >= n_end ? 0 : min(4, (n_end - c0 + 31) / 32);
        bool ok = true;
        for (int kb = 0; kb < e.kb; kb += p.part_blocks) {
          const bool got = mbar_wait_bounded(&tfull_bar[acc], acc_phase, abort_flag);
          if (!__all_sync(0xffffffffu, got)) {
            if (lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kTile + half * 128);
          if (kb == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(taddr + i * 32, x[i]);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(taddr + i * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) x[i][j] = __float_as_uint(__uint_as_float(x[i][j]) + __uint_as_float(r[j]));
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty_bar[acc]), 0));
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
        if (!ok) break;
        if (chunks == 0) continue;
        if (n_end - c0 < 128) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + i * 32 + j >= n_end) x[i][j] = 0xff800000u;  // -inf
        }
        const int off = tcol - c0;
        if (__any_sync(0xffffffffu, off >= 0 && off < 128)) {
          float t = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (i * 32 + j == off) t = __uint_as_float(x[i][j]);
          if (off >= 0 && off < 128) p.tlogit[row] = t;
        }
        float top4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) top4[i] = __uint_as_float(x[i][0]);
#pragma unroll
        for (int j = 1; j < 32; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) top4[i] = fmaxf(top4[i], __uint_as_float(x[i][j]));
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        const float base = top == -INFINITY ? 0.0f : top;
        if (p.keep) {
          if (lane == 0) tma_store_wait_read<0>();  // the staging tiles are free once the last group has been read
          __syncwarp();
        }
        float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr float kLift = BF ? 0.0f : 15.0f;  // FP16: exponentials times 2^15, so that small ones keep their digits
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float d = __uint_as_float(x[i][j]) - base;
            v[j] = ex2(BF ? d * k2 : fmaf(d, k2, kLift));
            s4[j & 3] += v[j];
          }
          if (p.keep) stage_row<BF>(st + i * 2048, lane, v);
        }
        const float sum = ((s4[0] + s4[1]) + (s4[2] + s4[3])) * (BF ? 1.0f : 1.0f / 32768.0f);
        if (row < live) p.part[static_cast<int64_t>(w.n0 / 128 + half) * p.part_ld + row] = make_float2(top, sum);
        if (p.keep) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < live) {
            for (int i = 0; i < chunks; ++i) tma_store_3d(&map_out, st + i * 2048, c0 + 32 * i, row0, 0);
            tma_store_commit();
          }
        }
        continue;
      }
      const bool got = mbar_wait_bounded(&tfull_bar[acc], acc_phase, abort_flag);
      if (!__all_sync(0xffffffffu, got)) {
        if (lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kTile + half * 128);
      const int chunks = c0 >= n_end ? 0 : min(4, (n_end - c0 + 31) / 32);
      uint32_t r[32];
      if (chunks > 0) tmem_ld_32x32b_x32(taddr, r);
      auto release = [&] {  // everything this warp needs from the accumulator is in registers
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty_bar[acc]), 0));
      };
      if ((MODE == kGrad || MODE == kWeightGrad) && chunks > 0) {
        if (lane == 0) tma_store_wait_read<0>();  // the staging tiles are free once the last group has been read
        __syncwarp();
      }
#pragma unroll 1
      for (int i = 0; i < chunks; ++i) {
        const int col0 = c0 + i * 32;
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        if (i + 1 < chunks) tmem_ld_32x32b_x32(taddr + (i + 1) * 32, r);
        else release();
        const int valid = min(32, n_end - col0);
        if constexpr (MODE == kGrad) {
          // rows that do not count, those behind the last one among them, are zeros whatever the product left there
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float g = -c * ex2(fmaf(v[j] - mine.x, k2, -mine.y));
            if (col0 + j == tcol) g += c;
            v[j] = counts ? g : 0.0f;
          }
          stage_row<BF>(st + i * 2048, lane, v);
        } else if constexpr (MODE == kInputGrad) {
          if (row < live) {
            if (e.slices > 1) {
              float* o = p.partial + (static_cast<int64_t>(w.slice) * p.cap + row) * p.width + col0;
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (4 * j < valid) *reinterpret_cast<float4*>(o + 4 * j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            } else {
              uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + at * p.out_ld + col0;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (8 * j < valid) {
                  uint4 q;
                  q.x = pack2<BF>(v[8 * j] * down, v[8 * j + 1] * down);
                  q.y = pack2<BF>(v[8 * j + 2] * down, v[8 * j + 3] * down);
                  q.z = pack2<BF>(v[8 * j + 4] * down, v[8 * j + 5] * down);
                  q.w = pack2<BF>(v[8 * j + 6] * down, v[8 * j + 7] * down);
                  *reinterpret_cast<uint4*>(o + 8 * j) = q;
                }
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = e.kb > 0 ? v[j] * down : 0.0f;  // no row counts: the accumulator was never written
          if (p.partial != nullptr) {  // FP32 rows that several launches add up in
            if (row < p.vocab) {
              float* o = p.partial + static_cast<int64_t>(row) * p.width + col0;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (4 * j < valid) {
                  float4 q = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                  if (p.add) {
                    const float4 was = *reinterpret_cast<const float4*>(o + 4 * j);
                    q.x += was.x; q.y += was.y; q.z += was.z; q.w += was.w;
                  }
                  *reinterpret_cast<float4*>(o + 4 * j) = q;
                }
              }
            }
          } else {
            stage_row<BF>(st + i * 2048, lane, v);
          }
        }
      }
      if (chunks == 0) release();
      if constexpr (MODE == kGrad || MODE == kWeightGrad) {
        if (chunks > 0 && (MODE == kGrad || p.partial == nullptr)) {
          fence_proxy_async_smem();
          __syncwarp();
          const int row_end = MODE == kGrad ? static_cast<int>(p.cap) : p.vocab;
          if (lane == 0 && row0 < row_end) {
            for (int i = 0; i < chunks; ++i) tma_store_3d(&map_out, st + i * 2048, c0 + 32 * i, row0, 0);
            tma_store_commit();
          }
        }
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (MODE != kInputGrad && lane == 0) tma_store_wait_all();  // the staging tiles die with the CTA
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0) {  // a wait ran out: copies still in flight land before the shared memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(2000);
    __syncthreads();
  }
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------ up to 64 rows
// Scoring beside decoding: the time is that of reading the weight once.  The weight's rows are the tall operand here: every SM takes one run of
// the vocabulary, in groups of 32 rows so that the runs differ by at most one group (with 256 x 256 tiles 50257 rows were 197 tiles for 74 pairs,
// three rounds for 2.7), and a lane of the epilogue keeps maximum and sum of one row of a tile for every token, over all tiles of the run; lanes
// meet once, at its end.  8 x 50257 x 1600 BF16: 35 us (4.6 TB/s of weights), 256 x 256 tiles 44.  The form for 64 tokens keeps 192 values per lane
// and spills (255 registers; 148 bytes stored, 164 loaded): 50 us with L2 flushed, where 32 tokens take 46 and a plain read of the weight 37.
constexpr int kFewRows = 64, kFewThreads = 192;  // warp 0: TMA, warp 1: MMA, warps 2..5: a quarter of the 128 lanes each
constexpr int kGroupBytes = 32 * kBK * 2, kFewAccumulators = 4;
template <int NT>
struct Few {
  static constexpr int kStageBytes = 4 * kGroupBytes + NT * kBK * 2;
  static constexpr int kStages = 200 * 1024 / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes;
  static constexpr int kTmemCols = kFewAccumulators * NT;
};

template <int NT, bool BF>
__global__ void __launch_bounds__(kFewThreads, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_h, const Params p, const uint32_t idesc) {
  using F = Few<NT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full_bar[F::kStages], empty_bar[F::kStages], tfull_bar[kFewAccumulators], tempty_bar[kFewAccumulators];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ int32_t target[NT];
  __shared__ float2 met[4][NT];
  volatile int* const abort_flag = &abort_word;
  if ((smem_u32(smem) & 1023u) != 0u) {  // the swizzle needs it
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kStatusBadArgument);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < F::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kFewAccumulators; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 4);
    }
    abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, F::kTmemCols);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_h);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  const int rows = static_cast<int>(p.rows), kb_all = (p.width + kBK - 1) / kBK;
  const int64_t groups = (p.vocab + 31) / 32;
  const int g0 = static_cast<int>(groups * blockIdx.x / gridDim.x), g1 = static_cast<int>(groups * (blockIdx.x + 1) / gridDim.x);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int g = g0; g < g1 && ok; g += 4) {
        const int here = min(4, g1 - g);
        for (int kb = 0; kb < kb_all; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            atomicCAS(p.status, 0, kStatusTimeoutProducer);
            break;
          }
          uint8_t* const sa = smem + stage * F::kStageBytes;
          mbar_arrive_expect_tx(&full_bar[stage], static_cast<uint32_t>(here * kGroupBytes + NT * kBK * 2));
          for (int i = 0; i < here; ++i) tma_load_3d(sa + i * kGroupBytes, &map_w, &full_bar[stage], kb * kBK, (g + i) * 32, 0);
          tma_load_3d(sa + 4 * kGroupBytes, &map_h, &full_bar[stage], kb * kBK, 0, 0);
          if (++stage == F::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int g = g0; g < g1 && ok; g += 4) {
      for (int kb = 0; kb < kb_all && ok;) {
        const int stop = min(kb_all, kb + p.part_blocks);
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1u, abort_flag))) {
          if (leader) atomicCAS(p.status, 0, kStatusTimeoutMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        for (const int first = kb; kb < stop; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full_bar[stage], phase, abort_flag))) {
            if (leader) atomicCAS(p.status, 0, kStatusTimeoutMma);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(smem + stage * F::kStageBytes);
          const uint64_t da = make_smem_desc_sw128(sa, 16, 1024), db = make_smem_desc_sw128(sa + 4 * kGroupBytes, 16, 1024);
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < kBK / 16; ++ks)
              umma_f16_ss(tmem_base + static_cast<uint32_t>(acc * NT), da + static_cast<uint64_t>(ks * 2), db + static_cast<uint64_t>(ks * 2), idesc,
                          (kb > first || ks > 0) ? 1u : 0u);
            umma_commit(&empty_bar[stage]);
          }
          __syncwarp();
          if (++stage == F::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (leader) umma_commit(&tfull_bar[acc]);
        __syncwarp();
        if (++acc == kFewAccumulators) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
    }
  } else {
    const int quarter = warp & 3;  // the lanes of tensor memory that this warp may read
    for (int j = threadIdx.x - 64; j < NT; j += 128) {
      int32_t t = -1;
      if (j < rows) {
        const int64_t tg = target_of(p.targets, p.targets_wide, j);
        if (tg != p.ignore && tg >= 0 && tg < p.vocab) t = static_cast<int32_t>(tg);
      }
      target[j] = t;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const float k2 = p.inv_temp * kLog2e;
    float top[NT], sum[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) top[j] = -INFINITY, sum[j] = 0.0f;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int g = g0; g < g1 && ok; g += 4) {
      uint32_t x[NT];
      for (int kb = 0; kb < kb_all; kb += p.part_blocks) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], acc_phase, abort_flag))) {
          if (lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t at = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * NT);
#pragma unroll
        for (int i = 0; i < NT / 16; ++i) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(at + i * 16, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            x[i * 16 + j] = kb == 0 ? r[j] : __float_as_uint(__uint_as_float(x[i * 16 + j]) + __uint_as_float(r[j]));
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty_bar[acc]);
        if (++acc == kFewAccumulators) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) break;
      // this lane's row of the vocabulary; groups that the last tile does not have hold what an earlier one left
      const int v = (g + quarter) * 32 + lane;
      if (g + quarter < g1 && v < p.vocab) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float l = __uint_as_float(x[j]);
          if (target[j] == v) p.tlogit[j] = l;
          const float m = fmaxf(top[j], l), base = m == -INFINITY ? 0.0f : m;
          sum[j] = sum[j] * ex2((top[j] - base) * k2) + ex2((l - base) * k2);
          top[j] = m;
        }
      }
    }
    // the lanes of a warp, then the warps
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float m = warp_max(top[j]);
      const float s = warp_sum(top[j] == -INFINITY ? sum[j] : sum[j] * ex2((top[j] - m) * k2));
      if (lane == 0) met[quarter][j] = make_float2(m, s);
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int j = threadIdx.x - 64; j < rows; j += 128) {
      float m = met[0][j].x, s = 0.0f;
      for (int w = 1; w < 4; ++w) m = fmaxf(m, met[w][j].x);
      for (int w = 0; w < 4; ++w) {
        const float2 v = met[w][j];
        s += v.x == -INFINITY ? v.y : v.y * ex2((v.x - m) * k2);
      }
      p.part[static_cast<int64_t>(blockIdx.x) * p.part_ld + j] = make_float2(m, s);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0) {  // a wait ran out: copies still in flight land before the shared memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(2000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, F::kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------ around the products
// index[0 .. count) = the rows whose target counts, in order; the others' logp is written.  One block: a thread takes a run of rows.
constexpr int kPickThreads = 1024;
__global__ void __launch_bounds__(kPickThreads) pick_rows_kernel(const void* __restrict__ targets, int wide, int64_t rows, int64_t ignore, int vocab,
                                                                 int32_t* __restrict__ index, int32_t* __restrict__ count, float* __restrict__ logp) {
  __shared__ int warp_total[32];
  pdl_dependency();
  pdl_trigger();
  const int64_t per = (rows + kPickThreads - 1) / kPickThreads, first = threadIdx.x * per, end = min(rows, first + per);
  int mine = 0;
  for (int64_t r = first; r < end; ++r) {
    const int64_t t = target_of(targets, wide, r);
    const bool in = t >= 0 && t < vocab;
    if (t != ignore && in) ++mine;
    else logp[r] = t == ignore ? 0.0f : NAN;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_total[warp] = upto;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < 32; ++i) {
    if (i < warp) before += warp_total[i];
    all += warp_total[i];
  }
  int at = before + upto - mine;
  for (int64_t r = first; r < end; ++r) {
    const int64_t t = target_of(targets, wide, r);
    if (t != ignore && t >= 0 && t < vocab) index[at++] = static_cast<int32_t>(r);
  }
  if (threadIdx.x == 0) *count = all;
}

// Row r of `out` = row index[r] of `h` for r < count, zeros up to the next multiple of 64 (the reduction of the weight gradient reads them)
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint4* __restrict__ h, int64_t ld, const int32_t* __restrict__ index,
                                                          const int32_t* __restrict__ count, uint4* __restrict__ out, int pieces, int64_t rows) {
  pdl_dependency();
  pdl_trigger();
  const int64_t n = *count, end = min((n + 63) / 64 * 64, rows);
  for (int64_t r = blockIdx.x; r < end; r += gridDim.x) {
    const uint4* src = r < n ? h + index[r] * ld : nullptr;
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) out[r * pieces + i] = src != nullptr ? src[i] : make_uint4(0, 0, 0, 0);
  }
}

// Joins the column tiles' maxima and sums of a row.  Eight rows per block (64 contiguous bytes of every tile), a quarter of a warp's lanes per row
// and four loads of each in flight: 1188 tiles of 380 rows took 24 us with 32 rows per block and a load at a time, 9 now.
constexpr int kJoinRows = 8;
__global__ void __launch_bounds__(1024) join_kernel(const Params p, int parts, float* __restrict__ logp, float2* __restrict__ stats) {
  __shared__ float2 share[32][kJoinRows + 1];
  pdl_dependency();
  pdl_trigger();
  const int64_t live = live_rows(p), row0 = static_cast<int64_t>(blockIdx.x) * kJoinRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in = lane & (kJoinRows - 1);
  if (row0 >= live) return;
  const float k2 = p.inv_temp * kLog2e;
  float top = -INFINITY, sum = 0.0f;
  auto take = [&](const float2 v) {
    if (v.x > top) {
      if (top != -INFINITY) sum *= ex2((top - v.x) * k2);
      top = v.x;
    }
    // a part of nothing but -inf has the sum 0 (or NaN)
    sum += v.x == -INFINITY ? v.y : v.y * ex2((v.x - top) * k2);
  };
  if (row0 + in < live) {
    const float2* const from = p.part + row0 + in;
    int i = threadIdx.x / kJoinRows;
    for (; i + 3 * 128 < parts; i += 4 * 128) {
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = from[(i + u * 128) * p.part_ld];
#pragma unroll
      for (int u = 0; u < 4; ++u) take(v[u]);
    }
    for (; i < parts; i += 128) take(from[i * p.part_ld]);
  }
  auto meet = [&](int o) {  // with the lane that is `o` away and has the same row
    const float2 v = make_float2(__shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, sum, o));
    const float m = fmaxf(top, v.x);
    sum = (top == -INFINITY ? sum : sum * ex2((top - m) * k2)) + (v.x == -INFINITY ? v.y : v.y * ex2((v.x - m) * k2));
    top = m;
  };
  meet(8);
  meet(16);
  if (lane < kJoinRows) share[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp >= kJoinRows) return;
  const float2 v = share[lane][warp];  // a warp takes a row, a lane a warp's share
  const float m = warp_max(v.x);
  const float s = warp_sum(v.x == -INFINITY ? v.y : v.y * ex2((v.x - m) * k2));
  const int64_t mine = row0 + warp;
  if (lane == 0 && mine < live) {
    const int64_t at = place(p, mine);
    const int64_t tg = target_of(p.targets, p.targets_wide, at);
    if (tg == p.ignore || tg < 0 || tg >= p.vocab) {
      logp[at] = tg == p.ignore ? 0.0f : NAN;
      return;
    }
    logp[at] = (p.tlogit[mine] - m) * p.inv_temp - logf(s);
    stats[p.row0 + mine] = make_float2(m, log2f(s));
  }
}

// scale = {2^e, 2^-e} with the largest |coef * inv_temp| * 2^e of the rows that count in [2^14, 2^15); one where none is positive and finite
__global__ void __launch_bounds__(1024) coef_scale_kernel(const float* __restrict__ coef, const void* __restrict__ targets, int wide, int64_t ignore,
                                                          int64_t n, float inv_temp, float* __restrict__ scale) {
  __shared__ float scratch[32];
  pdl_dependency();
  pdl_trigger();
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const float v = fabsf(coef[i]) * inv_temp;
    if (v <= 3.0e38f && target_of(targets, wide, i) != ignore) top = fmaxf(top, v);
  }
  top = block_max(top, scratch);
  if (threadIdx.x == 0) {
    int e = 0;
    if (top > 0.0f) {
      frexpf(top, &e);
      e = 15 - e;
      e = max(-100, min(100, e));
    }
    scale[0] = ldexpf(1.0f, e);
    scale[1] = ldexpf(1.0f, -e);
  }
}

template <bool BF>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  if constexpr (BF) {
    unpack_bf16x2(w, a, b);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
  }
}
template <bool BF>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3]), pack2<BF>(v[4], v[5]), pack2<BF>(v[6], v[7]));
}

// Exponentials relative to the largest logit of their row and 128 columns -> gradient of the logits: each times the row's coefficient and the
// 128 columns' share, the target's c more.  Rows up to the next multiple of 256 are cleared: the products read them.  from and to may be the same.
// 5376 x 32000 BF16 in place: 125 to 143 us, 4.8 to 5.5 TB/s, bound by these bytes.
template <bool BF>
__global__ void __launch_bounds__(256) weigh_kernel(const Params p, const uint4* from, uint4* to, int64_t ld) {
  pdl_dependency();
  pdl_trigger();
  const int64_t live = live_rows(p), end = min((live + kTile - 1) / kTile * kTile, p.cap);
  const float k2 = p.inv_temp * kLog2e, up = p.scale != nullptr ? p.scale[0] : 1.0f;
  const int pieces = (p.vocab + 7) / 8;
  for (int64_t r = blockIdx.x; r < end; r += gridDim.x) {
    uint4* const out = to + r * ld;
    int64_t tg = -1;
    float c = 0.0f;
    float2 mine = make_float2(0.0f, 0.0f);
    if (r < live) {
      const int64_t at = place(p, r);
      tg = target_of(p.targets, p.targets_wide, at);
      if (tg == p.ignore || tg < 0 || tg >= p.vocab) tg = -1;
      c = p.coef[at] * p.inv_temp * up;
      mine = p.stats[r];
    }
    if (tg < 0) {
      for (int i = threadIdx.x; i < pieces; i += blockDim.x) out[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const uint4* const in = from + r * ld;
    const int tpiece = static_cast<int>(tg >> 3);
    auto piece = [&](int i, const uint4& q, float share) {
      const float f = -c * ex2(fmaf(share - mine.x, k2, -mine.y)) * (BF ? 1.0f : 1.0f / 32768.0f);
      float v[8];
      unpack2<BF>(q.x, v[0], v[1]);
      unpack2<BF>(q.y, v[2], v[3]);
      unpack2<BF>(q.z, v[4], v[5]);
      unpack2<BF>(q.w, v[6], v[7]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * f;
      if (i == tpiece) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i * 8 + j == tg) v[j] += c;
      }
      out[i] = pack8<BF>(v);
    };
    const float2* const shares = p.part + r;
    int i = threadIdx.x;
    for (; i + 3 * 256 < pieces; i += 4 * 256) {
      uint4 q[4];
      float share[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        q[u] = in[i + u * 256];
        share[u] = shares[static_cast<int64_t>((i + u * 256) >> 4) * p.part_ld].x;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) piece(i + u * 256, q[u], share[u]);
    }
    for (; i < pieces; i += 256) piece(i, in[i], shares[static_cast<int64_t>(i >> 4) * p.part_ld].x);
  }
}

// Rows of dh = sum of the slices in order, times the inverse scale
template <bool BF>
__global__ void __launch_bounds__(128) slices_kernel(const Params p) {
  pdl_dependency();
  pdl_trigger();
  const int64_t live = live_rows(p);
  const Extent e = extent<kInputGrad>(p, static_cast<int>(live));
  if (e.slices == 1) return;  // the product has written the rows itself
  const float down = p.scale != nullptr ? p.scale[1] : 1.0f;
  for (int64_t r = blockIdx.x; r < live; r += gridDim.x) {
    uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + place(p, r) * p.out_ld;
    for (int i = threadIdx.x * 8; i < p.width; i += blockDim.x * 8) {
      float v[8] = {};
      for (int s = 0; s < e.slices; ++s) {
        const float4* q = reinterpret_cast<const float4*>(p.partial + (static_cast<int64_t>(s) * p.cap + r) * p.width + i);
        const float4 a = q[0], b = q[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= down;
      *reinterpret_cast<uint4*>(o + i) = pack8<BF>(v);
    }
  }
}

// Rows of dh whose target does not count (or lies outside the vocabulary): zeros
__global__ void __launch_bounds__(128) clear_rows_kernel(const void* __restrict__ targets, int wide, int64_t rows, int64_t ignore, int vocab,
                                                         uint4* __restrict__ out, int64_t ld, int pieces) {
  pdl_dependency();
  pdl_trigger();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t t = target_of(targets, wide, r);
    if (t != ignore && t >= 0 && t < vocab) continue;
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) out[r * ld + i] = make_uint4(0, 0, 0, 0);
  }
}

template <bool BF>
__global__ void __launch_bounds__(256) narrow_kernel(const float* __restrict__ x, uint4* __restrict__ out, int64_t pieces) {
  pdl_dependency();
  pdl_trigger();
  NX_GRID_STRIDE(i, pieces) {
    const float4 a = reinterpret_cast<const float4*>(x)[2 * i], b = reinterpret_cast<const float4*>(x)[2 * i + 1];
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    out[i] = pack8<BF>(v);
  }
}

// ------------------------------------------------------------------------------------------------ launches
template <int MODE, bool BF>
int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const Params& p, int64_t units, cudaStream_t st) {
  auto kern = head_kernel<MODE, BF>;
  NX_ALLOW_SMEM(kern, kSmemBytes);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(units, kNumSmsB200 / 2)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const uint32_t fmt = BF ? kFmtBF16 : kFmtF16;
  const uint32_t idesc = make_idesc(fmt, fmt, MODE == kWeightGrad, MODE == kInputGrad || MODE == kWeightGrad, kTile, kTile);
  if (cudaLaunchKernelEx(&cfg, kern, a, b, out, p, idesc) != cudaSuccess) {
    (void)cudaGetLastError();
    return -2;
  }
  return 0;
}

int64_t tiles(int64_t n) { return (n + kTile - 1) / kTile; }

template <int NT, bool BF>
int launch_few(const NxHeadArgs* a, const Params& p, int blocks, cudaStream_t st) {
  const CUtensorMapDataType dt = BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap w, h;
  int rc;
  if ((rc = make_tensor_map_3d(&w, dt, 2, a->weight, a->width, a->vocab, 1, a->ld_weight, 0, kBK, 32)) != 0 ||
      (rc = make_tensor_map_3d(&h, dt, 2, a->hidden, a->width, a->rows, 1, a->ld_hidden, 0, kBK, NT)) != 0)
    return rc;
  auto kern = few_rows_kernel<NT, BF>;
  NX_ALLOW_SMEM(kern, Few<NT>::kSmemBytes);
  const uint32_t fmt = BF ? kFmtBF16 : kFmtF16;
  return launch_pdl(kern, dim3(blocks), dim3(kFewThreads), Few<NT>::kSmemBytes, st, w, h, p, make_idesc(fmt, fmt, false, false, 128, NT));
}
template <bool BF>
int launch_few(const NxHeadArgs* a, const Params& p, int blocks, cudaStream_t st) {
  if (a->rows <= 16) return launch_few<16, BF>(a, p, blocks, st);
  return a->rows <= 32 ? launch_few<32, BF>(a, p, blocks, st) : launch_few<64, BF>(a, p, blocks, st);
}

// K-major operand of [rows][k], or MN-major of [k][mn]; 128-byte swizzle
int map_k(CUtensorMap* m, const NxHeadArgs* a, const void* base, int64_t k, int64_t rows, int64_t ld) {
  const CUtensorMapDataType dt = a->dtype == NX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return make_tensor_map_3d(m, dt, 2, base, k, rows, 1, ld, 0, kBK, 128);
}
int map_mn(CUtensorMap* m, const NxHeadArgs* a, const void* base, int64_t mn, int64_t k, int64_t ld) {
  const CUtensorMapDataType dt = a->dtype == NX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return make_tensor_map_3d(m, dt, 2, base, mn, k, 1, ld, 0, 64, kBK);
}
int map_store(CUtensorMap* m, const NxHeadArgs* a, const void* base, int64_t cols, int64_t rows, int64_t ld) {
  const CUtensorMapDataType dt = a->dtype == NX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return make_tensor_map_3d(m, dt, 2, base, cols, rows, 1, ld, 0, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

bool args_ok(const NxHeadArgs* a) {
  auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  auto split = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) != 0; };  // pairs of floats
  return a != nullptr && !split(a->stats) && !split(a->part) && (a->dtype == NX_BF16 || a->dtype == NX_F16) && a->rows > 0 &&
         a->rows <= (1 << 30) && a->width > 0 && a->width % 8 == 0 &&
         a->vocab > 0 && a->vocab <= (1 << 30) && a->hidden != nullptr && a->weight != nullptr && a->targets != nullptr && !off(a->hidden) &&
         !off(a->weight) && a->ld_hidden % 8 == 0 && a->ld_weight % 8 == 0 && a->ld_hidden >= a->width && a->ld_weight >= a->width &&
         a->stats != nullptr && a->status != nullptr && (a->index == nullptr) == (a->count == nullptr) &&
         (a->index == nullptr) == (a->gathered == nullptr) && !off(a->gathered) &&
         a->part_rows > 0 && a->part_rows % kTile == 0 &&
         (a->weights == nullptr || (!off(a->weights) && a->part_rows >= a->rows && a->ld_weights >= a->vocab && a->ld_weights % 64 == 0));
}

Params base_params(const NxHeadArgs* a) {
  Params p{};
  p.rows = a->rows;
  p.cap = a->rows;
  p.count = a->count;
  p.index = a->index;
  p.targets = a->targets;
  p.targets_wide = a->targets_wide;
  p.ignore = a->ignore_index;
  p.vocab = a->vocab;
  p.width = a->width;
  p.inv_temp = a->inv_temp;
  p.stats = reinterpret_cast<const float2*>(a->stats);
  p.status = a->status;
  p.slices = 1;
  p.part_blocks = 1024 / kBK;
  p.part = reinterpret_cast<float2*>(a->part);
  p.part_ld = a->part_rows;
  // row tiles whose part of h is about 40 MB pass over the vocabulary together
  p.group = static_cast<int>(std::max<int64_t>(1, (40ll << 20) / (static_cast<int64_t>(kTile) * a->width * 2)));
  return p;
}

int gather(const NxHeadArgs* a, cudaStream_t st) {
  const int pieces = a->width / 8;
  NX_PDL(gather_rows_kernel, static_cast<unsigned>(std::min<int64_t>(a->rows, kNumSmsB200 * 8)), 256, 0, st,
         reinterpret_cast<const uint4*>(a->hidden), a->ld_hidden / 8, a->index, a->count, reinterpret_cast<uint4*>(a->gathered), pieces,
         (a->rows + 63) / 64 * 64);
  return 0;
}
}  // namespace

#define NX_HEAD(MODE_, ...) (a->dtype == NX_BF16 ? launch<MODE_, true>(__VA_ARGS__) : launch<MODE_, false>(__VA_ARGS__))

extern "C" int nx_head_logprobs(const NxHeadArgs* a, float* logp, float* tlogit, nx_stream_t stream) {
  if (!args_ok(a) || logp == nullptr || a->part == nullptr || tlogit == nullptr) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc;
  if (a->index != nullptr) {
    NX_PDL(pick_rows_kernel, 1, kPickThreads, 0, st, a->targets, a->targets_wide, a->rows, a->ignore_index, a->vocab, a->index, a->count, logp);
    if ((rc = gather(a, st)) != 0) return rc;
  }
  Params p = base_params(a);
  p.tlogit = tlogit;
  auto join = [&](int64_t rows, int parts) {
    NX_PDL(join_kernel, static_cast<unsigned>((rows + kJoinRows - 1) / kJoinRows), 1024, 0, st, p, parts, logp, reinterpret_cast<float2*>(a->stats));
    return 0;
  };
  if (a->index == nullptr && a->rows <= kFewRows) {
    // a part for every SM; `part` has room for one per 128 columns
    const int blocks = static_cast<int>(std::min<int64_t>(kNumSmsB200, 2 * tiles(a->vocab)));
    rc = a->dtype == NX_BF16 ? launch_few<true>(a, p, blocks, st) : launch_few<false>(a, p, blocks, st);
    return rc != 0 ? rc : join(a->rows, blocks);
  }
  const void* h = a->index != nullptr ? a->gathered : a->hidden;
  const int64_t ldh = a->index != nullptr ? a->width : a->ld_hidden;
  CUtensorMap ma, mb;
  if ((rc = map_k(&mb, a, a->weight, a->width, a->vocab, a->ld_weight)) != 0) return rc;
  p.keep = a->weights != nullptr;
  for (; p.row0 < a->rows; p.row0 += a->part_rows) {  // as many rows at a time as `part` has room for
    const int64_t here = std::min(a->part_rows, a->rows - p.row0);
    if ((rc = map_k(&ma, a, static_cast<const uint16_t*>(h) + p.row0 * ldh, a->width, here, ldh)) != 0) return rc;
    CUtensorMap mo = ma;
    p.cap = tiles(here) * kTile;
    if (p.keep && (rc = map_store(&mo, a, a->weights, a->vocab, p.cap, a->ld_weights)) != 0) return rc;
    if ((rc = NX_HEAD(kStats, ma, mb, mo, p, tiles(here) * tiles(a->vocab), st)) != 0) return rc;
    // the last column tile may have no second half
    if ((rc = join(here, static_cast<int>((a->vocab + 127) / 128))) != 0) return rc;
  }
  return 0;
}

extern "C" int nx_head_logprobs_grad(const NxHeadArgs* a, const NxHeadGrad* g, nx_stream_t stream) {
  if (!args_ok(a) || a->index == nullptr || g == nullptr || g->coef == nullptr || g->logit_grad == nullptr || g->chunk < kTile ||
      g->chunk % kTile != 0 ||
      g->ld_logit_grad < a->vocab || g->ld_logit_grad % 64 != 0 || (reinterpret_cast<uintptr_t>(g->logit_grad) & 15) != 0 ||
      (a->dtype == NX_F16 && g->scale == nullptr) || g->slices < 1 || (g->slices > 1 && g->slice_sums == nullptr) ||
      (reinterpret_cast<uintptr_t>(g->d_hidden) & 15) != 0 || (reinterpret_cast<uintptr_t>(g->d_weight) & 15) != 0 ||
      (g->d_weight != nullptr && g->chunk < a->rows && g->weight_sums == nullptr) ||
      (a->weights != nullptr && (a->part == nullptr || g->chunk < a->rows || g->ld_logit_grad != a->ld_weights)))
    return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc;
  const bool half = a->dtype == NX_F16;
  if (half) NX_PDL(coef_scale_kernel, 1, 1024, 0, st, g->coef, a->targets, a->targets_wide, a->ignore_index, a->rows, a->inv_temp, g->scale);
  if (a->weights == nullptr && (rc = gather(a, st)) != 0) return rc;
  const void* h = a->gathered;
  const int64_t ldh = a->width;
  if (g->d_hidden != nullptr)
    NX_PDL(clear_rows_kernel, static_cast<unsigned>(std::min<int64_t>(a->rows, kNumSmsB200 * 16)), 128, 0, st, a->targets, a->targets_wide, a->rows,
           a->ignore_index, a->vocab, reinterpret_cast<uint4*>(g->d_hidden), static_cast<int64_t>(a->width / 8), a->width / 8);
  const bool sums = g->d_weight != nullptr && g->chunk < a->rows;  // several launches add up in FP32
  CUtensorMap w_k, w_mn, g_k, g_mn, g_out, dw_out;
  const int64_t ldg = g->ld_logit_grad;
  if ((rc = map_k(&w_k, a, a->weight, a->width, a->vocab, a->ld_weight)) != 0 ||
      (rc = map_mn(&w_mn, a, a->weight, a->width, a->vocab, a->ld_weight)) != 0 ||
      (rc = map_k(&g_k, a, g->logit_grad, a->vocab, g->chunk, ldg)) != 0 || (rc = map_mn(&g_mn, a, g->logit_grad, a->vocab, g->chunk, ldg)) != 0 ||
      (rc = map_store(&g_out, a, g->logit_grad, a->vocab, g->chunk, ldg)) != 0)
    return rc;
  dw_out = g_out;
  if (g->d_weight != nullptr && !sums && (rc = map_store(&dw_out, a, g->d_weight, a->width, a->vocab, a->width)) != 0) return rc;
  for (int64_t row0 = 0; row0 < a->rows; row0 += g->chunk) {
    Params p = base_params(a);
    p.row0 = row0;
    p.cap = g->chunk;
    p.coef = g->coef;
    p.scale = half ? g->scale : nullptr;
    const int64_t here = std::min(g->chunk, a->rows - row0);
    CUtensorMap h_k, h_mn;
    const uint16_t* hp = static_cast<const uint16_t*>(h) + row0 * ldh;
    if ((rc = map_k(&h_k, a, hp, a->width, here, ldh)) != 0 || (rc = map_mn(&h_mn, a, hp, a->width, here, ldh)) != 0) return rc;
    if (a->weights != nullptr) {
      const unsigned blocks_in = static_cast<unsigned>(std::min<int64_t>(p.cap, kNumSmsB200 * 16));
      const auto from = static_cast<const uint4*>(a->weights);
      const auto to = static_cast<uint4*>(g->logit_grad);
      if (half) NX_PDL((weigh_kernel<false>), blocks_in, 256, 0, st, p, from, to, ldg / 8);
      else NX_PDL((weigh_kernel<true>), blocks_in, 256, 0, st, p, from, to, ldg / 8);
    } else if ((rc = NX_HEAD(kGrad, h_k, w_k, g_out, p, tiles(here) * tiles(a->vocab), st)) != 0) {
      return rc;
    }
    if (g->d_hidden != nullptr) {
      p.out = g->d_hidden;
      p.out_ld = a->width;
      p.slices = g->slices;
      p.partial = g->slice_sums;
      if ((rc = NX_HEAD(kInputGrad, g_k, w_mn, g_out, p, tiles(here) * tiles(a->width) * p.slices, st)) != 0) return rc;
      if (p.slices > 1) {
        const unsigned blocks_out = static_cast<unsigned>(std::min<int64_t>(here, kNumSmsB200 * 16));
        if (half) NX_PDL((slices_kernel<false>), blocks_out, 128, 0, st, p);
        else NX_PDL((slices_kernel<true>), blocks_out, 128, 0, st, p);
      }
    }
    if (g->d_weight != nullptr) {
      p.slices = 1;
      p.partial = sums ? g->weight_sums : nullptr;
      p.add = row0 > 0;
      if ((rc = NX_HEAD(kWeightGrad, g_mn, h_mn, dw_out, p, tiles(a->vocab) * tiles(a->width), st)) != 0) return rc;
    }
  }
  if (sums) {
    const int64_t pieces = static_cast<int64_t>(a->vocab) * a->width / 8;
    if (half) NX_PDL((narrow_kernel<false>), blocks_for(pieces, 256), 256, 0, st, g->weight_sums, static_cast<uint4*>(g->d_weight), pieces);
    else NX_PDL((narrow_kernel<true>), blocks_for(pieces, 256), 256, 0, st, g->weight_sums, static_cast<uint4*>(g->d_weight), pieces);
  }
  return 0;
}
