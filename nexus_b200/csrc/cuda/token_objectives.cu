// Log-probabilities of given tokens, the clipped policy loss and the preference loss on logits, with their gradients.
//
//   x = logits * inv_temp,  m = max,  s = sum exp(x - m),  logp_j = x_j - m - ln s,  p_j = exp(logp_j),  H = ln s - sum p_j (x_j - m)
//   d logp_t / d x_j = delta_jt - p_j          d H / d x_j = -p_j (logp_j + H)
//
// Statistics are kept as one logit and log2 of the sum relative to it: with the difference taken before any product, p and logp have no
// rounding that grows with the logits (a sum m + ln s rounded to FP32 would put 2^-24 |lse| into the exponent of every p).
// Everything here is bound by the bytes of the logits.
#include "common.cuh"
#include "nx_api_objectives.h"
#include "row_vec.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace {
using namespace nx;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kThreads = 512;

// rows, and with them `per`, `adv_per` and `seq_len` that divide them, stay below 2^31
__device__ __forceinline__ uint32_t row_over(int64_t r, int64_t by) { return static_cast<uint32_t>(r) / static_cast<uint32_t>(by); }
__device__ __forceinline__ int64_t row_offset(const NxTokenRows& a, int64_t r) {
  const int64_t o = row_over(r, a.per);
  return o * a.stride_outer + (r - o * a.per) * a.stride_inner;
}
__device__ __forceinline__ int64_t target_at(const void* targets, int wide, int64_t r) {
  return wide ? reinterpret_cast<const int64_t*>(targets)[r] : static_cast<int64_t>(reinterpret_cast<const int32_t*>(targets)[r]);
}

// A row as 16-byte pieces between its first and last 16-byte boundary, and single elements before and behind them.
template <typename T>
struct RowSplit {
  static constexpr int kN = RowVec<T>::kN;
  int head, pieces, tail;  // elements, pieces, elements
  __device__ __forceinline__ RowSplit(const T* p, int count) {
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    head = min(off == 0 ? 0 : kN - off, count);
    pieces = (count - head) / kN;
    tail = count - head - pieces * kN;
  }
};

constexpr float kNoWeight = -160.0f;    // 2^t is zero
constexpr float kFarBelow = -1.0e30f;  // stands for a difference of -inf where a weight of zero multiplies it

// Running maximum, sum of exponentials and sum of exponentials times differences, of one thread's elements.
struct Online {
  float m = -INFINITY, s = 0.0f, h = 0.0f;
  __device__ __forceinline__ void raise(float to, float k) {  // a larger maximum: the sums so far are taken down to it
    const float old = m;
    m = to;
    if (old == -INFINITY) return;  // nothing but -inf so far: the sums are zero (or NaN) as they are
    const float d = fmaxf(old - to, kFarBelow);  // finite beside a masked lowest value, so that its weight of zero makes it zero
    const float f = ex2_approx(d * k);
    h = (h + d * s) * f;
    s *= f;
  }
  template <int N>
  __device__ __forceinline__ void absorb(const float (&v)[N], float k) {
    float vm = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) vm = fmaxf(vm, v[j]);
    if (vm > m) raise(vm, k);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float d = v[j] - base;
      // a masked -inf has the weight 0 and must not make 0 * -inf of it; NaN stays NaN
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(kFarBelow));
      const float e = ex2_approx(d * k);
      s += e;
      h = fmaf(e, d, h);
    }
  }
};

// ------------------------------------------------------------------------------------------------ gradients of rows
// Gradient of a row, four pieces of loads at a time: f(logit) for every element of the vocabulary, `extra` added at the target, zeros behind.
template <typename T, typename F>
__device__ __forceinline__ void write_row(const T* p, T* g, int vocab, int width, int tg, float extra, F f) {
  constexpr int VN = RowVec<T>::kN;
  const RowSplit<T> sp(p, vocab);
  const T* body = p + sp.head;
  T* gbody = g + sp.head;
  const int step = blockDim.x;
  const int tpiece = tg < sp.head ? -1 : (tg - sp.head) / VN;
  auto piece = [&](int i, const uint4& raw) {
    float v[VN];
    RowVec<T>::unpack(raw, v);
#pragma unroll
    for (int j = 0; j < VN; ++j) v[j] = f(v[j]);
    if (i == tpiece) {
#pragma unroll
      for (int j = 0; j < VN; ++j)
        if (sp.head + i * VN + j == tg) v[j] += extra;
    }
    RowVec<T>::store(gbody + static_cast<int64_t>(i) * VN, v);
  };
  int i = threadIdx.x;
  for (; i + 3 * step < sp.pieces; i += 4 * step) {
    uint4 raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = *reinterpret_cast<const uint4*>(body + static_cast<int64_t>(i + u * step) * VN);
#pragma unroll
    for (int u = 0; u < 4; ++u) piece(i + u * step, raw[u]);
  }
  for (; i < sp.pieces; i += step) piece(i, *reinterpret_cast<const uint4*>(body + static_cast<int64_t>(i) * VN));
  const int done = sp.head + sp.pieces * VN;
  int c = -1;
  if (static_cast<int>(threadIdx.x) < sp.head) c = threadIdx.x;
  else if (static_cast<int>(threadIdx.x) >= 32 && static_cast<int>(threadIdx.x) - 32 < sp.tail) c = done + threadIdx.x - 32;
  if (c >= 0) Num<T>::store(g + c, f(Num<T>::load(p + c)) + (c == tg ? extra : 0.0f));
  for (int w = vocab + threadIdx.x; w < width; w += step) Num<T>::store(g + w, 0.0f);
}

template <typename T>
__device__ __forceinline__ void clear_row(T* g, int width) {
  constexpr int VN = RowVec<T>::kN;
  const RowSplit<T> sp(g, width);
  for (int i = threadIdx.x; i < sp.pieces; i += blockDim.x)
    *reinterpret_cast<uint4*>(g + sp.head + static_cast<int64_t>(i) * VN) = make_uint4(0, 0, 0, 0);
  if (static_cast<int>(threadIdx.x) < sp.head) Num<T>::store(g + threadIdx.x, 0.0f);
  else if (static_cast<int>(threadIdx.x) >= 32 && static_cast<int>(threadIdx.x) - 32 < sp.tail)
    Num<T>::store(g + sp.head + static_cast<int64_t>(sp.pieces) * VN + threadIdx.x - 32, 0.0f);
}

// c (delta - p) of each row.  8192 x 50304 BF16 or FP16: 262 us, 6.3 TB/s read and written, bound by these bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_grad_kernel(const NxTokenRows a, const float2* __restrict__ stats,
                                                              const float* __restrict__ coef, int64_t coef_per,
                                                              const float* __restrict__ factor, T* __restrict__ grad) {
  pdl_dependency();
  pdl_trigger();
  const int64_t row = gridDim.x - 1 - blockIdx.x;  // the last rows first: the sums have left them in L2
  const int64_t tg = target_at(a.targets, a.targets_wide, row);
  const int64_t at = row_offset(a, row);
  T* g = grad + at;
  if (tg == a.ignore_index || tg < 0 || tg >= a.vocab) {
    clear_row(g, a.width);
    return;
  }
  const float c = coef[row_over(row, coef_per)] * (factor != nullptr ? *factor : 1.0f) * a.inv_temp;
  const float2 st = stats[row];
  const float k = a.inv_temp * kLog2e;
  write_row(reinterpret_cast<const T*>(a.logits) + at, g, a.vocab, a.width, static_cast<int>(tg), c,
            [&](float v) { return -c * ex2_approx(fmaf(v - st.x, k, -st.y)); });
}

// Gradient of the policy loss from what its forward pass left of each row: g = p (slope (v - x) + off) and c at the target, times the loss's own
// gradient before anything is rounded.  FP16 only, where a gradient that is rounded first and multiplied by a loss scale afterwards has lost all
// below 2^-25: one more read of the logits than writing it forward.  8192 x 50304: 264 us (6.2 TB/s) behind 166 of the forward pass; BF16, which has
// the range of FP32 and writes it forward, 299 for both.
template <typename T>
__global__ void __launch_bounds__(kThreads) policy_grad_kernel(const NxTokenRows a, const NxPolicySlope* __restrict__ slopes,
                                                               const float* __restrict__ factor, T* __restrict__ grad) {
  pdl_dependency();
  pdl_trigger();
  const int64_t row = gridDim.x - 1 - blockIdx.x;  // the last rows first: the sums have left them in L2
  const int64_t tg = target_at(a.targets, a.targets_wide, row);
  const int64_t at = row_offset(a, row);
  T* g = grad + at;
  if (tg == a.ignore_index || tg < 0 || tg >= a.vocab) {
    clear_row(g, a.width);
    return;
  }
  const NxPolicySlope st = slopes[row];
  const float f = *factor, k = a.inv_temp * kLog2e;
  const float slope = st.slope * f, off = st.off * f, least = 2.0f * kNoWeight / k;
  write_row(reinterpret_cast<const T*>(a.logits) + at, g, a.vocab, a.width, static_cast<int>(tg), st.c * f, [&](float v) {
    float d = v - st.x;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(least));  // no weight from here on, and small enough to be multiplied
    return ex2_approx(fmaf(d, k, -st.log2_s)) * fmaf(d, slope, off);
  });
}

// ------------------------------------------------------------------------------------------------ policy loss
// Sums over a few thousand to a million values by one cluster of eight blocks: partial sums meet in the first block's shared memory.
constexpr int kJoinBlocks = 8, kJoinThreads = 1024;

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// slot[rank] of the cluster's first block = v; one thread of each block, once every block of the cluster is known to run
__device__ __forceinline__ void put_in_first(double* slot, uint32_t rank, double v) {
  uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(slot + rank)), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(addr));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}

// totals[0] = rows that count, totals[1] = sequences with such rows, totals[2] = no block has ended (the policy kernel counts them there);
// counts[q] = rows of sequence q that count
__global__ void __cluster_dims__(kJoinBlocks, 1, 1) __launch_bounds__(kJoinThreads)
token_count_kernel(const void* __restrict__ targets, int wide, int64_t sequences, int64_t len, int64_t ignore, double* __restrict__ totals,
                   int32_t* __restrict__ counts) {
  __shared__ double tokens[kJoinBlocks], filled[kJoinBlocks];
  __shared__ double scratch[32];
  cluster_arrive();
  pdl_dependency();
  pdl_trigger();
  const uint32_t rank = cluster_ctarank();
  double mine = 0.0, full = 0.0;
  if (len >= 256) {
    for (int64_t q = rank; q < sequences; q += kJoinBlocks) {
      int n = 0;
      for (int64_t t = threadIdx.x; t < len; t += blockDim.x) n += target_at(targets, wide, q * len + t) != ignore;
      const double got = block_sum<double>(n, scratch);
      mine += got;
      full += got > 0.0;
      if (threadIdx.x == 0) counts[q] = static_cast<int32_t>(got);
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int64_t q = rank * 32 + (threadIdx.x >> 5); q < sequences; q += kJoinBlocks * 32) {
      int n = 0;
      for (int64_t t = lane; t < len; t += 32) n += target_at(targets, wide, q * len + t) != ignore;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) {
        mine += n;
        full += n > 0;
        counts[q] = n;
      }
    }
    mine = block_sum<double>(mine, scratch);
    full = block_sum<double>(full, scratch);
  }
  cluster_wait();
  if (threadIdx.x == 0) {
    put_in_first(tokens, rank, mine);
    put_in_first(filled, rank, full);
  }
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && threadIdx.x == 0) {
    double a = 0.0, b = 0.0;
    for (int i = 0; i < kJoinBlocks; ++i) {
      a += tokens[i];
      b += filled[i];
    }
    totals[0] = a;
    totals[1] = b;
    totals[2] = 0.0;
  }
}

struct PolicyRow {
  float c;       // d row loss / d logp, weighted
  float ent;     // entropy coefficient, weighted
  float loss, kl;
};
struct PolicyIn {
  float adv, old, ref, weight;
};
// A row's constants and weight: the whole batch's mean over tokens, the mean over sequences of the means over their tokens, or one.
__device__ __forceinline__ PolicyIn policy_in(const NxPolicyArgs& g, const double* totals, const int32_t* counts, int64_t row) {
  PolicyIn i;
  i.adv = g.advantages[row_over(row, g.adv_per)];
  i.old = g.old_logp[row];
  i.ref = g.ref_logp != nullptr ? g.ref_logp[row] : 0.0f;
  i.weight = g.scale;
  if (g.mean == NX_MEAN_TOKEN) i.weight = static_cast<float>(g.scale / totals[0]);
  if (g.mean == NX_MEAN_SEQUENCE) i.weight = static_cast<float>(g.scale / (totals[1] * counts[row_over(row, g.seq_len)]));
  return i;
}
__device__ __forceinline__ PolicyRow policy_row(const NxPolicyArgs& g, const PolicyIn& in, float logp, float entropy) {
  PolicyRow o;
  float ratio = expf(logp - in.old);
  if (in.adv == 0.0f && ratio == INFINITY) ratio = 1.0f;  // beyond FP32, and counted zero times
  const float free = ratio * in.adv, bound = fminf(fmaxf(ratio, 1.0f - g.clip_low), 1.0f + g.clip_high) * in.adv;
  // the unclipped term where it is the smaller one, or they are equal, or it is no number
  const bool follows = !(free > bound);
  float loss = follows ? -free : -bound, c = follows ? -free : 0.0f;
  o.kl = 0.0f;
  if (g.ref_logp != nullptr) {
    const float d = in.ref - logp;
    float slope;
    if (g.kl == NX_KL_K3) {
      const float e = expm1f(d);
      o.kl = e - d;
      slope = -e;
    } else if (g.kl == NX_KL_K2) {
      o.kl = 0.5f * d * d;
      slope = -d;
    } else {
      o.kl = -d;
      slope = 1.0f;
    }
    if (g.kl_coef != 0.0f) {  // an estimate that is only looked at may be infinite
      loss = fmaf(g.kl_coef, o.kl, loss);
      c = fmaf(g.kl_coef, slope, c);
    }
  }
  if (g.entropy_coef != 0.0f) loss -= g.entropy_coef * entropy;
  o.loss = loss * in.weight;
  o.c = c * in.weight;
  o.ent = g.entropy_coef * in.weight;
  return o;
}

// ------------------------------------------------------------------------------------------------ rows through shared memory
// A persistent block reads its rows through a ring of 16 KiB slots in shared memory, filled by one warp with bulk copies: what a row needs
// arrives while the block still works on the row before it.  Sums come from the first pass over a row's slots; where a gradient is written, the
// slots stay for a second pass, which frees them one by one for the next row: one read of the logits.  Of a row that is longer than the ring,
// the last slots stay and the others are read again, from L2.  Few rows are cut over a cluster of blocks, whose sums meet in each other's shared
// memory.
//
// Three shapes (BF16, B200; bytes read and written over the time):
//   sums only                 three blocks of four warps per SM      8192 x 50304: 146 us, 5.6 TB/s; two of eight warps 156, one of sixteen 180
//   gradient, rows to 112 KiB two blocks of eight warps              8192 x 50304: 283 us, 5.8 TB/s (to 304 in other runs); one of sixteen 336
//   gradient, longer rows     one block of sixteen warps, 208 KiB    2368 x 32000 FP32: 101 us, 6.0 TB/s; two of eight 114
// With sums and maxima kept per thread instead of a common base, 64-bit divisions per row in every thread and each row's target and constants
// loaded at its beginning, the same ring took 465 us for 8192 x 50304 (11 instructions per element and pass instead of 7).
constexpr int kSlotBytes = 16384, kSlotPieces = kSlotBytes / 16;
constexpr int kMaxCuts = 8;

template <int WORKERS, int SLOTS, int RESIDENT, bool WRITES>
struct Shape {
  static constexpr bool kWrites = WRITES;                            // a second pass writes the gradient
  static constexpr int kWorkers = WORKERS, kThreads = WORKERS + 32;  // and the warp that copies
  static constexpr int kSlots = SLOTS, kResident = RESIDENT;         // blocks per SM
};
using SumsShape = Shape<128, 4, 3, false>;
using ShortShape = Shape<256, 7, 2, true>;
using LongShape = Shape<512, 13, 1, true>;

// A row's sums relative to its target's logit:  s = sum 2^t,  h = sum t 2^t  with  t = v k - B,  B = x_t k rounded,  k = log2(e) inv_temp.  The
// base is the same for every thread and block, so joining is adding and no maximum is kept; the product is inside the fused multiply-add, so t
// is exact to its own last bit, and results are taken relative to B itself.  The target's own term is 2^(x_t k - B): with |B| up to kFastLimit, B is
// rounded by 2^-5 at most, and s is at least 0.97.  A row where a logit lies so far above its target's that the sums overflow (t of 120 and more), or
// where B would be too coarse (|x_t| or |B| above kFastLimit: at temperatures of 1e-8 the second from logits of 0.007 on; -inf, NaN), is done again
// in the form with running maxima and the difference first; and so is, where t is multiplied, one where the finite value that stands for -inf (an
// FP16 piece holds none below -65504) comes so near the target's logit, or is scaled down so far, that its weight is not zero.
// Where a second pass writes the gradient its factors are divided by s, and are normal numbers (the row's weight being 2^-66 or more) only while
// s stays below 2^60: t of 60 and more, targets of a log-probability below -41, are done again there.
constexpr float kFastLimit = 1.0e6f, kFastSum = 1.3e36f, kFastSumDivides = 0x1p60f;
// Stands for -inf (and all below it) where t is multiplied: the weight is zero either way, and zero times a finite product is zero.  Representable in
// BF16; no lower than it must be, so that k (up to 1.5e8) and the entropy's factors keep the products finite.
constexpr float kFloor = -998244352.0f;

struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void halves(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

// A 16-byte piece as pairs of FP32 values; kFloored: -inf (and anything below kFloor) becomes a finite value, NaN stays
template <typename T>
struct PieceOf;
template <>
struct PieceOf<__nv_bfloat16> {
  static constexpr int kPairs = 4;
  static constexpr float kLowest = kFloor;
  template <bool kFloored>
  static __device__ __forceinline__ void get(const uint4& q, Pair (&p)[4]) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kFloored) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(0xce6ece6eu));  // kFloor
      p[i] = pair_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
};
template <>
struct PieceOf<__half> {
  static constexpr int kPairs = 4;
  static constexpr float kLowest = -65504.0f;
  template <bool kFloored>
  static __device__ __forceinline__ void get(const uint4& q, Pair (&p)[4]) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kFloored) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(0xfbfffbffu));  // -65504
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      p[i] = pair_of(f.x, f.y);
    }
  }
};
template <>
struct PieceOf<float> {
  static constexpr int kPairs = 2;
  static constexpr float kLowest = kFloor;
  template <bool kFloored>
  static __device__ __forceinline__ void get(const uint4& q, Pair (&p)[2]) {
    float v[4] = {__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w)};
    if (kFloored) {
#pragma unroll
      for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(v[i]) : "f"(kFloor));
    }
    p[0] = pair_of(v[0], v[1]);
    p[1] = pair_of(v[2], v[3]);
  }
};

template <bool kEntropy>
struct Fast {
  Pair s{0}, h{0};
  template <typename T>
  __device__ __forceinline__ void absorb(const uint4& q, Pair kk, Pair minus_base) {
    constexpr int N = PieceOf<T>::kPairs;
    Pair p[N];
    PieceOf<T>::template get<kEntropy>(q, p);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Pair t = fma2(p[i], kk, minus_base);
      float a, b;
      halves(t, a, b);
      const Pair e = pair_of(ex2_approx(a), ex2_approx(b));
      s = add2(s, e);
      if (kEntropy) h = fma2(t, e, h);
    }
  }
  __device__ __forceinline__ void absorb_one(float v, float k, float base) {
    if (kEntropy) asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(kFloor));
    const float t = fmaf(v, k, -base), e = ex2_approx(t);
    s = add2(s, pair_of(e, 0.0f));
    if (kEntropy) h = fma2(pair_of(t, 0.0f), pair_of(e, 0.0f), h);
  }
};

// What the producer has gathered of a row by the time the workers come to it.
struct RowInfo {
  int64_t at;       // offset of the row in elements
  int32_t target;   // -1: ignored, -2: outside the vocabulary
  float x;          // the target's logit
  PolicyIn in;
};
// What the row's end makes of its sums, for every worker's second pass.
struct RowEnd {
  float c, c1, es, eb;   // g = 2^t (es t + eb), without an entropy term 2^t c1; c more at the target
  int32_t careful;       // or kStop: a wait has run out, nothing more is written
  float m, log2_s, slope, off;  // careful: g = 2^((v - m) k - log2_s) (slope (v - m) + off)
};
constexpr int kStop = 2;
constexpr int kAhead = 4;
template <typename S>
struct RingSpace {
  RowInfo info[kAhead];
  RowEnd end;
  float4 warps[S::kWorkers / 32];    // (m, s, h) of each warp, and whether one of its waits has run out
  float4 blocks[2][kMaxCuts];        // of each block of the cluster, in turns
  uint64_t full[S::kSlots], empty[S::kSlots], told[kAhead], heard[kAhead];
  uint64_t arrived;                  // counts the blocks that have put theirs in
  int abort_word;
};

template <typename S>
__device__ __forceinline__ void workers_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(S::kWorkers) : "memory");
}

// s and h are relative to a maximum m: brings them to `top`, differences in units of the logits
__device__ __forceinline__ void weigh(float4& v, float top, float k) {
  if (v.x == -INFINITY) return;  // nothing but -inf: zero (or NaN) as it is
  const float d = fmaxf(v.x - top, kFarBelow), f = ex2_approx(d * k);
  v.z = fmaf(d, v.y, v.z) * f;
  v.y *= f;
}
// (m, s, h) of 2^n lanes together; kMaxima: s and h are relative to m, otherwise m is not used
template <bool kMaxima, int kLanes>
__device__ __forceinline__ void join_lanes(float4& v, float k) {
  if (kMaxima) {
    float top = v.x;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    weigh(v, top, k);
    v.x = top;
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
  }
}

// Joins all threads' and blocks' sums of a row; the first warp gets them.  The last component is not zero where a wait of any thread or block has run
// out (`fine` is what this thread knows of it), so that all of them stop at the same row.
template <bool kMaxima, typename S>
__device__ __forceinline__ float4 join_all(float4 v, float k, RingSpace<S>* sp, int rank, int cuts, int& turn, bool& fine) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  join_lanes<kMaxima, 32>(v, k);
  v.w = __all_sync(0xffffffffu, fine) ? 0.0f : 1.0f;
  if (lane == 0) sp->warps[warp] = v;
  workers_sync<S>();
  const int side = turn & 1;
  if (cuts > 1) ++turn;
  if (warp != 0) return v;
  v = sp->warps[lane & (S::kWorkers / 32 - 1)];
  join_lanes<kMaxima, S::kWorkers / 32>(v, k);
  v.w = __any_sync(0xffffffffu, v.w != 0.0f) ? 1.0f : 0.0f;
  if (cuts > 1) {
    if (lane < cuts) {  // a lane per block of the cluster
      const uint32_t to = mapa_shared(smem_u32(&sp->blocks[side][rank]), lane);
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
      mbar_arrive_cluster(mapa_shared(smem_u32(&sp->arrived), lane));
    }
    uint32_t done = 0, tries = 0;
    uint64_t began = 0;
    while (!done) {
      asm volatile(
          "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(smem_u32(&sp->arrived)), "r"(static_cast<uint32_t>(side))
          : "memory");
      if (!done && (++tries & 63u) == 0) {
        const uint64_t now = globaltimer_ns();
        if (began == 0) began = now;
        if (*static_cast<volatile int*>(&sp->abort_word) != 0 || now - began > NX_WAIT_LIMIT_NS) {
          *static_cast<volatile int*>(&sp->abort_word) = 1;
          break;
        }
      }
    }
    if (!__all_sync(0xffffffffu, done != 0)) fine = false;
    v = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    if ((lane & (kMaxCuts - 1)) < cuts) v = sp->blocks[side][lane & (kMaxCuts - 1)];
    join_lanes<kMaxima, kMaxCuts>(v, k);
    v.w = !fine || __any_sync(0xffffffffu, v.w != 0.0f) ? 1.0f : 0.0f;
  }
  return v;
}

struct RingOut {
  float* logp;
  float2* stats;     // token log-probabilities: a logit x, log2 of the sum of exp((logit - x) inv_temp)
  double* wide;      // and, where given, logp before it is rounded to FP32
  float* kl;
  float* entropy;
  float* row_loss;
  NxPolicySlope* slopes;  // policy: where given, what a row's gradient is made of later
  const double* totals;
  const int32_t* counts;
  int* ended;        // policy: blocks that have ended, zero before; the last one adds up the rows' losses
  float* loss;
  int* status;
  int cuts;
};

template <typename T, bool kPolicy, typename S>
__global__ void __launch_bounds__(S::kThreads, S::kResident)
ring_kernel(const NxTokenRows a, const NxPolicyArgs g, const RingOut o, T* __restrict__ grad) {
  constexpr int kWorkers = S::kWorkers, kSlots = S::kSlots;
  constexpr int VN = RowVec<T>::kN, kPer = kSlotPieces / kWorkers;
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(16) RingSpace<S> space;
  RingSpace<S>* const sp = &space;
  volatile int* const abort_flag = &space.abort_word;
  const int cuts = o.cuts, rank = cuts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const uint32_t rows = static_cast<uint32_t>(a.rows), first = blockIdx.x / cuts, step = gridDim.x / cuts;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&sp->full[s], 1);
      mbar_init(&sp->empty[s], kWorkers / 32);
    }
    for (int s = 0; s < kAhead; ++s) {
      mbar_init(&sp->told[s], 1);
      mbar_init(&sp->heard[s], kWorkers / 32);
    }
    mbar_init(&sp->arrived, static_cast<uint32_t>(cuts));
    sp->abort_word = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (cuts > 1) cluster_sync_all();  // the others' barriers exist
  pdl_dependency();
  pdl_trigger();

  constexpr bool second = S::kWrites;
  static_assert(kPolicy || !second);
  // slots of `n` pieces that are freed in the first pass: all without a second one; with one, those that the ring has no room for (and of a long
  // row two more, so that copies go on while the sums are joined)
  auto freed = [&](int n) {
    const int all = (n + kSlotPieces - 1) / kSlotPieces;
    return !second ? all : (all <= kSlots ? 0 : all - (kSlots - 2));
  };
  const float k = a.inv_temp * kLog2e;
  const int shift = 31 - __clz(cuts);  // cuts is a power of two
  // this block's pieces of a row
  auto share = [&](const RowSplit<T>& r, int& lo, int& n) {
    lo = static_cast<int>(static_cast<uint64_t>(r.pieces) * rank >> shift);
    n = static_cast<int>(static_cast<uint64_t>(r.pieces) * (rank + 1) >> shift) - lo;
  };

  if (threadIdx.x >= kWorkers) {
    // The copying warp: 32 rows at a time, a lane gathers what is known of one; then the first lane tells the workers and fills slots, row by row.
    const int lane = threadIdx.x & 31;
    int slot = 0, seat = 0;
    uint32_t phase = 0, seat_phase = 0;
    bool ok = true;
    for (uint64_t batch = first; batch < rows; batch += 32ull * step) {
      const uint64_t row = batch + static_cast<uint64_t>(lane) * step;
      RowInfo info{};
      info.target = -1;
      if (row < rows) {
        const uint32_t r = static_cast<uint32_t>(row);
        const int64_t tg = target_at(a.targets, a.targets_wide, r);
        info.at = row_offset(a, r);
        info.target = tg == a.ignore_index ? -1 : (tg < 0 || tg >= a.vocab ? -2 : static_cast<int32_t>(tg));
        if (info.target >= 0) {
          info.x = Num<T>::load(reinterpret_cast<const T*>(a.logits) + info.at + info.target);
          if (kPolicy) info.in = policy_in(g, o.totals, o.counts, r);
        }
      }
      const int here = static_cast<int>(min(static_cast<uint64_t>(32), (rows - batch + step - 1) / step));
      for (int j = 0; j < here; ++j) {
        const int32_t tg = __shfl_sync(0xffffffffu, info.target, j);
        const int64_t at = __shfl_sync(0xffffffffu, info.at, j);
        ok = ok && mbar_wait_bounded(&sp->heard[seat], seat_phase ^ 1u, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          if (lane == j) sp->info[seat] = info;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sp->told[seat]);
        }
        if (++seat == kAhead) {
          seat = 0;
          seat_phase ^= 1u;
        }
        if (lane == 0 && ok && tg >= 0) {
          const T* p = reinterpret_cast<const T*>(a.logits) + at;
          const RowSplit<T> r(p, a.vocab);
          int lo, n;
          share(r, lo, n);
          const uint8_t* src = reinterpret_cast<const uint8_t*>(p + r.head) + static_cast<int64_t>(lo) * 16;
          const int slots = (n + kSlotPieces - 1) / kSlotPieces, loads = slots + (second ? freed(n) : 0);
          for (int d = 0; d < loads; ++d) {
            const int c = (d < slots ? d : d - slots) * kSlotPieces;
            if (!mbar_wait_bounded(&sp->empty[slot], phase ^ 1u, abort_flag)) {
              ok = false;
              break;
            }
            const uint32_t bytes = static_cast<uint32_t>(min(kSlotPieces, n - c)) * 16;
            mbar_arrive_expect_tx(&sp->full[slot], bytes);
            bulk_load(ring_smem + slot * kSlotBytes, src + static_cast<int64_t>(c) * 16, bytes, &sp->full[slot]);
            if (++slot == kSlots) {
              slot = 0;
              phase ^= 1u;
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (!ok) break;
    }
    if (!ok && lane == 0) atomicCAS(o.status, 0, kStatusTimeoutProducer);
  } else {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int slot = 0, turn = 0, seat = 0;
    uint32_t phase = 0, seat_phase = 0;
    bool fine = true, stopped = false;  // a wait of this thread has not run out; one of any has, and all warps have left at the same row
    auto wait = [&](uint64_t* bar, uint32_t ph) { fine = mbar_wait_bounded(bar, ph, abort_flag) && fine; };
    auto release = [&](int s) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sp->empty[s]);
    };
    auto stop = [&] {  // the first warp, between the two barriers of a join
      if (lane == 0) {
        sp->end.careful = kStop;
        *abort_flag = 1;
      }
    };
    const Pair kk = pair_of(k, k);
    for (uint64_t row = first; row < rows; row += step) {
      wait(&sp->told[seat], seat_phase);
      if (!__all_sync(0xffffffffu, fine)) break;  // nothing is known of this row; the others hear of it in their next join or behind the loop
      const int32_t tg = sp->info[seat].target;
      const int64_t at = sp->info[seat].at;
      const float xt = sp->info[seat].x;
      PolicyIn in{};
      if (kPolicy && warp == 0) in = sp->info[seat].in;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sp->heard[seat]);
      if (++seat == kAhead) {
        seat = 0;
        seat_phase ^= 1u;
      }
      if (tg < 0) {
        if (rank == 0 && tid == 0) {
          const float v = tg == -1 ? 0.0f : NAN;
          o.logp[row] = v;
          if constexpr (kPolicy) {
            o.kl[row] = o.entropy[row] = o.row_loss[row] = v;
          } else {
            o.stats[row] = make_float2(0.0f, 0.0f);
            if (o.wide != nullptr) o.wide[row] = v;
          }
        }
        if (second) {
          T* gr = grad + at;
          const RowSplit<T> r(gr, a.width);
          for (int i = rank * kWorkers + tid; i < r.pieces; i += cuts * kWorkers)
            *reinterpret_cast<uint4*>(gr + r.head + static_cast<int64_t>(i) * VN) = make_uint4(0, 0, 0, 0);
          if (rank == 0 && tid < r.head) Num<T>::store(gr + tid, 0.0f);
          if (rank == 0 && tid >= 32 && tid - 32 < r.tail) Num<T>::store(gr + r.head + static_cast<int64_t>(r.pieces) * VN + tid - 32, 0.0f);
        }
        continue;
      }
      const T* p = reinterpret_cast<const T*>(a.logits) + at;
      const RowSplit<T> r(p, a.vocab);
      int lo, n;
      share(r, lo, n);
      // single elements before the first and behind the last piece: one per thread of the first block
      int edge = -1;
      if (rank == 0) {
        if (tid < r.head) edge = tid;
        else if (tid >= 32 && tid - 32 < r.tail) edge = r.head + r.pieces * VN + tid - 32;
      }
      const float ev = edge >= 0 ? Num<T>::load(p + edge) : 0.0f;
      const float base = xt * k;
      const Pair bb = pair_of(-base, -base);

      Fast<kPolicy> on;
      const int slots = (n + kSlotPieces - 1) / kSlotPieces, free_now = freed(n);
      int s = slot, c = 0;
      uint32_t ph = phase;
      auto next = [&] {
        if (++s == kSlots) {
          s = 0;
          ph ^= 1u;
        }
        if (c / kSlotPieces + 1 == free_now) {  // the first slot that stays is the next one
          slot = s;
          phase = ph;
        }
      };
      for (; c + kSlotPieces <= n; c += kSlotPieces) {
        wait(&sp->full[s], ph);
        const uint4* data = reinterpret_cast<const uint4*>(ring_smem + s * kSlotBytes) + tid;
        uint4 q[kPer];
#pragma unroll
        for (int u = 0; u < kPer; ++u) q[u] = data[u * kWorkers];
#pragma unroll
        for (int u = 0; u < kPer; ++u) on.template absorb<T>(q[u], kk, bb);
        if (c < free_now * kSlotPieces) release(s);
        next();
      }
      if (c < n) {
        wait(&sp->full[s], ph);
        const uint4* data = reinterpret_cast<const uint4*>(ring_smem + s * kSlotBytes);
        for (int i = tid; i < n - c; i += kWorkers) on.template absorb<T>(data[i], kk, bb);
        if (c < free_now * kSlotPieces) release(s);
        next();
      }
      if (edge >= 0) on.absorb_one(ev, k, base);
      float s0, s1, h0, h1;
      halves(on.s, s0, s1);
      halves(on.h, h0, h1);
      float4 st = join_all<false, S>(make_float4(0.0f, s0 + s1, h0 + h1, 0.0f), k, sp, rank, cuts, turn, fine);
      // The first warp ends the row and tells the others how its gradient comes.  `m`, `sum` and `h` relative to it where done with maxima.
      auto end_row = [&](const float4& v, bool careful) {
        RowEnd e{};
        e.careful = careful;
        const float ln_s = logf(v.y), log2_s = log2f(v.y), coarse = fmaf(xt, k, -base);  // x_t k - B is the rounding of B
        const float lp = careful ? (xt - v.x) * a.inv_temp - ln_s : coarse * kLn2 - ln_s;
        if constexpr (!kPolicy) {
          if (rank == 0 && lane == 0) {
            o.logp[row] = lp;
            o.stats[row] = make_float2(careful ? v.x : xt, log2_s - (careful ? 0.0f : coarse));
            if (o.wide != nullptr)
              o.wide[row] = (careful ? (static_cast<double>(xt) - v.x) * a.inv_temp : coarse * 0.6931471805599453) - log(static_cast<double>(v.y));
          }
        } else {
          const float ent = careful ? ln_s - v.z / v.y * a.inv_temp : ln_s - v.z / v.y * kLn2;
          const PolicyRow pr = policy_row(g, in, lp, ent);
          if (rank == 0 && lane == 0) {
            o.logp[row] = lp;
            o.kl[row] = pr.kl;
            o.entropy[row] = ent;
            o.row_loss[row] = pr.loss;
            if (o.slopes != nullptr) {  // relative to the same logit as `stats` above; logp at it is -ln_s or lp
              const float c = pr.c * a.inv_temp, e0 = pr.ent * a.inv_temp;
              NxPolicySlope& to = o.slopes[row];
              to.x = careful ? v.x : xt;
              to.log2_s = log2_s - (careful ? 0.0f : coarse);
              to.c = c;
              to.slope = e0 * a.inv_temp;
              to.off = g.entropy_coef != 0.0f ? e0 * (ent + (careful ? -ln_s : lp)) - c : -c;
            }
          }
          const float inv_s = 1.0f / v.y, e1 = pr.ent * a.inv_temp;
          e.c = pr.c * a.inv_temp;
          e.c1 = -e.c * inv_s;
          e.es = e1 * inv_s * kLn2;
          e.eb = e1 * inv_s * (ent - ln_s) + e.c1;
          e.m = v.x;
          e.log2_s = log2_s;
          e.slope = e1 * a.inv_temp;
          e.off = g.entropy_coef != 0.0f ? e1 * (ent - ln_s) - e.c : -e.c;
          if (lane == 0) sp->end = e;
        }
      };
      if (warp == 0) {
        const bool careful = !(fabsf(xt) <= kFastLimit && fabsf(base) <= kFastLimit && st.y <= (second ? kFastSumDivides : kFastSum) &&
                               (!kPolicy || fmaf(PieceOf<T>::kLowest, k, -base) <= kNoWeight));
        if (st.w != 0.0f) stop();
        else if (!careful) end_row(st, false);
        else if (lane == 0) sp->end.careful = 1;
        if (!kPolicy && st.w == 0.0f && !careful && lane == 0) sp->end.careful = 0;
      }
      workers_sync<S>();
      if (sp->end.careful == kStop) {
        stopped = true;
        break;
      }
      if (sp->end.careful) {  // the same in every block of the cluster; from memory, with maxima and the difference first
        Online on2;
        const T* body = p + r.head + static_cast<int64_t>(lo) * VN;
        for (int i = tid; i < n; i += kWorkers) {
          float v[VN];
          RowVec<T>::load(body + static_cast<int64_t>(i) * VN, v);
          on2.absorb(v, k);
        }
        if (edge >= 0) {
          const float v[1] = {ev};
          on2.absorb(v, k);
        }
        st = join_all<true, S>(make_float4(on2.m, on2.s, on2.h, 0.0f), k, sp, rank, cuts, turn, fine);
        if (warp == 0) {
          if (st.w != 0.0f) stop();
          else end_row(st, true);
        }
        workers_sync<S>();
        if (sp->end.careful == kStop) {
          stopped = true;
          break;
        }
      }
      if constexpr (second) {
        const RowEnd e = sp->end;
        T* gr = grad + at;
        const int col0 = r.head + lo * VN;
        if (e.careful) {
          const float least = 2.0f * kNoWeight / k;  // no weight from here on (log2_s is not negative), and small enough to be multiplied
          auto one = [&](float v) {
            float d = v - e.m;
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(least));
            return ex2_approx(fmaf(d, k, -e.log2_s)) * (g.entropy_coef != 0.0f ? fmaf(d, e.slope, e.off) : e.off);
          };
          for (int i = tid; i < n; i += kWorkers) {
            float v[VN];
            RowVec<T>::load(p + col0 + static_cast<int64_t>(i) * VN, v);
#pragma unroll
            for (int j = 0; j < VN; ++j) v[j] = one(v[j]) + (col0 + i * VN + j == tg ? e.c : 0.0f);
            RowVec<T>::store(gr + col0 + static_cast<int64_t>(i) * VN, v);
          }
          if (edge >= 0) Num<T>::store(gr + edge, one(ev) + (edge == tg ? e.c : 0.0f));
          for (int d = 0; d < slots; ++d) {  // the slots were not needed
            wait(&sp->full[slot], phase);
            release(slot);
            if (++slot == kSlots) {
              slot = 0;
              phase ^= 1u;
            }
          }
        } else {
          const Pair cc = pair_of(e.c1, e.c1), ee = pair_of(e.es, e.es), eo = pair_of(e.eb, e.eb);
          uint4* const out = reinterpret_cast<uint4*>(gr + col0);
          auto second_pass = [&](auto entropy) {
            constexpr bool kEnt = decltype(entropy)::value;
            auto piece = [&](int i, const uint4& q) {
              constexpr int N = PieceOf<T>::kPairs;
              Pair v[N];
              PieceOf<T>::template get<kEnt>(q, v);
              float w[VN];
#pragma unroll
              for (int u = 0; u < N; ++u) {
                const Pair t = fma2(v[u], kk, bb);
                float x, y;
                halves(t, x, y);
                const Pair ex = pair_of(ex2_approx(x), ex2_approx(y));
                halves(mul2(ex, kEnt ? fma2(t, ee, eo) : cc), w[2 * u], w[2 * u + 1]);
              }
              RowVec<T>::store(reinterpret_cast<T*>(out + i), w);
            };
            for (int d = free_now; d < slots + free_now; ++d) {  // those that stayed, then those that come again
              c = (d < slots ? d : d - slots) * kSlotPieces;
              const uint4* data = reinterpret_cast<const uint4*>(ring_smem + slot * kSlotBytes);
              if (d >= slots) wait(&sp->full[slot], phase);
              if (!fine) {  // not there
              } else if (c + kSlotPieces <= n) {
                uint4 q[kPer];
#pragma unroll
                for (int u = 0; u < kPer; ++u) q[u] = data[tid + u * kWorkers];
#pragma unroll
                for (int u = 0; u < kPer; ++u) piece(c + tid + u * kWorkers, q[u]);
              } else {
                for (int i = tid; i < n - c; i += kWorkers) piece(c + i, data[i]);
              }
              release(slot);
              if (++slot == kSlots) {
                slot = 0;
                phase ^= 1u;
              }
            }
          };
          if (g.entropy_coef != 0.0f) second_pass(std::true_type{});
          else second_pass(std::false_type{});
          auto single = [&](float v) {
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(kFloor));
            const float t = fmaf(v, k, -base);
            return ex2_approx(t) * (g.entropy_coef != 0.0f ? fmaf(t, e.es, e.eb) : e.c1);
          };
          if (edge >= 0 && edge != tg) Num<T>::store(gr + edge, single(ev));
          // The target's element, by the thread that wrote its piece (or has it at the edge): once more, with c added before it is rounded.
          const int off = tg - col0;
          const bool at_edge = edge == tg;
          const bool in_piece = off >= 0 && off < n * VN && (off / VN) % kWorkers == tid;
          if (at_edge || in_piece) Num<T>::store(gr + tg, single(xt) + e.c);
        }
        for (int w = a.vocab + rank * kWorkers + tid; w < a.width; w += cuts * kWorkers) Num<T>::store(gr + w, 0.0f);
      }
    }
    if (!stopped) {  // the barriers of one more join: a warp that has left early meets the others here, or here those that are in a row
      const bool all = __all_sync(0xffffffffu, fine);
      if (lane == 0) sp->warps[warp].w = all ? 0.0f : 1.0f;
      workers_sync<S>();
      if (warp == 0 && __any_sync(0xffffffffu, sp->warps[lane & (kWorkers / 32 - 1)].w != 0.0f)) stop();
      workers_sync<S>();
    }
    if (!fine) atomicCAS(o.status, 0, kStatusTimeoutEpilogue);
  }
  __syncthreads();
  if (*abort_flag != 0) {  // a wait ran out: copies still in flight land before the shared memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(2000);
  }
  if constexpr (kPolicy) {
    __shared__ int last;
    __shared__ double scratch[32];
    if (threadIdx.x == 0) {  // the thread that wrote this block's losses
      __threadfence();
      last = atomicAdd(o.ended, 1) == static_cast<int>(gridDim.x) - 1;
      __threadfence();
    }
    __syncthreads();
    if (last) {
      double acc = 0.0;
      for (uint32_t i = threadIdx.x; i < rows; i += S::kThreads) acc += __ldcg(o.row_loss + i);
      acc = block_sum<double>(acc, scratch);
      if (threadIdx.x == 0) *o.loss = static_cast<float>(acc);
    }
  }
  if (cuts > 1) cluster_sync_all();  // no block leaves while another may still write to it
}

// Blocks that a row is cut over, while rows are too few for the SMs
inline int cuts_for(int64_t rows, int64_t pieces) {
  int cuts = 1;
  while (cuts < kMaxCuts && rows * cuts < kNumSmsB200 && pieces / cuts >= 512) cuts *= 2;
  return cuts;
}

template <typename T, bool kPolicy, typename S>
int launch_shape(const NxTokenRows& a, const NxPolicyArgs& g, RingOut o, T* grad, cudaStream_t st) {
  auto kern = ring_kernel<T, kPolicy, S>;
  constexpr int kRingBytes = S::kSlots * kSlotBytes;
  NX_ALLOW_SMEM(kern, kRingBytes);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(o.cuts);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = kRingBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = o.cuts > 1 ? 2 : 1;
  // All clusters at the same time: the GPCs' SMs do not divide by four and eight, and a cluster left over would double the time.
  static std::atomic<int> resident[4];
  int at = 0;
  while ((1 << at) < o.cuts) ++at;
  int most = o.cuts == 1 ? S::kResident * kNumSmsB200 : resident[at].load(std::memory_order_relaxed);
  if (most == 0) {
    cfg.gridDim = dim3(static_cast<unsigned>(S::kResident * kNumSmsB200 / o.cuts * o.cuts));
    if (cudaOccupancyMaxActiveClusters(&most, kern, &cfg) != cudaSuccess || most < 1) {
      (void)cudaGetLastError();
      return -2;
    }
    resident[at].store(most, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, most) * o.cuts));
  if (cudaLaunchKernelEx(&cfg, kern, a, g, o, grad) != cudaSuccess) {
    (void)cudaGetLastError();
    return -2;
  }
  return 0;
}

template <typename T, bool kPolicy>
int launch_ring(const NxTokenRows& a, const NxPolicyArgs& g, RingOut o, T* grad, cudaStream_t st) {
  const int64_t pieces = static_cast<int64_t>(a.vocab) * sizeof(T) / 16;
  o.cuts = cuts_for(a.rows, pieces);
  if constexpr (!kPolicy) {
    return launch_shape<T, false, SumsShape>(a, g, o, grad, st);
  } else {
    if (!g.write_grad) return launch_shape<T, true, SumsShape>(a, g, o, grad, st);
    if constexpr (std::is_same_v<T, __half>) return -1;  // nx_policy_loss_grad
    else if ((pieces + o.cuts - 1) / o.cuts + 1 <= ShortShape::kSlots * kSlotPieces) return launch_shape<T, true, ShortShape>(a, g, o, grad, st);
    else return launch_shape<T, true, LongShape>(a, g, o, grad, st);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) scale_unless_one_kernel(T* __restrict__ x, const float* __restrict__ factor, int64_t n, int64_t vec) {
  pdl_dependency();
  pdl_trigger();
  const float f = *factor;
  if (f == 1.0f) return;
  constexpr int VN = RowVec<T>::kN;
  NX_GRID_STRIDE(i, vec) {
    float v[VN];
    RowVec<T>::load(x + i * VN, v);
#pragma unroll
    for (int j = 0; j < VN; ++j) v[j] *= f;
    RowVec<T>::store(x + i * VN, v);
  }
  for (int64_t i = vec * VN + blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    Num<T>::store(x + i, Num<T>::load(x + i) * f);
}

// ------------------------------------------------------------------------------------------------ preference loss
// A pair's sums in FP64, of log-probabilities in FP64 (the margin is a difference of sums that are near each other), by a block (long sequences)
// or a warp; ln(1 + e^-|z|) and the sigmoid from one exponential.
__global__ void __cluster_dims__(kJoinBlocks, 1, 1) __launch_bounds__(kJoinThreads)
preference_kernel(const NxPreferenceArgs a, float* __restrict__ seq_logp, float* __restrict__ margin, float* __restrict__ coef,
                  float* __restrict__ loss) {
  __shared__ double part[kJoinBlocks], scratch[32];
  cluster_arrive();
  pdl_dependency();
  pdl_trigger();
  const uint32_t rank = cluster_ctarank();
  const bool by_block = a.seq_len >= 256;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = by_block ? rank : rank * 32 + warp, step = by_block ? kJoinBlocks : kJoinBlocks * 32;
  const int from = by_block ? threadIdx.x : lane, by = by_block ? blockDim.x : 32;
  double total = 0.0;
  for (int64_t q = first; q < a.pairs; q += step) {
    double s[2], n[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int64_t at = (q + side * a.pairs) * a.seq_len;
      double acc = 0.0;
      int got = 0;
      for (int64_t t = from; t < a.seq_len; t += by) {
        acc += a.logp[at + t];  // zero where the token does not count
        got += target_at(a.targets, a.targets_wide, at + t) != a.ignore_index;
      }
      s[side] = by_block ? block_sum<double>(acc, scratch) : warp_sum_d(acc);
      n[side] = by_block ? block_sum<double>(got, scratch) : warp_sum_d(got);
      n[side] = a.average ? fmax(n[side], 1.0) : 1.0;
      s[side] /= n[side];
    }
    if (by_block ? threadIdx.x != 0 : lane != 0) continue;
    double h = s[0] - s[1];
    if (a.ref_logp != nullptr) h = (s[0] - a.ref_logp[q]) - (s[1] - a.ref_logp[q + a.pairs]);
    double value, slope;
    if (a.kind == NX_PREF_IPO) {
      const double off = h - 0.5 / a.beta;
      value = off * off;
      slope = 2.0 * off;
    } else {
      const double z = a.beta * h - a.target_margin;
      if (a.kind == NX_PREF_HINGE) {
        value = z < 1.0 ? 1.0 - z : (z == z ? 0.0 : z);
        slope = z < 1.0 ? -a.beta : 0.0;
      } else {
        // -(1 - e) ln sig(z) - e ln sig(-z) = ln(1 + exp(-|z|)) + (e - 1 where z < 0, else e) z; z may be infinite (a sequence that cannot be)
        const double t = exp(-fabs(z)), sig = z >= 0.0 ? t / (1.0 + t) : 1.0 / (1.0 + t);  // sig = sigmoid(-z)
        value = log1p(t);
        if (z < 0.0) value += (a.smoothing - 1.0) * z;
        else if (a.smoothing != 0.0f) value += a.smoothing * z;
        slope = a.beta * (a.smoothing - sig);
      }
    }
    seq_logp[q] = static_cast<float>(s[0]);
    seq_logp[q + a.pairs] = static_cast<float>(s[1]);
    margin[q] = static_cast<float>(h);
    coef[q] = static_cast<float>(slope / (n[0] * a.pairs));
    coef[q + a.pairs] = static_cast<float>(-slope / (n[1] * a.pairs));
    total += value;
  }
  total = block_sum<double>(total, scratch);
  cluster_wait();
  if (threadIdx.x == 0) put_in_first(part, rank, total);
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < kJoinBlocks; ++i) sum += part[i];
    *loss = static_cast<float>(sum / a.pairs);
  }
}

bool rows_ok(const NxTokenRows* a) {
  return a != nullptr && a->rows >= 0 && a->rows <= 0x7fffffff && a->per > 0 && a->per <= 0x7fffffff && a->vocab > 0 && a->vocab <= a->width &&
         (a->rows == 0 || (a->logits != nullptr && a->targets != nullptr));
}
// the kernels write a row's gradient in the pieces that they read it in
bool same_lines(const void* a, const void* b) { return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0; }
}  // namespace

#define NX_BY_TYPE(CODE_, ...)               \
  switch (CODE_) {                           \
    case NX_BF16: {                          \
      using T = __nv_bfloat16;               \
      __VA_ARGS__;                           \
      break;                                 \
    }                                        \
    case NX_F16: {                           \
      using T = __half;                      \
      __VA_ARGS__;                           \
      break;                                 \
    }                                        \
    case NX_F32: {                           \
      using T = float;                       \
      __VA_ARGS__;                           \
      break;                                 \
    }                                        \
    default:                                 \
      return -1;                             \
  }

extern "C" int nx_token_logprobs(const NxTokenRows* a, float* logp, float* stats, double* wide, int* status, nx_stream_t stream) {
  if (!rows_ok(a) || logp == nullptr || stats == nullptr || ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(wide)) & 7) != 0 ||
      status == nullptr)
    return -1;
  if (a->rows == 0) return 0;
  RingOut o{};
  o.logp = logp;
  o.stats = reinterpret_cast<float2*>(stats);
  o.wide = wide;
  o.status = status;
  NX_BY_TYPE(a->dtype, return launch_ring<T, false>(*a, NxPolicyArgs{}, o, nullptr, static_cast<cudaStream_t>(stream)))
}

extern "C" int nx_token_logprobs_grad(const NxTokenRows* a, const float* stats, const float* coef, int64_t coef_per, const float* factor,
                                      void* grad, nx_stream_t stream) {
  if (!rows_ok(a) || stats == nullptr || (reinterpret_cast<uintptr_t>(stats) & 7) != 0 || coef == nullptr || coef_per < 1 || coef_per > 0x7fffffff ||
      grad == nullptr || !same_lines(a->logits, grad))
    return -1;
  if (a->rows == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NX_BY_TYPE(a->dtype, NX_PDL((token_grad_kernel<T>), a->rows, kThreads, 0, st, *a, reinterpret_cast<const float2*>(stats), coef, coef_per,
                              factor, static_cast<T*>(grad)))
  return 0;
}

extern "C" int nx_policy_loss(const NxTokenRows* a, const NxPolicyArgs* g, double* totals, int32_t* counts, float* logp, float* kl,
                              float* entropy, float* row_loss, float* loss, void* grad, NxPolicySlope* slopes, int* status, nx_stream_t stream) {
  if (!rows_ok(a) || a->rows == 0 || g == nullptr || (reinterpret_cast<uintptr_t>(slopes) & 3) != 0 ||
      totals == nullptr || (reinterpret_cast<uintptr_t>(totals) & 7) != 0 || counts == nullptr || loss == nullptr || status == nullptr ||
      g->adv_per < 1 || g->adv_per > 0x7fffffff || g->seq_len < 1 || g->seq_len > 0x7fffffff || a->rows % g->seq_len != 0 ||
      (g->write_grad && (grad == nullptr || !same_lines(a->logits, grad))))
    return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NX_PDL(token_count_kernel, kJoinBlocks, kJoinThreads, 0, st, a->targets, a->targets_wide, g->mean != NX_MEAN_NONE ? a->rows / g->seq_len : 0,
         g->seq_len, a->ignore_index, totals, counts);
  RingOut o{};
  o.logp = logp;
  o.kl = kl;
  o.entropy = entropy;
  o.row_loss = row_loss;
  o.slopes = slopes;
  o.totals = totals;
  o.counts = counts;
  o.ended = reinterpret_cast<int*>(totals + 2);
  o.loss = loss;
  o.status = status;
  NX_BY_TYPE(a->dtype, return (launch_ring<T, true>(*a, *g, o, static_cast<T*>(grad), st)))
}

extern "C" int nx_policy_loss_grad(const NxTokenRows* a, const NxPolicySlope* slopes, const float* factor, void* grad, nx_stream_t stream) {
  if (!rows_ok(a) || a->dtype != NX_F16 || slopes == nullptr || (reinterpret_cast<uintptr_t>(slopes) & 3) != 0 || factor == nullptr ||
      grad == nullptr || !same_lines(a->logits, grad))
    return -1;
  if (a->rows == 0) return 0;
  NX_PDL((policy_grad_kernel<__half>), a->rows, kThreads, 0, static_cast<cudaStream_t>(stream), *a, slopes, factor, static_cast<__half*>(grad));
  return 0;
}

extern "C" int nx_scale_unless_one(void* x, const float* factor, int dtype, int64_t n, nx_stream_t stream) {
  if (n < 0 || factor == nullptr || (n > 0 && x == nullptr) || (dtype != NX_BF16 && dtype != NX_F32)) return -1;
  if (n == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t vec = (reinterpret_cast<uintptr_t>(x) & 15) ? 0 : n / (dtype == NX_BF16 ? 8 : 4);
  const int blocks = blocks_for(std::max<int64_t>(vec, 1), 256);
  if (dtype == NX_BF16) NX_PDL((scale_unless_one_kernel<__nv_bfloat16>), blocks, 256, 0, st, static_cast<__nv_bfloat16*>(x), factor, n, vec);
  else NX_PDL((scale_unless_one_kernel<float>), blocks, 256, 0, st, static_cast<float*>(x), factor, n, vec);
  return 0;
}

extern "C" int nx_preference_loss(const NxPreferenceArgs* a, float* seq_logp, float* margin, float* coef, float* loss, nx_stream_t stream) {
  if (a == nullptr || a->logp == nullptr || a->targets == nullptr || a->pairs < 1 || a->seq_len < 0 || seq_logp == nullptr ||
      margin == nullptr || coef == nullptr || loss == nullptr || a->kind < 0 || a->kind > NX_PREF_IPO)
    return -1;
  NX_PDL(preference_kernel, kJoinBlocks, kJoinThreads, 0, static_cast<cudaStream_t>(stream), *a, seq_logp, margin, coef, loss);
  return 0;
}
