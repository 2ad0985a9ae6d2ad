// Log-probabilities of given tokens, the clipped policy loss and the preference loss on logits, with their gradients.
//
//   x = logits * inv_temp,  m = max,  s = sum exp(x - m),  logp_j = x_j - m - ln s,  p_j = exp(logp_j),  H = ln s - sum p_j (x_j - m)
//   d logp_t / d x_j = delta_jt - p_j          d H / d x_j = -p_j (logp_j + H)
//
// Statistics are kept as the largest logit and log2 of the sum: with the difference taken before any product, p and logp have no
// rounding that grows with the logits (a sum m + ln s rounded to FP32 would put 2^-24 |lse| into the exponent of every p).
// Everything here is bound by the bytes of the logits.
#include "common.cuh"
#include "nx_api_objectives.h"
#include "row_vec.cuh"

#include <algorithm>

namespace {
using namespace nx;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 512;

__device__ __forceinline__ int64_t row_offset(const NxTokenRows& a, int64_t r) {
  const int64_t o = r / a.per;
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

// Running maximum, sum of exponentials and, where asked for, sum of exponentials times differences, of one thread's elements.
template <bool kEntropy>
struct Online {
  float m = -INFINITY, s = 0.0f, h = 0.0f;
  __device__ __forceinline__ void raise(float to, float k) {  // a larger maximum: the sums so far are taken down to it
    const float old = m;
    m = to;
    if (old == -INFINITY) return;  // nothing but -inf so far: the sums are zero (or NaN) as they are
    const float d = fmaxf(old - to, -1e30f);  // finite beside a masked lowest value, so that its weight of zero makes it zero
    const float f = ex2_approx(d * k);
    if (kEntropy) h = (h + d * s) * f;
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
      if (kEntropy) asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(-1e30f));
      const float e = ex2_approx(d * k);
      s += e;
      if (kEntropy) h = fmaf(e, d, h);
    }
  }
};

template <typename T, bool kEntropy>
__device__ __forceinline__ void absorb_row(const T* p, int count, float k, Online<kEntropy>& on) {
  constexpr int VN = RowVec<T>::kN;
  const RowSplit<T> sp(p, count);
  const T* body = p + sp.head;
  const int step = blockDim.x;
  int i = threadIdx.x;
  for (; i + 3 * step < sp.pieces; i += 4 * step) {
    uint4 raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = *reinterpret_cast<const uint4*>(body + static_cast<int64_t>(i + u * step) * VN);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float v[VN];
      RowVec<T>::unpack(raw[u], v);
      on.absorb(v, k);
    }
  }
  for (; i < sp.pieces; i += step) {
    float v[VN];
    RowVec<T>::load(body + static_cast<int64_t>(i) * VN, v);
    on.absorb(v, k);
  }
  if (static_cast<int>(threadIdx.x) < sp.head) {
    const float v[1] = {Num<T>::load(p + threadIdx.x)};
    on.absorb(v, k);
  } else if (static_cast<int>(threadIdx.x) >= 32 && static_cast<int>(threadIdx.x) - 32 < sp.tail) {
    const float v[1] = {Num<T>::load(body + static_cast<int64_t>(sp.pieces) * VN + threadIdx.x - 32)};
    on.absorb(v, k);
  }
}

// Every thread gets the block's maximum and sums.
template <bool kEntropy>
__device__ __forceinline__ void join_block(Online<kEntropy>& on, float k, float* scratch) {
  const float top = block_max(on.m, scratch);
  if (on.m != top) on.raise(top, k);
  on.s = block_sum<float>(on.s, scratch);
  if (kEntropy) on.h = block_sum<float>(on.h, scratch);
}

// ------------------------------------------------------------------------------------------------ log-probabilities
template <typename T>
__global__ void __launch_bounds__(kThreads) token_stats_kernel(const NxTokenRows a, float* __restrict__ logp, float2* __restrict__ stats) {
  __shared__ float scratch[32];
  pdl_dependency();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const int64_t tg = target_at(a.targets, a.targets_wide, row);
  const bool inside = tg >= 0 && tg < a.vocab;
  if (tg == a.ignore_index || !inside) {
    if (threadIdx.x == 0) {
      logp[row] = tg == a.ignore_index ? 0.0f : NAN;
      stats[row] = make_float2(0.0f, 0.0f);
    }
    return;
  }
  const T* p = reinterpret_cast<const T*>(a.logits) + row_offset(a, row);
  Online<false> on;
  absorb_row(p, a.vocab, a.inv_temp * kLog2e, on);
  join_block(on, a.inv_temp * kLog2e, scratch);
  if (threadIdx.x == 0) {
    logp[row] = (Num<T>::load(p + tg) - on.m) * a.inv_temp - logf(on.s);
    stats[row] = make_float2(on.m, log2f(on.s));
  }
}

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

template <typename T>
__global__ void __launch_bounds__(kThreads) token_grad_kernel(const NxTokenRows a, const float2* __restrict__ stats,
                                                              const float* __restrict__ coef, int64_t coef_per,
                                                              const float* __restrict__ factor, T* __restrict__ grad) {
  pdl_dependency();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const int64_t tg = target_at(a.targets, a.targets_wide, row);
  const int64_t at = row_offset(a, row);
  T* g = grad + at;
  if (tg == a.ignore_index || tg < 0 || tg >= a.vocab) {
    clear_row(g, a.width);
    return;
  }
  const float c = coef[row / coef_per] * (factor != nullptr ? *factor : 1.0f) * a.inv_temp;
  const float2 st = stats[row];
  const float k = a.inv_temp * kLog2e;
  write_row(reinterpret_cast<const T*>(a.logits) + at, g, a.vocab, a.width, static_cast<int>(tg), c,
            [&](float v) { return -c * ex2_approx(fmaf(v - st.x, k, -st.y)); });
}

// ------------------------------------------------------------------------------------------------ policy loss
// Sums over a few thousand to a million values by one cluster of eight blocks: partial sums meet in the first block's shared memory.
constexpr int kJoinBlocks = 8, kJoinThreads = 1024;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// slot[rank] of the cluster's first block = v; one thread of each block, once every block of the cluster is known to run
__device__ __forceinline__ void put_in_first(double* slot, uint32_t rank, double v) {
  uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(slot + rank)), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(addr));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}

// totals[0] = rows that count, totals[1] = sequences with such rows; counts[q] = rows of sequence q that count
__global__ void __cluster_dims__(kJoinBlocks, 1, 1) __launch_bounds__(kJoinThreads)
token_count_kernel(const void* __restrict__ targets, int wide, int64_t sequences, int64_t len, int64_t ignore, double* __restrict__ totals,
                   int32_t* __restrict__ counts) {
  __shared__ double tokens[kJoinBlocks], filled[kJoinBlocks];
  __shared__ double scratch[32];
  cluster_arrive();
  pdl_dependency();
  pdl_trigger();
  const uint32_t rank = cluster_rank();
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
  }
}

// out = sum of x in a fixed order
__global__ void __cluster_dims__(kJoinBlocks, 1, 1) __launch_bounds__(kJoinThreads)
sum_kernel(const float* __restrict__ x, int64_t n, float* __restrict__ out) {
  __shared__ double part[kJoinBlocks], scratch[32];
  cluster_arrive();
  pdl_dependency();
  pdl_trigger();
  const uint32_t rank = cluster_rank();
  double acc = 0.0;
  for (int64_t i = rank * kJoinThreads + threadIdx.x; i < n; i += kJoinBlocks * kJoinThreads) acc += x[i];
  acc = block_sum<double>(acc, scratch);
  cluster_wait();
  if (threadIdx.x == 0) put_in_first(part, rank, acc);
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && threadIdx.x == 0) {
    double a = 0.0;
    for (int i = 0; i < kJoinBlocks; ++i) a += part[i];
    *out = static_cast<float>(a);
  }
}

struct PolicyRow {
  float c;       // d row loss / d logp, weighted
  float ent;     // entropy coefficient, weighted
  float loss, kl;
};
__device__ __forceinline__ PolicyRow policy_row(const NxPolicyArgs& g, int64_t row, float logp, float entropy, float weight) {
  PolicyRow o;
  const float adv = g.advantages[row / g.adv_per];
  const float ratio = expf(logp - g.old_logp[row]);
  const float free = ratio * adv, bound = fminf(fmaxf(ratio, 1.0f - g.clip_low), 1.0f + g.clip_high) * adv;
  const bool follows = free <= bound;  // the unclipped term is the smaller one, or they are equal
  float loss = follows ? -free : -bound, c = follows ? -free : 0.0f;
  o.kl = 0.0f;
  if (g.ref_logp != nullptr) {
    const float d = g.ref_logp[row] - logp;
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
    loss = fmaf(g.kl_coef, o.kl, loss);
    c = fmaf(g.kl_coef, slope, c);
  }
  if (g.entropy_coef != 0.0f) loss -= g.entropy_coef * entropy;
  o.loss = loss * weight;
  o.c = c * weight;
  o.ent = g.entropy_coef * weight;
  return o;
}

// Weight of a row: the whole batch's mean over tokens, the mean over sequences of the means over their tokens, or one.
__device__ __forceinline__ float policy_weight(const NxPolicyArgs& g, const double* totals, const int32_t* counts, int64_t row) {
  if (g.mean == NX_MEAN_NONE) return g.scale;
  if (g.mean == NX_MEAN_TOKEN) return static_cast<float>(g.scale / totals[0]);
  return static_cast<float>(g.scale / (totals[1] * counts[row / g.seq_len]));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) policy_kernel(const NxTokenRows a, const NxPolicyArgs g, const double* __restrict__ totals,
                                                          const int32_t* __restrict__ counts, float* __restrict__ logp, float* __restrict__ kl, float* __restrict__ entropy,
                                                          float* __restrict__ row_loss, T* __restrict__ grad) {
  __shared__ float scratch[32];
  pdl_dependency();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const int64_t tg = target_at(a.targets, a.targets_wide, row);
  const int64_t at = row_offset(a, row);
  if (tg == a.ignore_index || tg < 0 || tg >= a.vocab) {
    if (threadIdx.x == 0) {
      const float v = tg == a.ignore_index ? 0.0f : NAN;
      logp[row] = kl[row] = entropy[row] = row_loss[row] = v;
    }
    if (g.write_grad) clear_row(grad + at, a.width);
    return;
  }
  const float weight = policy_weight(g, totals, counts, row);
  const T* p = reinterpret_cast<const T*>(a.logits) + at;
  const float k = a.inv_temp * kLog2e;
  Online<true> on;
  absorb_row(p, a.vocab, k, on);
  join_block(on, k, scratch);
  const float ln_s = logf(on.s), log2_s = log2f(on.s);
  const float lp = (Num<T>::load(p + tg) - on.m) * a.inv_temp - ln_s;
  const float ent = ln_s - on.h / on.s * a.inv_temp;
  const PolicyRow r = policy_row(g, row, lp, ent, weight);
  if (threadIdx.x == 0) {
    logp[row] = lp;
    kl[row] = r.kl;
    entropy[row] = ent;
    row_loss[row] = r.loss;
  }
  if (!g.write_grad) return;
  const float c = r.c * a.inv_temp;
  if (g.entropy_coef == 0.0f) {
    write_row(p, grad + at, a.vocab, a.width, static_cast<int>(tg), c,
              [&](float v) { return -c * ex2_approx(fmaf(v - on.m, k, -log2_s)); });
  } else {
    const float e1 = r.ent * a.inv_temp, slope = e1 * a.inv_temp, base = e1 * (ent - ln_s) - c;
    write_row(p, grad + at, a.vocab, a.width, static_cast<int>(tg), c, [&](float v) {
      float d = v - on.m;
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(-1e30f));
      return ex2_approx(fmaf(d, k, -log2_s)) * fmaf(d, slope, base);
    });
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
// A pair's sums in FP64 by a block (long sequences) or a warp; ln(1 + e^-|z|) and the sigmoid from one exponential.
__global__ void __cluster_dims__(kJoinBlocks, 1, 1) __launch_bounds__(kJoinThreads)
preference_kernel(const NxPreferenceArgs a, float* __restrict__ seq_logp, float* __restrict__ margin, float* __restrict__ coef,
                  float* __restrict__ loss) {
  __shared__ double part[kJoinBlocks], scratch[32];
  cluster_arrive();
  pdl_dependency();
  pdl_trigger();
  const uint32_t rank = cluster_rank();
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
        // -(1 - e) ln sig(z) - e ln sig(-z) = ln(1 + exp(-|z|)) + max(-z, 0) + e z
        const double t = exp(-fabs(z)), sig = z >= 0.0 ? t / (1.0 + t) : 1.0 / (1.0 + t);  // sig = sigmoid(-z)
        value = log1p(t) + (z < 0.0 ? -z : 0.0) + a.smoothing * z;
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
  return a != nullptr && a->rows >= 0 && a->rows <= 0x7fffffff && a->per > 0 && a->vocab > 0 && a->vocab <= a->width &&
         (a->rows == 0 || (a->logits != nullptr && a->targets != nullptr));
}
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

extern "C" int nx_token_logprobs(const NxTokenRows* a, float* logp, float* stats, nx_stream_t stream) {
  if (!rows_ok(a) || logp == nullptr || stats == nullptr) return -1;
  if (a->rows == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NX_BY_TYPE(a->dtype, NX_PDL((token_stats_kernel<T>), a->rows, kThreads, 0, st, *a, logp, reinterpret_cast<float2*>(stats)))
  return 0;
}

extern "C" int nx_token_logprobs_grad(const NxTokenRows* a, const float* stats, const float* coef, int64_t coef_per, const float* factor,
                                      void* grad, nx_stream_t stream) {
  if (!rows_ok(a) || stats == nullptr || coef == nullptr || coef_per < 1 || grad == nullptr) return -1;
  if (a->rows == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NX_BY_TYPE(a->dtype, NX_PDL((token_grad_kernel<T>), a->rows, kThreads, 0, st, *a, reinterpret_cast<const float2*>(stats), coef, coef_per,
                              factor, static_cast<T*>(grad)))
  return 0;
}

extern "C" int nx_policy_loss(const NxTokenRows* a, const NxPolicyArgs* g, double* totals, int32_t* counts, float* logp, float* kl,
                              float* entropy, float* row_loss, float* loss, void* grad, nx_stream_t stream) {
  if (!rows_ok(a) || g == nullptr || totals == nullptr || counts == nullptr || loss == nullptr || g->adv_per < 1 || g->seq_len < 1 ||
      a->rows % g->seq_len != 0 || (g->write_grad && grad == nullptr))
    return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (g->mean != NX_MEAN_NONE)
    NX_PDL(token_count_kernel, kJoinBlocks, kJoinThreads, 0, st, a->targets, a->targets_wide, a->rows / g->seq_len, g->seq_len, a->ignore_index, totals, counts);
  if (a->rows > 0)
    NX_BY_TYPE(a->dtype, NX_PDL((policy_kernel<T>), a->rows, kThreads, 0, st, *a, *g, totals, counts, logp, kl, entropy, row_loss, static_cast<T*>(grad)))
  NX_PDL(sum_kernel, kJoinBlocks, kJoinThreads, 0, st, row_loss, a->rows, loss);
  return 0;
}

extern "C" int nx_scale_unless_one(void* x, const float* factor, int dtype, int64_t n, nx_stream_t stream) {
  if (n < 0 || factor == nullptr || (n > 0 && x == nullptr)) return -1;
  if (n == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NX_BY_TYPE(dtype, const int64_t vec = (reinterpret_cast<uintptr_t>(x) & 15) ? 0 : n / RowVec<T>::kN;
             NX_PDL((scale_unless_one_kernel<T>), blocks_for(std::max<int64_t>(vec, 1), 256), 256, 0, st, static_cast<T*>(x), factor, n, vec))
  return 0;
}

extern "C" int nx_preference_loss(const NxPreferenceArgs* a, float* seq_logp, float* margin, float* coef, float* loss, nx_stream_t stream) {
  if (a == nullptr || a->logp == nullptr || a->targets == nullptr || a->pairs < 1 || a->seq_len < 0 || seq_logp == nullptr ||
      margin == nullptr || coef == nullptr || loss == nullptr || a->kind < 0 || a->kind > NX_PREF_IPO)
    return -1;
  NX_PDL(preference_kernel, kJoinBlocks, kJoinThreads, 0, static_cast<cudaStream_t>(stream), *a, seq_logp, margin, coef, loss);
  return 0;
}
