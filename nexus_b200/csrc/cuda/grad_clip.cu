// Global norm of the gradients of many tensors, and the clipped gradients:  |g| = sqrt(sum g^2),  g <- min(1, max / (|g| + 1e-6)) g.
//
// Two launches for any list of up to kTableMax tensors (further launches of the same two kernels beyond): the descriptors travel as kernel
// arguments, so nothing is uploaded and a captured graph carries its own.  A block walks over pieces of kPiece elements, whatever tensors they
// belong to.  The second kernel's blocks each add up the first one's partial sums, in the same order, instead of a launch in between.
// Bound by bytes: every gradient is read twice and written once; the second pass walks backwards, so that it begins with what the first one
// left in L2.  8 x [4096, 4096] FP32: norm 82 us (6.5 TB/s), both passes to other memory 293 us (5.5 TB/s of two reads and a write); in place with
// a norm that is small enough 107.  Other shapes of blocks (256, 1024 threads; two or four pieces in flight) and stores past L2 were no faster.
#include "common.cuh"
#include "nx_api_objectives.h"
#include "row_vec.cuh"

#include <algorithm>

namespace {
using namespace nx;

constexpr int kPiece = 16384;     // elements of one block's turn
constexpr int kClipThreads = 512;
constexpr int kTableMax = 256;    // tensors of one launch: 7 KiB of arguments
constexpr int kClipBlocks = kNumSmsB200 * 4;

template <int N>
struct Table {
  const void* src[N];
  void* dst[N];
  int64_t count[N];
  int32_t last[N];    // pieces of the tensors up to this one, itself included
  uint8_t type[N];    // of src | of dst << 4
  int tensors, pieces;
};

struct Piece {
  int tensor;
  int64_t begin, count;
};
template <int N>
__device__ __forceinline__ Piece find_piece(const Table<N>& t, int piece) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t.last[mid] > piece) hi = mid;
    else lo = mid + 1;
  }
  Piece p;
  p.tensor = lo;
  const int first = lo == 0 ? 0 : t.last[lo - 1];
  p.begin = static_cast<int64_t>(piece - first) * kPiece;
  p.count = min(static_cast<int64_t>(kPiece), t.count[lo] - p.begin);
  return p;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    float a[4], b[4];
    RowVec<T>::load(p, a);
    RowVec<T>::load(p + 4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
    RowVec<T>::load(p, v);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    RowVec<T>::store(p, v);
  }
}

template <typename T>
__device__ __forceinline__ double square_sum(const T* p, int n) {
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const int head = min(n, off == 0 ? 0 : static_cast<int>(16 / sizeof(T)) - off), vec = (n - head) / 8;
  double acc = 0.0;
  for (int i = threadIdx.x; i < vec; i += blockDim.x) {
    float v[8];
    load8(p + head + i * 8, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc += static_cast<double>(v[j]) * v[j];
  }
  const int rest = head + (n - head - vec * 8);  // the elements before the first boundary and behind the last piece of eight
  for (int i = threadIdx.x; i < rest; i += blockDim.x) {
    const double v = Num<T>::load(p + (i < head ? i : vec * 8 + i));
    acc += v * v;
  }
  return acc;
}

template <int N>
__global__ void __launch_bounds__(kClipThreads) square_sum_kernel(const __grid_constant__ Table<N> t, double* __restrict__ partial) {
  __shared__ double scratch[32];
  pdl_dependency();
  pdl_trigger();
  double acc = 0.0;
  for (int i = blockIdx.x; i < t.pieces; i += gridDim.x) {
    const Piece p = find_piece(t, i);
    const int type = t.type[p.tensor] & 15;
    const int n = static_cast<int>(p.count);
    if (type == NX_F32) acc += square_sum(static_cast<const float*>(t.src[p.tensor]) + p.begin, n);
    else if (type == NX_BF16) acc += square_sum(static_cast<const __nv_bfloat16*>(t.src[p.tensor]) + p.begin, n);
    else acc += square_sum(static_cast<const __half*>(t.src[p.tensor]) + p.begin, n);
  }
  acc = block_sum<double>(acc, scratch);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__device__ __forceinline__ double total_of(const double* partial, int parts, double* scratch) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += blockDim.x) acc += partial[i];
  return block_sum<double>(acc, scratch);
}

template <typename S, typename D>
__device__ __forceinline__ void scaled(const S* s, D* d, int n, float f) {
  // an index from which on both sides are on 16-byte boundaries, if there is one
  int head = -1;
  for (int i = 0; i < 8 && head < 0; ++i)
    if (((reinterpret_cast<uintptr_t>(s + i) | reinterpret_cast<uintptr_t>(d + i)) & 15) == 0) head = i;
  const int start = head < 0 ? n : min(head, n), vec = (n - start) / 8;
  for (int i = threadIdx.x; i < vec; i += blockDim.x) {
    float v[8];
    load8(s + start + i * 8, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    store8(d + start + i * 8, v);
  }
  const int rest = n - vec * 8;
  for (int i = threadIdx.x; i < rest; i += blockDim.x) {
    const int at = i < start ? i : vec * 8 + i;
    Num<D>::store(d + at, Num<S>::load(s + at) * f);
  }
}
template <typename S>
__device__ __forceinline__ void scaled_to(const S* s, void* d, int type, int64_t at, int n, float f) {
  if (type == NX_F32) scaled(s + at, static_cast<float*>(d) + at, n, f);
  else if (type == NX_BF16) scaled(s + at, static_cast<__nv_bfloat16*>(d) + at, n, f);
  else scaled(s + at, static_cast<__half*>(d) + at, n, f);
}

// out[0] = sum of squares (FP64), then the norm (FP32); tensors of the table <- factor * themselves.  A norm that is not finite leaves them as
// they are.  `copy`: the results go to other memory, so a factor of 1 copies.
template <int N>
__global__ void __launch_bounds__(kClipThreads) clip_kernel(const __grid_constant__ Table<N> t, const double* __restrict__ partial, int parts,
                                                            double max_norm, int copy, double* __restrict__ out) {
  __shared__ double scratch[32];
  pdl_dependency();
  pdl_trigger();
  const double sq = total_of(partial, parts, scratch), norm = sqrt(sq);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    out[0] = sq;
    reinterpret_cast<float*>(out + 1)[0] = static_cast<float>(norm);
  }
  float f = 1.0f;
  if (isfinite(norm)) f = static_cast<float>(fmin(1.0, max_norm / (norm + 1e-6)));
  if (f == 1.0f && !copy) return;
  for (int i = blockIdx.x; i < t.pieces; i += gridDim.x) {
    const Piece p = find_piece(t, t.pieces - 1 - i);
    const int from = t.type[p.tensor] & 15, to = t.type[p.tensor] >> 4, n = static_cast<int>(p.count);
    if (from == NX_F32) scaled_to(static_cast<const float*>(t.src[p.tensor]), t.dst[p.tensor], to, p.begin, n, f);
    else if (from == NX_BF16) scaled_to(static_cast<const __nv_bfloat16*>(t.src[p.tensor]), t.dst[p.tensor], to, p.begin, n, f);
    else scaled_to(static_cast<const __half*>(t.src[p.tensor]), t.dst[p.tensor], to, p.begin, n, f);
  }
}

template <int N>
int fill(Table<N>* t, const NxGradTable* g, int64_t first, int64_t end) {
  int64_t pieces = 0;
  for (int64_t i = first; i < end; ++i) {
    const int k = static_cast<int>(i - first);
    t->src[k] = g->src[i];
    t->dst[k] = g->dst != nullptr ? g->dst[i] : const_cast<void*>(g->src[i]);
    t->count[k] = g->count[i];
    t->type[k] = static_cast<uint8_t>(g->type[i]);
    pieces += (g->count[i] + kPiece - 1) / kPiece;
    if (pieces > 0x7fffffff) return -1;
    t->last[k] = static_cast<int32_t>(pieces);
  }
  t->tensors = static_cast<int>(end - first);
  t->pieces = static_cast<int>(pieces);
  return 0;
}

template <int N>
int run(const NxGradTable* g, double max_norm, int clip, double* partial, double* out, cudaStream_t st) {
  Table<N> t;
  int parts = 0;
  for (int64_t first = 0; first < g->tensors; first += N) {
    if (fill(&t, g, first, std::min<int64_t>(g->tensors, first + N)) != 0) return -1;
    const int blocks = std::min(t.pieces, kClipBlocks);
    NX_PDL((square_sum_kernel<N>), blocks, kClipThreads, 0, st, t, partial + parts);
    parts += blocks;
  }
  if (!clip) {
    t.pieces = 0;
    NX_PDL((clip_kernel<N>), 1, kClipThreads, 0, st, t, partial, parts, max_norm, 0, out);
    return 0;
  }
  for (int64_t last = (g->tensors - 1) / N; last >= 0; --last) {
    if (fill(&t, g, last * N, std::min<int64_t>(g->tensors, last * N + N)) != 0) return -1;
    NX_PDL((clip_kernel<N>), std::min(t.pieces, kClipBlocks), kClipThreads, 0, st, t, partial, parts, max_norm, g->dst != nullptr ? 1 : 0, out);
  }
  return 0;
}
}  // namespace

extern "C" int nx_grad_clip(const NxGradTable* g, double max_norm, int clip, double* partial, double* out, nx_stream_t stream) {
  if (g == nullptr || g->tensors < 1 || g->src == nullptr || g->count == nullptr || g->type == nullptr || partial == nullptr || out == nullptr ||
      !(max_norm >= 0.0))
    return -1;
  for (int64_t i = 0; i < g->tensors; ++i)
    if (g->src[i] == nullptr || g->count[i] < 1 || (g->type[i] & 15) > NX_F16 || (g->type[i] >> 4) > NX_F16 ||
        (g->dst != nullptr && g->dst[i] == nullptr))
      return -1;
  return run<kTableMax>(g, max_norm, clip, partial, out, static_cast<cudaStream_t>(stream));
}
