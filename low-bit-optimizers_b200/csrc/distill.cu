// Distillation from a teacher's K stored top logits: the loss, its gradient, and both in one call.
//
//   p_k = exp(t_k / T) / sum_j exp(t_j / T)       over a row's K stored entries (index < 0 or t = -inf: no entry)
//   q_v = exp(x_v / T) / sum_u exp(x_u / T)       over the whole vocabulary
//   loss = w T^2 sum_k p_k (log p_k - log q_{i_k})
//   d loss / d x_v = w T (q_v - sum_{k: i_k = v} p_k)
//
// One CTA, or one cluster of CTAs that share the row's columns, takes a row: a pass with a running maximum and sum
// gives the softmax statistics; the gradient is a second pass over the same columns, which the first one has left in
// L2, then the K corrected entries are written over it.  All sums are fp32, the gradient is rounded once.
// Bound by memory: a logit is read once and its gradient written once; an exponential per logit and pass.
#include <cooperative_groups.h>

#include "loss_common.cuh"

namespace cg = cooperative_groups;

namespace lpmm_b200 {

enum { DISTILL_LOSS = 0, DISTILL_BOTH = 1, DISTILL_GRAD = 2 };

constexpr int MAX_K = LPMM_B200_DISTILL_MAX_K;
constexpr int HASH = 2 * MAX_K;  // at most half full

// saved per row for the gradient: maximum and sum of the student's exponentials, the same of the teacher's.  The
// teacher's sum is 0 for a row that has no part in the loss, NaN for one whose entries are invalid.
struct __align__(16) RowStats {
  float m, s, tm, ts;
};

struct DistillArgs {
  const void* logits;
  void* grad;
  const void* teacher;
  const void* index;
  const float* weights;
  const float* upstream;
  float* row_loss;
  RowStats* stats;
  const float* norm;  // 1 / sum of the weights, for the mean
  long long rows, inner, outer_stride, inner_stride;
  int vocab, k, teacher_dtype, index_bits, upstream_per_row;
  float temperature, c;  // c = log2(e) / T
  float scale;
  int slice;  // columns per CTA of the cluster
};

constexpr float LOWEST = -3.402823466e38f;

// (m, s) stands for s * 2^(m c).  m starts at the lowest finite value: a -inf logit then adds 2^-inf = 0, and a NaN or
// +inf reaches s.
struct Running {
  float m, s;
};

__device__ __forceinline__ Running join(const Running& a, const Running& b, float c) {
  Running r;
  r.m = fmaxf(a.m, b.m);
  r.s = a.s * ex2((a.m - r.m) * c) + b.s * ex2((b.m - r.m) * c);
  return r;
}

template <int N>
__device__ __forceinline__ void take(Running& a, const float* x, float c) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
  m = fmaxf(m, a.m);
  float s = a.s * ex2((a.m - m) * c);
#pragma unroll
  for (int i = 0; i < N; ++i) s += ex2((x[i] - m) * c);
  a.m = m;
  a.s = s;
}

struct DistillSmem {
  int idx[MAX_K];
  float p[MAX_K];
  float x[MAX_K];
  int hash[HASH];
  Running warp[32];
  float red[32];
  Running mine;  // this CTA's part of the row, read by the cluster
  int bad, twice;
};

__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) r = fmaxf(r, red[i]);
  return r;
}

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) r += red[i];
  return r;
}

// Columns [lo, hi) of a row in steps of 16 bytes: up to VE - 1 single columns before the first boundary, vectors, the
// rest singly.
struct Span {
  int lo, head, vecs, tail, tail_at;
};

template <typename T>
__device__ __forceinline__ Span span_of(const T* row, int lo, int hi) {
  constexpr int VE = Elem<T>::VE;
  Span s;
  s.lo = lo;
  const int n = hi - lo;
  const int off = (int)(((uintptr_t)(row + lo) & 15) / sizeof(T));
  s.head = off ? min(VE - off, n) : 0;
  s.vecs = (n - s.head) / VE;
  s.tail_at = lo + s.head + s.vecs * VE;
  s.tail = hi - s.tail_at;
  return s;
}

template <typename T, int MODE>
__global__ void __launch_bounds__(512) distill_kernel(const DistillArgs a) {
  using E = Elem<T>;
  constexpr int VE = E::VE;
  __shared__ DistillSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int lo = min(part * a.slice, a.vocab), hi = min(lo + a.slice, a.vocab);
  const T* x = reinterpret_cast<const T*>(a.logits) + (row / a.inner) * a.outer_stride + (row % a.inner) * a.inner_stride;
  T* g = MODE == DISTILL_LOSS ? nullptr : reinterpret_cast<T*>(a.grad) + row * a.vocab;
  const float w = a.weights ? a.weights[row] : 1.0f;

  // the teacher's entries; an index outside the vocabulary makes the row NaN and is not followed
  if (tid == 0) sm.bad = sm.twice = 0;
  if (MODE != DISTILL_LOSS)
    for (int i = tid; i < HASH; i += nthr) sm.hash[i] = -1;
  __syncthreads();
  float tm = LOWEST;
  bool any = false;
  for (int k = tid; k < a.k; k += nthr) {
    const long long i = load_index(a.index, row * a.k + k, a.index_bits);
    const float t = load_any(a.teacher, row * a.k + k, a.teacher_dtype);
    const bool entry = i >= 0 && t != -__int_as_float(0x7f800000);
    if (entry && i >= a.vocab) sm.bad = 1;
    sm.idx[k] = entry && i < a.vocab ? (int)i : -1;
    sm.p[k] = t;
    if (entry) {
      any = true;
      tm = fmaxf(tm, t);
    }
  }
  const bool live = __syncthreads_or(any) && w != 0.0f;
  const bool bad = sm.bad;
  if (!live) {  // uniform over the cluster: every CTA of it has read the same entries
    if (MODE != DISTILL_LOSS) {
      const Span o = span_of(g, lo, hi);
      if (tid < o.head) g[o.lo + tid] = E::narrow(0.0f);
      uint4* gv = reinterpret_cast<uint4*>(g + o.lo + o.head);
      for (int i = tid; i < o.vecs; i += nthr) gv[i] = make_uint4(0, 0, 0, 0);
      if (tid < o.tail) g[o.tail_at + tid] = E::narrow(0.0f);
    }
    if (MODE != DISTILL_GRAD && tid == 0 && part == 0) {
      a.row_loss[row] = 0.0f;
      a.stats[row] = RowStats{0.0f, 1.0f, 0.0f, 0.0f};
    }
    return;
  }
  float ts, m, s;
  if (MODE == DISTILL_GRAD) {
    const RowStats st = a.stats[row];
    tm = st.tm, ts = st.ts, m = st.m, s = st.s;
    for (int k = tid; k < a.k; k += nthr) sm.p[k] = sm.idx[k] >= 0 ? ex2((sm.p[k] - tm) * a.c) / ts : 0.0f;
  } else {
    tm = block_max(tm, sm.red);
    float sum = 0.0f;
    for (int k = tid; k < a.k; k += nthr)
      if (sm.idx[k] >= 0) sum += ex2((sm.p[k] - tm) * a.c);
    ts = block_sum(sum, sm.red);
    if (bad) ts = nan_f();

    // one pass over the row: running maximum and sum
    const Span o = span_of(x, lo, hi);
    Running r{LOWEST, 0.0f};
    if (tid < o.head) {
      const float v = E::widen(x[o.lo + tid]);
      take<1>(r, &v, a.c);
    }
    if (tid < o.tail) {
      const float v = E::widen(x[o.tail_at + tid]);
      take<1>(r, &v, a.c);
    }
    const uint4* xv = reinterpret_cast<const uint4*>(x + o.lo + o.head);
    int i = tid;
    for (; i + 3 * nthr < o.vecs; i += 4 * nthr) {
      float v[4 * VE];
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = xv[i + j * nthr];
#pragma unroll
      for (int j = 0; j < 4; ++j) E::unpack(u[j], v + j * VE);
      take<4 * VE>(r, v, a.c);
    }
    for (; i < o.vecs; i += nthr) {
      float v[VE];
      E::unpack(xv[i], v);
      take<VE>(r, v, a.c);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      Running b;
      b.m = __shfl_xor_sync(~0u, r.m, d);
      b.s = __shfl_xor_sync(~0u, r.s, d);
      r = join(r, b, a.c);
    }
    if ((tid & 31) == 0) sm.warp[tid >> 5] = r;
    __syncthreads();
    r = sm.warp[0];
    for (int j = 1; j < (nthr >> 5); ++j) r = join(r, sm.warp[j], a.c);
    if (parts > 1) {
      if (tid == 0) sm.mine = r;
      cluster.sync();
      r = *cluster.map_shared_rank(&sm.mine, 0);
      for (int j = 1; j < parts; ++j) r = join(r, *cluster.map_shared_rank(&sm.mine, j), a.c);
      cluster.sync();  // nobody leaves while its part is still read
    }
    m = r.m;
    s = r.s == 0.0f ? nan_f() : r.s;  // every logit -inf: no distribution

    if (part == 0) {
      const float inv_t = 1.0f / a.temperature, log_ts = logf(ts);
      float sum_l = 0.0f;
      for (int k = tid; k < a.k; k += nthr) {
        if (sm.idx[k] < 0) continue;
        const float z = sm.p[k] - tm, p = ex2(z * a.c) / ts;
        if (p != 0.0f) sum_l += p * ((z - (E::widen(x[sm.idx[k]]) - m)) * inv_t - log_ts);
      }
      sum_l = block_sum(sum_l, sm.red);
      if (tid == 0) {
        a.row_loss[row] = w * a.temperature * a.temperature * (sum_l + logf(s)) + (ts - ts);
        a.stats[row] = RowStats{m, s, tm, ts};
      }
    }
    if (MODE == DISTILL_LOSS) return;
    __syncthreads();
    for (int k = tid; k < a.k; k += nthr) sm.p[k] = sm.idx[k] >= 0 ? ex2((sm.p[k] - tm) * a.c) / ts : 0.0f;
  }

  // the gradient: q everywhere, then the entries of this part of the row
  float up = a.scale * (a.norm ? *a.norm : 1.0f);
  if (a.upstream) up *= a.upstream[a.upstream_per_row ? row : 0];
  const float G = up * w * a.temperature + (ts - ts);  // NaN for a row with invalid entries
  const float gs = G / s;
  for (int k = tid; k < a.k; k += nthr) {
    const int i = sm.idx[k];
    if (i < lo || i >= hi) continue;
    sm.x[k] = E::widen(x[i]);
    for (unsigned h = (unsigned)i * 2654435761u >> 16;; ++h) {  // ends: the table is at most half full
      const int was = atomicCAS(&sm.hash[h % HASH], -1, i);
      if (was == -1) break;
      if (was == i) {
        sm.twice = 1;
        break;
      }
    }
  }
  {
    const Span o = span_of(g, lo, hi);
    if (tid < o.head) g[o.lo + tid] = E::narrow(gs * ex2((E::widen(x[o.lo + tid]) - m) * a.c));
    if (tid < o.tail) g[o.tail_at + tid] = E::narrow(gs * ex2((E::widen(x[o.tail_at + tid]) - m) * a.c));
    uint4* gv = reinterpret_cast<uint4*>(g + o.lo + o.head);
    const T* xs = x + o.lo + o.head;
    if (((uintptr_t)xs & 15) == 0) {
      const uint4* xv = reinterpret_cast<const uint4*>(xs);
      for (int i = tid; i < o.vecs; i += nthr) {
        float v[VE];
        E::unpack(xv[i], v);
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = gs * ex2((v[j] - m) * a.c);
        gv[i] = E::pack(v);
      }
    } else {  // rows of logits and gradient that lie differently to the 16-byte boundaries: single loads
      for (int i = tid; i < o.vecs; i += nthr) {
        float v[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = gs * ex2((E::widen(xs[i * VE + j]) - m) * a.c);
        gv[i] = E::pack(v);
      }
    }
  }
  __syncthreads();
  const bool twice = sm.twice;
  for (int k = tid; k < a.k; k += nthr) {
    const int i = sm.idx[k];
    if (i < lo || i >= hi) continue;
    float p = sm.p[k];
    if (twice) {  // an index that occurs several times: its first entry writes for all, in their order
      bool first = true;
      for (int j = 0; j < k; ++j) first &= sm.idx[j] != i;
      if (!first) continue;
      for (int j = k + 1; j < a.k; ++j)
        if (sm.idx[j] == i) p += sm.p[j];
    }
    g[i] = E::narrow(gs * ex2((sm.x[k] - m) * a.c) - G * p);
  }
}

// One CTA: the sum of the weights and of the weighted row losses in a fixed order, in double.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ row_loss,
                                                              const float* __restrict__ weights, long long rows, int mean,
                                                              float* __restrict__ loss, float* __restrict__ norm) {
  __shared__ double red[2][32];
  double l = 0.0, w = 0.0;
  for (long long i = threadIdx.x; i < rows; i += blockDim.x) {
    if (row_loss) l += row_loss[i];
    if (mean && weights) w += weights[i];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    l += __shfl_xor_sync(~0u, l, o);
    w += __shfl_xor_sync(~0u, w, o);
  }
  if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = l, red[1][threadIdx.x >> 5] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    l = w = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) l += red[0][i], w += red[1][i];
    if (mean && !weights) w = (double)rows;
    const double n = !mean ? 1.0 : w == 0.0 ? 0.0 : 1.0 / w;
    if (norm) *norm = (float)n;
    if (loss) *loss = n == 0.0 ? 0.0f : (float)(l * n);
  }
}

static int distill_check(const lpmm_b200_distill* d, int mode) {
  if (!d) return LPMM_B200_ERR_NULL_POINTER;
  if (d->rows < 0 || d->inner < 1 || d->vocab < 1 || d->k < 1) return LPMM_B200_ERR_BAD_SIZE;
  if (d->dtype < 0 || d->dtype > 2 || d->teacher_dtype < 0 || d->teacher_dtype > 2) return LPMM_B200_ERR_BAD_KIND;
  if (d->index_bits != 32 && d->index_bits != 64) return LPMM_B200_ERR_BAD_KIND;
  if (d->reduction < 0 || d->reduction > 2) return LPMM_B200_ERR_BAD_KIND;
  if (!(d->temperature >= LPMM_B200_DISTILL_MIN_T && d->temperature <= LPMM_B200_DISTILL_MAX_T)) return LPMM_B200_ERR_BAD_SIZE;
  if (d->k > MAX_K || d->vocab > (1 << 30) || d->rows >= (1ll << 28)) return LPMM_B200_ERR_TOO_LARGE;
  if (d->rows && (!d->logits || !d->teacher || !d->index || !d->work)) return LPMM_B200_ERR_NULL_POINTER;
  if (d->rows && mode != DISTILL_LOSS && !d->grad) return LPMM_B200_ERR_NULL_POINTER;
  if (mode != DISTILL_GRAD && !d->loss && (d->rows || d->reduction != LPMM_B200_REDUCE_NONE)) return LPMM_B200_ERR_NULL_POINTER;
  if (mode == DISTILL_GRAD && !d->upstream) return LPMM_B200_ERR_NULL_POINTER;
  if ((uintptr_t)d->work & 15) return LPMM_B200_ERR_BAD_SIZE;
  return LPMM_B200_OK;
}

template <typename T, int MODE>
static cudaError_t distill_launch(DistillArgs& a, cudaStream_t stream) {
  // few rows: their columns are shared by clusters of up to 8 CTAs, so that all SMs have work
  int parts = 1;
  const int vecs = (a.vocab + Elem<T>::VE - 1) / Elem<T>::VE;
  while (parts < 8 && a.rows * parts < 2ll * num_sms() && vecs / (parts * 2) >= 512) parts *= 2;
  a.slice = ((vecs + parts - 1) / parts + 7) / 8 * 8 * Elem<T>::VE;
  const int per = a.slice / Elem<T>::VE;
  const int threads = per >= 2048 ? 512 : per >= 512 ? 256 : 128;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, MODE>, a);
}

template <int MODE>
static int distill_run(const lpmm_b200_distill* d, void* stream_) {
  const int bad = distill_check(d, MODE);
  if (bad) return bad;
  cudaStream_t stream = (cudaStream_t)stream_;
  const bool mean = d->reduction == LPMM_B200_REDUCE_MEAN, none = d->reduction == LPMM_B200_REDUCE_NONE;
  float* norm = d->work;
  DistillArgs a = {};
  a.logits = d->logits, a.grad = d->grad, a.teacher = d->teacher, a.index = d->index, a.weights = d->weights;
  a.upstream = MODE == DISTILL_GRAD ? d->upstream : nullptr;
  a.stats = reinterpret_cast<RowStats*>(d->work + 4);
  a.row_loss = none ? d->loss : d->work + 4 + 4 * d->rows;
  a.norm = mean ? norm : nullptr;
  a.rows = d->rows, a.inner = d->inner, a.outer_stride = d->outer_stride, a.inner_stride = d->inner_stride;
  a.vocab = (int)d->vocab, a.k = (int)d->k, a.teacher_dtype = d->teacher_dtype, a.index_bits = d->index_bits;
  a.upstream_per_row = none;
  a.temperature = d->temperature;
  a.c = (float)(1.4426950408889634 / (double)d->temperature);
  a.scale = d->grad_scale;
  if (d->rows == 0) {
    if (MODE != DISTILL_GRAD && !none) LPMM_CUDA_TRY(cudaMemsetAsync(d->loss, 0, sizeof(float), stream));
    return LPMM_B200_OK;
  }
  if (MODE == DISTILL_BOTH && mean) {
    distill_reduce_kernel<<<1, 1024, 0, stream>>>(nullptr, d->weights, d->rows, 1, nullptr, norm);
    LPMM_CUDA_TRY(cudaGetLastError());
  }
  cudaError_t e;
  if (d->dtype == LPMM_B200_DTYPE_FP32)
    e = distill_launch<float, MODE>(a, stream);
  else if (d->dtype == LPMM_B200_DTYPE_BF16)
    e = distill_launch<__nv_bfloat16, MODE>(a, stream);
  else
    e = distill_launch<__half, MODE>(a, stream);
  LPMM_CUDA_TRY(e);
  if (MODE != DISTILL_GRAD && !none) {
    distill_reduce_kernel<<<1, 1024, 0, stream>>>(a.row_loss, d->weights, d->rows, mean, d->loss, norm);
    LPMM_CUDA_TRY(cudaGetLastError());
  }
  return LPMM_B200_OK;
}

}  // namespace lpmm_b200

using namespace lpmm_b200;

extern "C" int64_t lpmm_b200_distill_work_floats(int64_t rows) { return rows < 0 ? LPMM_B200_ERR_BAD_SIZE : 4 + 5 * rows; }

extern "C" int lpmm_b200_distill_forward(const lpmm_b200_distill* d, void* stream) {
  return distill_run<DISTILL_LOSS>(d, stream);
}
extern "C" int lpmm_b200_distill_backward(const lpmm_b200_distill* d, void* stream) {
  return distill_run<DISTILL_GRAD>(d, stream);
}
extern "C" int lpmm_b200_distill_forward_backward(const lpmm_b200_distill* d, void* stream) {
  return distill_run<DISTILL_BOTH>(d, stream);
}
